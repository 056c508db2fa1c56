"""CPU: the device code of the 4-bit floating point kernels and of the norms around a block, run under the model of the CUDA execution
model (tests/cpu_emu/) against the definitions in 64 bits (tests/fp4_oracle.py)."""
import ctypes

import numpy as np
import pytest
import torch

from tests import fp4_oracle as O
from tests.test_cpu_emulated_kernels import _build, _build_short_waits

_vp, _sz, _ci, _cu, _cf = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_uint, ctypes.c_float
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def emu():
    L = _build("emu_fp4")
    L.emu_fp4_quantize.argtypes = [_vp, _ci, _sz, _sz, _sz, _ci, _vp, _ci, _ci, _cu, _vp, _vp]
    L.emu_fp4_dequantize.argtypes = [_vp, _vp, _vp, _sz, _sz, _ci, _ci, _ci, _vp]
    L.emu_fp4_forward.argtypes = [_vp, _vp, _vp, _vp, _vp, _ci, _ci, _ci, _ci, _ci, _ci, _vp, _sz, _ci, _cu]
    L.emu_residual_norm.argtypes = [_vp, _vp, _vp, _sz, _sz, _sz, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _ci, _ci, _ci, _ci, _cf, _cf, _cf, _ci, _ci, _ci, _ci,
                                    _ci, _cu]
    return L


def aligned(shape, dtype, align=64):
    """A CPU tensor on a 64-byte boundary, as the GPU's allocator gives them."""
    n = int(np.prod(shape)) * torch.empty((), dtype=dtype).element_size()
    raw = torch.zeros(n + align, dtype=torch.uint8)
    off = -raw.data_ptr() % align
    return raw[off:off + n].view(dtype).view(shape)


def special(rows, cols, dtype, seed):
    """Normal values with everything that a quantizer can get wrong among them: ties between codes, zeros of both signs, blocks of
    zeros, powers of two, the smallest and the largest numbers, infinities and NaN."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(2.0 * torch.randn(rows, 1, generator=g))
    x.view(-1)[::7] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0, 6.0, 7.0])[torch.arange(x.numel())[::7] % 11]
    if rows > 2:
        x[2, : min(cols, 40)] = 0.0
        x[2, : min(cols, 40)][::3] = -0.0
    if rows > 3:
        x[3] = torch.finfo(dtype).tiny * torch.arange(cols) / 8
    if rows > 4:
        x[4, 0] = float("inf")
        x[4, cols // 2] = float("nan")
    out = aligned((rows, cols), dtype)
    out.copy_(x.to(dtype))
    if rows > 5 and dtype is not torch.float16:
        out[5, cols - 1] = torch.finfo(dtype).max
    return out


def unsigned_zeros(codes):
    """Codes with the sign of zeros dropped, which is not specified."""
    lo, hi = codes & 15, codes >> 4
    return np.where(lo == 8, 0, lo) | np.where(hi == 8, 0, hi) << 4


def run_quantize(emu, x, nv, g=None, route=1, grid=3):
    rows, cols = x.shape
    kp = -(-cols // 32) * 32
    codes, scales = aligned((rows, kp // 2), torch.uint8), aligned((rows, kp // (16 if nv else 32)), torch.uint8)
    whole = torch.full((1,), 0.0 if g is None else g, dtype=torch.float32)
    rc = emu.emu_fp4_quantize(x.data_ptr(), DTYPES.index(x.dtype), rows, cols, x.stride(0), int(nv), whole.data_ptr(), int(nv and g is None), route, grid,
                              codes.data_ptr(), scales.data_ptr())
    assert rc == 0
    return codes, scales, whole


@pytest.mark.parametrize("nv", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,route", [(7, 64, 0), (33, 256, 0), (1, 32, 0), (6, 33, 1), (7, 64, 1), (1, 1, 1), (9, 1000, 1), (6, 2080, 1)])
def test_quantize_is_exact(emu, dtype, nv, rows, cols, route):
    x = special(rows, cols, dtype, rows * cols)
    codes, scales, whole = run_quantize(emu, x, nv, route=route)
    want_codes, want_scales, g, values = O.quantize(x.double().numpy(), nv)
    if nv:
        assert float(whole) == g
    np.testing.assert_array_equal(scales.numpy(), want_scales)
    np.testing.assert_array_equal(unsigned_zeros(codes.numpy()), unsigned_zeros(want_codes))
    out = aligned((rows, cols), torch.float32)
    assert emu.emu_fp4_dequantize(codes.data_ptr(), scales.data_ptr(), whole.data_ptr(), rows, cols, int(nv), route if cols % 32 == 0 else 1, 0, out.data_ptr()) == 0
    np.testing.assert_array_equal(out.numpy(), values.astype(np.float32))


@pytest.mark.parametrize("g", [0.37, 2.0 ** -10, 1e-6])
def test_a_given_tensor_scale(emu, g):
    x = special(6, 200, torch.float32, 5)
    x[5, -1] = 1.0
    codes, scales, _ = run_quantize(emu, x, True, g)
    want = O.quantize(x.double().numpy(), True, float(np.float32(g)))
    np.testing.assert_array_equal(scales.numpy(), want[1])
    np.testing.assert_array_equal(unsigned_zeros(codes.numpy()), unsigned_zeros(want[0]))


@pytest.mark.parametrize("grid,words", [(1, 1), (3, 1), (3, 3), (1, 2), (3, 4), (40, 64)])
@pytest.mark.parametrize("route", [0, 1])
def test_the_scale_of_small_and_of_zero_tensors(emu, route, grid, words):
    """In its own word and with words for the blocks' parts behind it."""
    x = aligned((5, 64), torch.float32)
    for top in (0.0, 1e-44, 2688.0, 2689.0, 3e38):
        x[3, 7] = top
        codes, scales, whole = aligned((5, 32), torch.uint8), aligned((5, 4), torch.uint8), torch.full((words + 1,), -5.0)
        assert emu.emu_fp4_quantize(x.data_ptr(), 0, 5, 64, 64, 1, whole.data_ptr(), words, route, grid, codes.data_ptr(), scales.data_ptr()) == 0
        want = O.quantize(x.double().numpy(), True)
        assert float(whole[0]) == want[2] and float(whole[words]) == -5.0
        np.testing.assert_array_equal(scales.numpy(), want[1])
        np.testing.assert_array_equal(unsigned_zeros(codes.numpy()), unsigned_zeros(want[0]))


@pytest.mark.parametrize("route", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_far_above_a_given_tensor_scale_saturate(emu, dtype, route):
    """x / g beyond f32 is still a finite x: the largest code and scale of its sign, not a NaN."""
    x = aligned((4, 64), dtype)
    x.copy_(torch.tensor([1e30, -1e30, 3e38, -1.0])[torch.arange(256) % 4].view(4, 64))
    x[1, 17] = float("inf")
    x[2, 40] = float("nan")
    x[3, 16:] = 0.0
    codes, scales, _ = run_quantize(emu, x, True, 2.0 ** -100, route=route)
    want_codes, want_scales = np.full((4, 32), 0xF7), np.full((4, 4), 0x7E)
    want_codes[1, 8:16], want_scales[1, 1] = 0, 0x7F
    want_codes[2, 16:24], want_scales[2, 2] = 0, 0x7F
    want_codes[3, 8:], want_scales[3, 1:] = 0, 0x38
    np.testing.assert_array_equal(codes.numpy(), want_codes)
    np.testing.assert_array_equal(scales.numpy(), want_scales)


def test_rows_with_a_stride(emu):
    wide = special(6, 200, torch.bfloat16, 3)
    for view in (wide[:, 8:72], wide[:, 1:100]):
        codes, scales, _ = run_quantize(emu, view, False)
        want = O.quantize(view.double().numpy(), False)
        np.testing.assert_array_equal(scales.numpy(), want[1])
        np.testing.assert_array_equal(unsigned_zeros(codes.numpy()), unsigned_zeros(want[0]))


def stored(rows, cols, nv, seed, spread=0):
    """Codes and scales of their own: any code, scales over `spread` octaves (MX) or the whole of E4M3 (NV)."""
    g = np.random.default_rng(seed)
    kp = -(-cols // 32) * 32
    code = g.integers(0, 16, (rows, kp), dtype=np.uint8)
    code[:, cols:] = 0
    scales = g.integers(1, 0x7F, (rows, kp // 16), dtype=np.uint8) if nv else (127 - g.integers(0, spread + 1, (rows, kp // 32))).astype(np.uint8)
    c, s = aligned((rows, kp // 2), torch.uint8), aligned(scales.shape, torch.uint8)
    c.copy_(torch.from_numpy(code[:, 0::2] | code[:, 1::2] << 4))
    s.copy_(torch.from_numpy(scales))
    return c, s, torch.tensor([0.5], dtype=torch.float32)


@pytest.mark.parametrize("nv", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols,route", [(64, 0), (1024, 0), (64, 1), (7, 1), (41, 1)])
def test_dequantize_rounds_once(emu, dtype, nv, cols, route):
    c, s, g = stored(5, cols, nv, 1, spread=30)
    s[0, 0] = 0x7F if nv else 255
    out = aligned((5, cols), dtype)
    assert emu.emu_fp4_dequantize(c.data_ptr(), s.data_ptr(), g.data_ptr(), 5, cols, int(nv), route, DTYPES.index(dtype), out.data_ptr()) == 0
    want = torch.from_numpy(O.dequantize(c.numpy(), s.numpy(), 0.5, cols, nv)).to(dtype)
    assert torch.equal(out.nan_to_num(77.0), want.nan_to_num(77.0)) and torch.equal(out.isnan(), want.isnan())


def forward(emu, emu_gemm, x, weights, biases, K, nv, relu=False, pad=0):
    """The kernel that takes so many tokens: a few by warp MMA, more on the tensor cores (there also with k split over a cluster of two)."""
    M, N = x.shape[0], weights[0][0].shape[0]
    table = lambda ts: (ctypes.c_void_p * 2)(*[None if t is None else t.data_ptr() for t in (list(ts) * 2)[:2]])  # noqa: E731
    args = (table([w[0] for w in weights]), table([w[1] for w in weights]), table([w[2] for w in weights]), table(biases), x.data_ptr(),
            int(x.dtype is torch.float32), M, N, K)
    y = torch.full((M, N + pad), -77.0)
    if M <= 4:
        assert emu.emu_fp4_forward(*args, int(nv), int(len(weights) == 2), y.data_ptr(), N + pad, int(relu), 5) == 0
    else:
        split = int(K > 128 and N % 2)
        assert emu_gemm.emu_gemm_w4_bf16(*args, 16 if M <= 16 else 32, int(nv), int(len(weights) == 2), y.data_ptr(), N + pad, int(relu), split, M % 3) == 0
    assert (y[:, N:] == -77.0).all()
    return y[:, :N].double().numpy()


@pytest.fixture(scope="module")
def emu_gemm():
    L = _build("emu_gemm_fp4")
    L.emu_gemm_fp4.argtypes = [_vp, _vp, _vp, _vp, _vp, _cf, _ci, _ci, _ci, _ci, _ci, _ci, _vp, _sz, _ci, _ci, _cu]
    L.emu_gemm_w4_bf16.argtypes = [_vp, _vp, _vp, _vp, _vp, _ci, _ci, _ci, _ci, _ci, _ci, _ci, _vp, _sz, _ci, _ci, _cu]
    return L


@pytest.mark.parametrize("nv", [False, True])
@pytest.mark.parametrize("M,N,K,x_dtype", [(1, 130, 256, torch.bfloat16), (3, 40, 1100, torch.bfloat16), (9, 129, 96, torch.float32), (20, 17, 33, torch.bfloat16),
                                           (32, 5, 2100, torch.bfloat16), (2, 1, 1, torch.float32)])
def test_forward(emu, emu_gemm, nv, M, N, K, x_dtype):
    g = torch.Generator().manual_seed(M * N + K)
    x = aligned((M, K), x_dtype)
    x.copy_(torch.randn(M, K, generator=g) * torch.exp(3 * torch.randn(M, 1, generator=g)))
    w, bias = stored(N, K, nv, N, spread=9), torch.randn(N, generator=g)
    y = forward(emu, emu_gemm, x, [w], [bias], K, nv, relu=N % 2 == 1, pad=3)
    xd, wd = x.double().numpy(), O.dequantize(w[0].numpy(), w[1].numpy(), 0.5, K, nv)
    want, bound = O.product(xd, wd, bias.numpy(), relu=N % 2 == 1), O.product_bound(xd, wd, K, bias=bias.numpy())
    assert (np.abs(y - want) <= bound).all()


@pytest.mark.parametrize("nv", [False, True])
@pytest.mark.parametrize("M", [3, 5, 30])
def test_gated_forward(emu, emu_gemm, nv, M):
    N, K = 70, 300
    g = torch.Generator().manual_seed(8)
    x = aligned((M, K), torch.bfloat16)
    x.copy_(torch.randn(M, K, generator=g))
    ws, biases = [stored(N, K, nv, s, spread=5 + 20 * s) for s in (0, 1)], [torch.randn(N, generator=g), None]
    for w in ws:
        w[2].fill_(2.0 ** -9 if nv else 1.0)
    y = forward(emu, emu_gemm, x, ws, biases, K, nv)
    xd = x.double().numpy()
    wd = [O.dequantize(w[0].numpy(), w[1].numpy(), 2.0 ** -9, K, nv) for w in ws]
    assert (np.abs(y - O.product(xd, wd[0], biases[0].numpy(), up=wd[1])) <= O.product_bound(xd, wd[0], K, up=wd[1], bias=biases[0].numpy())).all()


@pytest.mark.parametrize("M,N", [(3, 24), (7, 24), (20, 25)])
def test_scales_wider_than_a_window_and_activations_wider_than_a_term(emu, emu_gemm, M, N):
    """Block scales over 90 octaves and activations over 60: every product still counts, whatever large things stand beside it."""
    K = 320
    c, s, g1 = stored(N, K, False, 4, spread=90)
    x = aligned((M, K), torch.bfloat16)
    gen = torch.Generator().manual_seed(2)
    x.copy_(torch.randn(M, K, generator=gen) * torch.exp2(-torch.randint(0, 60, (M, K), generator=gen).float()))
    # rows whose large blocks meet zeros in x: what is left is small, and must be right
    s[:, 0], s[:, 1:] = 127, 127 - torch.randint(40, 90, (N, K // 32 - 1), generator=gen).to(torch.uint8)
    x[1, :32] = 0.0
    x[2, 40:] = 0.0
    x[2, 32] = 2.0 ** 20
    c[:, 16] = 0x00   # codes of columns 32, 33: the large activation of token 2 meets zeros
    y = forward(emu, emu_gemm, x, [(c, s, g1)], [None], K, False)
    xd, wd = x.double().numpy(), O.dequantize(c.numpy(), s.numpy(), 1.0, K, False)
    assert (np.abs(y - O.product(xd, wd)) <= O.product_bound(xd, wd, K)).all()


@pytest.mark.parametrize("M", [4, 9])
def test_infinities_and_nan_reach_their_outputs_only(emu, emu_gemm, M):
    N, K = 20, 64
    w = stored(N, K, False, 4, spread=3)
    w[1][7, 1] = 255                       # a NaN block of row 7
    x = aligned((M, K), torch.bfloat16)
    x.copy_(torch.randn(M, K, generator=torch.Generator().manual_seed(1)))
    x[2, 5] = float("inf")
    x[3, 9] = float("nan")
    y = forward(emu, emu_gemm, x, [w], [None], K, False)
    wd = O.dequantize(w[0].numpy(), w[1].numpy(), 1.0, K, False)
    want = O.product(x.double().numpy(), wd)
    np.testing.assert_array_equal(np.isnan(y), np.isnan(want))
    np.testing.assert_array_equal(y[np.isinf(want)], want[np.isinf(want)])


@pytest.mark.parametrize("x_dtype,b_dtype,h_dtype", [(0, 0, 0), (0, 1, 1), (1, 1, 1), (0, 0, 1)])
@pytest.mark.parametrize("M,D,V", [(3, 96, 1), (2, 256, 1), (2, 1000, 4), (2, 1100, 2), (1, 1, 1), (2, 1296, 2)])
@pytest.mark.parametrize("pre,post,gate_kind", [(1, 0, 0), (2, 1, 1), (1, 2, 2), (2, 2, 3), (0, 1, 1), (1, -1, 0)])
def test_residual_norm(emu, x_dtype, b_dtype, h_dtype, M, D, V, pre, post, gate_kind):
    """post -1: no branch.  Tolerance: r is a handful of f32 operations on a norm whose sums of D terms are good to (D + 16) 2^-24, relative to
    the largest terms; then one rounding to each output's type."""
    types = (torch.float32, torch.bfloat16)
    g = torch.Generator().manual_seed(D + pre)
    pad = 8 if D % 8 == 0 else 3
    x, b, gate_full = (aligned((M, D + pad), types[t]) for t in (x_dtype, b_dtype, b_dtype))
    for t in (x, b, gate_full):
        t.copy_(torch.randn(M, D + pad, generator=g) * 2 + 3)
    x, b, gate_full = x[:, :D], b[:, :D], gate_full[:, :D]
    gate = {0: None, 1: aligned((D,), types[b_dtype]), 2: aligned((M, 1), types[b_dtype]), 3: gate_full}[gate_kind]
    if gate_kind in (1, 2):
        gate.copy_(torch.randn(gate.shape, generator=g))
    vec = [aligned((D,), torch.float32) for _ in range(4)]
    for v in vec:
        v.copy_(torch.randn(D, generator=g))
    r, h = torch.zeros(M, D, dtype=types[x_dtype]), torch.zeros(M, D, dtype=types[h_dtype])
    r2, h2 = aligned((M, D), types[x_dtype]), aligned((M, D), types[h_dtype])
    no_branch = post < 0
    ldg = {0: 0, 1: 0, 2: 1, 3: gate_full.stride(0)}[gate_kind]
    is_vec = int(D % 8 == 0 and (D + pad) % 8 == 0)
    rc = emu.emu_residual_norm(x.data_ptr(), None if no_branch else b.data_ptr(), None if gate is None else gate.data_ptr(), x.stride(0), b.stride(0), ldg,
                               vec[0].data_ptr(), vec[1].data_ptr(), vec[2].data_ptr(), None, r2.data_ptr(), h2.data_ptr() if pre else None, M, D, max(post, 0), pre,
                               gate_kind, 1e-5, 0.75, 0.5, is_vec, x_dtype, b_dtype, h_dtype, V, 2)
    assert rc == 0
    n = [v.double().numpy() for v in vec]
    want_r, want_h = O.residual_norm(x.double().numpy(), None if no_branch else b.double().numpy(), None if gate is None else gate.double().numpy(),
                                     pre=(pre, n[2], None, 1e-5) if pre else None, post=(post, n[0], n[1], 1e-5) if post > 0 else None, residual_scale=0.75,
                                     branch_scale=0.5)
    eps = (D + 16) * 2.0 ** -24
    half = {0: 2.0 ** -24, 1: 2.0 ** -8}
    scale_r = np.abs(want_r) + np.abs(0.75 * x.double().numpy()) + 8.0 * (1 + (np.abs(n[0]).max() + np.abs(n[1]).max()) * (1 if gate is None else np.abs(gate.double().numpy()).max()))
    assert (np.abs(r2.double().numpy() - want_r) <= half[x_dtype] * np.abs(want_r) + eps * scale_r).all()
    if pre and D > 1:
        # an error of r moves h by at most |weight| / rms(r) times it, twice over for the statistics
        rms = np.sqrt(((want_r - (want_r.mean(-1, keepdims=True) if pre == 2 else 0)) ** 2).mean(-1, keepdims=True) + 1e-5)
        spread = np.abs(n[2]) * (scale_r.max(-1, keepdims=True) / rms) * (1 + np.abs(want_r) / rms)
        assert (np.abs(h2.double().numpy() - want_h) <= half[h_dtype] * np.abs(want_h) + 4 * eps * spread).all()


@pytest.mark.parametrize("nv", [False, True])
@pytest.mark.parametrize("M,N,K,tok,gated,split,seed", [(70, 130, 600, 64, False, 0, 0), (100, 129, 256, 128, False, 0, 3), (300, 40, 330, 256, False, 1, 0),
                                                        (33, 70, 1300, 64, True, 1, 5), (130, 128, 90, 128, True, 0, 0), (1, 1, 1, 64, False, 0, 0),
                                                        (200, 20, 2600, 256, False, 0, 7), (40, 20, 2600, 64, False, 1, 9), (130, 60, 520, 128, True, 1, 2),
                                                        (140, 270, 600, 256, False, 2, 0), (300, 100, 1700, 256, False, 2, 4), (200, 150, 300, 128, True, 2, 0),
                                                        (290, 30, 1600, 128, True, 2, 8)])
def test_four_bits_by_four_bits(emu_gemm, nv, M, N, K, tok, gated, split, seed):
    g = torch.Generator().manual_seed(M + K)
    x = aligned((M, K), torch.float32)
    x.copy_(torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g)))
    ws = [stored(N, K, nv, N + i, spread=6) for i in range(2 if gated else 1)]
    if nv:
        for w in ws:   # (moderate scales, so that silu's argument stays ordinary)
            w[1].copy_(torch.randint(0x20, 0x40, w[1].shape, generator=g).to(torch.uint8))
            w[2].fill_(2.0 ** -4)
    biases = [torch.randn(N, generator=g), None][: len(ws)]
    y = torch.full((M, N + 4), -77.0)
    table = lambda ts: (ctypes.c_void_p * 2)(*[None if t is None else t.data_ptr() for t in (list(ts) * 2)[:2]])  # noqa: E731
    rc = emu_gemm.emu_gemm_fp4(table([w[0] for w in ws]), table([w[1] for w in ws]), table([w[2] for w in ws]), table(biases), x.data_ptr(), 0.5, M, N, K, tok,
                               int(nv), int(gated), y.data_ptr(), N + 4, int(not gated and N % 2), split, seed)
    assert rc == 0 and (y[:, N:] == -77.0).all()
    xq = O.quantize(x.double().numpy(), nv, 0.5 if nv else None)[3]
    wd = [O.dequantize(w[0].numpy(), w[1].numpy(), float(w[2]), K, nv) for w in ws]
    up = wd[1] if gated else None
    want = O.product(xq, wd[0], biases[0].numpy(), up=up, relu=not gated and N % 2 == 1)
    bound = O.product_bound(xq, wd[0], K, up=up, bias=biases[0].numpy())
    assert (np.abs(y[:, :N].double().numpy() - want) <= bound).all()


@pytest.mark.parametrize("nv", [False, True])
@pytest.mark.parametrize("M,N,K,tok,x_dtype,gated,split,seed", [(70, 130, 600, 64, torch.bfloat16, False, 0, 0), (100, 129, 256, 128, torch.bfloat16, False, 1, 3),
                                                                (300, 40, 336, 256, torch.bfloat16, False, 1, 0), (33, 70, 1300, 64, torch.float32, True, 1, 5),
                                                                (130, 100, 96, 128, torch.bfloat16, True, 0, 0), (1, 1, 1, 64, torch.float32, False, 0, 0),
                                                                (200, 150, 1111, 256, torch.bfloat16, True, 1, 7), (65, 20, 900, 64, torch.float32, False, 0, 9)])
def test_four_bit_weights_on_the_tensor_cores(emu_gemm, nv, M, N, K, tok, x_dtype, gated, split, seed):
    g = torch.Generator().manual_seed(M + K)
    x = aligned((M, K), x_dtype)
    x.copy_(torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g)))
    ws = [stored(N, K, nv, N + i, spread=6) for i in range(2 if gated else 1)]
    if nv:
        for w in ws:
            w[1].copy_(torch.randint(0x20, 0x40, w[1].shape, generator=g).to(torch.uint8))
            w[2].fill_(2.0 ** -4)
    biases = [torch.randn(N, generator=g), None][: len(ws)]
    y = torch.full((M, N + 4), -77.0)
    table = lambda ts: (ctypes.c_void_p * 2)(*[None if t is None else t.data_ptr() for t in (list(ts) * 2)[:2]])  # noqa: E731
    rc = emu_gemm.emu_gemm_w4_bf16(table([w[0] for w in ws]), table([w[1] for w in ws]), table([w[2] for w in ws]), table(biases), x.data_ptr(),
                                   int(x_dtype is torch.float32), M, N, K, tok, int(nv), int(gated), y.data_ptr(), N + 4, int(not gated and N % 2), split, seed)
    assert rc == 0 and (y[:, N:] == -77.0).all()
    xd = x.double().numpy()
    wd = [O.dequantize(w[0].numpy(), w[1].numpy(), float(w[2]), K, nv) for w in ws]
    up = wd[1] if gated else None
    want = O.product(xd, wd[0], biases[0].numpy(), up=up, relu=not gated and N % 2 == 1)
    assert (np.abs(y[:, :N].double().numpy() - want) <= O.product_bound(xd, wd[0], K, up=up, bias=biases[0].numpy())).all()


@pytest.mark.parametrize("nv,K,x_dtype,spread", [(False, 96, torch.float32, 3), (True, 128, torch.float32, 0), (False, 256, torch.float32, 3), (False, 96, torch.bfloat16, 100),
                                                 (False, 200, torch.float32, 40)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.timeout(120)
def test_converters_that_come_late_to_a_pass(nv, K, x_dtype, spread, gated):
    """Several passes (terms of f32 activations, windows of scales) of a round or two: the warps that have nothing to convert in the first passes
    look at the accumulators' barrier long after those passes could be done."""
    L = _build_short_waits("emu_gemm_fp4", ("-DSHREWQ_SPIN_FAST_LIMIT=64", "-DSHREWQ_SPIN_SLOW_LIMIT=10000"), "second_waits")
    L.emu_gemm_w4_bf16.argtypes = [_vp, _vp, _vp, _vp, _vp, _ci, _ci, _ci, _ci, _ci, _ci, _ci, _vp, _sz, _ci, _ci, _cu]
    M, N = 9, 30
    g = torch.Generator().manual_seed(K)
    x = aligned((M, K), x_dtype)
    x.copy_(torch.randn(M, K, generator=g))
    ws = [stored(N, K, nv, i, spread=spread) for i in range(2 if gated else 1)]
    for w in ws:
        w[2].fill_(2.0 ** -9 if nv else 1.0)
    bias = torch.randn(N, generator=g)
    y = torch.full((M, N), -77.0)
    table = lambda ts: (ctypes.c_void_p * 2)(*[None if t is None else t.data_ptr() for t in (list(ts) * 2)[:2]])  # noqa: E731
    try:
        for first in (10, 6, 2):   # the third group of converters, then more of them
            L.emu_late_warps(first, 150)
            rc = L.emu_gemm_w4_bf16(table([w[0] for w in ws]), table([w[1] for w in ws]), table([w[2] for w in ws]), table([bias]), x.data_ptr(), int(x_dtype is torch.float32),
                                    M, N, K, 16, int(nv), int(gated), y.data_ptr(), N, 0, 0, 0)
            assert rc == 0
            xd, wd = x.double().numpy(), [O.dequantize(w[0].numpy(), w[1].numpy(), 2.0 ** -9, K, nv) for w in ws]
            up = dict(up=wd[1], bias_up=bias.numpy()) if gated else {}
            want, bound = O.product(xd, wd[0], bias.numpy(), **up), O.product_bound(xd, wd[0], K, bias=bias.numpy(), **up)
            assert (np.abs(y.double().numpy() - want) <= bound).all()
    finally:
        L.emu_late_warps(-1, 0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_inputs_of_a_stream_are_not_read_as_constant(emu, dtype):
    """Tensors, activations, branches and gates may be the output of the kernel before, which may still run when these kernels are launched early: no
    load of theirs goes through the read-only path, which is for data that nothing writes while the kernel is there."""
    emu.emu_read_only_loads.restype = ctypes.c_long
    emu.emu_read_only_loads()
    x = special(9, 64, dtype, 1)
    for nv in (False, True):
        for route in (0, 1):
            run_quantize(emu, x, nv, route=route)
    assert emu.emu_read_only_loads() == 0
    if dtype is torch.float16:
        return
    x, b, r, h = (aligned((3, 64), dtype) for _ in range(4))
    which, w = int(dtype is torch.bfloat16), aligned((64,), torch.float32)
    for gate_kind in (1, 3):
        assert emu.emu_residual_norm(x.data_ptr(), b.data_ptr(), b.data_ptr(), 64, 64, 64, w.data_ptr(), None, w.data_ptr(), None, r.data_ptr(), h.data_ptr(), 3, 64, 1, 1, gate_kind,
                                     1e-5, 1.0, 1.0, 1, which, which, which, 1, 2) == 0
    assert emu.emu_read_only_loads() == 0


@pytest.mark.parametrize("M", [3, 9])
def test_relu_keeps_nan(emu, emu_gemm, M):
    w = stored(20, 64, False, 4, spread=3)
    x = aligned((M, 64), torch.bfloat16)
    x.copy_(torch.randn(M, 64, generator=torch.Generator().manual_seed(1)))
    x[2, 9] = float("nan")
    y = forward(emu, emu_gemm, x, [w], [None], 64, False, relu=True)
    assert np.isnan(y[2]).all() and (y[:2] >= 0).all() and (y[3:] >= 0).all()
