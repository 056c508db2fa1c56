"""GPU: quantization to 4-bit microscaled floating point, Linear layers over it and the norms around a block, through the package's
public entry points, against the definitions in 64 bits (tests/fp4_oracle.py).  Tolerances: see product_bound there; a result of type t is
then rounded once, half a step."""
import numpy as np
import pytest
import torch

from shrew_b200 import (Fp4Format, Fp4Linear, Fp4Tensor, GatedMlp, Linear, Norm, NormKind, QuantConfig, QuantizedLinear, ShrewError, dequantize_fp4,
                        quantize_fp4, residual_norm, run_blocks)
from shrew_b200 import _lib
from shrew_b200.quantize import Device
from tests import fp4_oracle as O
from tests.test_fp4_emulated import special, unsigned_zeros

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
FORMATS = [Fp4Format.Mx, Fp4Format.Nv]


def near(y, want, bound):
    """|y - want| <= bound, then y's own rounding; infinities and NaN in the same places."""
    got = y.double().cpu().numpy()
    fine = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    assert (np.abs(got - want)[fine] <= (bound + HALF[y.dtype] * (np.abs(want) + bound))[fine]).all()


def layer(n, k, fmt, seed, bias=True, **options):
    """A layer over random codes and scales, its weights in 64 bits and its bias."""
    g = np.random.default_rng(seed)
    kp, nv = -(-k // 32) * 32, fmt is Fp4Format.Nv
    code = g.integers(0, 16, (n, kp), dtype=np.uint8)
    code[:, k:] = 0
    scales = g.integers(0x18, 0x50, (n, kp // 16), dtype=np.uint8) if nv else (127 - g.integers(0, 9, (n, kp // 32))).astype(np.uint8)
    codes = code[:, 0::2] | code[:, 1::2] << 4
    t = Fp4Tensor(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), torch.tensor([0.25], device="cuda") if nv else None, [n, k], F32, fmt)
    b = torch.from_numpy(g.standard_normal(n).astype(np.float32)).cuda() if bias else None
    return Fp4Linear(t, b, **options), O.dequantize(codes, scales, 0.25, k, nv), None if b is None else b.double().cpu().numpy()


def acts(m, k, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + m * k)
    return (torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g))).to(dtype).cuda()


# ---- quantize, dequantize -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (7, 64), (300, 4096), (129, 1000), (3, 20000), (50, 33)])
def test_quantize_is_exact(fmt, dtype, rows, cols):
    x = special(rows, cols, dtype, rows + cols)
    q = quantize_fp4(x.cuda(), fmt)
    codes, scales, g, values = O.quantize(x.double().numpy(), fmt is Fp4Format.Nv)
    np.testing.assert_array_equal(q.scales.cpu().numpy(), scales)
    np.testing.assert_array_equal(unsigned_zeros(q.codes.cpu().numpy()), unsigned_zeros(codes))
    assert (q.tensor_scale is None) == (fmt is Fp4Format.Mx) and (q.tensor_scale is None or float(q.tensor_scale) == g)
    back = dequantize_fp4(q)
    want = torch.from_numpy(values).to(F32).to(dtype)
    assert back.dtype is dtype and torch.equal(back.cpu().nan_to_num(9.0), want.nan_to_num(9.0)) and torch.equal(back.isnan().cpu(), want.isnan())


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_views_ranks_and_empty_tensors(fmt):
    wide = special(40, 200, BF16, 1).cuda()
    for view in (wide[:, 16:80], wide[:, 3:50], wide[::2, :64], wide.t(), wide.view(4, 10, 200), wide[0], wide[0, 0], wide[:0], wide[:, :0]):
        rows, cols = (1, 1) if view.dim() == 0 else (view.shape[0], int(np.prod(view.shape[1:])))
        q = quantize_fp4(view, fmt)
        assert q.shape == list(view.shape)
        if rows * cols:
            codes, scales, _, _ = O.quantize(view.double().cpu().numpy().reshape(rows, cols), fmt is Fp4Format.Nv)
            np.testing.assert_array_equal(q.scales.cpu().numpy(), scales)
            np.testing.assert_array_equal(unsigned_zeros(q.codes.cpu().numpy()), unsigned_zeros(codes))
        back = dequantize_fp4(q, F32)
        assert back.shape == view.shape and back.dtype is F32
    assert float(quantize_fp4(wide[:0], Fp4Format.Nv).tensor_scale) == 1.0


def test_a_given_tensor_scale():
    x = special(6, 300, F32, 2)
    x[5, -1] = 3.0
    g = torch.tensor([0.37], device="cuda")
    q = quantize_fp4(x.cuda(), Fp4Format.Nv, tensor_scale=g)
    want = O.quantize(x.double().numpy(), True, float(g))
    assert q.tensor_scale is g
    np.testing.assert_array_equal(q.scales.cpu().numpy(), want[1])
    np.testing.assert_array_equal(unsigned_zeros(q.codes.cpu().numpy()), unsigned_zeros(want[0]))


def test_quantize_on_streams_and_in_a_graph():
    xs = [special(64, 512, F32, s).cuda() for s in range(4)]
    want = [quantize_fp4(x, Fp4Format.Nv) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for s, x in zip(streams, xs):
        with torch.cuda.stream(s):
            got.append(quantize_fp4(x, Fp4Format.Nv))
    torch.cuda.synchronize()
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        back = dequantize_fp4(quantize_fp4(x, Fp4Format.Nv))
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and torch.equal(a.tensor_scale, b.tensor_scale)
        x.copy_(xs[i])
        graph.replay()
        assert torch.equal(back.nan_to_num(7.0), dequantize_fp4(b).nan_to_num(7.0))


def test_quantize_refusals():
    x = torch.zeros(4, 64, device="cuda")
    for bad, code in ((lambda: quantize_fp4(x.double()), _lib.ERR_UNSUPPORTED), (lambda: quantize_fp4(x.cpu()), _lib.ERR_NO_DEVICE),
                      (lambda: quantize_fp4(x, Fp4Format.Mx, torch.ones(1, device="cuda")), _lib.ERR_INVALID_ARG),
                      (lambda: quantize_fp4(x, Fp4Format.Nv, torch.ones(1)), _lib.ERR_INVALID_ARG),
                      (lambda: quantize_fp4(x, Fp4Format.Nv, torch.ones(2, device="cuda")), _lib.ERR_INVALID_ARG)):
        with pytest.raises(ShrewError) as e:
            bad()
        assert e.value.code == code
    q = quantize_fp4(x, Fp4Format.Nv)
    with pytest.raises(ShrewError):
        dequantize_fp4(q, torch.float64)
    q.scales = q.scales[:1]
    with pytest.raises(ShrewError):
        dequantize_fp4(q)


# ---- layers ------------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 256, 512), (2, 130, 1100), (7, 40, 96), (16, 129, 4096), (17, 300, 33), (32, 64, 2048), (33, 128, 256), (64, 200, 1000), (100, 513, 320),
          (128, 256, 4096), (130, 1000, 2080), (257, 136, 1024), (300, 50, 77), (1, 4100, 11008)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("x_dtype,y_dtype", [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_forward(fmt, x_dtype, y_dtype, m, n, k):
    lin, w, b = layer(n, k, fmt, m + n, bias=n % 2 == 0)
    x = acts(m, k, x_dtype)
    y = lin.forward(x, epilogue=_lib.EPILOGUE_RELU if n % 3 == 0 else _lib.EPILOGUE_NONE, out_dtype=y_dtype)
    assert y.dtype is y_dtype and list(y.shape) == [m, n]
    xd = x.double().cpu().numpy()
    near(y, O.product(xd, w, b, relu=n % 3 == 0), O.product_bound(xd, w, k, bias=b))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("x_dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_forward_with_quantized_activations(fmt, x_dtype, m, n, k):
    lin, w, b = layer(n, k, fmt, m + n, bias=n % 2 == 0, quantize_activations=True, activation_scale=0.5)
    x = acts(m, k, x_dtype)
    y = lin.forward(x, out_dtype=F32 if n % 3 else BF16)
    xq = O.quantize(x.double().cpu().numpy(), fmt is Fp4Format.Nv, 0.5)[3]
    near(y, O.product(xq, w, b), O.product_bound(xq, w, k, bias=b))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rounded", [False, True])
@pytest.mark.parametrize("x_dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gated_pair(fmt, rounded, x_dtype, m, n, k):
    options = dict(quantize_activations=True, activation_scale=0.5) if rounded else {}
    gate, wg, bg = layer(n, k, fmt, 1, **options)
    up, wu, bu = layer(n, k, fmt, 2, bias=False, **options)
    x = acts(m, k, x_dtype) / (8 * k ** 0.5)
    h = gate.forward_gate_up_silu(up, x)
    xd = x.double().cpu().numpy()
    xd = O.quantize(xd, fmt is Fp4Format.Nv, 0.5)[3] if rounded else xd
    near(h, O.product(xd, wg, bg, up=wu, bias_up=bu), O.product_bound(xd, wg, k, up=wu, bias=bg, bias_up=bu))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(129, 9473, 33), (140, 9600, 320), (300, 4900, 600), (513, 3400, 2080), (1100, 2000, 1600)])
def test_wide_products_of_quantized_activations(fmt, gated, m, n, k):
    """Outputs that fill the machine, in both directions."""
    lin, w, b = layer(n, k, fmt, m + n, quantize_activations=True, activation_scale=0.5)
    up, wu, bu = layer(n, k, fmt, 2, bias=False, quantize_activations=True, activation_scale=0.5)
    x = acts(m, k, BF16) / (8 * k ** 0.5)
    xq = O.quantize(x.double().cpu().numpy(), fmt is Fp4Format.Nv, 0.5)[3]
    y = lin.forward_gate_up_silu(up, x) if gated else lin.forward(x, out_dtype=F32)
    pair = dict(up=wu, bias_up=bu) if gated else {}
    near(y, O.product(xq, w, b, **pair), O.product_bound(xq, w, k, bias=b, **pair))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("off", [0, 8, 3])
def test_column_slice_of_a_wide_product(gated, dtype, off):
    n = 4801
    lin, _, _ = layer(n, 320, Fp4Format.Nv, 3, quantize_activations=True)
    up, _, _ = layer(n, 320, Fp4Format.Nv, 4, quantize_activations=True)
    x = acts(300, 320, BF16) * 0.01

    def run(out):
        return lin.forward_gate_up_silu(up, x, out=out) if gated else lin.forward(x, out=out)
    wide = torch.full((301, n + 23), -7.0, dtype=dtype, device="cuda")
    out = wide[:300, off:off + n]
    run(out)
    assert torch.equal(out, run(torch.empty(300, n, dtype=dtype, device="cuda")))
    mask = torch.ones_like(wide, dtype=torch.bool)
    mask[:300, off:off + n] = False
    assert (wide[mask] == -7.0).all()


@pytest.mark.parametrize("rounded", [False, True])
@pytest.mark.parametrize("m", [3, 40, 150])
def test_column_slice_of_a_wider_buffer(rounded, m):
    lin, w, b = layer(200, 320, Fp4Format.Mx, 3, quantize_activations=rounded)
    x = acts(m, 320, BF16)
    for off in (0, 8, 3):
        wide = torch.full((m + 1, 232), -7.0, dtype=BF16, device="cuda")
        out = wide[:m, off:off + 200]
        lin.forward(x, out=out)
        assert torch.equal(out, lin.forward(x))
        mask = torch.ones_like(wide, dtype=torch.bool)
        mask[:m, off:off + 200] = False
        assert (wide[mask] == -7.0).all()


@pytest.mark.parametrize("m", [2, 50])
def test_activations_off_their_boundaries(m):
    lin, w, b = layer(72, 256, Fp4Format.Nv, 3)
    rows = lin.forward(acts(m, 256, BF16))
    odd = torch.empty(m * 256 + 1, dtype=BF16, device="cuda")[1:].view(m, 256)
    odd.copy_(acts(m, 256, BF16))
    assert torch.equal(lin.forward(odd), rows)


def test_no_tokens():
    lin, _, _ = layer(8, 64, Fp4Format.Mx, 1)
    assert lin.forward(torch.empty(0, 64, device="cuda", dtype=BF16)).shape == (0, 8)


@pytest.mark.parametrize("m", [1, 40])
@pytest.mark.parametrize("rounded", [False, True])
def test_infinities_and_nan_stay_in_their_rows(m, rounded):
    lin, w, _ = layer(150, 256, Fp4Format.Mx, 5, bias=False, quantize_activations=rounded)
    x = acts(m + 2, 256, BF16)
    clean = lin.forward(x)
    x[m, 3] = float("inf")
    x[m + 1, 9] = float("nan")
    y = lin.forward(x)
    assert torch.equal(y[:m], clean[:m]) and not y[m:].isfinite().all()
    assert y[m + 1].isnan().all() and (rounded or not y[m].isfinite().any())


@pytest.mark.parametrize("m", [1, 40])
def test_a_nan_block_reaches_its_channel_only(m):
    lin, w, _ = layer(150, 256, Fp4Format.Mx, 5, bias=False)
    t = lin.weight_q
    scales = t.scales.clone()
    scales[77, 3] = 255
    bad = Fp4Linear(Fp4Tensor(t.codes, scales, None, t.shape, F32, Fp4Format.Mx))
    x = acts(m, 256, BF16)
    y, clean = bad.forward(x), lin.forward(x)
    assert y[:, 77].isnan().all()
    y[:, 77] = clean[:, 77]
    assert torch.equal(y, clean)


@pytest.mark.parametrize("m", [1, 20, 40])
def test_scales_of_any_size(m):
    """MX scales at both ends of E8M0, in one tensor and at once."""
    n, k = 64, 256
    g = np.random.default_rng(0)
    codes = g.integers(0, 256, (n, k // 2), dtype=np.uint8)
    for lo, hi in ((0, 5), (200, 240), (120, 220)):
        scales = g.integers(lo, hi, (n, k // 32), dtype=np.uint8)
        lin = Fp4Linear(Fp4Tensor(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), None, [n, k], F32, Fp4Format.Mx))
        x = (acts(m, k, BF16).double() * 2.0 ** -40).to(BF16) if hi > 200 else acts(m, k, BF16)
        w = O.dequantize(codes, scales, 1.0, k, False)
        xd = x.double().cpu().numpy()
        want, bound = O.product(xd, w), O.product_bound(xd, w, k)
        ok = np.abs(want) + bound < 3e38
        y = lin.forward(x, out_dtype=F32).double().cpu().numpy()
        assert ok.mean() > 0.5 and (np.abs(y - want)[ok] <= bound[ok] + 2.0 ** -148).all()


@pytest.mark.parametrize("rounded", [False, True])
@pytest.mark.parametrize("m", [1, 20, 64, 300])
def test_streams_graphs_and_repetition(rounded, m):
    """The same call twice, on another stream, captured and replayed with new data: the same bits each time."""
    gate, _, _ = layer(384, 1024, Fp4Format.Nv, 1, quantize_activations=rounded)
    up, _, _ = layer(384, 1024, Fp4Format.Nv, 2, quantize_activations=rounded)
    down, _, _ = layer(1024, 384, Fp4Format.Nv, 3, quantize_activations=rounded)
    xs = [acts(m, 1024, BF16, seed=s) * 0.01 for s in range(3)]

    def run(x):
        return down.forward(gate.forward_gate_up_silu(up, x))
    want = [run(x) for x in xs]
    assert all(torch.equal(run(x), w) for x, w in zip(xs, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [run(x) for x in xs]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    x, graph = xs[0].clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run(run(x) * 0.0 + x)
    for x_new, w in zip(xs, want):
        x.copy_(x_new)
        graph.replay()
        assert torch.equal(y, w)
    gate.device.synchronize()


@pytest.mark.parametrize("fmt", FORMATS)
def test_wide_products_captured_and_repeated(fmt):
    """Outputs that fill the machine, tile after tile: the same bits eagerly, on another stream and from a graph with new data."""
    gate, _, _ = layer(4900, 608, fmt, 1, quantize_activations=True)
    up, _, _ = layer(4900, 608, fmt, 2, quantize_activations=True)
    down, _, _ = layer(608, 4900, fmt, 3, quantize_activations=True)
    xs = [acts(700, 608, BF16, seed=s) * 0.01 for s in range(3)]

    def run(x):
        return down.forward(gate.forward_gate_up_silu(up, x))
    want = [run(x) for x in xs]
    for _ in range(20):
        assert all(torch.equal(run(x), w) for x, w in zip(xs, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [run(x) for x in xs]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    x, graph = xs[0].clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run(x)
    for x_new, w in zip(xs, want):
        x.copy_(x_new)
        graph.replay()
        assert torch.equal(y, w)
    gate.device.synchronize()


@pytest.mark.parametrize("rounded", [False, True])
@pytest.mark.parametrize("m", [4, 8, 16, 32, 64, 250])
def test_layers_of_different_widths_in_turn(rounded, m):
    """Two layers that share the context's workspace, laid out for another k each, over and over: the same bits each time."""
    gate, _, _ = layer(384, 1024, Fp4Format.Nv, 1, quantize_activations=rounded)
    up, _, _ = layer(384, 1024, Fp4Format.Nv, 2, quantize_activations=rounded)
    down, _, _ = layer(1024, 384, Fp4Format.Nv, 3, quantize_activations=rounded)
    xs = [acts(m, 1024, BF16, seed=s) * 0.01 for s in range(3)]
    want = []
    for x in xs:
        h = gate.forward_gate_up_silu(up, x)
        torch.cuda.synchronize()
        want.append(down.forward(h))
        torch.cuda.synchronize()
    for _ in range(30):
        got = [down.forward(gate.forward_gate_up_silu(up, x)) for x in xs]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_layer_surface_and_host_buffers():
    w = torch.randn(96, 160, device="cuda")
    b = torch.randn(96, device="cuda")
    lin = Fp4Linear.from_linear(Linear(w, b), Fp4Format.Nv, quantize_activations=True)
    assert lin.parameters() == [] and lin.num_parameters() == 0 and lin.memory_savings_bytes() == 96 * 160 * 4 - 96 * 160 * 9 // 16
    assert "Nv" in repr(lin) and lin.weight_quantized().compression_ratio() > 7
    x = acts(5, 160, BF16)
    y = lin.forward(x)
    assert torch.equal(lin.forward_host(x.cpu()), y.cpu())
    assert torch.equal(lin(x), y) and lin.last_kernel()


def test_layer_refusals():
    w = quantize_fp4(torch.randn(64, 96, device="cuda"), Fp4Format.Mx)
    v = quantize_fp4(torch.randn(64, 96, device="cuda"), Fp4Format.Nv)
    x = acts(4, 96, BF16)
    bad = [lambda: Fp4Linear(w, torch.zeros(3, device="cuda")), lambda: Fp4Linear(v, quantize_activations=True, activation_scale=0.0),
           lambda: Fp4Linear(v, quantize_activations=True, activation_scale=float("nan")), lambda: Fp4Linear(w).forward(x[:, :64]),
           lambda: Fp4Linear(w).forward(x.half()), lambda: Fp4Linear(w).forward(x.cpu()), lambda: Fp4Linear(w).forward_gate_up_silu(Fp4Linear(v), x),
           lambda: Fp4Linear(w).forward_gate_up_silu(Fp4Linear(w, quantize_activations=True), x),
           lambda: Fp4Linear(Fp4Tensor(w.codes, w.scales, v.tensor_scale, w.shape, F32, Fp4Format.Mx)),
           lambda: Fp4Linear(Fp4Tensor(v.codes, v.scales, None, v.shape, F32, Fp4Format.Nv)),
           lambda: Fp4Linear(Fp4Tensor(w.codes[:, :16], w.scales, None, w.shape, F32, Fp4Format.Mx)),
           lambda: Fp4Linear(Fp4Tensor(w.codes, w.scales[:, :1], None, w.shape, F32, Fp4Format.Mx)),
           lambda: Fp4Linear.new_int4_packed(w)]
    for f in bad:
        with pytest.raises(ShrewError):
            f()
    i8 = QuantizedLinear.from_linear(Linear(torch.randn(64, 96, device="cuda")), QuantConfig.int8_per_channel())
    with pytest.raises(ShrewError):
        i8.forward_gate_up_silu(Fp4Linear(w), x)
    # peers and the no-allocation form have no 4-bit kernel
    lin = Fp4Linear(w)
    y = torch.empty(4, 64, dtype=BF16, device="cuda")
    L = _lib.lib()
    assert L.shrewq_linear_forward_noalloc(lin._h, x.data_ptr(), 4, y.data_ptr(), _lib.BF16, 64, 0) == _lib.ERR_UNSUPPORTED
    import ctypes
    peers = (ctypes.c_void_p * 1)(y.data_ptr())
    assert L.shrewq_linear_forward_peers(lin._h, None, x.data_ptr(), _lib.BF16, 4, y.data_ptr(), peers, 1, _lib.BF16, 64, 0) == _lib.ERR_UNSUPPORTED


# ---- norms ----------------------------------------------------------------------------------------------------------------
def norm_pair(d, kind, seed, bias=True):
    g = torch.Generator().manual_seed(seed)
    w, b = 1 + torch.randn(d, generator=g), torch.randn(d, generator=g)
    return Norm(kind, w.cuda(), b.cuda() if bias else None), (kind.value, w.double().numpy(), b.double().numpy() if bias else None, 1e-5)


def check_norm(x, branch, gate, pre, post, residual_scale, branch_scale, out_dtype):
    """r is a few f32 operations on norms whose sums of D terms are good to (D + 16) 2^-24 of their largest terms; an error of r moves h by
    |weight| / spread(r) times it, and the statistics by as much again."""
    r, h = residual_norm(x, branch, gate, pre=pre and pre[0], post=post and post[0], residual_scale=residual_scale, branch_scale=branch_scale, out_dtype=out_dtype)
    f = [None if t is None else t.double().cpu().numpy() for t in (x, branch, gate)]
    want_r, want_h = O.residual_norm(*f, pre=pre and pre[1], post=post and post[1], residual_scale=float(np.float32(residual_scale)),
                                     branch_scale=float(np.float32(branch_scale)))
    d = x.shape[-1]
    eps = (d + 16) * 2.0 ** -24
    size = np.abs(want_r) + abs(residual_scale) * np.abs(f[0])
    if branch is not None:
        b = f[1] if post is None else O.norm(f[1], *post[1])
        gg = np.abs(f[2]) if gate is not None else 1.0
        size = size + abs(branch_scale) * np.abs(b) * gg
        if post is not None:
            rms = np.sqrt((f[1] ** 2).mean(-1, keepdims=True))
            s = np.sqrt(((f[1] - (f[1].mean(-1, keepdims=True) if post[1][0] == 2 else 0)) ** 2).mean(-1, keepdims=True) + 1e-5)
            size = size + abs(branch_scale) * gg * np.abs(post[1][1]) * (rms / s) * (1 + np.abs(f[1]) / s) + abs(branch_scale) * gg * np.abs(post[1][2] if post[1][2] is not None else 0)
    near(r, want_r, eps * size)
    if pre is None:
        assert h is None
        return r, h
    s = np.sqrt(((want_r - (want_r.mean(-1, keepdims=True) if pre[1][0] == 2 else 0)) ** 2).mean(-1, keepdims=True) + 1e-5)
    rms = np.sqrt((want_r ** 2).mean(-1, keepdims=True))
    spread = np.abs(pre[1][1]) / s * (size + rms + size.max(-1, keepdims=True) * (1 + np.abs(want_r) / s))
    near(h, want_h, 2 * eps * spread + 2.0 ** -22 * np.abs(want_h) + 2.0 ** -23 * (np.abs(pre[1][2]) if pre[1][2] is not None else 0.0))
    return r, h


@pytest.mark.parametrize("x_dtype,b_dtype,out_dtype", [(BF16, BF16, BF16), (F32, BF16, BF16), (F32, F32, F32), (BF16, F32, F32)])
@pytest.mark.parametrize("m,d", [(1, 4096), (3, 1), (9, 7), (5, 256), (17, 512), (8, 1000), (4, 1024), (3, 1032), (2, 5000), (2, 11008), (2, 16385), (1, 32768)])
@pytest.mark.parametrize("kinds,gate_kind", [(("rms", None), None), (("rms", "rms"), "channel"), (("layer", "layer"), "token"), ((None, "rms"), "full"), (("rms", None), "full")])
def test_residual_norm(x_dtype, b_dtype, out_dtype, m, d, kinds, gate_kind):
    if d == 1 and "layer" in kinds:
        kinds = ("rms", "rms")   # (a layer norm of one value is its bias, whatever rounding does to a difference of nothing)
    x, branch = acts(m, d, x_dtype) + 1, acts(m, d, b_dtype, seed=1) - 2
    gate = {None: None, "channel": acts(1, d, b_dtype, seed=2)[0], "token": acts(m, 1, b_dtype, seed=2), "full": acts(m, d, b_dtype, seed=2)}[gate_kind]
    kind = {"rms": NormKind.Rms, "layer": NormKind.Layer}
    pre, post = (None if k is None else norm_pair(d, kind[k], i, bias=k == "layer") for i, k in enumerate(kinds))
    check_norm(x, branch, gate, pre, post, 0.75, 0.22, out_dtype)


def test_norm_of_views_ranks_and_nothing():
    pre = norm_pair(96, NormKind.Rms, 1, bias=False)
    x = acts(12, 200, BF16)
    check_norm(x[:, 8:104], x[:, 100:196], None, pre, None, 1.0, 1.0, F32)
    check_norm(x[:, 1:97], x[:, 3:99], x[:, 5:101], pre, None, 1.0, 1.0, BF16)
    x3 = acts(24, 96, F32).view(2, 3, 4, 96)
    r, h = residual_norm(x3, x3, x3[..., :1].contiguous(), pre=pre[0])
    r2, h2 = residual_norm(x3.view(24, 96), x3.view(24, 96), x3.view(24, 96)[:, :1], pre=pre[0])
    assert r.shape == x3.shape and torch.equal(r.view(24, 96), r2) and torch.equal(h.view(24, 96), h2)
    one = x3.view(24, 96)[0]
    assert torch.equal(residual_norm(one, pre=pre[0])[1], residual_norm(one[None], pre=pre[0])[1][0])
    r, h = residual_norm(x, pre=None)
    assert r is x and h is None
    r, h = residual_norm(x[:0], x[:0], pre=Norm())
    assert r.shape == (0, 200) and h.shape == (0, 200)
    r, h = residual_norm(x, residual_scale=0.5)
    assert torch.equal(r, (x.float() * 0.5).to(BF16)) and h is None


def test_norm_of_far_and_constant_rows():
    """Rows far from zero (a layer norm must not cancel), of zeros, and with a NaN that stays in its row."""
    x = torch.randn(6, 1024, device="cuda")
    x[0] += 1e5
    x[1] = 0.0
    x[2] = 3.0
    _, h = residual_norm(x, pre=Norm(NormKind.Layer))
    want = O.norm(x.double().cpu().numpy(), 2)
    # the row at 1e5 keeps 2^-24 * 1e5 of each value: 0.006 of its spread
    assert np.abs(h.double().cpu().numpy() - want).max() <= 2.0 ** -24 * 1e5 * 3
    assert (h[1] == 0).all() and (h[2] == 0).all()
    x[3, 5] = float("nan")
    r, h2 = residual_norm(x, x, pre=Norm(NormKind.Rms))
    assert h2[3].isnan().all() and h2[:3].isfinite().all() and h2[4:].isfinite().all() and r[3].isnan().sum() == 1


def test_norm_refusals():
    x = torch.zeros(4, 64, device="cuda")
    n = Norm(NormKind.Rms, torch.ones(32, device="cuda"))
    for f in (lambda: residual_norm(x, pre=n), lambda: residual_norm(x, x[:2]), lambda: residual_norm(x, None, x), lambda: residual_norm(x, x, x.bfloat16()),
              lambda: residual_norm(x, x, x[:, :3]), lambda: residual_norm(x.half(), pre=Norm()), lambda: residual_norm(x, x.half()), lambda: residual_norm(x.cpu(), pre=Norm()),
              lambda: residual_norm(x, pre=Norm(), out_dtype=F16), lambda: residual_norm(x, post=Norm()), lambda: residual_norm(torch.zeros(2, 32769, device="cuda"), pre=Norm()),
              lambda: Norm(eps=-1.0), lambda: Norm(eps=float("nan"))):
        with pytest.raises(ShrewError):
            f()


# ---- together --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["mx", "nv", "mx rounded", "nv rounded", "int8"])
@pytest.mark.parametrize("m", [1, 12, 70, 300])
def test_blocks_together(kind, m):
    """Two gated blocks as a decoder runs them, against the same steps in 64 bits, one call at a time: each step is fed what the package's step before
    it gave, so each is held to its own tolerance; and the blocks' output is those steps' output, bit for bit."""
    d, ff = 256, 672
    fmt, rounded = (Fp4Format.Nv if "nv" in kind else Fp4Format.Mx), "rounded" in kind
    g = torch.Generator().manual_seed(m)

    def linear(n, k):
        w = (torch.randn(n, k, generator=g) * k ** -0.5).cuda()
        if kind == "int8":
            return QuantizedLinear.from_linear(Linear(w), QuantConfig.int8_per_channel()), None
        lin = Fp4Linear.from_linear(Linear(w), fmt, quantize_activations=rounded)
        return lin, dequantize_fp4(lin.weight_q, F32).double().cpu().numpy()

    blocks, parts = [], []
    for i in range(2):
        (gate, wg), (up, wu), (down, wd) = linear(ff, d), linear(ff, d), linear(d, ff)
        pre, post = norm_pair(d, NormKind.Rms, i, bias=False), norm_pair(d, NormKind.Rms, 7 + i, bias=False) if i else None
        cg = torch.randn(d, generator=g).cuda() if i else None
        blocks.append(GatedMlp(gate, up, down, pre[0], post and post[0], cg, 1.0, 0.5))
        parts.append((gate, up, down, wg, wu, wd, pre, post, cg))
    final = norm_pair(d, NormKind.Layer, 20)
    x = acts(m, d, F32)
    got_x, got_h = run_blocks(blocks, x, final[0], act_dtype=BF16)
    _, h = check_norm(x, None, None, parts[0][6], None, 1.0, 1.0, BF16)
    for i, (gate, up, down, wg, wu, wd, pre, post, cg) in enumerate(parts):
        a = gate.forward_gate_up_silu(up, h)
        b = down.forward(a)
        if wg is not None:
            hd, ad = h.double().cpu().numpy(), a.double().cpu().numpy()
            if rounded:
                hd, ad = (O.quantize(v, fmt is Fp4Format.Nv, 1.0)[3] for v in (hd, ad))
            near(a, O.product(hd, wg, up=wu), O.product_bound(hd, wg, d, up=wu))
            near(b, O.product(ad, wd), O.product_bound(ad, wd, ff))
        x, h = check_norm(x, b, None if cg is None else cg.to(BF16), parts[i + 1][6] if i == 0 else final, post, 1.0, 0.5, BF16)
    assert torch.equal(got_x, x) and torch.equal(got_h, h)
    assert torch.equal(blocks[0](acts(m, d, BF16)), run_blocks(blocks[:1], acts(m, d, BF16))[0])
    assert run_blocks([], x)[1] is None


def test_blocks_refuse_other_widths():
    w = Fp4Linear(quantize_fp4(torch.randn(64, 96, device="cuda")))
    with pytest.raises(ShrewError):
        GatedMlp(w, w, w, Norm())
