"""GPU: calls of the 4-bit operators that meet other calls: other quantizers of the context, captured graphs beside eager calls, values at the
ends of their ranges.  Through the package's public entry points, against the definitions in 64 bits (tests/fp4_oracle.py)."""
import numpy as np
import pytest
import torch

from shrew_b200 import Fp4Format, Fp4Linear, Fp4Tensor, Norm, QuantConfig, ShrewError, dequantize_fp4, quantize_fp4, quantize_tensor, run_blocks
from shrew_b200 import _lib
from shrew_b200.quantize import Device
from tests import fp4_oracle as O
from tests.test_gpu_fp4 import acts, layer, near

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def same(a, b):
    return torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and torch.equal(a.tensor_scale, b.tensor_scale)


# ---- the tensor's scale ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("config", [QuantConfig.int8(), QuantConfig.int4()])
def test_tensor_scales_leave_the_other_quantizers_alone(oracle, config):
    """Large NV tensors, more of them than a context has slots for per-tensor quantizing, then per-tensor integers of several blocks each."""
    g = torch.Generator().manual_seed(0)
    big = torch.randn(512, 2048, generator=g).cuda()
    small = [(torch.randn(300, 1000, generator=g) * (i + 1)).cuda() for i in range(9)]
    before = [quantize_tensor(x, config) for x in small]
    for i in range(17):
        quantize_fp4(big * (i + 1), Fp4Format.Nv)
    for x, b in zip(small, before):
        q = quantize_tensor(x, config)
        assert torch.equal(q.data, b.data) and torch.equal(q.scales, b.scales)
        assert float(q.scales[0]) == float(x.abs().max().double()) / (127.0 if config.bits.name == "Int8" else 7.0)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_tensor_scales_of_calls_in_flight_together(dtype):
    """A captured call replayed on one stream while eager calls run on another, and eager calls on many streams: every tensor gets its own scale."""
    g = torch.Generator().manual_seed(1)
    xs = [(torch.randn(300, 1024, generator=g) * 2.0 ** (3 * i - 12)).to(dtype).cuda() for i in range(9)]
    want = [quantize_fp4(x, Fp4Format.Nv) for x in xs]
    assert len({float(w.tensor_scale) for w in want}) == len(xs)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        captured = quantize_fp4(xs[-1], Fp4Format.Nv)
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        with torch.cuda.stream(side):
            for _ in range(40):
                graph.replay()
        got += [quantize_fp4(x, Fp4Format.Nv) for x in xs]
    torch.cuda.synchronize()
    assert same(captured, want[-1])
    assert all(same(q, want[i % len(xs)]) for i, q in enumerate(got))
    streams = [torch.cuda.Stream() for _ in range(24)]
    got = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            got.append(quantize_fp4(xs[i % len(xs)], Fp4Format.Nv))
    torch.cuda.synchronize()
    assert all(same(q, want[i % len(xs)]) for i, q in enumerate(got))


@pytest.mark.parametrize("shape", [(1, 1), (3, 40), (64, 64), (2000, 1024)])
def test_the_scale_of_nothing_but_zeros(shape):
    x = torch.zeros(shape, device="cuda")
    x[0, 0] = float("nan")   # (finite values count)
    q = quantize_fp4(x, Fp4Format.Nv)
    assert float(q.tensor_scale) == 1.0
    codes, scales, _, _ = O.quantize(x.double().cpu().numpy(), True)
    np.testing.assert_array_equal(q.scales.cpu().numpy(), scales)
    assert (dequantize_fp4(q).nan_to_num(0.0) == 0.0).all()


@pytest.mark.parametrize("words", [1, 2, 30, 92, 93, 2048])
def test_words_for_finding_a_scale(words):
    """As many as the caller gives (at 93 the parts of all 92 blocks fit): the same result, and nothing behind them is written."""
    x = torch.randn(367, 1024, generator=torch.Generator().manual_seed(3)).cuda()
    x[200, 5] = 1e4
    want = quantize_fp4(x, Fp4Format.Nv)
    whole = torch.full((words + 3,), -5.0, device="cuda")
    codes, scales = torch.empty_like(want.codes), torch.empty_like(want.scales)
    dev = Device.get(x.device)
    dev.bind_stream()
    args = (dev.handle, x.data_ptr(), _lib.F32, 367, 1024, 1024, _lib.FP4_NV, whole.data_ptr())
    assert _lib.lib().shrewq_quantize_fp4(*args, words, codes.data_ptr(), scales.data_ptr()) == _lib.OK
    assert float(whole[0]) == float(want.tensor_scale) == O.quantize(x.double().cpu().numpy(), True)[2]
    assert torch.equal(codes, want.codes) and torch.equal(scales, want.scales) and (whole[words:] == -5.0).all()
    assert _lib.lib().shrewq_quantize_fp4(*args, -1, codes.data_ptr(), scales.data_ptr()) == _lib.ERR_INVALID_ARG


def test_a_tensor_scale_beside_mx_is_refused():
    """As the quantizer and the layers refuse it, not left out."""
    q = quantize_fp4(torch.ones(4, 64, device="cuda"), Fp4Format.Mx)
    with pytest.raises(ShrewError) as e:
        dequantize_fp4(Fp4Tensor(q.codes, q.scales, torch.full((1,), 2.0, device="cuda"), q.shape, F32, Fp4Format.Mx))
    assert e.value.code == _lib.ERR_INVALID_ARG


# ---- layers -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("scale", [0.0, 0.5, -3.0, float("nan")])
@pytest.mark.parametrize("m", [1, 4, 8, 20, 40, 200])
def test_activations_as_they_come_have_no_scale(m, scale):
    gate, _, _ = layer(136, 320, Fp4Format.Nv, 1)
    up, _, _ = layer(136, 320, Fp4Format.Nv, 2)
    gate_s, up_s = Fp4Linear(gate.weight_q, gate.bias, activation_scale=scale), Fp4Linear(up.weight_q, up.bias, activation_scale=scale + 1.0)
    for x in (acts(m, 320, BF16), acts(m, 320, F32)):
        assert torch.equal(gate_s.forward(x), gate.forward(x))
        assert torch.equal(gate_s.forward_gate_up_silu(up_s, x), gate.forward_gate_up_silu(up, x))


@pytest.mark.parametrize("m", [3, 300])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_activations_far_above_their_scale_saturate(m, dtype):
    """Finite activations that activation_scale takes beyond f32 are the largest value that the format has beside it, not NaN."""
    lin, w, _ = layer(40, 96, Fp4Format.Nv, 1, bias=False, quantize_activations=True, activation_scale=1e-30)
    x = torch.full((m, 96), 1e20, dtype=dtype, device="cuda")
    x[1] = -1e20
    x[2, 32:] = 1e-30
    y = lin.forward(x, out_dtype=F32).double().cpu().numpy()
    s = float(np.float32(1e-30))
    xq = np.full((m, 96), 6.0 * 448.0 * s)
    xq[1] *= -1.0
    xq[2, 32:] = O.quantize(x[2:3, 32:].double().cpu().numpy(), True, s)[3][0]
    want = O.product(xq, w)
    assert (np.abs(y - want) <= O.product_bound(xq, w, 96) + 2.0 ** -24 * np.abs(want)).all()


@pytest.mark.parametrize("rounded", [False, True])
@pytest.mark.parametrize("m,n", [(2, 150), (9, 150), (40, 150), (300, 150), (300, 9000)])
@pytest.mark.parametrize("fmt", list(Fp4Format))
def test_relu_keeps_nan(fmt, m, n, rounded):
    lin, _, _ = layer(n, 256, fmt, 5, quantize_activations=rounded)
    x = acts(m, 256, BF16)
    x[1, 9] = float("nan")
    y, r = lin.forward(x), lin.forward(x, epilogue=_lib.EPILOGUE_RELU)
    assert r[1].isnan().all() and torch.equal(r[0], y[0].clamp(min=0.0)) and torch.equal(r[2:], y[2:].clamp(min=0.0))


@pytest.mark.parametrize("rounded,x_dtype,most", [(True, _lib.BF16, 2 ** 31 - 257), (True, _lib.F32, 2 ** 31 - 257), (False, _lib.BF16, 2 ** 31 - 257),
                                                  (False, _lib.F32, 715827626)])
def test_more_tokens_than_indexes_hold_are_refused(rounded, x_dtype, most):
    """On the host, before anything of them is read."""
    lin, _, _ = layer(1, 32, Fp4Format.Mx, 1, quantize_activations=rounded)
    x = torch.zeros(64, device="cuda")
    for m in (most + 1, 2 ** 31 - 1):
        assert _lib.lib().shrewq_linear_forward(lin._h, x.data_ptr(), x_dtype, m, x.data_ptr(), _lib.F32, 1, 0) == _lib.ERR_UNSUPPORTED


@pytest.mark.parametrize("m", [6, 20, 32])
def test_gated_layers_of_many_tiles_in_turn_captured_and_on_streams(m):
    """The kernels of 5 to 32 tokens over more tiles than SMs, and over few, one after the other: the same bits eagerly, on another stream and replayed."""
    gate, wg, _ = layer(9600, 2080, Fp4Format.Nv, 1, bias=False)
    up, wu, _ = layer(9600, 2080, Fp4Format.Nv, 2, bias=False)
    down, wd, _ = layer(2080, 9600, Fp4Format.Nv, 3, bias=False)
    xs = [acts(m, 2080, BF16, seed=s) * 0.01 for s in range(3)]

    def run(x):
        return down.forward(gate.forward_gate_up_silu(up, x))
    h = gate.forward_gate_up_silu(up, xs[0])
    assert gate.last_kernel() == "tcgen05-w4-f16"
    xd = xs[0].double().cpu().numpy()
    near(h, O.product(xd, wg, up=wu), O.product_bound(xd, wg, 2080, up=wu))
    want = [run(x) for x in xs]
    assert down.last_kernel() == "tcgen05-w4"
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


@pytest.mark.parametrize("name", [b"gemv", b"mma", b"tcgen05", b"simt"])
def test_forced_kernels_do_not_take_these_layers(name):
    lin, _, _ = layer(32, 64, Fp4Format.Mx, 1)
    x = acts(2, 64, BF16)
    want = lin.forward(x)
    assert _lib.lib().shrewq_force_kernel(name) == _lib.OK
    try:
        for call in (lambda: lin.forward(x), lambda: lin.forward_gate_up_silu(lin, x)):
            with pytest.raises(ShrewError) as e:
                call()
            assert e.value.code == _lib.ERR_UNSUPPORTED
    finally:
        assert _lib.lib().shrewq_force_kernel(b"auto") == _lib.OK
    assert torch.equal(lin.forward(x), want)


# ---- blocks -------------------------------------------------------------------------------------------------------------------
def test_no_blocks_and_their_type():
    x = acts(5, 64, F32)
    r, h = run_blocks([], x, Norm(), act_dtype=BF16)
    assert r is x and h.dtype is BF16 and torch.equal(h, run_blocks([], x, Norm())[1].to(BF16))
