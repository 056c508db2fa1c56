"""GPU: 4-bit layers and quantizers where the result is known bit for bit: products whose partial sums all fit f32, so that a dropped block, row, term
or bit shows whatever the size, and the quantizer at every scale and every border between codes.  Through the package's public entry points."""
import numpy as np
import pytest
import torch

from shrew_b200 import Fp4Format, Fp4Linear, Fp4Tensor, quantize_fp4
from shrew_b200.quantize import mlp_forward_host
from tests import fp4_oracle as O
from tests.test_gpu_fp4 import acts, layer

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
FORMATS = [Fp4Format.Mx, Fp4Format.Nv]
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def stored(code, fmt, scale_exponent=0, nan_block=None):
    """Codes [n, k] (0 .. 15) with every scale a power of two, as a layer's weight."""
    n, k = code.shape
    c = torch.zeros(n, -(-k // 32) * 32, dtype=torch.uint8)
    c[:, :k] = code
    nv = fmt is Fp4Format.Nv
    scales = torch.full((n, c.shape[1] // fmt.block), 0x38 if nv else 127 + scale_exponent, dtype=torch.uint8)
    if nan_block is not None:
        scales[nan_block] = 0x7F if nv else 255
    g = torch.tensor([2.0 ** scale_exponent]).cuda() if nv else None
    return Fp4Tensor((c[:, 0::2] | c[:, 1::2] << 4).cuda(), scales.cuda(), g, [n, k], F32, fmt)


def values(code):
    return torch.where(code >= 8, -1.0, 1.0) * GRID[(code & 7).long()]


def codes(n, k, seed):
    return torch.randint(0, 16, (n, k), generator=torch.Generator().manual_seed(seed), dtype=torch.uint8)


def tokens(m, k, dtype, seed):
    """Values of the 4-bit grid, a 6 in every block of 16: they are their own quantization, with scales of 1."""
    x = values(codes(m, k, seed))
    x[:, ::16] = 6.0
    return x.to(dtype).cuda()


MS = [1, 2, 4, 5, 16, 17, 32, 33, 64, 65, 128, 129, 300]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("k,n", [(1, 3), (33, 40), (257, 130), (2049, 70), (4096, 130), (11008, 9), (2080, 19100)])
@pytest.mark.parametrize("m", MS)
def test_sums_are_exact(fmt, m, n, k):
    """Multiples of 1/4 below 36 k < 2^19: every partial sum has less than 24 bits, so f32 sums in any order are the exact sum."""
    code = codes(n, k, n)
    want = values(code).double()
    w = stored(code, fmt)
    plain, rounded = Fp4Linear(w), Fp4Linear(w, quantize_activations=True)
    for dtype in (BF16, F32):
        x = tokens(m, k, dtype, m)
        y = x.double().cpu() @ want.t()
        for lin in (plain, rounded):
            assert torch.equal(lin.forward(x, out_dtype=F32).double().cpu(), y)
            assert torch.equal(lin.forward(x, out_dtype=BF16).cpu(), y.to(F32).to(BF16))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("k,n", [(2049, 70), (4096, 130), (480, 9500)])
@pytest.mark.parametrize("m", [1, 4, 5, 32, 33, 128, 300])
def test_gated_sums_are_exact(fmt, m, n, k):
    """As above for both sums of a gated pair; silu(g) * u then has the errors of its own operations: exp(-g) to (2 + 1.2 |g|) units, the
    addition, the division and the product to 2 units each at most, 2^-23 a unit."""
    if n * m > 1 << 20 and k > 1000:
        m = 129
    cg, cu = codes(n, k, 1), codes(n, k, 2)
    wg, wu = values(cg).double() * 2.0 ** -7, values(cu).double() * 2.0 ** -7
    x = tokens(m, k, F32, m)
    g, u = x.double().cpu() @ wg.t(), x.double().cpu() @ wu.t()
    want = torch.sigmoid(g) * g * u
    for rounded in (False, True):
        lin = [Fp4Linear(stored(c, fmt, -7), quantize_activations=rounded) for c in (cg, cu)]
        h = lin[0].forward_gate_up_silu(lin[1], x).double().cpu()
        assert ((h - want).abs() <= (8 + 1.2 * g.abs()) * 2.0 ** -23 * want.abs() + 2.0 ** -120).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("k,times", [(96, 1), (333, 1), (1056, 1), (2080, 10)])
@pytest.mark.parametrize("m", MS)
def test_every_column_and_every_bit(fmt, k, times, m):
    """Each channel is one column of x with a factor of 2: f32 activations with all their 24 bits, the smallest 2^-12 of the largest."""
    lin = Fp4Linear(stored((torch.eye(k, dtype=torch.uint8) * 4).repeat(times, 1), fmt))
    g = torch.Generator().manual_seed(m + k)
    x = (torch.rand(m, k, generator=g) + 1.0) * torch.exp2(-torch.randint(0, 13, (m, k), generator=g).float()) * torch.where(torch.rand(m, k, generator=g) < 0.5, -1.0, 1.0)
    x = x.cuda()
    want, want16 = (2.0 * x).repeat(1, times), (2.0 * x.to(BF16).float()).repeat(1, times)
    assert torch.equal(lin.forward(x), want)
    assert torch.equal(lin.forward(x, out_dtype=BF16), want.to(BF16))
    assert torch.equal(lin.forward(x.to(BF16), out_dtype=F32), want16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("k", [32, 96, 256, 4096, 8192])
@pytest.mark.parametrize("m,n", [(m, 70) for m in MS] + [(5, 9600), (20, 9600), (300, 9600)])
def test_low_bits_of_f32_activations_survive_long_sums(fmt, m, n, k):
    """x = 1 + 2^-12 + 2^-20 in every column and weights of 1 and -1: k times 21 bits, k one or three times a power of two, so that the sums of the
    leading and of the low parts fit f32 and so does their sum (23 bits); added up together, the low parts fall below the last place."""
    sign = torch.randint(0, 2, (n, 1), generator=torch.Generator().manual_seed(k), dtype=torch.uint8)
    lin = Fp4Linear(stored((2 + 8 * sign).expand(n, k).contiguous(), fmt))
    x = torch.full((m, k), 1.0 + 2.0 ** -12 + 2.0 ** -20, device="cuda")
    want = ((1.0 - 2.0 * sign.double()) * k * (1.0 + 2.0 ** -12 + 2.0 ** -20)).view(1, n).expand(m, n)
    assert torch.equal(want.float().double(), want)
    assert torch.equal(lin.forward(x).double().cpu(), want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rounded", [False, True])
@pytest.mark.parametrize("m,n", [(1, 150), (8, 150), (8, 19100), (40, 150), (200, 150), (300, 9500)])
def test_a_nan_block_stays_in_its_channel(fmt, rounded, m, n):
    code = codes(n, 320, 3)
    bad, clean = (Fp4Linear(stored(code, fmt, nan_block=b), quantize_activations=rounded) for b in ((77, 9), None))
    x = tokens(m, 320, BF16, 5)
    y, want = bad.forward(x), clean.forward(x)
    assert y[:, 77].isnan().all()
    y[:, 77] = want[:, 77]
    assert torch.equal(y, want)


@pytest.mark.parametrize("m", [1, 6, 20, 32, 40])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [50, 19100])
def test_scales_far_apart(dtype, n, m):
    """Block scales over 90 octaves: what stands in the blocks of small scales alone comes out as exactly as the rest."""
    k = 2080
    code = codes(n, k, 1)
    w = stored(code, Fp4Format.Mx)
    e = torch.randint(-90, 1, (n, k // 32), generator=torch.Generator().manual_seed(2))
    e[:, 0] = 0
    w.scales.copy_((127 + e).to(torch.uint8))
    lin = Fp4Linear(w)
    x = torch.zeros(m, k)
    block = 1 + torch.arange(m) % (k // 32 - 1)
    for i in range(m):   # (values of the grid, in one block each)
        x[i, 32 * block[i]:32 * block[i] + 32] = values(codes(1, 32, i))[0]
    y = lin.forward(x.to(dtype).cuda(), out_dtype=F32).double().cpu()
    wd = values(code).double().view(n, -1, 32) * torch.exp2(e.double())[..., None]
    assert torch.equal(y, x.double() @ wd.view(n, k).t())


@pytest.mark.parametrize("m,n,k,dtype,gated,name", [
    (4, 4096, 4096, BF16, False, "mma-fp4"), (4, 128, 11008, BF16, False, "tcgen05-w4"), (16, 4096, 4096, BF16, False, "tcgen05-w4"), (8, 9600, 4096, BF16, False, "tcgen05-w4-f16"),
    (16, 9600, 4096, BF16, False, "tcgen05-w4"), (8, 9600, 8192, BF16, False, "tcgen05-w4"), (32, 9536, 2048, BF16, True, "tcgen05-w4-f16"),
    (32, 9472, 2048, BF16, True, "tcgen05-w4"), (32, 19072, 2016, BF16, False, "tcgen05-w4"), (7, 19072, 64, BF16, False, "tcgen05-w4-f16"), (5, 9600, 4096, F32, False, "tcgen05-w4-f16"), (6, 9600, 4096, F32, False, "tcgen05-w4"), (33, 19072, 4096, BF16, False, "tcgen05-w4")])
def test_which_kernel_takes_a_call(m, n, k, dtype, gated, name):
    """On the 148 SMs of a B200."""
    lin = Fp4Linear(stored(torch.zeros(n, k, dtype=torch.uint8), Fp4Format.Mx))
    x = torch.zeros(m, k, dtype=dtype, device="cuda")
    y = lin.forward_gate_up_silu(lin, x) if gated else lin.forward(x)
    assert lin.last_kernel() == name and (y == 0).all()


# ---- the quantizer ------------------------------------------------------------------------------------------------------------
def borders(s):
    """For block scales s: values that ask for them and every border between codes, on it and next to it."""
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    at = (s[:, None] * ties).float()
    rows = []
    for shift in (at, torch.nextafter(at, torch.tensor(float("inf"))), torch.nextafter(at, torch.tensor(0.0))):
        block = torch.zeros(s.numel(), 16)
        block[:, 0] = 6.0 * s.float()
        block[:, 1:8], block[:, 8:15] = shift, -shift
        rows.append(block)
    return torch.cat(rows)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("given", [False, True])
def test_nv_at_every_scale_and_border(dtype, given):
    """All 126 scales of E4M3 with every border of their codes, and every border between two scales; as one stream of rows and row by row."""
    e4m3 = torch.from_numpy(O.E4M3[1:])
    between = 6.0 * (e4m3[1:] + e4m3[:-1]) / 2.0
    tops = torch.cat([between, torch.nextafter(between.float(), torch.tensor(0.0)).double(), torch.nextafter(between.float(), torch.tensor(float("inf"))).double()])
    tail = torch.zeros(tops.numel(), 16)
    tail[:, 3] = tops.float()
    tail[:, 4:] = tops.float()[:, None] * torch.linspace(-1, 1, 12)
    x = torch.cat([borders(e4m3), tail]).to(dtype).view(-1)
    x = torch.cat([x, torch.zeros(-x.numel() % 32, dtype=dtype)])
    for cols in (32, 16, x.numel()):
        t = x.view(-1, cols)
        q = quantize_fp4(t.cuda(), Fp4Format.Nv, torch.ones(1, device="cuda") if given else None)
        c, s, g, _ = O.quantize(t.double().numpy(), True, 1.0 if given else None)
        assert given or float(q.tensor_scale) == g == 1.0
        np.testing.assert_array_equal(q.scales.cpu().numpy(), s)
        got, want = q.codes.cpu().numpy(), c
        for shift in (0, 4):   # (the sign of a zero is not specified)
            a, b = got >> shift & 15, want >> shift & 15
            np.testing.assert_array_equal(np.where(a == 8, 0, a), np.where(b == 8, 0, b))


# ---- host buffers ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rounded", [False, True])
@pytest.mark.parametrize("m", [1, 7, 50])
def test_a_block_on_host_buffers(fmt, rounded, m):
    (gate, _, _), (up, _, _), (down, _, _) = (layer(n, k, fmt, i, quantize_activations=rounded) for i, (n, k) in enumerate(((136, 96), (136, 96), (96, 136))))
    xs = [acts(m, 96, BF16, seed=s) * 0.05 for s in range(5)]
    want = [down.forward(gate.forward_gate_up_silu(up, x)).cpu() for x in xs]
    assert all(torch.equal(mlp_forward_host(gate, up, down, x.cpu()), w) for x, w in zip(xs, want))
    pinned = [x.cpu().pin_memory() for x in xs]
    out = [torch.empty(m, 96, dtype=BF16).pin_memory() for _ in xs]
    for x, y in zip(pinned, out):
        mlp_forward_host(gate, up, down, x, out=y, synchronize=False)
    gate.device.synchronize()
    assert all(torch.equal(y, w) for y, w in zip(out, want))
    y32 = mlp_forward_host(gate, up, down, xs[0].cpu(), out_dtype=F32)
    assert torch.equal(y32.to(BF16), want[0])
