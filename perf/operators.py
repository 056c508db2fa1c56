"""The measured operators: 4-bit microscaled weights, their products, and the norms around a block.

  roundtrip   quantize_fp4 of a tensor and dequantize_fp4 of the result: a checkpoint's weight on its way in, checked or served
  dequantize  dequantize_fp4 of a stored weight
  linear      Fp4Linear.forward, or forward_gate_up_silu of two: activations as they come, or rounded to 4 bits as well
  norm        residual_norm: what stands between two blocks: the norm after one, its gate and the residual scale, the norm before the next

Formats: "mx" has blocks of 32 along a row with a power-of-two scale (E8M0), "nv" blocks of 16 with an E4M3 scale and one f32
scale for the tensor; the codes are E2M1, two to a byte, rows padded to whole 32s.
"""
import math

import torch

own = False

_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one large f32 weight of a model that is being quantized
        dict(name="roundtrip_mx_f32_8192x8192", kind="roundtrip", rows=8192, cols=8192, x="f32", format="mx"),
        # the up projection of a Llama-shaped block from a bf16 checkpoint, with its tensor scale found on the way
        dict(name="roundtrip_nv_bf16_11008x4096", kind="roundtrip", rows=11008, cols=4096, x="bf16", format="nv"),
        # a narrow vocabulary head with an odd number of rows, back to f32
        dict(name="dequantize_mx_50257x256", kind="dequantize", rows=50257, cols=256, y="f32", format="mx"),
        # a stored down projection back to bf16
        dict(name="dequantize_nv_4096x11008", kind="dequantize", rows=4096, cols=11008, y="bf16", format="nv"),
        # a decoding step: one projection for one token
        dict(name="linear_mx_4096_m1", kind="linear", n=4096, k=4096, m=1, x="bf16", y="bf16", format="mx", round_x=False,
             gated=False, bias=True, relu=False),
        # 16 sequences decoded together through the gate and up projections
        dict(name="gate_up_nv_11008x4096_m16", kind="linear", n=11008, k=4096, m=16, x="bf16", y="bf16", format="nv", round_x=False,
             gated=True, bias=False, relu=False),
        # a prompt of ragged length through a down projection
        dict(name="linear_mx_4096x11008_m250", kind="linear", n=4096, k=11008, m=250, x="bf16", y="bf16", format="mx", round_x=False,
             gated=False, bias=True, relu=False),
        # 32 sequences decoded with activations in 4 bits too
        dict(name="linear4_mx_4096_m32", kind="linear", n=4096, k=4096, m=32, x="bf16", y="bf16", format="mx", round_x=True,
             gated=False, bias=True, relu=False),
        # prefill of 512 tokens through gate and up, 4 bits by 4 bits
        dict(name="gate_up4_nv_11008x4096_m512", kind="linear", n=11008, k=4096, m=512, x="bf16", y="bf16", format="nv", round_x=True,
             gated=True, bias=False, relu=False),
        # the largest: a long prefill through a down projection, 4 bits by 4 bits
        dict(name="linear4_mx_4096x11008_m4096", kind="linear", n=4096, k=11008, m=4096, x="bf16", y="bf16", format="mx", round_x=True,
             gated=False, bias=False, relu=False),
        # between two blocks of a decoding step, one token: all latency
        dict(name="norm_rms_m1_4096", kind="norm", m=1, d=4096, x="bf16", branch="bf16", y="bf16", pre="rms", post="none", gate="none",
             residual_scale=1.0, branch_scale=1.0),
        # the same place in a prefill of 4096 tokens, with a norm after the block, a gate for each channel and a scaled residual
        dict(name="norm_rms_post_m4096_4096", kind="norm", m=4096, d=4096, x="f32", branch="bf16", y="bf16", pre="rms", post="rms",
             gate="channel", residual_scale=1.0, branch_scale=0.5),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A layer width: mostly a multiple of 64, as model widths are, sometimes only of 16, sometimes any number."""
    v, r = _log_int(rng, lo, hi), rng.random()
    step = 64 if r < 0.7 else (16 if r < 0.85 else 1)
    return max(step, v // step * step)


def draw(rng):
    kind = rng.choices(["roundtrip", "dequantize", "linear", "norm"], [3, 2, 7, 3])[0]
    fmt = rng.choice(["mx", "nv"])
    if kind in ("roundtrip", "dequantize"):
        cols = _width(rng, 16, 16384)
        rows = _log_int(rng, 1, min(60000, (1 << 26) // cols))
        if kind == "roundtrip":
            return dict(kind=kind, rows=rows, cols=cols, x=rng.choice(["f32", "bf16", "f16"]), format=fmt)
        return dict(kind=kind, rows=rows, cols=cols, y=rng.choice(["f32", "bf16", "f16"]), format=fmt)
    if kind == "norm":
        d = _width(rng, 16, 16384)
        m = _log_int(rng, 1, min(16384, (1 << 25) // d))
        post, x = rng.choice(["none", "rms", "layer"]), rng.choice(["f32", "bf16"])
        return dict(kind=kind, m=m, d=d, x=x, branch=rng.choice(["f32", "bf16"]), y=rng.choice(["f32", "bf16"]),
                    pre=rng.choice(["rms", "rms", "layer"]), post=post, gate=rng.choice(["none", "channel", "token", "full"]),
                    residual_scale=rng.choice([1.0, 1.0, 0.75]), branch_scale=rng.choice([1.0, 0.5, 0.22]))
    round_x = rng.random() < 0.5
    gated = rng.random() < 0.35
    n, k, m = _width(rng, 16, 16384), _width(rng, 64, 11008), _log_int(rng, 1, 4096)
    n = min(n, (1 << 26) // k)
    x = rng.choice(["bf16", "bf16", "bf16", "f32"])
    most = 1 << 37 if round_x else 1 << (35 if x == "bf16" else 33)
    m = max(1, min(m, most // (n * k * (2 if gated else 1))))
    return dict(kind="linear", n=n, k=k, m=m, x=x, y=x if gated else rng.choice([x, x, "f32"]), format=fmt, round_x=round_x,
                gated=gated, bias=rng.random() < 0.5, relu=not gated and rng.random() < 0.25)


# ---- inputs -------------------------------------------------------------------------------------------------------
def _weight(g, rows, cols, dtype):
    """Weights: normal, rows of different size, a few large entries."""
    w = torch.randn(rows, cols, generator=g, device="cuda") * 0.02
    w *= torch.exp(0.3 * torch.randn(rows, 1, generator=g, device="cuda"))
    w *= 1.0 + 5.0 * (torch.rand(rows, cols, generator=g, device="cuda") < 1e-4)
    return w.to(dtype)


def _acts(g, rows, cols, dtype):
    """Activations: normal, with a few channels much larger than the rest."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    return (x * (1.0 + 10.0 * (torch.rand(1, cols, generator=g, device="cuda") < 0.005))).to(dtype)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "roundtrip":
        return {"x": _weight(g, case["rows"], case["cols"], _DTYPE[case["x"]])}
    if kind == "dequantize":
        return {"w": [_weight(g, case["rows"], case["cols"], torch.float32)]}
    if kind == "linear":
        n, k, m = case["n"], case["k"], case["m"]
        layers = 2 if case["gated"] else 1
        return {"w": [_weight(g, n, k, torch.float32) for _ in range(layers)],
                "bias": [0.1 * torch.randn(n, generator=g, device="cuda") if case["bias"] else None for _ in range(layers)],
                "x": _acts(g, m, k, _DTYPE[case["x"]])}
    m, d = case["m"], case["d"]
    one = {"channel": (d,), "token": (m, 1), "full": (m, d)}
    return {"x": _acts(g, m, d, _DTYPE[case["x"]]), "branch": _acts(g, m, d, _DTYPE[case["branch"]]),
            "gate": torch.randn(one[case["gate"]], generator=g, device="cuda").to(_DTYPE[case["branch"]]) if case["gate"] != "none" else None,
            "pre": [1.0 + 0.1 * torch.randn(d, generator=g, device="cuda"), 0.1 * torch.randn(d, generator=g, device="cuda")],
            "post": [1.0 + 0.1 * torch.randn(d, generator=g, device="cuda"), 0.1 * torch.randn(d, generator=g, device="cuda")]}


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    if "w" in s:  # stored weights: codes and scales
        s["w"] = [_pack(*_quantize(w, case["format"])) for w in s["w"]]
    if not own:
        return s
    from shrew_b200 import Fp4Format, Fp4Linear, Fp4Tensor, Norm, NormKind
    fmt = {"mx": Fp4Format.Mx, "nv": Fp4Format.Nv}
    if case["kind"] == "roundtrip":
        s["format"] = fmt[case["format"]]
    if "w" in s:
        shape = [case["rows"], case["cols"]] if case["kind"] == "dequantize" else [case["n"], case["k"]]
        dtype = _DTYPE[case.get("y", "f32")]
        s["w"] = [Fp4Tensor(codes, scales, whole, shape, dtype, fmt[case["format"]]) for codes, scales, whole in s["w"]]
    if case["kind"] == "linear":
        s["layers"] = [Fp4Linear(w, b, quantize_activations=case["round_x"]) for w, b in zip(s["w"], s["bias"])]
    if case["kind"] == "norm":
        kinds = {"rms": NormKind.Rms, "layer": NormKind.Layer}
        for which in ("pre", "post"):
            kind = case[which]
            s["norm_" + which] = None if kind == "none" else Norm(kinds[kind], s[which][0], s[which][1] if kind == "layer" else None, eps=1e-5)
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        from shrew_b200 import dequantize_fp4, quantize_fp4, residual_norm
        if kind == "roundtrip":
            return dequantize_fp4(quantize_fp4(s["x"], s["format"]))
        if kind == "dequantize":
            return dequantize_fp4(s["w"][0])
        if kind == "linear":
            if case["gated"]:
                return s["layers"][0].forward_gate_up_silu(s["layers"][1], s["x"])
            return s["layers"][0].forward(s["x"], epilogue=1 if case["relu"] else 0, out_dtype=_DTYPE[case["y"]])
        return residual_norm(s["x"], s["branch"], s["gate"], pre=s["norm_pre"], post=s["norm_post"], residual_scale=case["residual_scale"],
                             branch_scale=case["branch_scale"], out_dtype=_DTYPE[case["y"]])
    if kind == "roundtrip":
        return _values(*_quantize(s["x"], case["format"])[:3])[:, :case["cols"]].to(s["x"].dtype)
    if kind == "dequantize":
        return _unpack(s["w"][0], case["format"])[:, :case["cols"]].to(_DTYPE[case["y"]])
    if kind == "linear":
        x = s["x"].float()
        if case["round_x"]:
            x = _values(*_quantize(s["x"], case["format"], whole=torch.ones(1, device="cuda"))[:3])[:, :case["k"]]
        y = [_plain_linear(x, w, b, case) for w, b in zip(s["w"], s["bias"])]
        if case["gated"]:
            return (y[0] / (1.0 + torch.exp(-y[0])) * y[1]).to(_DTYPE[case["y"]])
        return (torch.clamp(y[0], min=0.0) if case["relu"] else y[0]).to(_DTYPE[case["y"]])
    b = s["branch"].float()
    if case["post"] != "none":
        b = _plain_norm(b, case["post"], *s["post"])
    if s["gate"] is not None:
        b = b * s["gate"].float()
    r = case["residual_scale"] * s["x"].float() + case["branch_scale"] * b
    return r.to(s["x"].dtype), _plain_norm(r, case["pre"], *s["pre"]).to(_DTYPE[case["y"]])


# ---- the plain forms ------------------------------------------------------------------------------------------------
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _power(e):
    """2^e as f32 for whole e in [-149, 127]."""
    return torch.ldexp(torch.ones_like(e, dtype=torch.float64), e).float()


def _over(a, b):
    """a / b rounded once (a division by a plain number multiplies by its rounded reciprocal on the GPU)."""
    return a / torch.full_like(a, b)


def _quantize(x, fmt, whole=None):
    """E2M1 codes [rows, blocks, block] (0..15), block scales as f32, the tensor scale, and the scales' bytes."""
    block = 32 if fmt == "mx" else 16
    x = torch.nn.functional.pad(x.float(), (0, -x.shape[1] % 32)).view(x.shape[0], -1, block)
    if fmt == "nv":
        if whole is None:  # the smallest power of two that brings the largest block scale under 448
            mant, e = torch.frexp(_over(x.abs().max(), 2688.0))
            whole = torch.where(mant > 0, _power(torch.where(mant == 0.5, e - 1, e)), 1.0).view(1)
        x = x * (1.0 / whole)
    amax = x.abs().amax(-1, keepdim=True)
    mant, e = torch.frexp(amax)
    if fmt == "mx":  # the largest value's power of two, brought under E2M1's (2^2)
        e = torch.where(amax > 0, torch.clamp(e - 3, min=-127), 0)
        scale, byte = _power(e), (e + 127).to(torch.uint8)
    else:  # amax / 6, to three bits after the point (fewer below 2^-6); a scale of 1 for a block of zeros
        want = torch.clamp(_over(amax, 6.0), min=2.0 ** -9, max=448.0)
        step = _power(torch.clamp(torch.frexp(want)[1] - 1, min=-6) - 3)
        scale = torch.where(amax > 0, torch.clamp(torch.round(want / step) * step, max=448.0), 1.0)
        byte = scale.to(torch.float8_e4m3fn).view(torch.uint8)
    v = x / scale
    a = v.abs()  # ties go to the even code
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return code + 8 * (torch.signbit(x)).to(torch.uint8), scale, whole, byte


def _values(code, scale, whole):
    grid = torch.tensor(_GRID + tuple(-v for v in _GRID), device=code.device)
    v = grid[code.int()] * scale
    return (v if whole is None else v * whole).flatten(1)


def _pack(code, scale, whole, byte):
    code = code.flatten(1)
    return (code[:, 0::2] + 16 * code[:, 1::2]).contiguous(), byte.flatten(1).contiguous(), whole


def _unpack(stored, fmt):
    codes, scales, whole = stored
    code = torch.stack((codes % 16, codes // 16), -1).view(codes.shape[0], -1, 32 if fmt == "mx" else 16)
    scale = _power(scales.int() - 127) if fmt == "mx" else scales.view(torch.float8_e4m3fn).float()
    return _values(code, scale.view(code.shape[0], -1, 1), whole)


def _plain_linear(x, stored, bias, case):
    y = x @ _unpack(stored, case["format"])[:, :case["k"]].t()
    return y if bias is None else y + bias


def _plain_norm(v, kind, weight, bias):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
        return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-5) * weight + bias
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-5) * weight


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def _stored_bytes(rows, cols, fmt):
    blocks = -(-cols // 32)
    return rows * blocks * (16 + (1 if fmt == "mx" else 2))


def work(case):
    kind = case["kind"]
    if kind in ("roundtrip", "dequantize"):
        values = case["rows"] * case["cols"]
        stored = _stored_bytes(case["rows"], case["cols"], case["format"])
        return {"bytes": stored + values * (2 * _SIZE[case["x"]] if kind == "roundtrip" else _SIZE[case["y"]]), "flops": 0}
    if kind == "linear":
        n, k, m, layers = case["n"], case["k"], case["m"], 2 if case["gated"] else 1
        return {"bytes": layers * (_stored_bytes(n, k, case["format"]) + (4 * n if case["bias"] else 0)) + m * k * _SIZE[case["x"]] +
                m * n * _SIZE[case["y"]], "flops": 2 * layers * m * n * k}
    m, d = case["m"], case["d"]
    gate = {"none": 0, "channel": d, "token": m, "full": m * d}[case["gate"]]
    vectors = (1 if case["pre"] == "rms" else 2) + {"none": 0, "rms": 1, "layer": 2}[case["post"]]
    return {"bytes": m * d * (2 * _SIZE[case["x"]] + _SIZE[case["branch"]] + _SIZE[case["y"]]) + gate * _SIZE[case["branch"]] + 4 * d * vectors,
            "flops": 0}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------
def _exact_round(v):
    """To the nearest of 0, 0.5 .. 2 by halves, 2 .. 4 by ones, 4 and 6: ties to the even multiple of the step."""
    a = v.abs()
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0)).double()
    return torch.sign(v) * torch.clamp(torch.round(a / step) * step, max=6.0)


def _exact_floor2(v):
    """The largest power of two that is not above v > 0 (its exponent field alone), in 64 bits."""
    return ((v.view(torch.int64) >> 52) << 52).view(torch.float64)


def _exact_quantized(x, fmt, whole=None):
    """The values that a quantized x stands for, [rows, cols] in 64 bits."""
    rows, cols = x.shape
    block = 32 if fmt == "mx" else 16
    blocks = -(-cols // block)
    v = torch.zeros(rows, blocks * block, dtype=torch.float64, device=x.device)
    v[:, :cols] = x.double()
    if fmt == "nv" and whole is None:
        top = float(v.abs().max())
        whole = 2.0 ** -126
        while whole * 2688.0 < top:
            whole *= 2.0
        whole = whole if top > 0 else 1.0
    whole = 1.0 if whole is None else whole
    v = (v / whole).view(rows, blocks, block)
    amax = v.abs().amax(-1, keepdim=True)
    if fmt == "mx":
        scale = _exact_floor2(torch.clamp(amax, min=2.0 ** -125)) / 4.0
    else:
        s = torch.clamp(amax / torch.full_like(amax, 6.0), min=2.0 ** -9, max=448.0)
        step = torch.clamp(_exact_floor2(s), min=2.0 ** -6) / 8.0
        scale = torch.clamp(torch.round(s / step) * step, max=448.0)
    scale = torch.where(amax > 0, scale, torch.ones_like(scale))
    return (_exact_round(v / scale) * scale * whole).view(rows, -1)[:, :cols]


def _exact_norm(v, kind, weight, bias):
    if kind == "layer":
        return (v - v.mean(-1, keepdim=True)) / torch.sqrt(v.var(-1, unbiased=False, keepdim=True) + 1e-5) * weight.double() + bias.double()
    return v / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-5) * weight.double()


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "roundtrip":
        return _exact_quantized(s["x"], case["format"])
    if kind == "dequantize":
        return _exact_quantized(s["w"][0], case["format"])
    if kind == "linear":
        x = _exact_quantized(s["x"], case["format"], whole=1.0) if case["round_x"] else s["x"].double()
        y = [torch.matmul(x, _exact_quantized(w, case["format"]).T) + (0.0 if b is None else b.double()) for w, b in zip(s["w"], s["bias"])]
        if case["gated"]:
            return torch.sigmoid(y[0]) * y[0] * y[1]
        return y[0].relu() if case["relu"] else y[0]
    b = s["branch"].double()
    if case["post"] != "none":
        b = _exact_norm(b, case["post"], *s["post"])
    if s["gate"] is not None:
        b = b * s["gate"].double()
    r = s["x"].double() * case["residual_scale"] + b * case["branch_scale"]
    return r, _exact_norm(r, case["pre"], *s["pre"])
