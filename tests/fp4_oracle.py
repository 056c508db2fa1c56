"""The 4-bit microscaled formats, the products over them and the norms around a block in 64 bits, from their definitions
(include/shrewq.h).  Test infrastructure: numpy only, no code of the package."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([np.ldexp((b & 7) / 8 + (1 if b >> 3 else 0), (b >> 3) - 7 + (0 if b >> 3 else 1)) for b in range(127)])  # 0 .. 448


def nearest(values, table):
    """Index of the nearest entry of an ascending table, ties to the even index, saturating."""
    hi = np.clip(np.searchsorted(table, values), 1, len(table) - 1)
    lo = hi - 1
    a, b = values - table[lo], table[hi] - values
    return np.where((a < b) | ((a == b) & (lo % 2 == 0)), lo, hi)


def quantize(x, nv, g=None):
    """x [rows, cols] -> (codes [rows, kp/2] u8, scales u8, g or None, values f64 [rows, cols])."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    block, kp = (16 if nv else 32), -(-cols // 32) * 32
    v = np.zeros((rows, kp))
    v[:, :cols] = x
    if nv and g is None:
        finite = np.abs(v[np.isfinite(v)])
        top = finite.max() if finite.size else 0.0
        g = 1.0
        if top > 0:
            g = 2.0 ** -126
            while g * 2688.0 < top:
                g *= 2.0
    if nv:
        with np.errstate(over="ignore", invalid="ignore"):
            v = (v.astype(np.float32) * np.float32(1.0) * (np.float32(1.0) / np.float32(g))).astype(np.float64)  # the one rounding in f32 before the blocks
    v = v.reshape(rows, -1, block)
    amax = np.abs(v).max(-1)
    bad = ~np.isfinite(amax)
    safe = np.where(bad | (amax == 0), 1.0, amax)
    if nv:
        byte = nearest(np.clip(safe / 6.0, 2.0 ** -9, 448.0), E4M3)
        byte = np.where(amax == 0, 0x38, byte)
        scale = E4M3[byte]
        byte = np.where(bad, 0x7F, byte)
    else:
        e = np.clip(np.frexp(safe)[1] - 3, -127, 127)
        e = np.where(amax == 0, 0, e)
        scale = np.ldexp(1.0, e)
        byte = np.where(bad, 255, e + 127)
    clean = np.where(bad[..., None], 0.0, v)
    code = nearest(np.abs(clean) / scale[..., None], GRID) + 8 * (np.signbit(clean) & ~bad[..., None])
    values = np.where(code >= 8, -1.0, 1.0) * GRID[code & 7] * np.where(bad, np.nan, scale)[..., None]
    code = code.reshape(rows, kp)
    values = values.reshape(rows, kp)[:, :cols]
    if nv:
        values = values * float(np.float32(g))
    return (code[:, 0::2] | code[:, 1::2] << 4).astype(np.uint8), byte.astype(np.uint8), g, values


def dequantize(codes, scales, g, cols, nv):
    """Values in 64 bits of any codes and scales."""
    rows = codes.shape[0]
    code = np.stack([codes & 15, codes >> 4], -1).reshape(rows, -1)
    v = np.where(code >= 8, -1.0, 1.0) * GRID[code & 7]
    if nv:
        table = np.append(E4M3, np.nan)
        s = np.where(scales & 0x80, -1.0, 1.0) * table[scales & 0x7F]
    else:
        s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    v = v * np.repeat(s, 16 if nv else 32, axis=1)
    return (v * (float(np.float32(g)) if nv else 1.0))[:, :cols]


def product(x, w, bias=None, up=None, bias_up=None, relu=False):
    """x [M, K] . w [N, K]^T in 64 bits, with the epilogue of the layer or of a gated pair."""
    with np.errstate(invalid="ignore", over="ignore"):
        y = x @ w.T + (0 if bias is None else bias.astype(np.float64))
        if up is not None:
            u = x @ up.T + (0 if bias_up is None else bias_up.astype(np.float64))
            return y / (1.0 + np.exp(-y)) * u
        return np.maximum(y, 0.0) if relu else y


def product_bound(x, w, k, up=None, bias=None, bias_up=None):
    """How far f32 sums of k exact products may be from the exact sum, element by element: (k + 24) * 2^-24 * sum |x| |w|, the bound of
    any order of summation (each of at most k additions is off by 2^-24 of a partial sum, and no partial sum is larger; the matrix
    instructions may truncate instead, 2^-23, which the factor 2 covers), plus the scaling and the bias."""
    def one(w, b):
        return 2.0 * (k + 24) * 2.0 ** -24 * (np.abs(x) @ np.abs(w).T + (0 if b is None else np.abs(b)))
    if up is None:
        return one(w, bias)
    # silu(y) * u: |d silu| <= 1.1 |dy|, |silu(y)| <= |y|; exp and the division are good to a few ulp: 2^-20 of the value
    y, u = x @ w.T + (0 if bias is None else bias), x @ up.T + (0 if bias_up is None else bias_up)
    return 1.1 * one(w, bias) * np.abs(u) + np.abs(y) * one(up, bias_up) + 1.1 * one(w, bias) * one(up, bias_up) + 2.0 ** -20 * np.abs(y * u)


def norm(v, kind, weight=None, bias=None, eps=1e-5):
    """kind: 1 RMS, 2 layer."""
    if kind == 2:
        v = v - v.mean(-1, keepdims=True)
    v = v / np.sqrt((v * v).mean(-1, keepdims=True) + eps)
    return v * (1.0 if weight is None else weight) + (0.0 if bias is None else bias)


def residual_norm(x, branch=None, gate=None, pre=None, post=None, residual_scale=1.0, branch_scale=1.0):
    """pre, post: None or (kind, weight, bias, eps).  -> (r, h or None)"""
    r = residual_scale * x
    if branch is not None:
        b = branch if post is None else norm(branch, *post)
        r = r + branch_scale * (b if gate is None else b * gate)
    return r, None if pre is None else norm(r, *pre)
