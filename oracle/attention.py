"""Plain forms of the attention operators (include/consumer_int8_attention.h), on the CPU.

`norm_rope32` and `fp4_quantize` follow the operators' stated FP32 roundings one by one, so
codes can be compared bit for bit; `norm_rope64` and `attention64` are the formulas in 64
bits, with the magnitudes that error bounds are made of.
"""

import numpy as np

F32 = np.float32
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
BF16_ROUND = 2.0**-8  # largest relative error of a rounding to BF16's 8 significant bits


def bf16_half_ulp(x):
    """Largest error of rounding a value of magnitude up to |x| to BF16: half the spacing of
    its binade."""
    _, exp = np.frexp(np.abs(x))
    return np.ldexp(1.0, np.maximum(exp, -125) - 9)


def fp4_scale_bytes(amax):
    """E8M0 bytes of blocks with the largest magnitudes amax (FP32): the smallest e with
    amax <= 7 * 2^e, held in -125 .. 125; 255 where amax is infinite or NaN."""
    amax = np.asarray(amax, dtype=np.float64)
    bad = ~np.isfinite(amax)
    safe = np.where(bad, 1.0, amax)
    mant, exp = np.frexp(safe)  # safe = mant * 2^exp, 0.5 <= mant < 1
    e = np.clip(np.where(safe > 0, exp - 3 + (mant > 0.875), -125), -125, 125)
    return np.where(bad, 255, e + 127).astype(np.uint8)


def fp4_quantize(x):
    """x FP32 [..., dim] -> packed codes uint8 [..., dim/2] and scales uint8 [..., dim/32]."""
    x = np.asarray(x, dtype=F32)
    blocks = x.reshape(*x.shape[:-1], -1, 32)
    magnitude = np.abs(blocks)
    amax = np.where(np.isnan(magnitude).any(-1), np.nan, magnitude.max(-1))
    scales = fp4_scale_bytes(amax)
    e = scales.astype(np.int64) - 127
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.ldexp(magnitude.astype(np.float64), -e[..., None])
        # thresholds between neighbouring codes; a tie goes to the even one
        code = ((y > 0.25).astype(np.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5)
                + (y >= 3.5) + (y > 5))
    code = code + 8 * np.signbit(blocks)
    code = np.where(scales[..., None] == 255, 0, code).astype(np.uint8).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def fp4_values(codes, scales):
    """The values of packed codes [..., dim/2] and scales [..., dim/32], float64."""
    codes = np.asarray(codes)
    dim = 2 * codes.shape[-1]
    both = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], dim)
    value = np.where(both & 8, -1.0, 1.0) * E2M1[both & 7]
    unit = np.where(np.asarray(scales) == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (value.reshape(*value.shape[:-1], dim // 32, 32) * unit[..., None]).reshape(value.shape)


def _angles(table, rot, positions, axes, dtype):
    """Cosines and sines [T, rot/2]; NaN outside the table."""
    table, positions = np.asarray(table), np.atleast_2d(positions)
    which = np.zeros(rot // 2, dtype=np.int64) if axes is None else np.asarray(axes)
    known = (which >= 0) & (which < len(positions))
    at = positions[np.where(known, which, 0)].T  # [T, rot/2]
    inside = known & (at >= 0) & (at < len(table))
    row, col = np.where(inside, at, 0), np.arange(rot // 2)
    cos, sin = table[row, col].astype(dtype), table[row, rot // 2 + col].astype(dtype)
    return np.where(inside, cos, np.nan), np.where(inside, sin, np.nan)


def _pair_index(rot, interleaved):
    i = np.arange(rot // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def norm_rope32(x, weight, eps, table, rot, positions, axes, interleaved):
    """x FP32 [T, H, dim], each operation rounded to FP32 in the operators' order."""
    x = np.asarray(x, dtype=F32)
    with np.errstate(all="ignore"):
        if weight is not None:
            s = x * x
            while s.shape[-1] > 1:
                s = s[..., 0::2] + s[..., 1::2]
            inv = F32(1) / np.sqrt(s * F32(1 / x.shape[-1]) + F32(eps))
            x = x * inv * np.asarray(weight, dtype=F32)
        if not rot:
            return x
        cos, sin = (v[:, None] for v in _angles(table, rot, positions, axes, F32))
        a, b = _pair_index(rot, interleaved)
        y = x.copy()
        y[..., a] = x[..., a] * cos - x[..., b] * sin
        y[..., b] = x[..., b] * cos + x[..., a] * sin
    assert y.dtype == F32
    return y


def norm_rope64(x, weight, eps, table, rot, positions, axes, interleaved):
    """The formula in 64 bits, and the sum of the magnitudes of each output's terms."""
    x = np.asarray(x, dtype=np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    if not rot:
        return x, np.abs(x)
    cos, sin = (v[:, None] for v in _angles(table, rot, positions, axes, np.float64))
    a, b = _pair_index(rot, interleaved)
    y, size = x.copy(), np.abs(x)
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    size[..., a] = np.abs(x[..., a] * cos) + np.abs(x[..., b] * sin)
    size[..., b] = np.abs(x[..., b] * cos) + np.abs(x[..., a] * sin)
    return y, size


def norm_rope_bound(y, size, dim):
    """How far a BF16 output may be from y: the rounding to BF16, and FP32 roundings of each
    term: the tree of log2(dim) sums and 4 more in the norm factor (halved by the root), 3
    products and 1 sum."""
    fp32 = size * (np.log2(dim) + 10) * 2.0**-24
    return bf16_half_ulp(np.abs(y) + fp32) + fp32


def attention64(q, k, v, high, low, scale):
    """One sequence and key head in 64 bits. q [R, dim], k and v [C, dim]; row r attends to
    tokens low[r] .. high[r]-1 (token t of `k` holding NaN rows is a caller's hole). Returns
    out, lse, the mean |v| under the weights, and how far a score may be off by the FP32 sums
    of its products (any order: dim - 1 additions of terms up to their sum of magnitudes, and
    2 roundings of the scaled score)."""
    q, k, v = (np.asarray(a, dtype=np.float64) for a in (q, k, v))
    t = np.arange(len(k))
    seen = (t >= np.asarray(low)[:, None]) & (t < np.asarray(high)[:, None])
    with np.errstate(all="ignore"):
        s = np.where(seen, q @ k.T * scale, -np.inf)
        off = np.where(seen, (np.abs(q) @ np.abs(k).T) * abs(scale), 0) * (k.shape[1] + 2) * 2.0**-24
        top = s.max(-1, keepdims=True, initial=-np.inf)
        top = np.where(np.isneginf(top), 0, top)
        w = np.exp(s - top)
        total = w.sum(-1, keepdims=True)
        p = np.where(seen, w / np.where(total == 0, 1, total), 0)
        out, mean = p @ v, p @ np.abs(v)
        lse = np.log(total[:, 0]) + top[:, 0]
    return out, lse, mean, off.max(-1, initial=0)


def attention_bounds(out, lse, mean, off):
    """How far out (BF16) and lse (FP32) may be: each weight is off by its score's error twice
    (once in the weight, once in the sum), by the base-2 exponentials (2^-21 for 2 of them
    with their arguments' roundings, of scores within 2^7 of the largest that count) and by its
    rounding to BF16; sums and joins of parts in FP32 stay under 2^-16; then one rounding."""
    weight = 2 * off[:, None] + BF16_ROUND + 2.0**-15
    inner = mean * weight
    return (bf16_half_ulp(np.abs(out) + inner) + inner,
            off + 2.0**-15 + np.abs(np.where(np.isfinite(lse), lse, 0)) * 2.0**-21)
