"""The paged cache's operators in numpy: blocks by GGUF's fp32 rules, rotation and attention in 64 bits."""
import numpy as np

F16, Q4_0, Q8_0 = 0, 1, 5
UNIT = {F16: 16, Q4_0: 4, Q8_0: 8}


def bf16_round(x):
    """fp32 to the nearest bf16 (ties to even), as fp32."""
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), np.float32(np.nan), r)


def rotate(x, pos, inv_freq, gain, dim, halves):
    """x fp32 [rows, heads, head_dim] -> fp32, rotated in 64 bits."""
    if dim == 0:
        return x.copy()
    ang = pos.astype(np.float64)[:, None] * inv_freq
    c, s = (np.cos(ang) * gain)[:, None], (np.sin(ang) * gain)[:, None]
    y, x = x.copy(), x.astype(np.float64)
    n = dim // 2
    a, b = (slice(0, n), slice(n, dim)) if halves else (slice(0, dim, 2), slice(1, dim, 2))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def codes(x, fmt):
    """fp32 [..., 32 n] -> whole numbers (q, not biased) and fp16 scales [..., n]."""
    blk = np.asarray(x, dtype=np.float32).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        bad = ~np.isfinite(blk).all(-1, keepdims=True)
        size = np.abs(blk)
        first = np.argmax(np.where(np.isnan(size), -1, size), -1)[..., None]  # numpy takes the lowest index of equals
        top = np.take_along_axis(blk, first, -1)
        d = top / np.float32(-8) if fmt == Q4_0 else np.abs(top) / np.float32(127)
        most = np.float32(8188) if fmt == Q4_0 else np.float32(515.5)  # values within fp16's range
        d = np.clip(d, -most, most).astype(np.float32)
        inv = np.where(d == 0, np.float32(0), np.float32(1) / d)
        y = blk * inv
        if fmt == Q4_0:
            q = np.clip(np.floor(y + np.float32(8.5)), 0, 15) - 8
        else:
            q = np.copysign(np.minimum(np.floor(np.abs(y) + np.float32(0.5)), 127), y)
        q, d = np.where(bad, 0, q), np.where(bad, np.nan, d)
    return q.reshape(x.shape), d[..., 0].astype(np.float16)


def stored(x, fmt):
    """The values a cache holds for fp32 x [..., head_dim], as fp64."""
    if fmt == F16:
        with np.errstate(over="ignore"):
            return np.asarray(x, np.float32).astype(np.float16).astype(np.float64)
    q, d = codes(x, fmt)
    return q * np.repeat(d.astype(np.float64), 32, -1)


def tile_bytes(fmt, hd):
    return 2 * (64 * (hd // 32) * UNIT[fmt] + (0 if fmt == F16 else hd))


def tile_value(tile, fmt, hd, keys, token, dim):
    """One value of a tile's bytes, by the header's formulas."""
    nb, unit = hd // 32, UNIT[fmt]
    lane = nb * unit
    vec = 16 if lane % 16 == 0 else 8 if lane % 8 == 0 else 4
    plane, scales = 64 * lane, 0 if fmt == F16 else hd
    b = dim // 32
    if keys:
        j, p, r, e = token // 8, 4 * (token % 8) + dim // 8 % 4, dim // 2 % 4, dim % 2
    else:
        j, p, r, e = token // 8, 4 * (dim // 4 % 8) + token // 2 % 4, dim % 4, token % 2
    first = 0 if keys else plane + scales

    def at(x):
        X = b * unit + x
        return first + j * 32 * lane + X // vec * 32 * vec + p * vec + X % vec

    if fmt == F16:
        o = at(2 * (2 * r + e))
        return float(tile[o:o + 2].view(np.float16)[0])
    o = first + plane + ((((token // 2 % 4) * 2 + token // 8) * nb + b) * 2 + token % 2) * 2
    d = float(tile[o:o + 2].view(np.float16)[0])
    if fmt == Q8_0:
        return (int(tile[at(2 * r + e)]) - 128) * d
    return ((int(tile[at((r >> 1) + 2 * e)]) >> (4 * (r & 1)) & 15) - 8) * d


def attention(q, keys, values, kv_len, scale, window=0):
    """q [n, heads, hd], keys and values [kv_len, kv_heads, hd] in 64 bits; row i sits at kv_len - n + i."""
    n, heads, hd = q.shape
    group = heads // keys.shape[1]
    out = np.zeros((n, heads, hd))
    for i in range(n):
        pos = kv_len - n + i
        lo = max(0, pos - window + 1) if window else 0
        if pos < 0:
            continue
        for h in range(heads):
            s = keys[lo:pos + 1, h // group] @ q[i, h].astype(np.float64) * scale
            p = np.exp(s - s.max())
            out[i, h] = p @ values[lo:pos + 1, h // group] / p.sum()
    return out


def attention_bound(q, keys, values, scale, bf16_out, half_operands=False):
    """How far a result may be off, from the arithmetic.  A score is a sum of head_dim products of q's two fp16 parts (2^-22 of
    q) with codes whose offset is taken back (at most 16 steps where a value is 8 or fewer: three times the sum of
    magnitudes bounds it), added in fp32 with truncation: head_dim * 2^-23 of that sum.  It moves every probability by
    its own size, so the result by twice that of the largest value.  Probabilities: two fp16 parts times a scale, relative to
    the largest scale seen, 2^-21; exponentials 2^-21; their sums in fp32 over the tokens, 2^-24 each in the mean.  bf16
    rounds by half a step, 2^-8 of the value.  With fp16 operands (half_operands) q, keys, probabilities and values are off
    by 2^-11 each."""
    size = np.abs(values).max() if values.size else 0.0
    dots = scale * np.abs(q).reshape(-1, q.shape[-1]).sum(-1).max() * np.abs(keys).max() if keys.size else 0.0
    ds = dots * 3 * (2.0 ** -22 + q.shape[-1] * 2.0 ** -23)
    rest = 2.0 ** -19 + len(keys) * 2.0 ** -24
    if half_operands:
        ds += dots * 2 * 2.0 ** -11
        rest += 2 * 2.0 ** -11
    return size * (2 * ds + rest + (2.0 ** -8 if bf16_out else 0.0))


def norm_bound(hd, q_size, k_size, half_operands):
    """2-norm of the error over the result's, for independent roundings: bf16's result is off by at most 2^-8 of itself; with
    fp16 operands each of hd products of a score is off by 2^-11 of itself twice, hd^(1/2) of that in their sum, and
    probabilities and values by 2^-11 each.  Twice the sum: an upper bound with room for the maxima."""
    score = 2 * 2.0 ** -11 * q_size * k_size * hd ** 0.5 * hd ** -0.5
    return 2.0 ** -8 + 2 * (score + 2 * 2.0 ** -11 if half_operands else 2.0 ** -19)


def fp32_norm_bound(score_size):
    """2-norm of an fp32 result's error over the result's, scores of standard deviation `score_size` (natural logarithms).
    An error of a score is one of its probability, and independent ones of all tokens pass into the result with the weights that
    the values themselves have.  A score is a sum over hd / 32 blocks, each of four products on the tensor cores (two steps of
    16 dimensions, q's two fp16 parts) whose running sum is cut at 2^-23 of itself; codes with their offset are 2.4 times as
    large as without, and a block's sum is score_size / (hd / 32)^(1/2): together 2 * 2.4 * 2^-23 score_size, with the blocks'
    sums in fp32 2^-20.5 score_size.  exp2, the two parts of a probability and of its product with a scale: 2^-21.
    Four times the sum, for what is not independent and for the largest of many."""
    return 4 * (score_size * 2.0 ** -20.5 + 2.0 ** -21)
