"""Plain 64-bit forms of the NVFP4 cache and of attention with capped, biased and masked scores, for their tests."""
import numpy as np

F32, BF16 = 0, 1                  # XTG_X_*
KV = {"bf16": 0, "fp8": 1, "nvfp4": 2}


def bf16_bits(a):
    """BF16 bits (uint16) of FP32 values, to nearest even; NaN and infinities stay what they are."""
    b = np.ascontiguousarray(a, dtype=np.float32).view(np.uint32).astype(np.uint64)
    nan = (b & 0x7fffffff) > 0x7f800000
    r = ((b + 0x7fff + ((b >> np.uint64(16)) & np.uint64(1))) >> np.uint64(16)).astype(np.uint16)
    return np.where(nan, ((b >> np.uint64(16)) | np.uint64(0x40)).astype(np.uint16), r)


def bf16_values(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def bf16(a):
    return bf16_values(bf16_bits(a))


def rows(a, x_dtype):
    """What a call is given for FP32 values a, and the values that it means."""
    return (bf16_bits(a), bf16(a)) if x_dtype == BF16 else (np.ascontiguousarray(a, np.float32), np.asarray(a, np.float32))


def nearest(y, bits, low):
    """y >= 0 to `bits` significant bits with a step of at least `low`, ties to even (in 64 bits: exact here)."""
    e = np.frexp(y)[1]
    step = np.maximum(np.ldexp(1.0, e - bits), low)
    return np.rint(y / step) * step


def stored_nvfp4(x, glob=1.0):
    """The values an NVFP4 cache holds of one array's rows [...][d]; rows that are not finite are left to the caller."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], x.shape[-1] // 16, 16) / glob
    amax = np.abs(b).max(axis=-1, keepdims=True)
    with np.errstate(all="ignore"):
        s = np.where(amax >= 2688, 448.0, nearest(np.minimum(amax, 2688) / 6, 4, 2.0 ** -9))
        s = np.where(amax > 0, np.maximum(s, 2.0 ** -9), 1.0)
        c = np.minimum(nearest(np.abs(b) / s, 2, 0.5), 6.0)
    return (c * s * np.sign(b) * glob).reshape(x.shape)


def stored_pair(k, v, dtype, globals_=(1.0, 1.0)):
    """(K, V) rows [n][kv][d] as a cache of `dtype` holds them, in 64 bits."""
    if dtype == "bf16":
        return bf16(k).astype(np.float64), bf16(v).astype(np.float64)
    if dtype == "fp8":
        return stored_fp8(k), stored_fp8(v)
    bad = ~(np.isfinite(k).all(-1, keepdims=True) & np.isfinite(v).all(-1, keepdims=True))
    return tuple(np.where(bad, np.nan, stored_nvfp4(np.where(bad, 0, x), g)) for x, g in zip((k, v), globals_))


def stored_fp8(x):
    """E4M3 codes of x / scale with scale amax / 448 per (row, head), computed as the store does in FP32; a NaN is
    one itself and does not count for its row's scale."""
    x = np.asarray(x, np.float32)
    amax = np.fmax.reduce(np.abs(x), axis=-1, keepdims=True, initial=np.float32(0))
    s = np.where(amax > 0, amax / np.float32(448), np.float32(1)).astype(np.float32)
    y = (x * (np.float32(1) / s)).astype(np.float64)
    return np.minimum(nearest(np.abs(y), 4, 2.0 ** -9), 448.0) * np.sign(y) * s.astype(np.float64)


def attend(q, k, v, at, pos0, scale, window=0, softcap=0.0, slopes=None, first=None, end=None):
    """q [n][heads][d] over keys k, v [m][kv][d] at positions `at` [m] (64-bit values). Returns the outputs, the sum of
    |weight * value| that each is made of with 2^-32 of the sum of |value| (weights are at least the size of f16's
    smallest step, 2^-24, or lost: with the largest at 2^7 or more, by half a step, 2^-32 of it), and the largest sum
    of |q.k| * scale of a score (for tolerances)."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    n, heads, d = q.shape
    kvh = k.shape[1]
    t = pos0 + np.arange(n)
    lo = np.zeros(n) if first is None else np.maximum(np.asarray(first, np.float64), 0)
    if window > 0:
        lo = np.maximum(lo, t - window + 1)
    hi = t + 1 if end is None else np.asarray(end)
    seen = (at[None, :] >= lo[:, None]) & (at[None, :] < hi[:, None]) & (at[None, :] >= 0)
    out, size, floor, most = np.zeros_like(q), np.zeros_like(q), np.zeros_like(q), 0.0
    with np.errstate(all="ignore"):
        for h in range(heads):
            kh, vh = k[:, h * kvh // heads], v[:, h * kvh // heads]
            for i in range(n):   # only what the row sees: values in masked places do not count
                w = seen[i]
                if not w.any():
                    continue
                s = (kh[w] @ q[i, h]) * scale
                part = np.abs(kh[w]) @ np.abs(q[i, h]) * abs(scale)
                most = max(most, float(np.max(part[np.isfinite(part)], initial=0.0)))
                if softcap > 0:
                    s = softcap * np.tanh(s / softcap)
                if slopes is not None:
                    bias = float(slopes[h]) * np.abs(t[i] - at[w])
                    s = s - bias
                    most = max(most, float(bias.max()))
                p = np.exp(s - s.max())
                p /= p.sum()
                out[i, h] = (p[:, None] * vh[w]).sum(0)
                size[i, h] = (p[:, None] * np.abs(vh[w])).sum(0)
                floor[i, h] = np.abs(vh[w]).sum(0) * 2.0 ** -32
    return out, (size, floor), most


def tolerance(out, size, most, d, weight_bits, x_dtype):
    """How far an output may be off. The softmax weights are rounded to weight_bits significant bits (half a step:
    2^-weight_bits of each); a score is a sum of d products in FP32 and a few further FP32 roundings of its value, each
    at most 2^-24 of the terms' sum `most`, and an error e of a score is one of about e of its weight and of their sum;
    the product with V and the sum of the weights are FP32 sums, whose error grows with their length (below 2^15
    terms: 2^-9 of the largest bound, 2^-17 in practice for sums of mixed order: 2^-14 is allowed); BF16 rows are
    rounded once more, by half a step, 2^-8."""
    e = (d + 16) * 2.0 ** -24 * (most + 1.0)
    tol = size[0] * (2.0 ** -weight_bits + 2 * e + 2.0 ** -14) + size[1] + 1e-30
    return tol + (np.abs(out) + tol) * 2.0 ** -8 if x_dtype == BF16 else tol
