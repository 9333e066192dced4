"""Feed-forward operators restated in 64 bits (numpy): the Philox4x32-10 keep mask, activation + dropout, residual join
with its norms (both directions, from the formulas), and the rounding to e4m3 with block scales."""
import math

import numpy as np

M32 = np.uint64(0xFFFFFFFF)


def philox4x32(counter, key, rounds=10):
    """counter: four uint64 arrays of 32-bit words, key: two ints -> four arrays (Salmon, Moraes, Dror, Shaw 2011)."""
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k0, k1 = key
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & M32, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & M32]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def threshold(p):
    return int(p) * 65536 if p in (0, 1) else min(65535, max(1, round(p * 65536)))


def keep_mask(index, p, seed, offset, call):
    """bool per linear element index (any int array)."""
    index = np.asarray(index, dtype=np.uint64)
    j = index >> np.uint64(3)
    counter = (j & M32, ((j >> np.uint64(32)) & np.uint64(0xFFFF)) | np.uint64(call << 16),
               np.full_like(j, offset & 0xFFFFFFFF), np.full_like(j, (offset >> 32) & 0xFFFFFFFF))
    w = np.stack(philox4x32(counter, (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF)), -1)
    i = (index & np.uint64(7)).astype(np.int64)
    word = np.take_along_axis(w, (i >> 1)[..., None], -1)[..., 0]
    return ((word >> (np.uint64(16) * (i & 1).astype(np.uint64))) & np.uint64(0xFFFF)) >= np.uint64(threshold(p))


def drop_scale(p, seed, offset, call, shape, start=0):
    """keep * 65536 / (65536 - T) of a tensor's elements."""
    n = int(np.prod(shape))
    if p == 0:
        return np.ones(shape)
    t = threshold(p)
    k = keep_mask(np.arange(start, start + n, dtype=np.uint64), p, seed, offset, call).reshape(shape)
    return np.where(k, 65536.0 / max(65536 - t, 1), 0.0)


_erf = np.vectorize(math.erf, otypes=[np.float64])


def act(x, kind):
    if kind == "relu":
        return np.maximum(x, 0)
    if kind == "gelu":
        return x * 0.5 * (1 + _erf(x / math.sqrt(2)))
    return x


def act_grad(x, kind):
    if kind == "relu":
        return (x > 0).astype(np.float64)
    if kind == "gelu":
        return 0.5 * (1 + _erf(x / math.sqrt(2))) + x * np.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    return np.ones_like(x)


def normalise(t, kind, eps):
    """(normalised rows, mean, factor)."""
    mean = t.mean(-1, keepdims=True) if kind == "layer" else np.zeros_like(t[..., :1])
    if kind in ("layer", "rms"):
        r = 1 / np.sqrt(((t - mean) ** 2).mean(-1, keepdims=True) + eps)
    else:
        r = np.ones_like(mean)
    return (t - mean) * r, mean, r


def normalise_grad(t, n, r, kind):
    if kind not in ("layer", "rms"):
        return t
    m1 = t.mean(-1, keepdims=True) if kind == "layer" else 0.0
    return r * (t - m1 - n * (t * n).mean(-1, keepdims=True))


# ---- e4m3 with block scales --------------------------------------------------------------------------------------------
def block_exponents(x, rows):
    """int [ceil(R / rows), ceil(C / 128)]: smallest e >= -126 with max |finite| <= 448 * 2^e."""
    R, C = x.shape
    v = np.where(np.isfinite(x), np.abs(x), 0.0)
    v = np.pad(v, ((0, -R % rows), (0, -C % 128))).reshape(-(-R // rows), rows, -(-C // 128), 128).max((1, 3))
    m, e = np.frexp(v / 448.0)                       # exact: 448 = 7 * 64 divides into doubles of fp32 values to < 1 ulp
    e = np.where(m > 0.5, e, e - 1)
    e = np.where(v <= 448.0 * np.exp2((e - 1).astype(np.float64)), e - 1, e)
    e = np.where(v > 448.0 * np.exp2(e.astype(np.float64)), e + 1, e)
    return np.maximum(np.where(v > 0, e, -126), -126).astype(np.int64)


def round_e4m3(t):
    """nearest e4m3 value, ties to even; non-finite and beyond the range -> NaN."""
    t = np.asarray(t, dtype=np.float64)
    with np.errstate(invalid="ignore"):
        _, e = np.frexp(np.where(np.isfinite(t), t, 0.0))
        step = np.exp2(np.maximum(e, -5).astype(np.float64) - 4)
        q = np.round(t / step) * step
        return np.where(np.isfinite(t) & (np.abs(q) <= 448), q, np.nan)


def quantise(x, rows=1):
    """[R, C] -> what its e4m3 bytes and scales stand for."""
    x = np.asarray(x, dtype=np.float64)
    R, C = x.shape
    s = np.exp2(block_exponents(x, rows).astype(np.float64)).repeat(rows, 0)[:R].repeat(128, 1)[:, :C]
    return round_e4m3(x / s) * s
