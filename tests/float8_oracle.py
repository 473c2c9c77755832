"""Plain numpy statements of the block-scaled 8-bit operations, in 64 bits except where the definition itself is a float
operation. Test infrastructure."""
import numpy as np

import ocean_hip as oh

E4M3, E5M2 = oh.FLOAT8_E4M3, oh.FLOAT8_E5M2
HALF, FLOAT, BF16 = oh.HALF, oh.FLOAT, oh.BFLOAT16
CODE_NAMES = {E4M3: "e4m3", E5M2: "e5m2"}
WIDE_NAMES = {HALF: "half", FLOAT: "float", BF16: "bfloat16"}
MOST = {E4M3: 448.0, E5M2: 57344.0}
# half a step of rounding, relative to the value, and half the smallest step
HALF_STEP = {HALF: 2.0 ** -11, FLOAT: 2.0 ** -24, BF16: 2.0 ** -8, E4M3: 2.0 ** -4, E5M2: 2.0 ** -3}
HALF_SMALLEST = {HALF: 2.0 ** -25, FLOAT: 2.0 ** -150, BF16: 2.0 ** -134, E4M3: 2.0 ** -10, E5M2: 2.0 ** -17}
STORAGE = {HALF: np.uint16, BF16: np.uint16, FLOAT: np.float32}


def _table(code):
    exponent_bits, mantissa_bits, bias = (4, 3, 7) if code == E4M3 else (5, 2, 15)
    out = np.zeros(256)
    for i in range(256):
        e, m = (i >> mantissa_bits) & ((1 << exponent_bits) - 1), i & ((1 << mantissa_bits) - 1)
        if code == E4M3 and (i & 0x7F) == 0x7F:
            v = np.nan
        elif code == E5M2 and e == 31:
            v = np.inf if m == 0 else np.nan
        else:
            v = (m / (1 << mantissa_bits)) * 2.0 ** (1 - bias) if e == 0 else (1 + m / (1 << mantissa_bits)) * 2.0 ** (e - bias)
        out[i] = -v if i & 0x80 else v
    return out


TABLE = {c: _table(c) for c in (E4M3, E5M2)}


def decode(q, code):
    return TABLE[code][np.asarray(q, np.uint8)]


def encode(v, code):
    """Nearest code of finite values within the code's range, ties to the even code; the sign of zero is kept."""
    v = np.asarray(v, np.float64)
    positive = TABLE[code][:128]
    positive = positive[np.isfinite(positive)]
    a = np.abs(v)
    hi = np.clip(np.searchsorted(positive, a), 0, len(positive) - 1)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - positive[lo], positive[hi] - a
    pick = np.where((dh < dl) | ((dh == dl) & (hi % 2 == 0)), hi, lo)
    return (pick | np.where(np.signbit(v), 0x80, 0)).astype(np.uint8)


def to_wide(x, dtype):
    """float values in the storage of a wide type (half and bfloat16 as 16-bit patterns), rounded to nearest even."""
    x = np.asarray(x)
    with np.errstate(over="ignore", invalid="ignore"):
        if dtype == FLOAT:
            return x.astype(np.float32)
        if dtype == HALF:
            return x.astype(np.float16).view(np.uint16)
        bits = np.ascontiguousarray(x.astype(np.float32)).view(np.uint32)
    nan = np.isnan(x)
    out = ((bits + 0x7FFF + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(nan, np.uint16(0x7FC0), out)


def from_wide(s, dtype):
    s = np.asarray(s)
    if dtype == FLOAT:
        return s.astype(np.float64)
    if dtype == HALF:
        return s.view(np.float16).astype(np.float64)
    return (s.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def spread(s, bm, bn, M, N):
    """The scale of every element: s [ceil(N / bn), ceil(M / bm)] -> [N, M] (rows of a numpy array are columns of the matrix)."""
    return np.repeat(np.repeat(s, bn, 0)[:N], bm, 1)[:, :M]


def block_maxima(x, bm, bn):
    """Largest magnitude of every block of x [N, M]; NaN where a block holds a NaN."""
    N, M = x.shape
    p = np.zeros((-(-N // bn) * bn, -(-M // bm) * bm), x.dtype)
    p[:N, :M] = np.abs(x)
    return p.reshape(p.shape[0] // bn, bn, p.shape[1] // bm, bm).max(axis=(1, 3))


def quantize(x, bm, bn, code):
    """Codes and scales of x [N, M] exactly as the operation is defined: in float32, one rounding per operation."""
    x = np.asarray(x, np.float32)
    N, M = x.shape
    amax = block_maxima(x, bm, bn)
    bad = ~np.isfinite(amax)
    a = np.maximum(np.where(bad, np.float32(1), amax), np.float32(2.0 ** -100))
    most = np.float32(MOST[code])
    scale, factor = np.where(bad, np.float32(np.nan), a / most), most / a
    with np.errstate(invalid="ignore", over="ignore"):
        t = np.clip(x * spread(factor, bm, bn, M, N), -most, most)
    wide_bad = spread(bad, bm, bn, M, N)
    q = np.where(wide_bad, np.uint8(0x7F), encode(np.where(wide_bad, 0, t), code))
    return q.astype(np.uint8), scale.astype(np.float32)


def values(q, s, bm, bn, code):
    return decode(q, code) * spread(s.astype(np.float64), bm, bn, q.shape[1], q.shape[0])


def norm(x, r, w, eps, dtype):
    """h, rstd, y of rows x [rows, n] (values of the wide type): the sum is rounded to the type, the rest is in 64 bits."""
    h = x if r is None else from_wide(to_wide((x.astype(np.float32) + r.astype(np.float32)), dtype), dtype)
    h = h.astype(np.float64)
    rstd = 1.0 / np.sqrt((h * h).mean(1) + np.float64(np.float32(eps)))
    return h, rstd, h * rstd[:, None] * w


def norm_grad(dy, h, w, rstd, dh):
    u = h * rstd[:, None]
    g = dy * w
    dx = rstd[:, None] * (g - u * (g * u).mean(1, keepdims=True))
    return dx + dh, (dy * u).sum(0)
