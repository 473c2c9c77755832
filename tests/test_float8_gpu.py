"""The block-scaled 8-bit operations on the device against plain numpy statements of them (float8_oracle).

Tolerances. A rounding is off by at most half a step, u = 2^-24 relative for float. quantize_blocks is defined by single
float operations: codes and scales are equal bit for bit. The other operations sum in float: a sum of n terms in any order
is within d u sum|terms| of the exact one, d the longest chain of additions; the chains are at most 8 per vector, one
addition per vector that a thread takes (n / 2048 at the longest rows, 16 below 32768), and 16 to join threads."""
import ctypes as C

import numpy as np
import pytest

import float8_oracle as F
import ocean_hip as oh

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
WIDE = [F.HALF, F.BF16, F.FLOAT]
CODES = [F.E4M3, F.E5M2]
name_of = lambda v: F.WIDE_NAMES.get(v) or F.CODE_NAMES.get(v) or str(v)      # noqa: E731


def chain(n):
    return 40 + n / 2048


class Matrix:
    """cols columns of `rows` elements with leading dimension ld, inside a buffer whose other bytes hold a pattern; the
    first element lies `shift` elements into the buffer."""

    def __init__(self, stream, rows, cols, dtype, ld=None, shift=0, data=None):
        self.rows, self.cols, self.dtype, self.ld = rows, cols, np.dtype(dtype), ld or max(rows, 1)
        self.shift = shift
        n = shift + self.ld * max(cols, 1) + 64
        self.host = np.full(n * self.dtype.itemsize, 0xA5, np.uint8).view(self.dtype)
        if data is not None:
            self._view(self.host)[...] = data
        self.buf = oh.to_device(self.host.view(np.uint8), stream)

    def _view(self, flat):
        return np.lib.stride_tricks.as_strided(flat[self.shift:], (self.cols, self.rows), (self.ld * self.dtype.itemsize, self.dtype.itemsize))

    @property
    def ptr(self):
        return C.c_void_p(self.buf.address + self.shift * self.dtype.itemsize)

    def read(self):
        """The matrix as [cols, rows]; checks that no byte around it was written."""
        flat = self.buf.download(np.uint8, self.host.nbytes).view(self.dtype)
        around, before = flat.copy(), self.host.copy()
        self._view(around)[...] = 0
        self._view(before)[...] = 0
        assert np.array_equal(around.view(np.uint8), before.view(np.uint8)), "bytes outside the matrix were written"
        return self._view(flat).copy()

    def free(self):
        self.buf.free()


def wide_data(rng, cols, rows, dtype, scale=1.0):
    """Values as a layer sees them: features of different size."""
    feature = np.exp(0.7 * rng.standard_normal(rows))
    return F.to_wide(rng.standard_normal((cols, rows)) * feature * scale, dtype)


# ---- quantize_blocks --------------------------------------------------------------------------------------------------

def run_quantize(stream, x, dtype, code, bm, bn, ldx=None, ldq=None, lds=None, shift=0):
    N, M = x.shape
    X = Matrix(stream, M, N, F.STORAGE[dtype], ldx, shift, x)
    Q = Matrix(stream, M, N, np.uint8, ldq, shift)
    S = Matrix(stream, -(-M // bm), -(-N // bn), np.float32, lds, shift)
    oh.check(oh.lib.och_quantize_blocks(dtype, code, M, N, X.ptr, X.ld, bm, bn, Q.ptr, Q.ld, S.ptr, S.ld, stream.handle))
    q, s = Q.read(), S.read()
    for m in (X, Q, S):
        m.free()
    return q, s


def same_codes(got, want):
    q, s = got
    wq, ws = want
    assert np.array_equal(s.view(np.uint32) & 0x7FFFFFFF, ws.view(np.uint32) & 0x7FFFFFFF)
    assert np.array_equal(q, wq)


@pytest.mark.parametrize("bm,bn", [(128, 1), (1, 128), (128, 128)])
@pytest.mark.parametrize("code", CODES, ids=name_of)
@pytest.mark.parametrize("dtype", WIDE, ids=name_of)
def test_quantize(hip, stream, dtype, code, bm, bn):
    rng = np.random.default_rng(dtype * 100 + code + bm)
    for M, N, pad, shift in [(1, 1, 0, 0), (128, 1, 0, 0), (129, 128, 0, 0), (256, 129, 8, 8), (1000, 37, 3, 1), (4, 300, 1, 3), (2048, 130, 0, 0), (4111, 2, 0, 5)]:
        x = wide_data(rng, N, M, dtype)
        got = run_quantize(stream, x, dtype, code, bm, bn, M + pad, M + pad + 1, -(-M // bm) + pad, shift)
        same_codes(got, F.quantize(F.from_wide(x, dtype), bm, bn, code))


@pytest.mark.parametrize("bm,bn", [(128, 1), (1, 128), (128, 128)])
@pytest.mark.parametrize("dtype", WIDE, ids=name_of)
def test_quantize_special_values(hip, stream, dtype, bm, bn):
    """Zeros, subnormal blocks, the type's largest value, infinities and NaN: a block with one of the last two is NaN
    throughout, its neighbours are as without it."""
    rng = np.random.default_rng(5)
    M, N = 640, 270
    v = rng.standard_normal((N, M))
    v[:, :128] = 0
    v[:130, 128:256] *= 2.0 ** -120 if dtype != F.HALF else 2.0 ** -24
    v[140:, 256:300] = {F.HALF: 65504.0, F.BF16: 3.3895313892515355e38, F.FLOAT: np.finfo(np.float32).max}[dtype]
    v[3, 400], v[200, 401], v[7, 639] = np.inf, -np.inf, np.nan
    x = F.to_wide(v, dtype)
    for code in CODES:
        q, s = run_quantize(stream, x, dtype, code, bm, bn)
        want = F.quantize(F.from_wide(x, dtype), bm, bn, code)
        same_codes((q, np.where(np.isnan(s), np.float32(np.nan), s)), want)
        assert np.isnan(s).sum() == np.isnan(want[1]).sum() > 0


@pytest.mark.parametrize("code", CODES, ids=name_of)
def test_every_rounding_of_a_code(hip, stream, code):
    """All codes, the middles between them and their neighbours, in blocks whose factor is exactly 1."""
    positive = F.TABLE[code][:128]
    positive = positive[np.isfinite(positive)]
    middle = ((positive[1:] + positive[:-1]) / 2).astype(np.float32)
    v = np.concatenate([positive.astype(np.float32), middle, np.nextafter(middle, np.float32(1e9)), np.nextafter(middle, np.float32(0))])
    v = np.concatenate([v, -v])
    v = np.concatenate([v, np.zeros(-len(v) % 127, np.float32)]).reshape(-1, 127)
    x = np.concatenate([np.full((len(v), 1), F.MOST[code], np.float32), v], 1)
    q, s = run_quantize(stream, x, F.FLOAT, code, 128, 1)
    assert (s == 1).all()
    assert np.array_equal(q, F.encode(x, code))


# ---- rms_norm ---------------------------------------------------------------------------------------------------------

def run_norm(stream, x, r, w, dtype, dtype_w, dtype_y, eps=1e-5, pad=0, shift=0, in_place=None, want_h=True, want_rstd=True):
    rows, n = x.shape
    st, coded = F.STORAGE[dtype], dtype_y != dtype
    X = Matrix(stream, n, rows, st, n + pad, shift, x)
    R = Matrix(stream, n, rows, st, n + 2 * pad, shift, r) if r is not None else None
    H = {"x": X, "r": R}.get(in_place) or (Matrix(stream, n, rows, st, n + pad, 0) if want_h else None)
    W = Matrix(stream, n, 1, F.STORAGE[dtype_w], None, shift, w) if w is not None else None
    Y = X if in_place == "y" else Matrix(stream, n, rows, np.uint8 if coded else st, n + pad, shift)
    S = Matrix(stream, -(-n // 128), rows, np.float32, -(-n // 128) + pad) if coded else None
    T = Matrix(stream, rows, 1, np.float32) if want_rstd else None
    at = lambda m: m.ptr if m is not None else None      # noqa: E731
    ld = lambda m: m.ld if m is not None else 0          # noqa: E731
    oh.check(oh.lib.och_rms_norm(dtype, n, rows, X.ptr, X.ld, at(R), ld(R), at(H), ld(H), dtype_w, at(W), eps, dtype_y, Y.ptr, Y.ld, at(S), ld(S), at(T), stream.handle))
    out = {"y": Y.read(), "h": H.read() if H is not None else None, "s": S.read() if coded else None, "rstd": T.read()[0] if T is not None else None}
    for m in {id(m): m for m in (X, R, H, W, Y, S, T) if m is not None}.values():
        m.free()
    return out


def check_norm(out, x, r, w, dtype, dtype_w, dtype_y, eps=1e-5):
    xv, rv = F.from_wide(x, dtype), None if r is None else F.from_wide(r, dtype)
    wv = np.ones(x.shape[1]) if w is None else F.from_wide(w, dtype_w)
    h, rstd, y = F.norm(xv, rv, wv, eps, dtype)
    n = x.shape[1]
    near = (chain(n) / 2 + 6) * U             # the sum's error halves in the root; root, division, mean, eps and the products round once each
    if out["h"] is not None:
        want = F.to_wide(h, dtype)
        assert np.array_equal(out["h"], want)                            # one float addition and one rounding
    if out["rstd"] is not None:
        assert np.abs(out["rstd"] - rstd).max(initial=0) <= near * np.abs(rstd).max(initial=0)
        assert (np.abs(out["rstd"] - rstd) <= near * rstd).all()
    if dtype_y == dtype:
        got = F.from_wide(out["y"], dtype)
        assert (np.abs(got - y) <= (F.HALF_STEP[dtype] * (1 + near) + near) * np.abs(y) + F.HALF_SMALLEST[dtype]).all()
    else:
        scale = np.maximum(F.block_maxima(y, 128, 1), 2.0 ** -100) / F.MOST[dtype_y]
        assert (np.abs(out["s"] - scale) <= (near + 2 * U) * scale).all()
        wide = F.spread(out["s"].astype(np.float64), 128, 1, n, len(y))
        got = F.decode(out["y"], dtype_y) * wide
        assert (np.abs(got - y) <= (F.HALF_STEP[dtype_y] + 4 * near) * np.abs(y) + F.HALF_SMALLEST[dtype_y] * wide * (1 + near)).all()


SHAPES = [(1, 1), (1, 64), (3, 127), (200, 128), (77, 129), (5, 256), (9, 500), (2, 1000), (33, 1024), (4, 2048), (17, 2560), (300, 4096), (3, 5003),
          (2, 8192), (1, 16384), (2, 16385), (2, 20001), (1, 40000)]


@pytest.mark.parametrize("dtype_y", ["same"] + CODES, ids=name_of)
@pytest.mark.parametrize("dtype", WIDE, ids=name_of)
def test_norm(hip, stream, dtype, dtype_y):
    rng = np.random.default_rng(dtype + 7)
    dtype_y = dtype if dtype_y == "same" else dtype_y
    for k, (rows, n) in enumerate(SHAPES):
        dtype_w = dtype if k % 2 else F.FLOAT
        x, r = wide_data(rng, rows, n, dtype), wide_data(rng, rows, n, dtype, 3.0) if k % 3 else None
        w = F.to_wide(1 + 0.2 * rng.standard_normal(n), dtype_w) if k % 5 else None
        pad, shift = [(0, 0), (8, 8), (3, 1)][k % 3]
        out = run_norm(stream, x, r, w, dtype, dtype_w, dtype_y, pad=pad, shift=shift, want_h=bool(r is not None or k % 2), want_rstd=bool(k % 4))
        check_norm(out, x, r, w, dtype, dtype_w, dtype_y)


@pytest.mark.parametrize("n", [96, 640, 3000, 24000])
@pytest.mark.parametrize("where", ["x", "r", "y"])
def test_norm_in_place(hip, stream, where, n):
    """The sum over X or R, and the output over X."""
    rng = np.random.default_rng(n)
    dtype = F.BF16
    x, r = wide_data(rng, 5, n, dtype), wide_data(rng, 5, n, dtype)
    w = F.to_wide(1 + 0.2 * rng.standard_normal(n), F.FLOAT)
    if where == "y":
        out = run_norm(stream, x, None, w, dtype, F.FLOAT, dtype, in_place="y", want_h=False)
        check_norm(out, x, None, w, dtype, F.FLOAT, dtype)
    else:
        out = run_norm(stream, x, r, w, dtype, F.FLOAT, F.E4M3, in_place=where)
        check_norm(out, x, r, w, dtype, F.FLOAT, F.E4M3)


@pytest.mark.parametrize("n", [128, 1000, 20000])
def test_norm_special_rows(hip, stream, n):
    """A row of zeros is finite (eps), a NaN or an infinity stays in its own row, eps = 0 is allowed."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((6, n)).astype(np.float32)
    x[1], x[2, n // 2], x[4, n - 1] = 0, np.nan, np.inf
    out = run_norm(stream, x, None, None, F.FLOAT, F.FLOAT, F.FLOAT)
    coded = run_norm(stream, x, None, None, F.FLOAT, F.FLOAT, F.E4M3)
    good = [0, 1, 3, 5]
    check_norm({"h": None, "rstd": out["rstd"][good], "y": out["y"][good]}, x[good], None, None, F.FLOAT, F.FLOAT, F.FLOAT)
    check_norm({"h": None, "rstd": coded["rstd"][good], "y": coded["y"][good], "s": coded["s"][good]}, x[good], None, None, F.FLOAT, F.FLOAT, F.E4M3)
    assert (out["y"][1] == 0).all() and (coded["y"][1] & 0x7F == 0).all() and np.isfinite(coded["s"][1]).all()
    assert np.isnan(out["y"][2]).all() and np.isnan(coded["s"][2]).all() and (coded["y"][2] == 0x7F).all()
    assert np.isnan(out["y"][4, n - 1]) and (out["y"][4, :n - 1] == 0).all()          # finite / infinity, infinity / infinity
    out = run_norm(stream, x[:1], None, None, F.FLOAT, F.FLOAT, F.FLOAT, eps=0.0)
    check_norm(out, x[:1], None, None, F.FLOAT, F.FLOAT, F.FLOAT, eps=0.0)


# ---- rms_norm_grad ----------------------------------------------------------------------------------------------------

def run_grad(stream, dy, h, w, rstd, dh, dtype, dtype_w, pad=0, shift=0, in_place=None, want_dw=True):
    rows, n = h.shape
    st = F.STORAGE[dtype]
    dY, H = Matrix(stream, n, rows, st, n + pad, shift, dy), Matrix(stream, n, rows, st, n + 2 * pad, shift, h)
    dH = Matrix(stream, n, rows, st, n + pad, shift, dh) if dh is not None else None
    W = Matrix(stream, n, 1, F.STORAGE[dtype_w], None, shift, w) if w is not None else None
    T = Matrix(stream, rows, 1, np.float32, data=rstd.astype(np.float32))
    dX = {"dy": dY, "dh": dH}.get(in_place) or Matrix(stream, n, rows, st, n + pad, shift)
    dW = Matrix(stream, n, 1, np.float32) if want_dw else None
    oh.check(oh.lib.och_rms_norm_grad(dtype, n, rows, dY.ptr, dY.ld, H.ptr, H.ld, T.ptr, dtype_w, W.ptr if W else None, dH.ptr if dH else None, dH.ld if dH else 0,
                                      dX.ptr, dX.ld, dW.ptr if dW else None, stream.handle))
    out = dX.read(), dW.read()[0] if dW else None
    for m in {id(m): m for m in (dY, H, dH, W, T, dX, dW) if m is not None}.values():
        m.free()
    return out


def check_grad(got, dy, h, w, rstd, dh, dtype, dtype_w):
    rows, n = h.shape
    hv, dyv = F.from_wide(h, dtype), F.from_wide(dy, dtype)
    wv = np.ones(n) if w is None else F.from_wide(w, dtype_w)
    dhv = np.zeros((rows, n)) if dh is None else F.from_wide(dh, dtype)
    r = rstd.astype(np.float32).astype(np.float64)
    dx, dw = F.norm_grad(dyv, hv, wv, r, dhv)
    u, g = hv * r[:, None], dyv * wv
    size = r[:, None] * (np.abs(g) + np.abs(u) * np.abs(g * u).mean(1, keepdims=True))
    tol = F.HALF_STEP[dtype] * np.abs(dx) + F.HALF_SMALLEST[dtype] + (chain(n) + 8) * U * size + 2 * U * (np.abs(dhv) + np.abs(dx))
    assert (np.abs(F.from_wide(got[0], dtype) - dx) <= tol).all()
    if got[1] is not None:
        assert (np.abs(got[1] - dw) <= (rows + 4) * U * np.abs(dyv * u).sum(0)).all()         # any order of the rows


@pytest.mark.parametrize("dtype", WIDE, ids=name_of)
def test_norm_grad(hip, stream, dtype):
    rng = np.random.default_rng(dtype + 70)
    for k, (rows, n) in enumerate(SHAPES + [(1500, 96), (2100, 256), (1111, 1100)]):
        dtype_w = dtype if k % 2 else F.FLOAT
        h, dy = wide_data(rng, rows, n, dtype), wide_data(rng, rows, n, dtype, 0.5)
        dh = wide_data(rng, rows, n, dtype, 0.5) if k % 3 else None
        w = F.to_wide(1 + 0.2 * rng.standard_normal(n), dtype_w) if k % 5 else None
        rstd = 1 / np.sqrt((F.from_wide(h, dtype) ** 2).mean(1) + 1e-5)
        pad, shift = [(0, 0), (8, 8), (3, 1)][k % 3]
        got = run_grad(stream, dy, h, w, rstd, dh, dtype, dtype_w, pad, shift, want_dw=bool(k % 7 or k == 0))
        check_grad(got, dy, h, w, rstd, dh, dtype, dtype_w)


@pytest.mark.parametrize("n", [96, 640, 3000, 24000])
@pytest.mark.parametrize("where", ["dy", "dh"])
def test_norm_grad_in_place(hip, stream, where, n):
    rng = np.random.default_rng(n + 1)
    dtype, rows = F.HALF, 7
    h, dy, dh = wide_data(rng, rows, n, dtype), wide_data(rng, rows, n, dtype), wide_data(rng, rows, n, dtype)
    rstd = 1 / np.sqrt((F.from_wide(h, dtype) ** 2).mean(1) + 1e-5)
    w = F.to_wide(1 + 0.2 * rng.standard_normal(n), dtype)
    check_grad(run_grad(stream, dy, h, w, rstd, dh, dtype, dtype, in_place=where), dy, h, w, rstd, dh, dtype, dtype)


def test_norm_grad_against_differences(hip, stream):
    """The gradients of sum(y * c) + sum(h * d) by central differences of the 64-bit forward formula."""
    rng = np.random.default_rng(11)
    rows, n, eps, step = 3, 130, 1e-5, 1e-5
    x, c, d = (rng.standard_normal((rows, n)).astype(np.float32) for _ in range(3))
    w = (1 + 0.2 * rng.standard_normal(n)).astype(np.float32)

    def loss(xv, wv):
        rstd = 1 / np.sqrt((xv * xv).mean(1) + eps)
        return (xv * rstd[:, None] * wv * c).sum() + (xv * d).sum()
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    rstd = 1 / np.sqrt((x64 * x64).mean(1) + eps)
    dx, dw = run_grad(stream, c, x, w, rstd, d, F.FLOAT, F.FLOAT)
    for i in range(rows):
        for j in range(0, n, 7):
            e = np.zeros((rows, n)); e[i, j] = step
            # the differences are good to step^2 (third derivatives of order 1) and to 2^-52 |loss| / step
            assert abs((loss(x64 + e, w64) - loss(x64 - e, w64)) / (2 * step) - dx[i, j]) <= 1e-6 + 64 * U * (1 + abs(dx[i, j])) * 4
    for j in range(0, n, 7):
        e = np.zeros(n); e[j] = step
        assert abs((loss(x64, w64 + e) - loss(x64, w64 - e)) / (2 * step) - dw[j]) <= 1e-6 + 64 * U * (1 + abs(dw[j])) * 4


def test_norm_grad_of_no_rows_is_zero(hip, stream):
    dW = Matrix(stream, 300, 1, np.float32)
    oh.check(oh.lib.och_rms_norm_grad(F.BF16, 300, 0, None, 300, None, 300, None, F.FLOAT, None, None, 0, None, 300, dW.ptr, stream.handle))
    assert (dW.read() == 0).all()
    dW.free()


# ---- gemm_scaled ------------------------------------------------------------------------------------------------------

def stored(v, contiguous_k):
    """op(.) as [rows, k] -> the numpy array whose rows are the columns of the stored matrix."""
    return v if contiguous_k else np.ascontiguousarray(v.T)


def run_gemm(stream, ca, cb, dtype, ta, tb, a, sa, ba, b, sb, bb, alpha=1.0, beta=0.0, c0=None, pad=(0, 0, 0), shift=(0, 0, 0), spad=0):
    """a [M, K], b [N, K] codes; sa [ceil(M / ba), ceil(K / 128)], sb alike; returns C as [N, M] in the storage of its type"""
    M, K = a.shape
    N = b.shape[0]
    A, B = stored(a, ta == "T"), stored(b, tb == "N")
    SA, SB = stored(sa, ta == "T"), stored(sb, tb == "N")
    dA = Matrix(stream, A.shape[1], A.shape[0], np.uint8, A.shape[1] + pad[0], shift[0], A)
    dB = Matrix(stream, B.shape[1], B.shape[0], np.uint8, B.shape[1] + pad[1], shift[1], B)
    dSA = Matrix(stream, SA.shape[1], SA.shape[0], np.float32, SA.shape[1] + spad, spad, SA)
    dSB = Matrix(stream, SB.shape[1], SB.shape[0], np.float32, SB.shape[1] + spad, spad, SB)
    dC = Matrix(stream, M, N, F.STORAGE[dtype], M + pad[2], shift[2], c0)
    oh.check(oh.lib.och_gemm_scaled(ca, cb, dtype, ta.encode(), tb.encode(), M, N, K, alpha, dA.ptr, dA.ld, dSA.ptr, dSA.ld, ba, dB.ptr, dB.ld, dSB.ptr, dSB.ld, bb,
                                    beta, dC.ptr, dC.ld, stream.handle))
    out = dC.read()
    for m in (dA, dB, dSA, dSB, dC):
        m.free()
    return out


def wide_scales(s, block, rows, K):
    return np.repeat(np.repeat(s.astype(np.float64), block, 0)[:rows], 128, 1)[:, :K]


def check_gemm(got, ca, cb, dtype, a, sa, ba, b, sb, bb, alpha=1.0, beta=0.0, c0=None):
    """Every block's sum of 128 products and the sum over the blocks may round (or cut off) at every addition: 2^-23 of the
    sum of magnitudes each; then the products with the scales, alpha and beta, and the rounding to the type. Results of 16
    bits come from an instruction that adds eight neighbouring k at a time and cuts off, of each of the eight products and of
    what it adds them to, less than 2^-13 of the power of two in the largest product: at most 9 * 2^-13 max of the eight."""
    M, K = a.shape
    N = b.shape[0]
    av, bv = F.decode(a, ca) * wide_scales(sa, ba, M, K), F.decode(b, cb) * wide_scales(sb, bb, N, K)
    want, size = alpha * (bv @ av.T), abs(alpha) * (np.abs(bv) @ np.abs(av).T)
    cut = 0
    if dtype != F.FLOAT:
        p = -(-K // 8)
        a8, b8 = np.zeros((M, 8 * p)), np.zeros((N, 8 * p))
        a8[:, :K], b8[:, :K] = np.abs(av), np.abs(bv)
        for i in range(p):                       # one scale per eight: the largest scaled product is the scaled largest
            cut = cut + (b8[:, None, 8 * i:8 * i + 8] * a8[None, :, 8 * i:8 * i + 8]).max(2)
        cut = abs(alpha) * 9 * 2.0 ** -13 * cut
    if beta:
        old = F.from_wide(c0, dtype)
        want, size = want + beta * old, size + np.abs(beta * old)
    tol = (132 + -(-K // 128)) * 2.0 ** -23 * size + cut + F.HALF_STEP[dtype] * (np.abs(want) * 1.001 + cut) + F.HALF_SMALLEST[dtype]
    value = F.from_wide(got, dtype)
    assert (np.abs(value - want) <= tol).all(), np.abs((value - want) / np.maximum(tol, 1e-300)).max()


def random_codes(rng, rows, k, code):
    q = rng.integers(0, 256, (rows, k)).astype(np.uint8)
    return np.where(np.isfinite(F.TABLE[code][q]), q, 0).astype(np.uint8)


def random_scales(rng, rows, block, k):
    return np.exp(rng.standard_normal((-(-rows // block), -(-k // 128)))).astype(np.float32) * np.float32(0.01)


TRANS = [("T", "N"), ("N", "N"), ("N", "T"), ("T", "T")]
GEMM_SHAPES = [(1, 1, 1), (16, 1, 128), (5, 3, 127), (64, 64, 256), (65, 130, 129), (200, 17, 384), (128, 33, 1000), (300, 70, 40), (256, 256, 512), (272, 300, 640),
               (129, 2, 2048), (33, 9, 5000)]


@pytest.mark.parametrize("ta,tb", TRANS)
@pytest.mark.parametrize("dtype", WIDE, ids=name_of)
def test_gemm(hip, stream, dtype, ta, tb):
    rng = np.random.default_rng(ord(ta) * 3 + ord(tb) + dtype)
    for k, (M, N, K) in enumerate(GEMM_SHAPES):
        ca, cb = CODES[k % 2], CODES[k // 2 % 2]
        ba, bb = [(128, 1), (1, 1), (1, 128), (128, 128)][(k + k // 4) % 4]
        a, b = random_codes(rng, M, K, ca), random_codes(rng, N, K, cb)
        if dtype == F.HALF:                       # stay below half's largest value: e5m2 codes reach 57344
            sa, sb = random_scales(rng, M, ba, K) * (1e-4 if ca == F.E5M2 else 1e-2), random_scales(rng, N, bb, K) * (1e-4 if cb == F.E5M2 else 1e-2)
            sa, sb = sa.astype(np.float32), sb.astype(np.float32)
        else:
            sa, sb = random_scales(rng, M, ba, K), random_scales(rng, N, bb, K)
        pad = [(0, 0, 0), (16, 16, 8), (1, 3, 5)][k % 3]
        shift = [(0, 0, 0), (16, 16, 8), (3, 1, 1)][k % 3]
        got = run_gemm(stream, ca, cb, dtype, ta, tb, a, sa, ba, b, sb, bb, pad=pad, shift=shift, spad=k % 3)
        check_gemm(got, ca, cb, dtype, a, sa, ba, b, sb, bb)


def exact_case(rng, M, N, K, ba, bb):
    """Small whole numbers and scales that are powers of two: every sum is exact in float whatever its order. (At most 4
    blocks with scales 1/2 .. 2: products below 2^6, sums below 2^6 K 2^2.)"""
    grid = F.encode(np.array([-8, -4, -3, -2, -1, 0, 1, 2, 3, 4, 8]), F.E4M3)
    a, b = rng.choice(grid, (M, K)), rng.choice(grid, (N, K))
    sa = 2.0 ** rng.integers(-1, 2, (-(-M // ba), -(-K // 128)))
    sb = 2.0 ** rng.integers(-1, 2, (-(-N // bb), -(-K // 128)))
    return a, sa.astype(np.float32), b, sb.astype(np.float32)


@pytest.mark.parametrize("dtype", [F.FLOAT, F.BF16], ids=name_of)
@pytest.mark.parametrize("ba,bb", [(128, 1), (1, 1), (1, 128), (128, 128)])
@pytest.mark.parametrize("ta,tb", TRANS)
def test_gemm_exact(hip, stream, ta, tb, ba, bb, dtype):
    """Bit for bit, over the sizes at which kernels, tiles and shares of K change. (The products of a block lie within 2^6 of
    one another: no instruction cuts any of them.)"""
    rng = np.random.default_rng(ba + 2 * bb + ord(ta))
    for M, N, K, pad in [(64, 64, 128, 0), (256, 256, 256, 0), (256, 512, 1024, 0), (512, 256, 4096, 16), (300, 1, 4096, 0), (1024, 16, 2048, 0), (513, 40, 1040, 16),
                         (384, 640, 1168, 0), (260, 272, 208, 16), (1000, 1000, 1000, 8), (129, 200, 4100, 1), (2048, 128, 512, 0), (2080, 96, 2064, 0)]:
        a, sa, b, sb = exact_case(rng, M, N, K, ba, bb)
        got = run_gemm(stream, F.E4M3, F.E4M3, dtype, ta, tb, a, sa, ba, b, sb, bb, pad=(pad, pad, pad))
        av, bv = F.decode(a, F.E4M3) * wide_scales(sa, ba, M, K), F.decode(b, F.E4M3) * wide_scales(sb, bb, N, K)
        want = (bv.astype(np.float32) @ av.astype(np.float32).T)
        assert np.array_equal(got, F.to_wide(want, dtype)), (M, N, K)


@pytest.mark.parametrize("dtype", WIDE, ids=name_of)
@pytest.mark.parametrize("M,N,K", [(96, 5, 300), (256, 256, 256), (300, 100, 4096), (520, 260, 384)])
def test_gemm_alpha_beta(hip, stream, dtype, M, N, K):
    rng = np.random.default_rng(M + K)
    a, sa, b, sb = exact_case(rng, M, N, K, 128, 1)
    c0 = F.to_wide(rng.standard_normal((N, M)) * 30, dtype)
    for alpha, beta in ((0.5, 0.0), (-1.25, 1.0), (1.0, -0.75), (0.0, 2.0)):
        got = run_gemm(stream, F.E4M3, F.E4M3, dtype, "T", "N", a, sa, 128, b, sb, 1, alpha, beta, c0, pad=(0, 0, 8))
        check_gemm(got, F.E4M3, F.E4M3, dtype, a, sa, 128, b, sb, 1, alpha, beta, c0)


def test_gemm_of_no_k_and_beta_zero_reads_nothing(hip, stream):
    """K = 0 leaves beta * C; beta = 0 does not read C (NaN there do not survive)."""
    c0 = np.arange(40 * 3, dtype=np.float32).reshape(3, 40)
    for beta, want in ((0.0, 0 * c0), (2.0, 2 * c0)):
        C0 = Matrix(stream, 40, 3, np.float32, 44, 1, c0)
        oh.check(oh.lib.och_gemm_scaled(F.E4M3, F.E4M3, F.FLOAT, b"T", b"N", 40, 3, 0, 1.0, None, 0, None, 0, 128, None, 0, None, 0, 1, beta, C0.ptr, C0.ld, stream.handle))
        assert np.array_equal(C0.read(), want)
        C0.free()
    rng = np.random.default_rng(1)
    for M, N, K in ((300, 9, 512), (512, 512, 512)):
        a, sa, b, sb = exact_case(rng, M, N, K, 128, 1)
        nan = np.full((N, M), np.nan, np.float32)
        assert np.isfinite(run_gemm(stream, F.E4M3, F.E4M3, F.FLOAT, "T", "N", a, sa, 128, b, sb, 1, c0=nan)).all()


@pytest.mark.parametrize("M,N,K", [(130, 3, 400), (384, 300, 512)])
@pytest.mark.parametrize("ta,tb", TRANS)
def test_gemm_nan_and_infinity_stay_in_their_rows(hip, stream, ta, tb, M, N, K):
    """A NaN code, a NaN scale and an infinite e5m2 code reach the elements that are computed from them and no others."""
    rng = np.random.default_rng(9)
    a, sa, b, sb = exact_case(rng, M, N, K, 1, 1)
    b = F.encode(np.where(F.decode(b, F.E4M3) == 0, 1, F.decode(b, F.E4M3)), F.E5M2)
    b[N - 1, 5] = 0x7C                                       # infinity
    a = np.where(F.decode(a, F.E4M3) == 0, F.encode(1.0, F.E4M3), a).astype(np.uint8)
    a[3, K - 1], sa[M - 2, 1] = 0x7F, np.nan
    got = run_gemm(stream, F.E4M3, F.E5M2, F.FLOAT, ta, tb, a, sa, 1, b, sb, 1)
    nan = np.isnan(got)
    assert nan[:, 3].all() and nan[:, M - 2].all()
    rest = np.delete(got, [3, M - 2], 1)
    assert np.isinf(rest[N - 1]).all() and np.isfinite(rest[:N - 1]).all()


def test_gemm_is_reproducible(hip, stream):
    rng = np.random.default_rng(2)
    for M, N, K in ((512, 7, 8192), (640, 130, 8192), (768, 1024, 2048)):
        a, b = random_codes(rng, M, K, F.E4M3), random_codes(rng, N, K, F.E4M3)
        sa, sb = random_scales(rng, M, 128, K), random_scales(rng, N, 1, K)
        first = run_gemm(stream, F.E4M3, F.E4M3, F.FLOAT, "T", "N", a, sa, 128, b, sb, 1)
        for _ in range(3):
            assert np.array_equal(first.view(np.uint32), run_gemm(stream, F.E4M3, F.E4M3, F.FLOAT, "T", "N", a, sa, 128, b, sb, 1).view(np.uint32))


@pytest.mark.parametrize("dtype", [F.FLOAT, F.HALF], ids=name_of)
@pytest.mark.parametrize("ba,bb", [(128, 1), (1, 1), (128, 128)])
def test_gemm_few_columns(hip, stream, dtype, ba, bb):
    """One to a few columns, bit for bit: every number of tiles of 16 columns, K from one code to many slabs with ends of all
    lengths, M that leaves rows of the last tile empty, odd leading dimensions."""
    rng = np.random.default_rng(dtype + ba + bb)
    for k, (M, N, K) in enumerate([(1, 1, 1), (17, 1, 5), (16, 2, 15), (40, 3, 17), (128, 1, 127), (130, 5, 129), (96, 15, 255), (64, 16, 1000), (200, 17, 1025),
                                   (48, 31, 2047), (33, 33, 640), (256, 48, 4096), (100, 63, 3333), (1040, 64, 384), (4100, 1, 4112), (5000, 40, 208)]):
        a, sa, b, sb = exact_case(rng, M, N, K, ba, bb)
        pad = [0, 16, 3][k % 3]
        got = run_gemm(stream, F.E4M3, F.E4M3, dtype, "T", "N", a, sa, ba, b, sb, bb, pad=(pad, pad, pad), shift=(pad, 2 * pad, pad), spad=k % 2)
        av, bv = F.decode(a, F.E4M3) * wide_scales(sa, ba, M, K), F.decode(b, F.E4M3) * wide_scales(sb, bb, N, K)
        assert np.array_equal(got, F.to_wide(bv.astype(np.float32) @ av.astype(np.float32).T, dtype)), (M, N, K)


@pytest.mark.parametrize("ba,bb", [(128, 1), (1, 1)])
@pytest.mark.parametrize("ta,tb", TRANS)
def test_gemm_large(hip, stream, ta, tb, ba, bb):
    """Products of several hundred large tiles, whole and ragged, bit for bit against the product of the exact values by
    probes: C x for a vector of small whole numbers (every number below 2^53), and a few columns in full."""
    rng = np.random.default_rng(ba + ord(tb))
    for M, N, K in [(4096, 4096, 256), (4096 + 16, 3840 + 272, 400), (3856, 4352, 144)]:
        a, sa, b, sb = exact_case(rng, M, N, K, ba, bb)
        got = F.from_wide(run_gemm(stream, F.E4M3, F.E4M3, F.BF16, ta, tb, a, sa, ba, b, sb, bb), F.BF16)
        av = (F.decode(a, F.E4M3) * wide_scales(sa, ba, M, K)).astype(np.float32)
        bv = (F.decode(b, F.E4M3) * wide_scales(sb, bb, N, K)).astype(np.float32)
        want = F.from_wide(F.to_wide(bv @ av.T, F.BF16), F.BF16)        # whole multiples of 1/4 below 2^22: exact in float
        assert np.array_equal(got, want), (M, N, K, np.argwhere(got != want)[:5])


@pytest.mark.parametrize("dtype", [F.FLOAT, F.BF16], ids=name_of)
@pytest.mark.parametrize("ba", [1, 128])
@pytest.mark.parametrize("ta,tb", TRANS)
def test_gemm_exact_with_halves_of_k(hip, stream, ta, tb, ba, dtype):
    """Where two groups of waves share a tile: even and odd numbers of blocks, K that ends inside one, shares of K whose last is
    shorter. (Sums stay below 2^6 K 2^2 < 2^21: exact in float.)"""
    rng = np.random.default_rng(ba + ord(tb))
    for M, N, K, pad in [(640, 640, 896, 0), (1024, 1024, 1152, 16), (130, 140, 896, 3), (2048, 130, 4224, 0), (300, 1000, 2688, 5), (1500, 1400, 256, 0), (256, 384, 8064, 1), (700, 700, 1000, 4),
                         (1024, 700, 1030, 0), (2000, 1900, 130, 0), (300, 200, 4001, 1), (130, 900, 8200, 8)]:
        a, sa, b, sb = exact_case(rng, M, N, K, ba, 1)
        got = run_gemm(stream, F.E4M3, F.E4M3, dtype, ta, tb, a, sa, ba, b, sb, 1, pad=(pad, pad, pad), shift=(pad, pad, pad))
        av, bv = F.decode(a, F.E4M3) * wide_scales(sa, ba, M, K), F.decode(b, F.E4M3) * wide_scales(sb, 1, N, K)
        want = (bv.astype(np.float32) @ av.astype(np.float32).T)
        assert np.array_equal(got, F.to_wide(want, dtype)), (M, N, K)
