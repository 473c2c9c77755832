"""The block-scaled 8-bit operations where counts pass 32 bits: columns more than 2^32 bytes apart, and more rows than one
launch has threads for. Expected values come from the same entries on small, ordinary operands, which test_float8_gpu checks
against the oracle: the results must be equal bit for bit."""
import ctypes as C

import numpy as np
import pytest

import float8_oracle as F
import ocean_hip as oh
import test_float8_gpu as T

pytestmark = pytest.mark.gpu
L = oh.lib


class Far:
    """Columns of a matrix `ld` elements apart in a buffer of which only the columns are touched."""

    def __init__(self, stream, rows, cols, dtype, ld, data=None):
        self.rows, self.cols, self.dtype, self.ld = rows, cols, np.dtype(dtype), ld
        self.buf = oh.DeviceBuffer(((cols - 1) * ld + rows) * self.dtype.itemsize, stream)
        for j in range(cols):
            self.buf.upload(data[j] if data is not None else np.zeros(rows, dtype), j * ld * self.dtype.itemsize)
        self.ptr = self.buf.ptr

    def read(self):
        return np.stack([self.buf.download(self.dtype, self.rows, j * self.ld * self.dtype.itemsize) for j in range(self.cols)])


def test_columns_far_apart(hip, stream):
    rng = np.random.default_rng(0)
    n, cols, wide, bytes_ = 300, 3, (1 << 31) + 8, (1 << 32) + 16
    x = T.wide_data(rng, cols, n, F.HALF)
    X, Q, Y = Far(stream, n, cols, np.uint16, wide, x), Far(stream, n, cols, np.uint8, bytes_), Far(stream, n, cols, np.uint16, wide)
    S, R = T.Matrix(stream, 3, cols, np.float32), T.Matrix(stream, cols, 1, np.float32)
    oh.check(L.och_quantize_blocks(F.HALF, F.E4M3, n, cols, X.ptr, X.ld, 128, 1, Q.ptr, Q.ld, S.ptr, S.ld, stream.handle))
    q, s = Q.read(), S.read()
    T.same_codes((q, s), F.quantize(F.from_wide(x, F.HALF), 128, 1, F.E4M3))
    oh.check(L.och_rms_norm(F.HALF, n, cols, X.ptr, X.ld, None, 0, None, 0, F.FLOAT, None, 1e-5, F.HALF, Y.ptr, Y.ld, None, 0, R.ptr, stream.handle))
    near = T.run_norm(stream, x, None, None, F.HALF, F.FLOAT, F.HALF)
    assert np.array_equal(Y.read(), near["y"]) and np.array_equal(R.read()[0], near["rstd"])
    T.check_norm({"h": None, "rstd": near["rstd"], "y": near["y"]}, x, None, None, F.HALF, F.FLOAT, F.HALF)
    dw = T.Matrix(stream, n, 1, np.float32)
    oh.check(L.och_rms_norm_grad(F.HALF, n, cols, X.ptr, X.ld, X.ptr, X.ld, R.ptr, F.FLOAT, None, None, 0, Y.ptr, Y.ld, dw.ptr, stream.handle))
    T.check_grad((Y.read(), dw.read()[0]), x, x, None, near["rstd"].astype(np.float64), None, F.HALF, F.FLOAT)
    # the codes as both operands, contiguous along k (C's columns far apart too) and along the rows
    for ta, tb, M, N, K in (("T", "N", cols, cols, n), ("N", "T", n, n, cols)):
        Cm = Far(stream, M, N, np.float32, wide if ta == "T" else n + 5)
        along = ta == "T"
        if not along:
            qt, st = T.run_quantize(stream, x, F.HALF, F.E4M3, 1, 128)
            for j in range(cols):
                Q.buf.upload(qt[j], j * bytes_)
            S.free()
            S = T.Matrix(stream, n, 1, np.float32, data=st)
        oh.check(L.och_gemm_scaled(F.E4M3, F.E4M3, F.FLOAT, ta.encode(), tb.encode(), M, N, K, 1.0, Q.ptr, Q.ld, S.ptr, S.ld, 1, Q.ptr, Q.ld, S.ptr, S.ld, 1, 0.0,
                                   Cm.ptr, Cm.ld, stream.handle))
        a, sa = (q, s) if along else (np.ascontiguousarray(qt.T), np.ascontiguousarray(st.T))
        T.check_gemm(Cm.read(), F.E4M3, F.E4M3, F.FLOAT, a, sa, 1, a, sa, 1)
        Cm.buf.free()
    for b in (X.buf, Q.buf, Y.buf, S, R, dw):
        b.free()


def repeated(pattern, count, got):
    """got is `pattern` over and over, `count` elements."""
    whole = count // len(pattern) * len(pattern)
    return np.array_equal(got[:whole].reshape(-1, len(pattern)), np.broadcast_to(pattern, (whole // len(pattern), len(pattern)))) and np.array_equal(got[whole:count], pattern[:count - whole])


def test_more_rows_than_a_launch_has_threads(hip, stream):
    rng = np.random.default_rng(1)
    rows, period = (1 << 29) + 33, 4099                                     # eight threads a row: 2^32 and more
    x = F.to_wide(rng.standard_normal((period, 1)) * 3, F.HALF)
    near = T.run_norm(stream, x, None, None, F.HALF, F.FLOAT, F.HALF)
    T.check_norm({"h": None, "rstd": near["rstd"], "y": near["y"]}, x, None, None, F.HALF, F.FLOAT, F.HALF)
    X, Y, R = oh.to_device(np.resize(x[:, 0], rows), stream), oh.DeviceBuffer(2 * rows, stream), oh.DeviceBuffer(4 * rows, stream)
    oh.check(L.och_rms_norm(F.HALF, 1, rows, X.ptr, 1, None, 0, None, 0, F.FLOAT, None, 1e-5, F.HALF, Y.ptr, 1, None, 0, R.ptr, stream.handle))
    assert repeated(near["y"][:, 0], rows, Y.download(np.uint16)) and repeated(near["rstd"], rows, R.download(np.float32))
    for b in (X, Y, R):
        b.free()


def test_more_blocks_than_a_launch_has_threads(hip, stream):
    rng = np.random.default_rng(2)
    cols, period = (1 << 29) + 77, 4099                                     # eight threads a block: 2^32 and more
    x = F.to_wide(rng.standard_normal((period, 1)) * 3, F.HALF)
    q, s = T.run_quantize(stream, x, F.HALF, F.E5M2, 128, 1)
    T.same_codes((q, s), F.quantize(F.from_wide(x, F.HALF), 128, 1, F.E5M2))
    X, Q, S = oh.to_device(np.resize(x[:, 0], cols), stream), oh.DeviceBuffer(cols, stream), oh.DeviceBuffer(4 * cols, stream)
    oh.check(L.och_quantize_blocks(F.HALF, F.E5M2, 1, cols, X.ptr, 1, 128, 1, Q.ptr, 1, S.ptr, 1, stream.handle))
    assert repeated(q[:, 0], cols, Q.download(np.uint8)) and repeated(s[:, 0], cols, S.download(np.float32))
    for b in (X, Q, S):
        b.free()


@pytest.mark.parametrize("bm,bn", [(128, 1), (1, 128), (128, 128)])
@pytest.mark.parametrize("dtype", T.WIDE, ids=T.name_of)
def test_large_aligned_matrices_are_quantized_alike(hip, stream, dtype, bm, bn):
    """Large matrices whose columns are whole cache lines go past the caches: the same codes and scales, block for block."""
    rng = np.random.default_rng(dtype + bn)
    M, period, N = 4096, 256, 8320
    x = T.wide_data(rng, period, M, dtype)
    x[5, 100] = F.to_wide(np.array(np.nan), dtype)
    q, s = T.run_quantize(stream, x, dtype, F.E4M3, bm, bn)
    want = F.quantize(F.from_wide(x, dtype), bm, bn, F.E4M3)
    T.same_codes((q, np.where(np.isnan(s), np.float32(np.nan), s)), want)
    X, Q, S = oh.to_device(np.resize(x, (N, M)), stream), oh.DeviceBuffer(N * M, stream), oh.DeviceBuffer(4 * -(-N // bn) * -(-M // bm), stream)
    assert X.address % 128 == 0 and Q.address % 128 == 0
    oh.check(L.och_quantize_blocks(dtype, F.E4M3, M, N, X.ptr, M, bm, bn, Q.ptr, M, S.ptr, -(-M // bm), stream.handle))
    assert np.array_equal(Q.download(np.uint8).reshape(N, M), np.resize(q, (N, M)))
    got = S.download(np.float32).reshape(-(-N // bn), -(-M // bm))
    assert np.array_equal(got, np.resize(s, got.shape), equal_nan=True)
    for b in (X, Q, S):
        b.free()


@pytest.mark.parametrize("n", [2048, 3968, 5888, 8192, 16384])
@pytest.mark.parametrize("dtype,dtype_y", [(F.BF16, F.E4M3), (F.HALF, F.HALF), (F.FLOAT, F.E5M2)])
def test_large_aligned_norms_are_alike(hip, stream, dtype, dtype_y, n):
    rng = np.random.default_rng(n + dtype)
    period, rows = 33, (36 << 20) // n
    x, r = T.wide_data(rng, period, n, dtype), T.wide_data(rng, period, n, dtype)
    w = F.to_wide(1 + 0.2 * rng.standard_normal(n), F.FLOAT)
    near = T.run_norm(stream, x, r, w, dtype, F.FLOAT, dtype_y)
    T.check_norm(near, x, r, w, dtype, F.FLOAT, dtype_y)
    coded, es, st = dtype_y != dtype, F.STORAGE[dtype]().itemsize, F.STORAGE[dtype]
    X, R, W = oh.to_device(np.resize(x, (rows, n)), stream), oh.to_device(np.resize(r, (rows, n)), stream), oh.to_device(w, stream)
    Y, S = oh.DeviceBuffer(rows * n * (1 if coded else es), stream), oh.DeviceBuffer(4 * rows * (n // 128), stream)
    assert Y.address % 128 == 0 and R.address % 128 == 0
    oh.check(L.och_rms_norm(dtype, n, rows, X.ptr, n, R.ptr, n, R.ptr, n, F.FLOAT, W.ptr, 1e-5, dtype_y, Y.ptr, n, S.ptr if coded else None, n // 128, None, stream.handle))
    assert np.array_equal(Y.download(np.uint8 if coded else st).reshape(rows, n), np.resize(near["y"], (rows, n)))
    assert np.array_equal(R.download(st).reshape(rows, n), np.resize(near["h"], (rows, n)))
    if coded:
        assert np.array_equal(S.download(np.float32).reshape(rows, n // 128), np.resize(near["s"], (rows, n // 128)))
    for b in (X, R, W, Y, S):
        b.free()


@pytest.mark.parametrize("N", [1, 40])
@pytest.mark.parametrize("dtype", [F.HALF, F.FLOAT], ids=T.name_of)
def test_weights_larger_than_the_caches(hip, stream, dtype, N):
    """Rows of A that repeat give rows of C that repeat; sums are exact in every order (few enough magnitudes to stay finite in
    half: products below 2^6 in 17 blocks of 128, scaled by 2^-8)."""
    rng = np.random.default_rng(N)
    M, K, period = 98_321, 2064, 96
    a, sa, b, sb = T.exact_case(rng, period, N, K, 1, 1)
    sa = (sa * 2.0 ** -8).astype(np.float32)
    want = T.run_gemm(stream, F.E4M3, F.E4M3, dtype, "T", "N", a, sa, 1, b, sb, 1)
    T.check_gemm(want, F.E4M3, F.E4M3, dtype, a, sa, 1, b, sb, 1)
    A, SA = oh.to_device(np.resize(a, (M, K)), stream), oh.to_device(np.resize(sa, (M, sa.shape[1])), stream)
    B, SB, Cm = oh.to_device(b, stream), oh.to_device(sb, stream), T.Matrix(stream, M, N, F.STORAGE[dtype])
    oh.check(L.och_gemm_scaled(F.E4M3, F.E4M3, dtype, b"T", b"N", M, N, K, 1.0, A.ptr, K, SA.ptr, sa.shape[1], 1, B.ptr, K, SB.ptr, sb.shape[1], 1, 0.0, Cm.ptr, Cm.ld,
                               stream.handle))
    got = Cm.read()
    assert np.array_equal(got, np.resize(want.T, (M, N)).T)
    for x in (A, SA, B, SB, Cm):
        x.free()
