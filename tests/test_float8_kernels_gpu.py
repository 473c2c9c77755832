"""Each kernel of the block-scaled product over its own types, orders, ends and epilogues, bit for bit where every sum is exact
(test_float8_gpu.exact_case). Which kernel a product runs on:

  few columns   N <= 64, both operands contiguous along k, pointers and leading dimensions multiples of 16
  256 x 256     half and bfloat16 results, the same alignment, an operand contiguous along its rows has a multiple of 16 of
                them, and tiles enough: at the sizes here over 512 of 128 x 128, at most 256 of 256 x 256
  128 x 128     the rest
"""
import ctypes as C

import numpy as np
import pytest

import float8_oracle as F
import ocean_hip as oh
import test_float8_gpu as T

pytestmark = pytest.mark.gpu
L = oh.lib
PAIRS = [(F.E4M3, F.E4M3), (F.E4M3, F.E5M2), (F.E5M2, F.E4M3), (F.E5M2, F.E5M2)]
pair_name = lambda p: "%s_%s" % (F.CODE_NAMES[p[0]], F.CODE_NAMES[p[1]])      # noqa: E731


def exact_codes(rng, M, N, K, ba, bb, ca, cb):
    """exact_case in the given code types (its whole numbers are values of both)."""
    a, sa, b, sb = T.exact_case(rng, M, N, K, ba, bb)
    return F.encode(F.decode(a, F.E4M3), ca), sa, F.encode(F.decode(b, F.E4M3), cb), sb


def aligned(rows, more=0):
    """What brings a leading dimension of `rows` to a multiple of 16."""
    return -rows % 16 + more


def exact_result(dtype, a, sa, ba, b, sb, bb, ca, cb, alpha=1.0, beta=0.0, c0=None):
    """alpha, beta and the sums have few enough bits that every product is exact; the addition of beta * C rounds once, to
    float, and the result once more, to its type."""
    M, K = a.shape
    N = b.shape[0]
    av = (F.decode(a, ca) * T.wide_scales(sa, ba, M, K)).astype(np.float32)
    bv = (F.decode(b, cb) * T.wide_scales(sb, bb, N, K)).astype(np.float32)
    s = bv @ av.T
    assert np.abs(s).max() < 2.0 ** 19                       # multiples of 1/4: three bits are left for alpha
    v = alpha * s.astype(np.float64)
    if beta:
        v = v + beta * F.from_wide(c0, dtype)
    return F.to_wide(v.astype(np.float32), dtype)


FEW = [(1, 1, 1), (17, 1, 5), (40, 16, 130), (200, 3, 9000), (100, 17, 261), (33, 31, 2047), (96, 32, 129), (50, 33, 1000), (64, 48, 127), (64, 49, 515), (130, 64, 384),
       (4113, 17, 300), (4200, 32, 143), (4100, 48, 271), (4128, 49, 200), (4500, 64, 1037)]


@pytest.mark.parametrize("pair", PAIRS, ids=pair_name)
@pytest.mark.parametrize("dtype", T.WIDE, ids=T.name_of)
def test_few_columns_of_every_type(hip, stream, dtype, pair):
    """Aligned operands: every number of tiles of 16 columns, single tiles of rows and pairs (over 16 rows per compute unit),
    ends of K of all lengths, one wave to sixteen, alpha and beta."""
    rng = np.random.default_rng(dtype + 3 * pair[0] + pair[1])
    for k, (M, N, K) in enumerate(FEW):
        ba, bb = [(128, 1), (1, 1), (1, 128), (128, 128)][(k + k // 4) % 4]
        a, sa, b, sb = exact_codes(rng, M, N, K, ba, bb, *pair)
        alpha, beta = [(1.0, 0.0), (-1.25, 0.75), (0.5, 1.0)][k % 3]
        c0 = F.to_wide(rng.integers(-40, 41, (N, M)) / 4, dtype)
        more = 16 * (k % 2)
        got = T.run_gemm(stream, *pair, dtype, "T", "N", a, sa, ba, b, sb, bb, alpha, beta, c0, pad=(aligned(K, more), aligned(K, 2 * more), k % 5), shift=(more, 0, k % 3),
                         spad=k % 2)
        assert np.array_equal(got, exact_result(dtype, a, sa, ba, b, sb, bb, *pair, alpha, beta, c0)), (M, N, K)


LARGE = [(4112, 2192, 261), (4096, 2176, 128), (2320, 4000, 100), (3856, 2320, 1037)]


@pytest.mark.parametrize("pair", PAIRS, ids=pair_name)
@pytest.mark.parametrize("ta,tb", T.TRANS)
def test_large_tiles_of_every_type(hip, stream, ta, tb, pair):
    """Aligned products on 256 x 256 tiles: both code types in both places, half and bfloat16, alpha and beta, K that ends inside
    a block and inside a chunk of 16, no whole block of K, rows and columns that end inside a tile."""
    rng = np.random.default_rng(ord(ta) + 2 * ord(tb) + 5 * pair[0] + pair[1])
    first = T.TRANS.index((ta, tb)) + PAIRS.index(pair)
    for k in (first % 4, (first + 2) % 4):
        M, N, K = LARGE[k]
        assert -(-M // 128) * -(-N // 128) > 512 and -(-M // 256) * -(-N // 256) <= 256
        N -= 5 if tb == "N" and k % 2 else 0
        M -= 3 if ta == "T" and k == 3 else 0
        dtype = [F.HALF, F.BF16][(k // 2 + (ta == "T") + pair[1]) % 2]
        ba, bb = [(128, 1), (1, 1), (1, 128), (128, 128)][(k + pair[0]) % 4]
        a, sa, b, sb = exact_codes(rng, M, N, K, ba, bb, *pair)
        alpha, beta = [(-1.25, 0.75), (1.0, 0.0), (0.5, 1.0), (1.0, -2.0)][k]
        c0 = F.to_wide(rng.integers(-40, 41, (N, M)) / 4, dtype)
        pad = (aligned(K if ta == "T" else M, 16 * (k % 2)), aligned(K if tb == "N" else N), k)
        got = T.run_gemm(stream, *pair, dtype, ta, tb, a, sa, ba, b, sb, bb, alpha, beta, c0, pad=pad, shift=(0, 16 * (k % 2), k % 3), spad=k % 2)
        want = exact_result(dtype, a, sa, ba, b, sb, bb, *pair, alpha, beta, c0)
        assert np.array_equal(got, want), (M, N, K, np.argwhere(got != want)[:5])


@pytest.mark.parametrize("dtype", [F.HALF, F.BF16], ids=T.name_of)
@pytest.mark.parametrize("M,N,K", [(130, 3, 400), (130, 40, 300), (384, 300, 512), (384, 300, 130), (1200, 2000, 256), (4112, 2192, 272)])
@pytest.mark.parametrize("ta,tb", T.TRANS)
def test_nan_and_infinity_stay_in_their_rows_of_16_bit_results(hip, stream, ta, tb, M, N, K, dtype):
    """A NaN code, a NaN scale and an infinite e5m2 code, through the 8-bit matrix instructions: few columns, tiles for pairs of
    groups, tiles, large tiles."""
    rng = np.random.default_rng(M + N)
    a, sa, b, sb = T.exact_case(rng, M, N, K, 1, 1)
    b = F.encode(np.where(F.decode(b, F.E4M3) == 0, 1, F.decode(b, F.E4M3)), F.E5M2)
    b[N - 1, 5] = 0x7C                                       # infinity
    a = np.where(F.decode(a, F.E4M3) == 0, F.encode(1.0, F.E4M3), a).astype(np.uint8)
    a[3, K - 1], sa[M - 2, 1] = 0x7F, np.nan
    # half: products below 2^6 in at most 5 blocks of 128 (scales up to 4), by 2^-3: below 2^15
    got = F.from_wide(T.run_gemm(stream, F.E4M3, F.E5M2, dtype, ta, tb, a, sa, 1, b, sb, 1, 0.125, pad=(aligned(K if ta == "T" else M), aligned(K if tb == "N" else N), 0)), dtype)
    nan = np.isnan(got)
    assert nan[:, 3].all() and nan[:, M - 2].all()
    rest = np.delete(got, [3, M - 2], 1)
    assert np.isinf(rest[N - 1]).all() and np.isfinite(rest[:N - 1]).all()
    plain = exact_result(dtype, np.where(a == 0x7F, 0, a).astype(np.uint8), np.where(np.isnan(sa), 1, sa).astype(np.float32), 1, np.where(b == 0x7C, 0, b).astype(np.uint8), sb, 1,
                         F.E4M3, F.E5M2, 0.125)
    assert np.array_equal(rest[:N - 1], F.from_wide(np.delete(plain, [3, M - 2], 1)[:N - 1], dtype))


def product(stream, dtype, ta, tb, M, N, K, mats, alpha=1.0):
    A, SA, B, SB, Cm = mats
    oh.check(L.och_gemm_scaled(F.E4M3, F.E4M3, dtype, ta.encode(), tb.encode(), M, N, K, alpha, A.ptr, A.ld, SA.ptr, SA.ld, 128, B.ptr, B.ld, SB.ptr, SB.ld, 1, 0.0, Cm.ptr, Cm.ld,
                               stream.handle))


def operands(stream, rng, dtype, ta, tb, M, N, K):
    a, sa, b, sb = T.exact_case(rng, M, N, K, 128, 1)
    stored = [T.stored(a, ta == "T"), T.stored(sa, ta == "T"), T.stored(b, tb == "N"), T.stored(sb, tb == "N")]
    mats = [T.Matrix(stream, v.shape[1], v.shape[0], v.dtype, v.shape[1] + (aligned(v.shape[1]) if v.dtype == np.uint8 else 0), 0, v) for v in stored]
    mats.append(T.Matrix(stream, M, N, F.STORAGE[dtype]))
    return mats, exact_result(dtype, a, sa, 128, b, sb, 1, F.E4M3, F.E4M3)


def test_few_columns_replayed_from_a_graph(hip, stream):
    """Columns of one to four tiles, K with an end, single tiles of rows and pairs, and tiles with shares of K between them."""
    rng = np.random.default_rng(78)
    shapes = [(F.FLOAT, "T", "N", 300, 40, 1000), (F.HALF, "T", "N", 4200, 20, 300), (F.BF16, "T", "N", 4128, 64, 271), (F.FLOAT, "T", "N", 256, 200, 8192), (F.BF16, "T", "N", 40, 30, 5000)]
    cases = [(s, *operands(stream, rng, *s)) for s in shapes]

    def run():
        for s, mats, _ in cases:
            product(stream, *s, mats)

    def check_and_clear():
        for s, mats, want in cases:
            assert np.array_equal(mats[-1].read(), want), s
            mats[-1].buf.upload(mats[-1].host.view(np.uint8))
        stream.synchronize()
    run()
    check_and_clear()
    oh.check(L.och_stream_begin_capture(stream.handle))
    run()
    graph = C.c_void_p()
    oh.check(L.och_stream_end_capture(stream.handle, C.byref(graph)))
    for _ in range(3):
        oh.check(L.och_graph_launch(graph, stream.handle))
        check_and_clear()
        run()
        check_and_clear()
    oh.check(L.och_graph_destroy(graph))
    for _, mats, _ in cases:
        for m in mats:
            m.free()


def test_two_streams_interleaved_call_by_call(hip, stream):
    """Products that are cut along K and norm gradients on two streams, the calls issued in turns without a wait: both streams have
    partial sums in their workspaces at all times, so results from a workspace in common could not be right."""
    second, rng = oh.Stream(), np.random.default_rng(79)

    class Side:
        def __init__(self, on, shapes, norms):
            self.on, self.calls, self.checks, self.outputs, self.all = on, [], [], [], []
            for s in shapes:
                mats, want = operands(on, rng, *s)
                self.calls.append(lambda s=s, mats=mats: product(on, *s, mats))
                self.outputs.append(mats[-1])
                self.checks.append(lambda got, want=want: np.array_equal(got[0], want))
                self.all += mats
            for rows, n in norms:
                h, dy = T.wide_data(rng, rows, n, F.BF16), T.wide_data(rng, rows, n, F.BF16)
                rstd = (1 / np.sqrt((F.from_wide(h, F.BF16) ** 2).mean(1) + 1e-5)).astype(np.float32)
                H, dY, R, dX, dW = (T.Matrix(on, n, rows, np.uint16, data=h), T.Matrix(on, n, rows, np.uint16, data=dy), T.Matrix(on, rows, 1, np.float32, data=rstd),
                                    T.Matrix(on, n, rows, np.uint16), T.Matrix(on, n, 1, np.float32))
                self.calls.append(lambda H=H, dY=dY, R=R, dX=dX, dW=dW, n=n, rows=rows: oh.check(L.och_rms_norm_grad(
                    F.BF16, n, rows, dY.ptr, n, H.ptr, n, R.ptr, F.FLOAT, None, None, 0, dX.ptr, n, dW.ptr, on.handle)))
                self.outputs.append((dX, dW))
                self.checks.append(lambda got, h=h, dy=dy, rstd=rstd: T.check_grad((got[0], got[1][0]), dy, h, None, rstd.astype(np.float64), None, F.BF16, F.FLOAT) is None)
                self.all += [H, dY, R, dX, dW]

        def read(self):
            self.on.synchronize()
            return [[m.read() for m in (o if isinstance(o, tuple) else (o,))] for o in self.outputs]

        def clear(self):
            for o in self.outputs:
                for m in o if isinstance(o, tuple) else (o,):
                    m.buf.upload(m.host.view(np.uint8))
            self.on.synchronize()
    a = Side(stream, [(F.FLOAT, "N", "T", 256, 200, 8192), (F.BF16, "T", "N", 300, 129, 12288)], [(4000, 1024), (3000, 2048)])
    b = Side(second, [(F.BF16, "N", "N", 384, 130, 9000), (F.FLOAT, "T", "N", 200, 260, 8000)], [(3500, 1536), (4100, 640)])
    alone = []
    for side in (a, b):
        for call in side.calls:
            call()
        alone.append(side.read())
        assert all(check(got) for check, got in zip(side.checks, alone[-1]))
    for turn in range(4):
        a.clear()
        b.clear()
        for k in range(24):
            a.calls[k % len(a.calls)]()
            b.calls[(k + turn) % len(b.calls)]()
        for side, want in ((a, alone[0]), (b, alone[1])):
            for got, one in zip(side.read(), want):
                assert all(np.array_equal(g, w) for g, w in zip(got, one)), turn
    for m in a.all + b.all:
        m.free()
    second.synchronize()
    second.destroy()


@pytest.mark.parametrize("dtype", T.WIDE, ids=T.name_of)
def test_results_repeat_bit_for_bit(hip, stream, dtype):
    """Random codes, whose sums depend on the order of the additions: every kernel gives the same bits every time."""
    rng = np.random.default_rng(80)
    for ta, tb, M, N, K in [("T", "N", 512, 16, 8192), ("T", "N", 4200, 40, 2064), ("T", "N", 640, 144, 8192), ("N", "T", 768, 1024, 2000), ("T", "N", 4096, 2176, 1040)]:
        a, b = T.random_codes(rng, M, K, F.E4M3), T.random_codes(rng, N, K, F.E4M3)
        scale = np.float32(2e-4 if dtype == F.HALF else 1)
        sa, sb = T.random_scales(rng, M, 128, K) * scale, T.random_scales(rng, N, 1, K)
        run = lambda: T.run_gemm(stream, F.E4M3, F.E4M3, dtype, ta, tb, a, sa, 128, b, sb, 1)      # noqa: E731
        first = run()
        for _ in range(3):
            assert np.array_equal(first, run()), (M, N, K)


@pytest.mark.parametrize("n", [48, 640, 4096, 8192, 20000])
def test_norms_repeat_bit_for_bit(hip, stream, n):
    rng = np.random.default_rng(n)
    rows = 700
    x, r, dy = (T.wide_data(rng, rows, n, F.BF16) for _ in range(3))
    w = F.to_wide(1 + 0.2 * rng.standard_normal(n), F.FLOAT)
    rstd = 1 / np.sqrt((F.from_wide(x, F.BF16) ** 2).mean(1) + 1e-5)
    first = None
    for _ in range(3):
        out = T.run_norm(stream, x, r, w, F.BF16, F.FLOAT, F.E4M3)
        got = [out["y"], out["s"], out["h"], out["rstd"], *T.run_grad(stream, dy, x, w, rstd, r, F.BF16, F.FLOAT)]
        first = first or got
        assert all(np.array_equal(p, q) for p, q in zip(got, first))
