"""Sums of few columns: half and bfloat16 results of up to 32 columns are float sums, rounded once. Products of very different size
lie next to each other here, which the 8-bit matrix instruction would cut off (by up to 2^-13 of the largest of eight)."""
import numpy as np
import pytest

import float8_oracle as F
import test_float8_gpu as T
from test_float8_kernels_gpu import PAIRS, aligned, pair_name

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pair", PAIRS, ids=pair_name)
@pytest.mark.parametrize("dtype", [F.HALF, F.BF16], ids=T.name_of)
def test_small_products_beside_large_ones_that_cancel(hip, stream, dtype, pair):
    """In every eight neighbouring k: 448 x 448 and 448 x -448 (448 is a code of both types), and 1 x 1 to 3 x 2 beside them, which 2^-13
    of the largest passes. The large ones cancel within the eight; all partial sums of a block are whole numbers below 2^22 in any
    order, those of blocks small: exact in float."""
    rng = np.random.default_rng(dtype + pair[0] + 2 * pair[1])
    for M, N, K in [(40, 1, 128), (33, 5, 1000), (300, 16, 4096), (17, 31, 264), (4200, 32, 520), (96, 20, 40)]:
        av, bv = rng.choice([1.0, 2.0, 3.0, -1.0], (M, K)), rng.choice([1.0, 2.0, -1.0, -2.0], (N, K))
        av[:, 0::8], av[:, 3::8] = 448, 448
        bv[:, 0::8], bv[:, 3::8] = 448, -448
        whole = K // 8 * 8
        want = bv @ av.T
        assert np.abs(want).max() <= 6 * K and whole == K
        sa, sb = np.ones((M, -(-K // 128)), np.float32), np.ones((N, -(-K // 128)), np.float32)
        got = T.run_gemm(stream, *pair, dtype, "T", "N", F.encode(av, pair[0]), sa, 1, F.encode(bv, pair[1]), sb, 1, pad=(aligned(K), aligned(K), 0))
        assert np.array_equal(got, F.to_wide(want.astype(np.float32), dtype)), (M, N, K)


@pytest.mark.parametrize("dtype", [F.HALF, F.BF16], ids=T.name_of)
def test_random_codes_are_summed_as_for_a_float_result(hip, stream, dtype):
    """The bound of float results (test_float8_gpu.check_gemm) and one rounding to the type; for bfloat16 also bit for bit the float
    result, rounded: the same kernel adds the same numbers in the same order."""
    rng = np.random.default_rng(dtype)
    for M, N, K in [(14336, 1, 4096), (640, 16, 2064), (4200, 32, 1037), (130, 17, 300)]:
        a, b = T.random_codes(rng, M, K, F.E4M3), T.random_codes(rng, N, K, F.E4M3)
        sa, sb = T.random_scales(rng, M, 128, K) * np.float32(0.01), T.random_scales(rng, N, 1, K) * np.float32(0.01)
        args = ("T", "N", a, sa, 128, b, sb, 1)
        pad = (aligned(K), aligned(K), 0)
        wide = T.run_gemm(stream, F.E4M3, F.E4M3, F.FLOAT, *args, pad=pad)
        T.check_gemm(wide, F.E4M3, F.E4M3, F.FLOAT, a, sa, 128, b, sb, 1)
        assert np.array_equal(T.run_gemm(stream, F.E4M3, F.E4M3, dtype, *args, pad=pad), F.to_wide(wide, dtype)), (M, N, K)
