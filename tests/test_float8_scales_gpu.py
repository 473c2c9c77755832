"""The range of the scales of a scaled product: single scales may lie far out as long as the product of the two scales of a
block is a normal float number; a block of zeros counts as zero under any product of scales that is finite."""
import numpy as np
import pytest

import float8_oracle as F
import test_float8_gpu as T

pytestmark = pytest.mark.gpu
# few columns, 128 x 128 tiles (unaligned; with halves of K; with shares of K), 256 x 256 tiles
SHAPES = [(130, 3, 400, (0, 0, 0)), (4200, 40, 272, (0, 0, 0)), (129, 131, 400, (1, 3, 0)), (640, 640, 896, (0, 0, 0)), (256, 200, 8192, (0, 0, 0)), (4096, 2176, 256, (0, 0, 0))]


@pytest.mark.parametrize("x,y", [(100, -100), (-100, 100), (119, -109), (-62, -62), (-109, -15), (70, 30), (10, 90)])
@pytest.mark.parametrize("ba", [1, 128])
def test_products_of_scales_within_the_range(hip, stream, ba, x, y):
    """Exact sums (test_float8_gpu.exact_case, scales between 1/2 and 2) times powers of two."""
    rng = np.random.default_rng(x * x + ba)
    for M, N, K, pad in SHAPES:
        a, sa, b, sb = T.exact_case(rng, M, N, K, ba, 1)
        a[5, 128:256] = 0                                                     # zeros as the quantizer leaves them, where the scale is that row's alone
        if ba == 1:
            sa[5, 1] = np.float32(2.0 ** -100) / np.float32(448) / np.float32(2.0) ** np.float32(x)
        av, bv = F.decode(a, F.E4M3) * T.wide_scales(sa, ba, M, K), F.decode(b, F.E4M3) * T.wide_scales(sb, 1, N, K)
        want = (bv.astype(np.float32) @ av.astype(np.float32).T).astype(np.float64) * 2.0 ** (x + y)
        big = (sa.astype(np.float64) * 2.0 ** x).astype(np.float32), (sb.astype(np.float64) * 2.0 ** y).astype(np.float32)
        assert np.isfinite(big[0]).all() and np.isfinite(big[1]).all()
        for dtype in (F.FLOAT, F.BF16) + ((F.HALF,) if x + y == 0 else ()):
            got = T.run_gemm(stream, F.E4M3, F.E4M3, dtype, "T", "N", a, big[0], ba, b, big[1], 1, pad=pad)
            assert np.array_equal(got, F.to_wide(want.astype(np.float32), dtype)), (M, N, K, dtype)


def test_quantized_matrices_of_very_different_size(hip, stream):
    """The quantizer's scales of values around 1e30 and 1e-25, and a matrix with blocks of zeros, through products of every kernel."""
    rng = np.random.default_rng(5)
    for M, N, K, pad in SHAPES:
        w, v = T.wide_data(rng, M, K, F.BF16, 1e30), T.wide_data(rng, N, K, F.BF16, 1e-25)
        w[7, :] = 0
        v[1, 128:256] = 0
        a, sa = F.quantize(F.from_wide(w, F.BF16), 128, 1, F.E4M3)
        b, sb = F.quantize(F.from_wide(v, F.BF16), 128, 1, F.E4M3)
        if M * N > 1 << 20:                                                   # (check_gemm holds K / 8 planes of the result's size)
            a, sa, b, sb = a[:2320], sa[:2320], b[:100], sb[:100]
        for dtype in (F.FLOAT, F.BF16):
            got = T.run_gemm(stream, F.E4M3, F.E4M3, dtype, "T", "N", a, sa, 1, b, sb, 1, pad=pad)
            assert np.isfinite(F.from_wide(got, dtype)).all() and (got[:, 7] & 0x7FFF == 0 if dtype == F.BF16 else got[:, 7] == 0).all()
            T.check_gemm(got, F.E4M3, F.E4M3, dtype, a, sa, 1, b, sb, 1)
