"""Calls of the block-scaled 8-bit operations that are allowed and easily forgotten: in place through the device module, on views,
on the default stream, with the longest rows that have a gradient of the weights."""
import numpy as np
import pytest

import float8_oracle as F
import ocean_gpu as ocean
import ocean_hip as oh
import ocean_host as host
import test_float8_gpu as T
from test_float8_host import half, on_gpu

pytestmark = pytest.mark.gpu
L = oh.lib
bits = lambda a: np.ascontiguousarray(a).view(np.uint16)      # noqa: E731


@pytest.mark.parametrize("n", [256, 1001, 20000])
def test_in_place_through_the_device_module(hip, n):
    """The sum over the residual and over the input, the output over the input, the gradient over either of its terms."""
    rng = np.random.default_rng(n)
    x, r, gain = half(rng, 9, n), half(rng, 9, n), (1 + 0.2 * rng.standard_normal(n)).astype(np.float32)
    gg, lib = on_gpu(gain), host.lib
    for over in ("residual", "input"):
        gx, gr = on_gpu(x), on_gpu(r)
        h = gr if over == "residual" else gx
        y, s, rstd = ocean.zeros((n, 9), ocean.uint8), ocean.zeros((-(-n // 128), 9), ocean.float), ocean.zeros((9,), ocean.float)
        y, s, rstd = (ocean.gpu[0](t) for t in (y, s, rstd))
        host.check(lib.OcTensorGPU_rmsNorm(gx._h, gr._h, gg._h, 1e-5, F.E4M3, h._h, y._h, s._h, rstd._h))
        T.check_norm({"h": bits(h.asnumpy()), "rstd": rstd.asnumpy(), "y": y.asnumpy(), "s": s.asnumpy()}, bits(x), bits(r), gain, F.HALF, F.FLOAT, F.E4M3)
        assert np.array_equal((gx if over == "residual" else gr).asnumpy(), x if over == "residual" else r)
    gx = on_gpu(x)
    host.check(lib.OcTensorGPU_rmsNorm(gx._h, None, gg._h, 1e-5, 0, None, gx._h, None, None))
    T.check_norm({"h": None, "rstd": None, "y": bits(gx.asnumpy())}, bits(x), None, gain, F.HALF, F.FLOAT, F.HALF)
    root = 1 / np.sqrt((x.astype(np.float64) ** 2).mean(1) + 1e-5)
    for over in (0, 1):
        dy, dh, dw, gx, gt = on_gpu(r), on_gpu(x), ocean.gpu[0](ocean.zeros((n,), ocean.float)), on_gpu(x), on_gpu(root.astype(np.float32))
        dx = (dy, dh)[over]
        host.check(lib.OcTensorGPU_rmsNormGradient(dy._h, gx._h, gt._h, gg._h, dh._h, dx._h, dw._h))
        T.check_grad((bits(dx.asnumpy()), dw.asnumpy()), bits(r), bits(x), gain, root, bits(x), F.HALF, F.FLOAT)


def test_norm_and_product_of_views(hip):
    """Columns and rows out of the middle of larger matrices, in every place of the calls."""
    rng = np.random.default_rng(6)
    x, r = half(rng, 40, 700), half(rng, 40, 700)
    gain = (1 + 0.2 * rng.standard_normal(700)).astype(np.float32)
    cut, take = slice(100, 483), slice(3, 33)
    view = lambda a: on_gpu(a)[cut, take]      # noqa: E731
    y = ocean.rmsNorm(view(x), on_gpu(gain)[cut], 1e-5, residual=view(r), code="e4m3")
    xs, rs, gs = (np.ascontiguousarray(a) for a in (x[take, cut], r[take, cut], gain[cut]))
    T.check_norm({"h": bits(y.sum.asnumpy()), "rstd": y.rstd.asnumpy(), "y": y.y.asnumpy(), "s": y.scales.asnumpy()}, bits(xs), bits(rs), gs, F.HALF, F.FLOAT, F.E4M3)
    dx, dw = ocean.rmsNormGradient(view(r), y.sum, y.rstd, on_gpu(gain)[cut], view(x))
    T.check_grad((bits(dx.asnumpy()), dw.asnumpy()), bits(rs), bits(y.sum.asnumpy()), gs, y.rstd.asnumpy().astype(np.float64), bits(xs), F.HALF, F.FLOAT)
    # the product of every other block of columns: codes and scales cut alike
    w = rng.standard_normal((512, 383)).astype(np.float32) / 20
    q, s = ocean.quantizeBlocks(on_gpu(w), (128, 128))
    z = ocean.gemmScaled(1.0, q[:, 128:384], s[:, 1:3], y.y[:, 5:25], y.scales[:, 5:25], transA="T", dt=ocean.half)
    T.check_gemm(bits(z.asnumpy()), F.E4M3, F.E4M3, F.HALF, q.asnumpy()[128:384], s.asnumpy()[1:3], 128, y.y.asnumpy()[5:25], y.scales.asnumpy()[5:25], 1)


def test_default_stream(hip):
    """A quantization, a product that is cut along K and a norm's gradient, on the null stream."""
    rng = np.random.default_rng(7)

    class Null:
        handle = None
    null = Null()
    stream = oh.Stream()
    M, N, K, n, rows = 256, 200, 8192, 640, 300
    a, sa, b, sb = T.exact_case(rng, M, N, K, 128, 1)
    x, dy = T.wide_data(rng, rows, n, F.BF16), T.wide_data(rng, rows, n, F.BF16)
    rstd = (1 / np.sqrt((F.from_wide(x, F.BF16) ** 2).mean(1) + 1e-5)).astype(np.float32)
    A, SA, B, SB, X, dY, R = (T.Matrix(stream, v.shape[1], v.shape[0], v.dtype, data=v) for v in (a, sa, b, sb, x, dy, rstd[None]))
    Cm, Q, S, dX, dW = (T.Matrix(stream, r, c, t) for r, c, t in ((M, N, np.float32), (n, rows, np.uint8), (5, rows, np.float32), (n, rows, np.uint16), (n, 1, np.float32)))
    stream.synchronize()
    for _ in range(2):
        oh.check(L.och_gemm_scaled(F.E4M3, F.E4M3, F.FLOAT, b"T", b"N", M, N, K, 1.0, A.ptr, K, SA.ptr, K // 128, 128, B.ptr, K, SB.ptr, K // 128, 1, 0.0, Cm.ptr, M, null.handle))
        oh.check(L.och_rms_norm_grad(F.BF16, n, rows, dY.ptr, n, X.ptr, n, R.ptr, F.FLOAT, None, None, 0, dX.ptr, n, dW.ptr, null.handle))
        oh.check(L.och_quantize_blocks(F.BF16, F.E4M3, n, rows, X.ptr, n, 128, 1, Q.ptr, n, S.ptr, 5, null.handle))
    oh.check(L.och_stream_synchronize(None))
    av, bv = F.decode(a, F.E4M3) * T.wide_scales(sa, 128, M, K), F.decode(b, F.E4M3) * T.wide_scales(sb, 1, N, K)
    assert np.array_equal(Cm.read(), bv.astype(np.float32) @ av.astype(np.float32).T)
    T.check_grad((dX.read(), dW.read()[0]), dy, x, None, rstd.astype(np.float64), None, F.BF16, F.FLOAT)
    T.same_codes((Q.read(), S.read()), F.quantize(F.from_wide(x, F.BF16), 128, 1, F.E4M3))
    for m in (A, SA, B, SB, X, dY, R, Cm, Q, S, dX, dW):
        m.free()
    oh.check(L.och_stream_release_workspace(None))
    stream.synchronize()
    stream.destroy()


def test_longest_rows_with_a_gradient_of_the_weights(hip, stream):
    """2^24 features: one workgroup's sums fill the workspace. One feature more has a gradient of the input only."""
    rng = np.random.default_rng(8)
    n = 1 << 24
    for n, want_dw in ((n, True), (n + 1, False)):
        h, dy = (np.resize(F.to_wide(rng.standard_normal((1, 4099)), F.HALF), (2, n)) for _ in range(2))
        rstd = 1 / np.sqrt((F.from_wide(h, F.HALF) ** 2).mean(1) + 1e-5)
        got = T.run_grad(stream, dy, h, None, rstd, None, F.HALF, F.FLOAT, want_dw=want_dw)
        T.check_grad(got, dy, h, None, rstd, None, F.HALF, F.FLOAT)


def test_norms_of_one_value(hip, stream):
    """One feature, many rows, to codes: sixteen rows a workgroup."""
    rng = np.random.default_rng(9)
    x = F.to_wide(rng.standard_normal((5000, 1)) * 3, F.FLOAT)
    for dtype_y in (F.FLOAT, F.E4M3, F.E5M2):
        out = T.run_norm(stream, x, None, None, F.FLOAT, F.FLOAT, dtype_y)
        T.check_norm(out, x, None, None, F.FLOAT, F.FLOAT, dtype_y)
