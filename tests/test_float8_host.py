"""The block-scaled 8-bit operations through the device module (OcTensorGPU_quantizeBlocks, rmsNorm, rmsNormGradient,
gemmScaled) and its Python surface: results against the library's oracle, views, refusals. Arithmetic and tolerances are
those of test_float8_gpu."""
import numpy as np
import pytest

import float8_oracle as F
import ocean_gpu as ocean
import ocean_host as host


def test_refusals_without_a_device():
    """On host tensors every function is refused before anything runs."""
    x, w = ocean.asTensor(np.ones((3, 256), np.float32)), ocean.asTensor(np.ones(256, np.float32))
    q, s = ocean.zeros((256, 3), ocean.uint8), ocean.zeros((2, 3), ocean.float)
    for call in (lambda: ocean.quantizeBlocks(x), lambda: ocean.rmsNorm(x, w), lambda: ocean.rmsNorm(x, w, code="e4m3"),
                 lambda: ocean.rmsNormGradient(x, x, ocean.zeros((3,)), w), lambda: ocean.gemmScaled(1.0, q, s, q, s, transA="T")):
        with pytest.raises(host.OceanError, match="same GPU"):
            call()
    for missing in ((None, q._h, s._h), (x._h, None, s._h), (x._h, q._h, None)):
        assert host.lib.OcTensorGPU_quantizeBlocks(missing[0], 33, 128, 1, missing[1], missing[2]) == -1
    assert b"missing" in host.lib.OcError_lastMessage()
    assert host.lib.OcTensorGPU_rmsNorm(x._h, x._h, None, 1e-5, 0, None, x._h, None, None) == -1        # a residual without a place for the sum
    assert host.lib.OcTensorGPU_rmsNormGradient(x._h, x._h, None, None, None, x._h, None) == -1
    assert host.lib.OcTensorGPU_gemmScaled(1.0, q._h, 33, b"T", s._h, q._h, 33, b"N", None, 0.0, x._h) == -1
    with pytest.raises(ValueError, match="e4m3"):
        ocean.quantizeBlocks(x, code="fp8")
    with pytest.raises(ValueError, match="128"):
        ocean.quantizeBlocks(x, block=(0, 1))
    with pytest.raises(ValueError, match="beta"):
        ocean.gemmScaled(1.0, q, s, q, s, beta=1.0)


def on_gpu(a, dt=None):
    return ocean.gpu[0](ocean.asTensor(a)) if dt is None else ocean.asTensor(a, dt, ocean.gpu[0])


def half(rng, rows, n):
    return (rng.standard_normal((rows, n)) * np.exp(0.7 * rng.standard_normal(n))).astype(np.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("block", [(128, 1), (1, 128), (128, 128)])
@pytest.mark.parametrize("code", ["e4m3", "e5m2"])
def test_quantize(hip, code, block):
    rng = np.random.default_rng(3)
    for x, dt in ((half(rng, 70, 300), F.HALF), (half(rng, 5, 129).astype(np.float32), F.FLOAT)):
        q, s = ocean.quantizeBlocks(on_gpu(x), block, code)
        want = F.quantize(F.from_wide(F.to_wide(x.astype(np.float64), dt), dt), *block, {"e4m3": F.E4M3, "e5m2": F.E5M2}[code])
        assert q.dtype == ocean.uint8 and s.dtype == ocean.float
        assert np.array_equal(q.asnumpy(), want[0]) and np.array_equal(s.asnumpy(), want[1])
    v = on_gpu(x[0])                                                       # one column, as a vector
    q, s = ocean.quantizeBlocks(v, (128, 1), code)
    assert q.size == (129,) and s.size == (2,)
    assert np.array_equal(q.asnumpy(), F.quantize(x[:1], 128, 1, {"e4m3": F.E4M3, "e5m2": F.E5M2}[code])[0][0])


@pytest.mark.gpu
def test_layer(hip):
    """Norm, product, gradients, each tensor on its own stream."""
    import test_float8_gpu as T
    rng = np.random.default_rng(8)
    n, m, t = 384, 256, 140
    x, r, gain, w, dz = half(rng, t, n), half(rng, t, n), (1 + 0.2 * rng.standard_normal(n)).astype(np.float32), rng.standard_normal((m, n)).astype(np.float32) / 20, half(rng, t, m)
    bits = lambda a: a.view(np.uint16)      # noqa: E731
    wq, ws = ocean.quantizeBlocks(on_gpu(w), (128, 128))
    gx, gr, gg = on_gpu(x), on_gpu(r), on_gpu(gain)
    y = ocean.rmsNorm(gx, gg, 1e-5, residual=gr, code="e4m3")
    z = ocean.gemmScaled(1.0, wq, ws, y.y, y.scales, transA="T", dt=ocean.half)
    dq, ds = ocean.quantizeBlocks(on_gpu(dz), (128, 1), "e5m2")
    dy = ocean.gemmScaled(0.5, wq, ws, dq, ds, codeB="e5m2", dt=ocean.half)
    dx, dw = ocean.rmsNormGradient(dy, y.sum, y.rstd, gg, on_gpu(x))
    T.check_norm({"h": bits(y.sum.asnumpy()), "rstd": y.rstd.asnumpy(), "y": y.y.asnumpy(), "s": y.scales.asnumpy()}, bits(x), bits(r), gain, F.HALF, F.FLOAT, F.E4M3)
    T.check_gemm(bits(z.asnumpy()), F.E4M3, F.E4M3, F.HALF, wq.asnumpy(), ws.asnumpy(), 128, y.y.asnumpy(), y.scales.asnumpy(), 1)
    T.check_gemm(bits(dy.asnumpy()), F.E4M3, F.E5M2, F.HALF, np.ascontiguousarray(wq.asnumpy().T), np.ascontiguousarray(ws.asnumpy().T), 128, dq.asnumpy(), ds.asnumpy(), 1, 0.5)
    T.check_grad((bits(dx.asnumpy()), dw.asnumpy()), bits(dy.asnumpy()), bits(y.sum.asnumpy()), gain, y.rstd.asnumpy().astype(np.float64), bits(x), F.HALF, F.FLOAT)
    plain = ocean.rmsNorm(gx, None, 1e-5)
    assert plain.scales is None and plain.sum is None
    T.check_norm({"h": None, "rstd": plain.rstd.asnumpy(), "y": bits(plain.y.asnumpy())}, bits(x), None, None, F.HALF, F.FLOAT, F.HALF)
    # accumulation into C, whose columns lie inside a larger matrix
    c = on_gpu(np.ones((m, 2 * n), np.float32))
    part = c[:n, :]
    yq, ys = ocean.quantizeBlocks(plain.y, (1, 128))
    zq, zs = ocean.quantizeBlocks(on_gpu(dz), (1, 128), "e5m2")
    assert ocean.gemmScaled(1.0, yq, ys, zq, zs, beta=2.0, c=part, transB="T", codeB="e5m2") is part
    out = c.asnumpy()
    assert (out[:, n:] == 1).all()
    T.check_gemm(out[:, :n], F.E4M3, F.E5M2, F.FLOAT, np.ascontiguousarray(yq.asnumpy().T), np.ascontiguousarray(ys.asnumpy().T), 1, np.ascontiguousarray(zq.asnumpy().T),
                 np.ascontiguousarray(zs.asnumpy().T), 1, 1.0, 2.0, np.ones((m, n), np.float32))


@pytest.mark.gpu
def test_views_and_refusals(hip):
    rng = np.random.default_rng(4)
    x = half(rng, 12, 400)
    g = on_gpu(x)
    q, s = ocean.quantizeBlocks(g[100:356, 2:9])
    want = F.quantize(x[2:9, 100:356].astype(np.float32), 128, 1, F.E4M3)
    assert np.array_equal(q.asnumpy(), want[0]) and np.array_equal(s.asnumpy(), want[1])
    refused = lambda match: pytest.raises(host.OceanError, match=match)      # noqa: E731
    f = on_gpu(x.astype(np.float32))
    with refused("columns of X must be dense"):
        ocean.quantizeBlocks(g.T)
    with refused("columns of X must be dense"):
        ocean.quantizeBlocks(g[::2, :])
    with refused("half or float"):
        ocean.quantizeBlocks(on_gpu(x.astype(np.float64)))
    with refused("128 x 1, 1 x 128 or 128 x 128"):
        ocean.quantizeBlocks(g, (64, 1))
    with refused("same GPU"):
        ocean.rmsNorm(g, ocean.asTensor(np.ones(400, np.float32)))
    with refused("must be 400 x 1"):
        ocean.rmsNorm(g, on_gpu(np.ones(401, np.float32)))
    with refused("must be 400 x 12"):
        ocean.rmsNorm(g, residual=g[:, :11])
    with refused("must be of type half"):
        ocean.rmsNorm(g, residual=f)
    with refused("eps"):
        ocean.rmsNorm(g, eps=-1.0)
    y = ocean.rmsNorm(g)
    with refused("must be of type half"):
        ocean.rmsNormGradient(f, g, y.rstd)
    with refused("must be 12 x 1"):
        ocean.rmsNormGradient(g, g, y.rstd[:11])
    q, s = ocean.quantizeBlocks(g)
    with refused("sizes"):
        ocean.gemmScaled(1.0, q, s, q[:399, :], s, transA="T")
    with refused("scales do not fit"):
        ocean.gemmScaled(1.0, q, s, q, s[:2, :], transA="T")
    with refused("type uint8"):
        ocean.gemmScaled(1.0, g, s, q, s, transA="T")
    with refused("half or float"):
        ocean.gemmScaled(1.0, q, s, q, s, transA="T", dt=ocean.double)
    with refused("native byte order"):
        swapped = f.clone()
        host.lib.OcTensor_setByteswapped(swapped._h, 1)
        ocean.quantizeBlocks(swapped)
    # nothing to do
    assert ocean.quantizeBlocks(g[:, 3:3])[0].size == (400, 0)
    assert ocean.rmsNormGradient(g[:, 3:3], g[:, 3:3], y.rstd[3:3])[1].asnumpy().tolist() == [0.0] * 400
