"""The block-scaled 8-bit operations as they are used together: a layer's forward and backward pass, launched one by one and
replayed from a graph; and two streams at once.

Each stage is checked against the 64-bit statement of it on the stage's actual inputs, with the tolerances of
test_float8_gpu; the layer's output also against the layer without any rounding to 8 bits."""
import ctypes as C

import numpy as np
import pytest

import float8_oracle as F
import ocean_hip as oh
import test_float8_gpu as T

pytestmark = pytest.mark.gpu
L = oh.lib


class Layer:
    """x, r -> h = x + r, y = norm(h) in codes, z = W' y; and back: dz, dh -> dy = W dz, dx, the gradients of the norm's
    weights and, added to a running sum, of W. Features n, outputs m, tokens t."""

    def __init__(self, stream, rng, n, m, t):
        self.stream, self.n, self.m, self.t = stream, n, m, t
        up, g = (lambda v: -(-v // 128)), T.wide_data
        self.start = {"X": g(rng, t, n, F.BF16), "R": g(rng, t, n, F.BF16), "gain": F.to_wide(1 + 0.2 * rng.standard_normal((1, n)), F.FLOAT),
                      "W": (rng.standard_normal((m, n)) / np.sqrt(n)).astype(np.float32), "dZ": g(rng, t, m, F.BF16), "dH": g(rng, t, n, F.BF16)}
        shapes = {"WQ": (m, n, np.uint8), "WS": (up(m), up(n), np.float32), "YQ": (t, n, np.uint8), "YS": (t, up(n), np.float32), "Y": (t, n, np.uint16),
                  "rstd": (1, t, np.float32), "YT": (t, n, np.uint8), "YTS": (up(t), n, np.float32), "Z": (t, m, np.uint16), "dZQ": (t, m, np.uint8),
                  "dZS": (t, up(m), np.float32), "dZT": (t, m, np.uint8), "dZTS": (up(t), m, np.float32), "dY": (t, n, np.uint16), "dX": (t, n, np.uint16),
                  "dgain": (1, n, np.float32), "dW": (m, n, np.float32)}
        for k, (c, r, d) in shapes.items():
            self.start[k] = np.zeros((c, r), d)
        self.at = {k: T.Matrix(stream, v.shape[1], v.shape[0], v.dtype, data=v) for k, v in self.start.items()}

    def run(self):
        n, m, t, h, a = self.n, self.m, self.t, self.stream.handle, self.at
        arg = lambda k: (a[k].ptr, a[k].ld)      # noqa: E731
        ok = oh.check
        ok(L.och_quantize_blocks(F.FLOAT, F.E4M3, n, m, *arg("W"), 128, 128, *arg("WQ"), *arg("WS"), h))
        ok(L.och_rms_norm(F.BF16, n, t, *arg("X"), *arg("R"), *arg("R"), F.FLOAT, a["gain"].ptr, 1e-5, F.E4M3, *arg("YQ"), *arg("YS"), a["rstd"].ptr, h))
        ok(L.och_gemm_scaled(F.E4M3, F.E4M3, F.BF16, b"T", b"N", m, t, n, 1.0, *arg("WQ"), *arg("WS"), 128, *arg("YQ"), *arg("YS"), 1, 0.0, *arg("Z"), h))
        ok(L.och_rms_norm(F.BF16, n, t, *arg("R"), None, 0, None, 0, F.FLOAT, a["gain"].ptr, 1e-5, F.BF16, *arg("Y"), None, 0, None, h))
        ok(L.och_quantize_blocks(F.BF16, F.E4M3, n, t, *arg("Y"), 1, 128, *arg("YT"), *arg("YTS"), h))
        ok(L.och_quantize_blocks(F.BF16, F.E5M2, m, t, *arg("dZ"), 128, 1, *arg("dZQ"), *arg("dZS"), h))
        ok(L.och_quantize_blocks(F.BF16, F.E5M2, m, t, *arg("dZ"), 1, 128, *arg("dZT"), *arg("dZTS"), h))
        ok(L.och_gemm_scaled(F.E4M3, F.E5M2, F.BF16, b"N", b"N", n, t, m, 1.0, *arg("WQ"), *arg("WS"), 128, *arg("dZQ"), *arg("dZS"), 1, 0.0, *arg("dY"), h))
        ok(L.och_rms_norm_grad(F.BF16, n, t, *arg("dY"), *arg("R"), a["rstd"].ptr, F.FLOAT, a["gain"].ptr, *arg("dH"), *arg("dX"), a["dgain"].ptr, h))
        ok(L.och_gemm_scaled(F.E4M3, F.E5M2, F.FLOAT, b"N", b"T", n, m, t, 1.0, *arg("YT"), *arg("YTS"), 1, *arg("dZT"), *arg("dZTS"), 1, 1.0, *arg("dW"), h))

    def read(self):
        self.stream.synchronize()
        return {k: v.read() for k, v in self.at.items()}

    def reset(self):
        for k, v in self.at.items():
            v.buf.upload(v.host.view(np.uint8))
        self.stream.synchronize()

    def free(self):
        for v in self.at.values():
            v.free()


def check_layer(got, start, dw_before):
    x, r, gain, w, dz = (start[k] for k in ("X", "R", "gain", "W", "dZ"))
    h = got["R"]                                                          # the sum, in place of the residual
    T.same_codes((got["WQ"], got["WS"]), F.quantize(w, 128, 128, F.E4M3))
    T.check_norm({"h": h, "rstd": got["rstd"][0], "y": got["YQ"], "s": got["YS"]}, x, r, gain[0], F.BF16, F.FLOAT, F.E4M3)
    T.check_norm({"h": None, "rstd": None, "y": got["Y"]}, h, None, gain[0], F.BF16, F.FLOAT, F.BF16)
    T.same_codes((got["YT"], got["YTS"]), F.quantize(F.from_wide(got["Y"], F.BF16), 1, 128, F.E4M3))
    T.same_codes((got["dZQ"], got["dZS"]), F.quantize(F.from_wide(dz, F.BF16), 128, 1, F.E5M2))
    T.same_codes((got["dZT"], got["dZTS"]), F.quantize(F.from_wide(dz, F.BF16), 1, 128, F.E5M2))
    T.check_gemm(got["Z"], F.E4M3, F.E4M3, F.BF16, got["WQ"], got["WS"], 128, got["YQ"], got["YS"], 1)
    T.check_gemm(got["dY"], F.E4M3, F.E5M2, F.BF16, np.ascontiguousarray(got["WQ"].T), np.ascontiguousarray(got["WS"].T), 128, got["dZQ"], got["dZS"], 1)
    T.check_grad((got["dX"], got["dgain"][0]), got["dY"], h, gain[0], got["rstd"][0].astype(np.float64), start["dH"], F.BF16, F.FLOAT)
    T.check_gemm(got["dW"], F.E4M3, F.E5M2, F.FLOAT, np.ascontiguousarray(got["YT"].T), np.ascontiguousarray(got["YTS"].T), 1, np.ascontiguousarray(got["dZT"].T),
                 np.ascontiguousarray(got["dZTS"].T), 1, 1.0, 1.0, dw_before)
    # the output without 8 bits: a code is off by half a step, 2^-4 of the value or 2^-10 scales, whichever is larger; 1 % of
    # that for scales, factors and float sums, 2^-9 * 9/8 for the instruction that cuts off (9 * 2^-13 of the largest of eight)
    # and 2^-8 for the result
    _, _, y = F.norm(F.from_wide(x, F.BF16), F.from_wide(r, F.BF16), gain[0].astype(np.float64), 1e-5, F.BF16)
    w64 = w.astype(np.float64)
    near = lambda v, s: 1.01 * (2.0 ** -4 * np.abs(v) + 2.0 ** -10 * s)      # noqa: E731
    ey = near(y, F.spread(got["YS"].astype(np.float64), 128, 1, y.shape[1], len(y)))
    ew = near(w64, F.spread(got["WS"].astype(np.float64), 128, 128, w64.shape[1], len(w64)))
    size = (np.abs(y) + ey) @ (np.abs(w64) + ew).T
    tol = ey @ np.abs(w64).T + np.abs(y) @ ew.T + ey @ ew.T + (2.0 ** -8 + 9 * 2.0 ** -13 + 2.0 ** -15) * size + F.HALF_SMALLEST[F.BF16]
    assert (np.abs(F.from_wide(got["Z"], F.BF16) - y @ w64.T) <= tol).all()


@pytest.mark.parametrize("n,m,t", [(512, 384, 260), (1100, 272, 5), (640, 1024, 1)])
def test_layer(hip, stream, n, m, t):
    layer = Layer(stream, np.random.default_rng(n), n, m, t)
    layer.run()
    got = layer.read()
    check_layer(got, layer.start, layer.start["dW"])
    layer.free()


@pytest.mark.parametrize("n,m,t", [(512, 384, 260), (2048, 512, 7)])
def test_layer_replayed_from_a_graph(hip, stream, n, m, t):
    """R (the residual stream) and dW (a running sum) change with every run; every replay equals the eager run bit for bit,
    with eager work of the same kind, which uses the same workspace, between the replays."""
    layer, other = Layer(stream, np.random.default_rng(n + 1), n, m, t), Layer(stream, np.random.default_rng(n + 2), 640, 256, 130)
    eager = []
    for _ in range(4):
        layer.run()
        eager.append(layer.read())
    assert not np.array_equal(eager[0]["dW"], eager[1]["dW"])
    layer.reset()
    oh.check(L.och_stream_begin_capture(stream.handle))
    layer.run()
    graph = C.c_void_p()
    oh.check(L.och_stream_end_capture(stream.handle, C.byref(graph)))
    for k in range(4):
        oh.check(L.och_graph_launch(graph, stream.handle))
        got = layer.read()
        for name in got:
            assert np.array_equal(got[name], eager[k][name], equal_nan=True), "replay %d: %s differs from the eager launches" % (k, name)
        other.run()
        stream.synchronize()
    oh.check(L.och_graph_destroy(graph))
    layer.free()
    other.free()


def test_every_product_kernel_replayed_from_a_graph(hip, stream):
    """Few columns, few columns' shares of K, tiles with shares of K, tiles, and large tiles."""
    rng = np.random.default_rng(77)
    cases = []
    for dtype, ta, tb, M, N, K, pad in [(F.BF16, "T", "N", 512, 1, 4096, 0), (F.FLOAT, "T", "N", 300, 40, 1000, 16), (F.FLOAT, "N", "N", 256, 200, 8192, 0),
                                        (F.HALF, "N", "T", 400, 129, 2000, 1), (F.BF16, "T", "N", 4096, 4352, 256, 0), (F.FLOAT, "N", "T", 2048, 2304, 384, 0)]:
        a, sa, b, sb = T.exact_case(rng, M, N, K, 128, 1)
        A, B, SA, SB = T.stored(a, ta == "T"), T.stored(b, tb == "N"), T.stored(sa, ta == "T"), T.stored(sb, tb == "N")
        mats = [T.Matrix(stream, v.shape[1], v.shape[0], v.dtype, v.shape[1] + pad, pad, v) for v in (A, SA, B, SB)]
        mats.append(T.Matrix(stream, M, N, F.STORAGE[dtype], M + pad, pad))
        cases.append((dtype, ta, tb, M, N, K, mats))

    def run():
        for dtype, ta, tb, M, N, K, (A, SA, B, SB, Cm) in cases:
            oh.check(L.och_gemm_scaled(F.E4M3, F.E4M3, dtype, ta.encode(), tb.encode(), M, N, K, 0.25, A.ptr, A.ld, SA.ptr, SA.ld, 128, B.ptr, B.ld, SB.ptr, SB.ld, 1,
                                       0.0, Cm.ptr, Cm.ld, stream.handle))

    def clear():
        for c in cases:
            c[-1][-1].buf.upload(c[-1][-1].host.view(np.uint8))
        stream.synchronize()
    run()
    want = [c[-1][-1].read() for c in cases]
    clear()
    oh.check(L.och_stream_begin_capture(stream.handle))
    run()
    graph = C.c_void_p()
    oh.check(L.och_stream_end_capture(stream.handle, C.byref(graph)))
    for k in range(3):
        oh.check(L.och_graph_launch(graph, stream.handle))
        for c, w in zip(cases, want):
            assert np.array_equal(c[-1][-1].read(), w), (k, c[:6])
        clear()
        run()
        for c, w in zip(cases, want):
            assert np.array_equal(c[-1][-1].read(), w), (k, c[:6])
        clear()
    oh.check(L.och_graph_destroy(graph))
    for c in cases:
        for m in c[-1]:
            m.free()


def test_two_streams_at_once(hip, stream):
    """Layers on two streams, interleaved call by call in turns: each has its own workspace."""
    second = oh.Stream()
    a, b = Layer(stream, np.random.default_rng(5), 1024, 512, 300), Layer(second, np.random.default_rng(6), 768, 640, 260)
    a.run()
    want_a = a.read()
    b.run()
    want_b = b.read()
    for _ in range(3):
        a.reset()
        b.reset()
        a.run()
        b.run()
        got_b, got_a = b.read(), a.read()
        for k in got_a:
            assert np.array_equal(got_a[k], want_a[k], equal_nan=True) and np.array_equal(got_b[k], want_b[k], equal_nan=True), k
    a.free()
    b.free()
    second.synchronize()
    second.destroy()
