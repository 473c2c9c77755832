"""Recording the block-scaled 8-bit operations with the runtime's own graphs, not through och_stream_begin_capture, as a
program does that captures with another library: a call that would have to allocate its stream's scratch while the stream
records is refused; with the scratch reserved before, every replay equals the eager calls."""
import ctypes as C

import numpy as np
import pytest

import float8_oracle as F
import ocean_hip as oh
import test_float8_gpu as T

pytestmark = pytest.mark.gpu
L = oh.lib
RT = C.CDLL(oh.LIB_PATH)                # the runtime's functions, from the library that the device library was linked to
for name, args in {"hipStreamBeginCapture": [C.c_void_p, C.c_int], "hipStreamEndCapture": [C.c_void_p, C.POINTER(C.c_void_p)], "hipGraphDestroy": [C.c_void_p],
                   "hipGraphInstantiate": [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t],
                   "hipGraphLaunch": [C.c_void_p, C.c_void_p], "hipGraphExecDestroy": [C.c_void_p]}.items():
    getattr(RT, name).argtypes = args
THREAD_LOCAL = 1


def begin(stream):
    assert RT.hipStreamBeginCapture(stream.handle, THREAD_LOCAL) == 0


def end(stream):
    graph = C.c_void_p()
    assert RT.hipStreamEndCapture(stream.handle, C.byref(graph)) == 0
    return graph


def discard(graph):
    assert not graph or RT.hipGraphDestroy(graph) == 0


class Work:
    """A product that is cut along K and a norm's gradient with dw: both keep partial sums in the stream's workspace."""

    def __init__(self, stream, seed, M=256, N=200, K=8192, n=640, rows=300):
        rng = np.random.default_rng(seed)
        self.stream, self.size, self.norm = stream, (M, N, K), (n, rows)
        a, sa, b, sb = T.exact_case(rng, M, N, K, 128, 1)
        self.h, self.dy = T.wide_data(rng, rows, n, F.BF16), T.wide_data(rng, rows, n, F.BF16)
        self.rstd = (1 / np.sqrt((F.from_wide(self.h, F.BF16) ** 2).mean(1) + 1e-5)).astype(np.float32)
        self.want = (F.decode(b, F.E4M3) * T.wide_scales(sb, 1, N, K)).astype(np.float32) @ (F.decode(a, F.E4M3) * T.wide_scales(sa, 128, M, K)).astype(np.float32).T
        self.inputs = [T.Matrix(stream, v.shape[1], v.shape[0], v.dtype, data=v) for v in (a, sa, b, sb, self.h, self.dy, self.rstd[None])]
        self.outputs = [T.Matrix(stream, M, N, np.float32), T.Matrix(stream, n, rows, np.uint16), T.Matrix(stream, n, 1, np.float32)]

    def product(self):
        A, SA, B, SB = self.inputs[:4]
        Cm = self.outputs[0]
        return L.och_gemm_scaled(F.E4M3, F.E4M3, F.FLOAT, b"T", b"N", *self.size, 1.0, A.ptr, A.ld, SA.ptr, SA.ld, 128, B.ptr, B.ld, SB.ptr, SB.ld, 1, 0.0, Cm.ptr, Cm.ld,
                                 self.stream.handle)

    def gradient(self):
        H, dY, rstd = self.inputs[4:]
        _, dX, dW = self.outputs
        return L.och_rms_norm_grad(F.BF16, *self.norm, dY.ptr, dY.ld, H.ptr, H.ld, rstd.ptr, F.FLOAT, None, None, 0, dX.ptr, dX.ld, dW.ptr, self.stream.handle)

    def run(self):
        oh.check(self.product())
        oh.check(self.gradient())

    def read(self):
        self.stream.synchronize()
        return [m.read() for m in self.outputs]

    def clear(self):
        for m in self.outputs:
            m.buf.upload(m.host.view(np.uint8))
        self.stream.synchronize()

    def check(self, got):
        assert np.array_equal(got[0], self.want)
        T.check_grad((got[1], got[2][0]), self.dy, self.h, None, self.rstd.astype(np.float64), None, F.BF16, F.FLOAT)

    def free(self):
        for m in self.inputs + self.outputs:
            m.free()


def refused(status):
    assert status == -1 and "och_stream_reserve_workspace" in L.och_last_error().decode(), L.och_last_error()


def test_a_recording_stream_gets_no_scratch(hip):
    """On a stream that the library has not seen, on one whose reductions have their scratch but which has no workspace, and
    after the workspace has been given back: refused, and the recording goes on."""
    stream = oh.Stream()
    work = Work(stream, 1)
    begin(stream)
    refused(work.product())
    refused(work.gradient())
    refused(L.och_stream_reserve_workspace(stream.handle))
    discard(end(stream))
    x, out = T.Matrix(stream, 300, 1, np.float32, data=np.ones((1, 300), np.float32)), T.Matrix(stream, 1, 1, np.float32)
    oh.check(L.och_reduce_all_device(oh.R["sum"], oh.FLOAT, 1, oh.sizes([300]), oh.strides([4]), x.ptr, None, None, 0.0, out.ptr, None, stream.handle))
    stream.synchronize()
    for _ in range(2):
        begin(stream)
        refused(work.product())
        refused(work.gradient())
        discard(end(stream))
        work.run()                                                   # now there is a workspace
        work.check(work.read())
        begin(stream)
        assert L.och_stream_release_workspace(stream.handle) == -1 and "records" in L.och_last_error().decode()
        discard(end(stream))
        work.clear()
        work.run()
        work.check(work.read())
        oh.check(L.och_stream_release_workspace(stream.handle))
    for m in (work, x, out):
        m.free()
    stream.synchronize()
    stream.destroy()


def test_recorded_behind_the_reservation(hip):
    stream = oh.Stream()
    oh.check(L.och_stream_reserve_workspace(stream.handle))
    oh.check(L.och_stream_reserve_workspace(stream.handle))          # a second time: nothing to do
    work, other = Work(stream, 2), Work(stream, 3, 300, 140, 6000, 1000, 77)
    begin(stream)
    work.run()
    graph = end(stream)
    run = C.c_void_p()
    assert RT.hipGraphInstantiate(C.byref(run), graph, None, None, 0) == 0 and RT.hipGraphDestroy(graph) == 0
    first = None
    for k in range(4):
        work.clear()
        assert RT.hipGraphLaunch(run, stream.handle) == 0
        got = work.read()
        work.check(got)
        first = first or got
        other.clear()
        other.run()                                                  # eager work that uses the same workspace
        other.check(other.read())
        work.clear()
        work.run()
        for a, b, c in zip(got, work.read(), first):
            assert np.array_equal(a, b) and np.array_equal(a, c), k
    assert RT.hipGraphExecDestroy(run) == 0
    work.free()
    other.free()
    stream.synchronize()
    stream.destroy()


def test_a_reservation_without_a_device_call_is_enough_for_a_reduction(hip):
    """The reservation also creates the reductions' scratch: a reduction is the stream's first recorded call."""
    stream = oh.Stream()
    x, out = T.Matrix(stream, 5000, 1, np.float32, data=np.ones((1, 5000), np.float32)), T.Matrix(stream, 1, 1, np.float32)
    oh.check(L.och_stream_reserve_workspace(stream.handle))
    stream.synchronize()
    begin(stream)
    oh.check(L.och_reduce_all_device(oh.R["sum"], oh.FLOAT, 1, oh.sizes([5000]), oh.strides([4]), x.ptr, None, None, 0.0, out.ptr, None, stream.handle))
    graph = end(stream)
    run = C.c_void_p()
    assert RT.hipGraphInstantiate(C.byref(run), graph, None, None, 0) == 0 and RT.hipGraphDestroy(graph) == 0
    for _ in range(3):
        out.buf.upload(out.host.view(np.uint8))
        assert RT.hipGraphLaunch(run, stream.handle) == 0
        stream.synchronize()
        assert out.read()[0, 0] == 5000
    assert RT.hipGraphExecDestroy(run) == 0
    x.free()
    out.free()
    stream.synchronize()
    stream.destroy()
