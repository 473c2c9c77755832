"""Refusals of the block-scaled 8-bit operations, which are made on the host before a device is touched, and the oracle's
own rounding against the code tables."""
import ctypes as C

import numpy as np
import pytest

import float8_oracle as F
import ocean_hip as oh

P = C.c_void_p(0x1000)          # never dereferenced: every call below is refused, or has nothing to do
L = oh.lib


def refused(status, *words):
    assert status == -1
    message = L.och_last_error().decode()
    assert all(w in message for w in words), message


def quantize(dtype=F.BF16, code=F.E4M3, M=256, N=4, X=P, ldX=256, bm=128, bn=1, Q=P, ldQ=256, S=P, ldS=2):
    return L.och_quantize_blocks(dtype, code, M, N, X, ldX, bm, bn, Q, ldQ, S, ldS, None)


def test_quantize_refusals():
    refused(quantize(dtype=oh.DOUBLE), "half, bfloat16 and float")
    refused(quantize(dtype=oh.FLOAT8_E4M3), "half, bfloat16 and float")
    refused(quantize(code=oh.UINT8), "float8")
    for bm, bn in ((1, 1), (64, 1), (128, 2), (0, 128), (256, 1)):
        refused(quantize(bm=bm, bn=bn), "128 x 1, 1 x 128 or 128 x 128")
    refused(quantize(X=None), "null pointer")
    refused(quantize(Q=None), "null pointer")
    refused(quantize(S=None), "null pointer")
    refused(quantize(ldX=255), "leading dimension")
    refused(quantize(ldQ=255), "leading dimension")
    refused(quantize(ldS=1), "leading dimension")
    refused(quantize(ldX=-256), "leading dimension")
    refused(quantize(X=C.c_void_p(0x1001)), "misaligned")
    refused(quantize(S=C.c_void_p(0x1002)), "misaligned")
    refused(quantize(M=1 << 31, ldX=1 << 31, ldQ=1 << 31, ldS=1 << 30), "too long")
    assert quantize(M=0) == 0 and quantize(N=0) == 0


def norm(dtype=F.BF16, n=256, rows=4, X=P, ldX=256, R=None, ldR=0, H=None, ldH=0, dtype_w=F.FLOAT, W=P, eps=1e-6, dtype_y=F.E4M3, Y=P, ldY=256, S=P, ldS=2, rstd=P):
    return L.och_rms_norm(dtype, n, rows, X, ldX, R, ldR, H, ldH, dtype_w, W, eps, dtype_y, Y, ldY, S, ldS, rstd, None)


def test_norm_refusals():
    refused(norm(dtype=oh.DOUBLE), "half, bfloat16 and float")
    refused(norm(dtype_y=F.FLOAT), "output")
    refused(norm(dtype_y=oh.INT8), "output")
    refused(norm(eps=-1e-6), "eps")
    refused(norm(eps=float("nan")), "eps")
    refused(norm(X=None), "null pointer")
    refused(norm(Y=None), "null pointer")
    refused(norm(S=None), "null pointer")
    refused(norm(R=P, ldR=256), "null pointer")                       # the sum needs a place
    refused(norm(ldX=255), "leading dimension")
    refused(norm(ldY=255), "leading dimension")
    refused(norm(ldS=1), "leading dimension")
    refused(norm(R=P, ldR=255, H=P, ldH=256), "leading dimension")
    refused(norm(R=P, ldR=256, H=P, ldH=255), "leading dimension")
    refused(norm(dtype_w=F.HALF), "weights")
    refused(norm(W=C.c_void_p(0x1002)), "misaligned")
    refused(norm(X=C.c_void_p(0x1001)), "misaligned")
    refused(norm(rstd=C.c_void_p(0x1002)), "misaligned")
    refused(norm(rows=1 << 31), "too long")
    assert norm(n=0) == 0 and norm(rows=0) == 0


def grad(dtype=F.BF16, n=256, rows=4, dY=P, lddY=256, H=P, ldH=256, rstd=P, dtype_w=F.FLOAT, W=P, dH=None, lddH=0, dX=P, lddX=256, dW=P):
    return L.och_rms_norm_grad(dtype, n, rows, dY, lddY, H, ldH, rstd, dtype_w, W, dH, lddH, dX, lddX, dW, None)


def test_norm_grad_refusals():
    refused(grad(dtype=oh.INT32), "half, bfloat16 and float")
    for name in ("dY", "H", "rstd", "dX"):
        refused(grad(**{name: None}), "null pointer")
    refused(grad(lddY=255), "leading dimension")
    refused(grad(ldH=255), "leading dimension")
    refused(grad(lddX=255), "leading dimension")
    refused(grad(dH=P, lddH=255), "leading dimension")
    refused(grad(dtype_w=F.HALF), "weights")
    refused(grad(dW=C.c_void_p(0x1002)), "misaligned")
    refused(grad(n=(1 << 24) + 1, lddY=1 << 25, ldH=1 << 25, lddX=1 << 25), "too long")
    assert grad(n=0) == 0 and grad(rows=0, dW=None) == 0


def gemm(ca=F.E4M3, cb=F.E4M3, dtype=F.BF16, ta=b"T", tb=b"N", M=256, N=8, K=384, A=P, ldA=384, SA=P, ldSA=3, ba=128, B=P, ldB=384, SB=P, ldSB=3, bb=1, beta=0.0, Cc=P, ldC=256):
    return L.och_gemm_scaled(ca, cb, dtype, ta, tb, M, N, K, 1.0, A, ldA, SA, ldSA, ba, B, ldB, SB, ldSB, bb, beta, Cc, ldC, None)


def test_gemm_refusals():
    refused(gemm(ca=oh.INT8), "operands")
    refused(gemm(cb=F.HALF), "operands")
    refused(gemm(dtype=oh.DOUBLE), "result")
    refused(gemm(dtype=F.E4M3), "result")
    refused(gemm(ta=b"C"), "transposition")
    refused(gemm(tb=b"n"), "transposition")
    refused(gemm(ba=64), "1 or 128")
    refused(gemm(bb=0), "1 or 128")
    for name in ("A", "SA", "B", "SB", "Cc"):
        refused(gemm(**{name: None}), "null pointer")
    refused(gemm(ldA=383), "ldA")
    refused(gemm(ta=b"N", ldA=255), "ldA")
    refused(gemm(tb=b"T", ldB=7), "ldB")
    refused(gemm(ldSA=2), "ldSA")
    refused(gemm(ta=b"N", ldSA=1), "ldSA")
    refused(gemm(ldSB=2), "ldSB")
    refused(gemm(ldC=255), "ldC")
    refused(gemm(Cc=C.c_void_p(0x1001)), "misaligned")
    refused(gemm(SA=C.c_void_p(0x1001)), "misaligned")
    refused(gemm(M=1 << 31, ldC=1 << 31), "too long")
    assert gemm(M=0) == 0 and gemm(N=0) == 0


@pytest.mark.parametrize("code", [F.E4M3, F.E5M2])
def test_oracle_rounds_to_the_nearest_code(code):
    finite = np.flatnonzero(np.isfinite(F.TABLE[code]))
    assert np.array_equal(F.encode(F.TABLE[code][finite], code), finite)
    positive = F.TABLE[code][:128]
    positive = positive[np.isfinite(positive)]
    middle = (positive[1:] + positive[:-1]) / 2
    assert np.array_equal(F.encode(middle, code) % 2, np.zeros(len(middle)))        # ties to the even code
    assert np.array_equal(F.encode(np.nextafter(middle, 1e9), code), np.arange(1, len(positive)))
    assert np.array_equal(F.encode(np.nextafter(middle, 0), code), np.arange(0, len(positive) - 1))


def test_refusals_of_operations_in_place():
    other = C.c_void_p(0x10000)
    refused(norm(R=other, ldR=256, H=P, ldH=264, Y=C.c_void_p(0x20000)), "in place")
    refused(norm(R=other, ldR=256, H=other, ldH=264, Y=C.c_void_p(0x20000)), "in place")
    refused(norm(), "X's place")                                       # codes over X
    refused(norm(dtype_y=F.BF16, ldY=264), "X's place")
    refused(norm(dtype_y=F.BF16, R=other, ldR=256, H=other, ldH=256), "X's place")
    refused(grad(lddX=264), "place of dY")
    refused(grad(dY=other, dH=P, lddH=256, lddX=264), "place of dY")
