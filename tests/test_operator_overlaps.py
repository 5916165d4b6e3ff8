"""Outputs that lie on what another workgroup of the same call reads or writes: refused, without a GPU."""
from __future__ import annotations

import ctypes

import pytest

INVALID = 1  # hipErrorInvalidValue
NULL = ctypes.c_void_p(0)
AT = 1 << 20  # where a call's first tensor lies; the others a megabyte apart


@pytest.fixture(scope="module")
def L():
    from hyperkernels_amd import _lib

    return _lib.lib()


def _forward(L, M=64, N=32, K=16, batch=2, ta=0, tb=0, **kw):
    """z = A B + bias and C = act(z) + residual of two batches, each tensor in memory of its own."""
    a = dict(A=AT, lda=M if ta else K, sA=M * K, B=2 * AT, ldb=K if tb else N, sB=K * N, bias=3 * AT, sBias=0,
             R=4 * AT, ldr=N, sR=M * N, Z=5 * AT, ldz=N, sZ=M * N, C=6 * AT, ldc=N, sC=M * N) | kw
    return L.hk_bgemm_act(ta, tb, M, N, K, 0x3F80, a["A"], a["lda"], a["sA"], a["B"], a["ldb"], a["sB"], a["bias"],
                          a["sBias"], 2, a["R"], a["ldr"], a["sR"], a["Z"], a["ldz"], a["sZ"], a["C"], a["ldc"],
                          a["sC"], batch, NULL, 0, NULL)


def _backward(L, M=64, N=32, K=16, batch=2, **kw):
    a = dict(A=AT, B=2 * AT, Z=5 * AT, ldz=N, sZ=M * N, C=6 * AT, ldc=N, sC=M * N, db=7 * AT, sD=N) | kw
    return L.hk_bgemm_act_backward(0, 0, M, N, K, 0x3F80, a["A"], K, M * K, a["B"], N, K * N, 2, a["Z"], a["ldz"],
                                   a["sZ"], a["C"], a["ldc"], a["sC"], a["db"], a["sD"], 0, batch, NULL, 0, NULL)


C = 6 * AT
LAST = 2 * (2 * 64 * 32 - 1)  # of two batches, the last element's first byte


@pytest.mark.parametrize("bad", [
    # a residual at C's address whose rows, or batches, are elsewhere
    dict(R=C, ldr=40), dict(R=C, sR=0), dict(R=C, sR=64 * 32 + 8), dict(R=C, ldc=40, sC=64 * 40),
    # and one some elements on, or back
    dict(R=C + 2), dict(R=C - 16), dict(R=C + 64), dict(R=C + LAST), dict(R=C - LAST),
    # the pre-activation, bias, weights and input on C, and on the pre-activation
    dict(Z=C), dict(Z=C + 2), dict(Z=C + LAST), dict(Z=C, ldz=64, sZ=64 * 64), dict(bias=C + 640), dict(bias=C - 62),
    dict(A=C + 100), dict(A=C - 2 * (2 * 64 * 16 - 1)), dict(B=C + 128), dict(B=C - 2 * (2 * 16 * 32 - 1)),
    dict(A=5 * AT + 4), dict(B=5 * AT + 4), dict(bias=5 * AT + 4), dict(R=5 * AT + 4), dict(R=5 * AT),
    # batches of an output on each other
    dict(sC=32), dict(sC=63 * 32), dict(sC=8), dict(sZ=32), dict(sZ=-8), dict(sC=0), dict(sZ=0),
    # one batch
    dict(batch=1, R=C + 2), dict(batch=1, R=C, ldr=33), dict(batch=1, Z=C + 2), dict(batch=1, A=C + 2)])
def test_gemm_with_an_epilogue(L, bad):
    assert _forward(L, **bad) == INVALID


@pytest.mark.parametrize("bad", [
    dict(Z=C, ldz=40), dict(Z=C, sZ=0), dict(Z=C + 2), dict(Z=C - 64), dict(Z=C + LAST), dict(A=C + 64),
    dict(B=C + 64), dict(db=C), dict(db=C + 400), dict(db=C - 124), dict(db=5 * AT + 64), dict(db=AT), dict(db=2 * AT + 4),
    dict(sC=32), dict(batch=1, db=C + 4), dict(batch=1, db=C - 124), dict(db=C - 4 * 63, sD=32), dict(db=C - 124, sD=0)])
def test_gradient_with_an_epilogue(L, bad):
    assert _backward(L, **bad) == INVALID
