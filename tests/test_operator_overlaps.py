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


def _qk(L, backward, kind=1, **kw):
    """16-bit q [2, 4, 8, 64] and k [2, 2, 8, 64] by token, each tensor in memory of its own."""
    from hyperkernels_amd.kernels import QkNormRopeParams

    B, T, H, K, d = 2, 8, 4, 2, 64
    a = dict(q=AT, k=2 * AT, q_weight=3 * AT, k_weight=4 * AT, cos=5 * AT, sin=6 * AT, positions=7 * AT, q_out=8 * AT,
             k_out=9 * AT, dq_out=10 * AT, dk_out=11 * AT, dq=12 * AT, dk=13 * AT, dq_weight=14 * AT, dk_weight=15 * AT,
             B=B, T=T, q_heads=H, k_heads=K, head_dim=d, rotary_dim=32, eps=1e-6, table_rows=20, table_stride=16,
             pos_strideB=T)
    for n, h in (("q", H), ("k", K), ("qo", H), ("ko", K), ("dq", H), ("dk", K)):
        a |= {f"{n}_strideB": T * h * d, f"{n}_strideM": h * d, f"{n}_strideH": d}
    p = ctypes.byref(QkNormRopeParams(**a | kw))
    if backward:
        return L.hk_qk_norm_rope_backward(p, kind, NULL, 0, NULL)
    return L.hk_qk_norm_rope_forward(p, kind, NULL)


Q, K, QO, KO, DQ, DK = AT, 2 * AT, 8 * AT, 9 * AT, 12 * AT, 13 * AT
Q_LAST, K_LAST = 2 * (2 * 4 * 8 * 64 - 1), 2 * (2 * 2 * 8 * 64 - 1)
DENSE = {"strideM": 64, "strideH": 8 * 64}  # [B, heads, T, d] in order


def _as(name, strides):
    return {f"{name}_{s}": v for s, v in strides.items()}


@pytest.mark.parametrize("bad", [
    # in place with other strides, or with elements of another size
    dict(q_out=Q, **_as("qo", DENSE)), dict(k_out=K, ko_strideM=144, ko_strideB=8 * 144), dict(q_out=Q, f32_io=True),
    dict(k_out=K, f32_io=True), dict(q_out=Q, T=4, q_heads=4, qo_strideM=64, qo_strideH=256),
    # shifted
    dict(q_out=Q + 2), dict(q_out=Q - 128), dict(q_out=Q + Q_LAST), dict(k_out=K + 64), dict(k_out=K - K_LAST),
    # on the other side, on what both sides read, and on itself
    dict(q_out=K + 4), dict(k_out=Q + Q_LAST), dict(k_out=Q), dict(k_out=QO + 64), dict(q_out=3 * AT), dict(k_out=4 * AT + 64),
    dict(q_out=5 * AT + 1200), dict(q_out=6 * AT + 64), dict(k_out=7 * AT + 64), dict(qo_strideM=63, qo_strideH=512),
    dict(qo_strideH=32), dict(ko_strideB=1000), dict(qo_strideM=0), dict(ko_strideH=-8)])
def test_query_and_key_norms(L, bad):
    assert _qk(L, False, **bad) == INVALID


@pytest.mark.parametrize("bad", [
    dict(dq=Q, **_as("dq", DENSE)), dict(dq=10 * AT, **_as("dq", DENSE)), dict(dk=11 * AT, f32_io=True),
    dict(dq=10 * AT, f32_io=True), dict(dq=Q + 2), dict(dk=11 * AT - 128), dict(dq=10 * AT + Q_LAST), dict(dq=K),
    dict(dk=10 * AT + 64), dict(dq=11 * AT), dict(dk=DQ + 640), dict(dq_strideM=32), dict(dk_strideB=4),
    dict(dq_weight=15 * AT - 252), dict(dq_weight=DQ + 64), dict(dk_weight=DQ + 64), dict(dk_weight=Q + 64),
    dict(dq_weight=11 * AT + 64), dict(dq_weight=3 * AT), dict(dk_weight=5 * AT + 64), dict(dq=3 * AT), dict(dk=6 * AT)])
def test_gradients_of_query_and_key_norms(L, bad):
    assert _qk(L, True, **bad) == INVALID


def _arr(*xs):
    return (ctypes.c_void_p * len(xs))(*xs)


@pytest.mark.parametrize("kind,grads,ok", [
    (0, (AT + 4, 4 * AT), False), (0, (AT - 4 * 299, 4 * AT), False), (0, (3 * AT, AT + 1196), False),
    (0, (2 * AT, 4 * AT), False), (1, (AT, 4 * AT), False), (1, (3 * AT, 4 * AT + 2), True), (0, (AT, 4 * AT), True),
    (1, (3 * AT, 5 * AT + 600), True),  # behind the copy's 600 bytes
    (1, (3 * AT, 5 * AT + 598), False), (1, (5 * AT - 2 * 299, 4 * AT), False), (0, (6 * AT + 508, 4 * AT), False),
    (0, (7 * AT, 4 * AT), False), (0, (3 * AT, 8 * AT + 12), False), (2, (3 * AT, 9 * AT), False)])
def test_gradients_on_what_a_step_writes(L, kind, grads, ok):
    """Two tensors of 300 elements with a copy of the second; states of four blocks."""
    plan = ctypes.c_void_p(1)
    status = L.hk_adam8_plan_create(2, _arr(AT, 2 * AT), _arr(*grads), kind, _arr(0, 5 * AT),
                                    (ctypes.c_int64 * 2)(300, 300), 6 * AT, 7 * AT, 8 * AT, 9 * AT,
                                    ctypes.byref(plan))
    assert (status != INVALID) == ok
    if status == 0:
        L.hk_adam8_plan_destroy(plan)


@pytest.mark.parametrize("name", ["hk_adam8_quantize", "hk_adam8_dequantize"])
@pytest.mark.parametrize("at", [(1, 1, 3, 4, 5, 6), (1, 2, 1, 4, 5, 6), (1, 2, 3, 2, 5, 6), (1, 2, 3, 4, 1, 6),
                                (1, 2, 3, 4, 5, 5), (1, 2, 3, 3, 5, 6), (1, 2, 3, 4, 3, 6)])
@pytest.mark.parametrize("shift", [0, 4])
def test_conversions(L, name, at, shift):
    """300 elements: fp32 moments of 1,200 bytes, codes of 512, scales of 8."""
    m, v, a, b, c, d = (AT * x + shift * at[:i].count(x) for i, x in enumerate(at))
    if name == "hk_adam8_quantize":
        assert L.hk_adam8_quantize(m, v, 300, a, b, c, d, NULL) == INVALID
    else:
        assert L.hk_adam8_dequantize(a, b, c, d, 300, m, v, NULL) == INVALID
