"""What the operators refuse, checked without a GPU: the C ABI rejects bad arguments before any device
work, and the torch front end what is no device tensor."""
from __future__ import annotations

import ctypes
import pathlib
import subprocess

import pytest
import torch

INVALID = 1  # hipErrorInvalidValue
NULL = ctypes.c_void_p(0)


@pytest.fixture(scope="module")
def L():
    from hyperkernels_amd import _lib

    return _lib.lib()


def _arr(*xs):
    return (ctypes.c_void_p * len(xs))(*xs)


def test_adam8_plan_refuses(L):
    plan = ctypes.c_void_p(1)
    sizes = (ctypes.c_int64 * 1)(300)

    def create(n=1, params=_arr(1 << 20), grads=_arr(1 << 21), kind=0, copies=NULL, sz=sizes,
               states=(1 << 12, 1 << 13, 1 << 14, 1 << 15)):
        return L.hk_adam8_plan_create(n, params, grads, kind, copies, sz, *states,
                                      ctypes.byref(plan))

    for bad in (dict(n=-1), dict(kind=3), dict(kind=-1), dict(params=NULL), dict(grads=NULL),
                dict(sz=NULL), dict(params=_arr(0)), dict(grads=_arr(0)), dict(params=_arr(66)),
                dict(grads=_arr(66)), dict(grads=_arr(65), kind=1), dict(copies=_arr(65)),
                dict(sz=(ctypes.c_int64 * 1)(-1)), dict(sz=(ctypes.c_int64 * 1)(1 << 60)),
                dict(states=(0, 1 << 13, 1 << 14, 1 << 15)), dict(states=(1 << 12, 0, 1 << 14, 1 << 15)),
                dict(states=(1 << 12, 1 << 13, 0, 1 << 15)), dict(states=(1 << 12, 1 << 13, 1 << 14, 0)),
                dict(states=(4098, 1 << 13, 1 << 14, 1 << 15)),
                dict(states=(1 << 12, 8194, 1 << 14, 1 << 15)),
                # memory that two parts of a step would write
                dict(n=2, params=_arr(1 << 20, (1 << 20) + 1196), grads=_arr(1 << 21, 1 << 22),
                     sz=(ctypes.c_int64 * 2)(300, 300)),
                dict(copies=_arr((1 << 20) + 1198)), dict(copies=_arr((1 << 20) - 598)),
                dict(states=(1 << 12, (1 << 12) + 508, 1 << 14, 1 << 15)),
                dict(states=(1 << 12, 1 << 13, 1 << 14, (1 << 14) + 4)),
                dict(states=(1 << 20, 1 << 13, 1 << 14, 1 << 15))):
        assert create(**bad) == INVALID, bad
        assert plan.value is None  # no plan is handed out
    assert L.hk_adam8_plan_create(0, NULL, NULL, 0, NULL, NULL, *([NULL] * 4), NULL) == INVALID
    assert L.hk_adam8_plan_step(NULL, *([0.1] * 7), NULL) == INVALID
    assert L.hk_adam8_plan_num_blocks(NULL) == 0
    assert L.hk_adam8_plan_destroy(NULL) == 0


@pytest.mark.parametrize("name", ["hk_adam8_quantize", "hk_adam8_dequantize"])
def test_adam8_conversion_refuses(L, name):
    fn = getattr(L, name)

    def go(n, ptrs):
        m, v, a, b, c, d = ptrs
        return fn(m, v, n, a, b, c, d, NULL) if name == "hk_adam8_quantize" else fn(
            a, b, c, d, n, m, v, NULL)

    assert go(-1, [64] * 6) == INVALID
    assert go(1 << 50, [64] * 6) == INVALID
    for i in range(6):
        assert go(10, [64 if j != i else 0 for j in range(6)]) == INVALID
        assert go(10, [64 if j != i else 66 for j in range(6)]) == INVALID
    assert go(0, [0] * 6) == 0  # nothing to do


def test_adam8_front_end_refuses_host_tensors():
    from hyperkernels_amd import kernels as hk

    x = torch.zeros(300)
    state = hk.adam8_states([300], "cpu")
    assert state[0].numel() == 512 and state[2].numel() == 2
    with pytest.raises(ValueError):
        hk.Adam8Plan([x], [x], *state)
    with pytest.raises(ValueError):
        hk.adam8_quantize(x, x)
    with pytest.raises(ValueError):
        hk.adam8_dequantize(*state)
    with pytest.raises(ValueError):
        hk.Adam8Plan([x], [x, x], *state)


def _qk(**kw):
    from hyperkernels_amd.kernels import QkNormRopeParams

    base = dict(q=64, k=128, cos=192, sin=256, q_out=320, k_out=384, dq_out=448, dk_out=512, dq=576, dk=640,
                B=1, T=4, q_heads=2, k_heads=1, head_dim=64, rotary_dim=64, eps=1e-6, table_rows=4,
                table_stride=32, qo_strideM=128, qo_strideH=64, ko_strideM=64, dq_strideM=128,
                dq_strideH=64, dk_strideM=64)
    return QkNormRopeParams(**{**base, **kw})


@pytest.mark.parametrize("backward", [False, True])
def test_qk_norm_rope_refuses(L, backward):
    def go(kind=0, **kw):
        p = ctypes.byref(_qk(**kw))
        if not backward:
            return L.hk_qk_norm_rope_forward(p, kind, NULL)
        assert L.hk_qk_norm_rope_workspace(p, kind) == -1
        return L.hk_qk_norm_rope_backward(p, kind, NULL, 0, NULL)

    bad = [dict(B=-1), dict(T=-1), dict(q_heads=-1), dict(k_heads=-1), dict(head_dim=0),
           dict(head_dim=257), dict(rotary_dim=3), dict(rotary_dim=66), dict(rotary_dim=-2),
           dict(kind=3), dict(kind=-1), dict(cos=0), dict(sin=0), dict(cos=66), dict(table_rows=3),
           dict(table_stride=31), dict(positions=68), dict(q=0), dict(k=0), dict(q=66), dict(q=65, kind=1),
           dict(q_weight=66), dict(B=1 << 20, T=1 << 20, positions=64)]
    if backward:
        bad += [dict(dq=0), dict(dk=0), dict(dq_out=0), dict(dq=66), dict(dq_weight=66),
                dict(dk_out=66, kind=1, f32_io=True)]
    else:
        bad += [dict(q_out=0), dict(k_out=0), dict(q_out=66), dict(q_out=66, kind=1, f32_io=True)]
    for kw in bad:
        assert go(**kw) == INVALID, kw
    if backward:
        assert L.hk_qk_norm_rope_backward(NULL, 0, NULL, 0, NULL) == INVALID
        assert L.hk_qk_norm_rope_workspace(ctypes.byref(_qk()), 0) == 0  # no weight gradients
        p = _qk(dq_weight=64)
        n = L.hk_qk_norm_rope_workspace(ctypes.byref(p), 0)
        assert n > 0
        assert L.hk_qk_norm_rope_backward(ctypes.byref(p), 0, 64, n - 1, NULL) == INVALID
        assert L.hk_qk_norm_rope_backward(ctypes.byref(p), 0, 66, n, NULL) == INVALID
    else:
        assert L.hk_qk_norm_rope_forward(NULL, 0, NULL) == INVALID
        assert L.hk_qk_norm_rope_forward(ctypes.byref(_qk(B=0, q=0, k=0)), 0, NULL) == 0


@pytest.mark.parametrize("backward", [False, True])
def test_qk_refuses_rows_written_twice(L, backward):
    q, k = ("dq", "dk") if backward else ("qo", "ko")
    bad = [{f"{q}_strideM": 0}, {f"{q}_strideH": 0}, {f"{k}_strideM": 0}, dict(B=2),
           {"B": 2, f"{q}_strideB": 512}, {"k_heads": 2}]
    if backward:
        bad += [dict(dq_weight=4096, dk_weight=4096), dict(dq_weight=4096, dk_weight=4096 + 252),
                dict(dq=640), dict(dq=128), dict(dk=64), dict(dq=512), dict(dk=448)]
    else:
        bad += [dict(q_out=384), dict(q_out=128), dict(k_out=64)]
    for kw in bad:
        p = ctypes.byref(_qk(**kw))
        status = L.hk_qk_norm_rope_backward(p, 0, NULL, 0, NULL) if backward else (
            L.hk_qk_norm_rope_forward(p, 0, NULL))
        assert status == INVALID, kw


def test_qk_front_end_refuses_host_tensors():
    from hyperkernels_amd import kernels as hk

    q = torch.zeros(1, 2, 4, 64)
    with pytest.raises(ValueError):
        hk.qk_norm_rope_forward(q, q)
    with pytest.raises(ValueError):
        hk.qk_norm_rope_backward(q, q, q, q)
    with pytest.raises(ValueError):
        hk.qk_norm_rope_forward(None, None)


def test_qk_parameter_block_matches_the_header(tmp_path):
    from hyperkernels_amd.kernels import QkNormRopeParams as P

    root = pathlib.Path(__file__).resolve().parents[1]
    fields = [n for n, _ in P._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "hk.h"\nint main(void) {\n'
                   '  printf("%zu", sizeof(hk_qk_norm_rope_params));\n' + "".join(
                       f'  printf(" %zu", offsetof(hk_qk_norm_rope_params, {n}));\n'
                       for n in fields) + "  return 0;\n}\n")
    subprocess.run(["gcc", "-D__HIP_PLATFORM_AMD__", f"-I{root / 'include'}", "-I/opt/rocm/include",
                    str(src), "-o", str(tmp_path / "probe")], check=True)
    got = list(map(int, subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True,
                                       check=True).stdout.split()))
    assert got == [ctypes.sizeof(P)] + [getattr(P, n).offset for n in fields]


@pytest.mark.parametrize("backward", [False, True])
def test_bgemm_act_refuses(L, backward):
    def go(ta=0, tb=0, M=4, N=8, K=16, A=64, lda=16, B=1024, ldb=8, act=2, res=2048, ldr=8, Z=4096,
           ldz=8, C=8192, ldc=8, dbias=64, batch=1, ws=0, ws_bytes=0):
        if backward:
            return L.hk_bgemm_act_backward(ta, tb, M, N, K, 0x3F80, A, lda, 0, B, ldb, 0, act, Z, ldz,
                                           0, C, ldc, 0, dbias, 0, 0, batch, ws, ws_bytes, NULL)
        return L.hk_bgemm_act(ta, tb, M, N, K, 0x3F80, A, lda, 0, B, ldb, 0, 64, 0, act, res, ldr, 0,
                              Z, ldz, 0, C, ldc, 0, batch, ws, ws_bytes, NULL)

    bad = [dict(ta=3), dict(ta=-1), dict(tb=3), dict(M=-1), dict(N=-1), dict(K=-1), dict(A=0),
           dict(B=0), dict(C=0), dict(lda=15), dict(ldb=7), dict(ldc=7), dict(act=4), dict(act=-1),
           dict(batch=-1), dict(batch=65536), dict(ldz=7), dict(ta=1, lda=3), dict(tb=1, ldb=15)]
    bad += [dict(C=64), dict(C=1024)]
    bad += [dict(Z=0), dict(dbias=66)] if backward else [dict(ldr=7), dict(Z=64), dict(Z=1024),
                                                         dict(Z=2048), dict(Z=8192)]
    for kw in bad:
        assert go(**kw) == INVALID, kw
    if not backward:
        assert go(M=0, A=0, B=0, C=0) == 0 and go(N=0) == 0 and go(batch=0) == 0
    for n in ((3, 0, 4, 8, 16, 1, 0), (0, -1, 4, 8, 16, 1, 0), (0, 0, -1, 8, 16, 1, 0),
              (0, 0, 4, -8, 16, 1, 0), (0, 0, 4, 8, -1, 1, 0), (0, 0, 4, 8, 16, -1, 0),
              (0, 0, 4, 8, 16, 65536, 0)):
        assert L.hk_bgemm_act_workspace(*n) == -1
    assert L.hk_bgemm_act_workspace(0, 0, 0, 8, 16, 1, 1) == 0
    assert L.hk_bgemm_act_workspace(0, 0, 4, 8, 16, 1, 1) > 0


def test_bgemm_act_refuses_overlapping_outputs_and_huge_sides(L):
    def fwd(M=4, N=8, K=16, sZ=32, sC=32, batch=2):
        return L.hk_bgemm_act(0, 0, M, N, K, 0x3F80, 64, K, 0, 1024, N, 0, 64, 0, 2, 2048, N, 0, 4096, N, sZ,
                              8192, N, sC, batch, NULL, 0, NULL)

    def bwd(N=8, sC=32, sD=8, batch=2):
        return L.hk_bgemm_act_backward(0, 0, 4, N, 16, 0x3F80, 64, 16, 0, 1024, N, 0, 2, 4096, N, 0, 8192, N,
                                       sC, 64, sD, 0, batch, NULL, 0, NULL)

    huge = 2 ** 31 - 2 ** 16 + 1
    for status in (fwd(sC=0), fwd(sZ=0), fwd(M=huge), fwd(N=huge), fwd(K=huge), bwd(sC=0), bwd(sD=7),
                   bwd(sD=-7), bwd(N=huge)):
        assert status == INVALID
    for n in ((huge, 8, 16), (4, huge, 16), (4, 8, huge)):
        assert L.hk_bgemm_act_workspace(0, 0, *n, 1, 0) == -1


def test_bgemm_act_front_end_refuses():
    from hyperkernels_amd import kernels as hk

    bf = torch.bfloat16
    a, b = torch.zeros(4, 16, dtype=bf), torch.zeros(16, 8, dtype=bf)
    with pytest.raises(ValueError):
        hk.bgemm_act(a, b)  # host tensors
    with pytest.raises(ValueError):
        hk.bgemm_act(a, b, activation="tanh")
    with pytest.raises(ValueError):
        hk.bgemm_act(a[None], b)
    with pytest.raises(ValueError):
        hk.bgemm_act_backward(a, b)


def test_qk_packed_block_is_the_structure():
    """The packed parameter block has the structure's layout, field by field."""
    from hyperkernels_amd import kernels as hk

    names = [n for n, _ in hk.QkNormRopeParams._fields_]
    values = {n: i + 1 for i, n in enumerate(names)}
    values |= dict(interleaved=True, f32_io=False, accumulate=True, eps=0.5)
    got = hk.QkNormRopeParams.from_buffer_copy(
        hk._QK_PACK(*values.values()).ljust(ctypes.sizeof(hk.QkNormRopeParams), b"\0"))
    assert len(hk._QK_PACK(*values.values())) == ctypes.sizeof(hk.QkNormRopeParams)
    for n in names:
        assert getattr(got, n) == values[n], n
