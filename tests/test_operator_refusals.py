"""What the operators refuse, checked without a GPU: the C ABI rejects bad arguments before any device
work, and the torch front end what is no device tensor."""
from __future__ import annotations

import ctypes

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

    def create(n=1, params=_arr(64), grads=_arr(64), kind=0, copies=NULL, sz=sizes,
               states=(64, 64, 64, 64)):
        return L.hk_adam8_plan_create(n, params, grads, kind, copies, sz, *states,
                                      ctypes.byref(plan))

    for bad in (dict(n=-1), dict(kind=3), dict(kind=-1), dict(params=NULL), dict(grads=NULL),
                dict(sz=NULL), dict(params=_arr(0)), dict(grads=_arr(0)), dict(params=_arr(66)),
                dict(grads=_arr(66)), dict(grads=_arr(65), kind=1), dict(copies=_arr(65)),
                dict(sz=(ctypes.c_int64 * 1)(-1)), dict(sz=(ctypes.c_int64 * 1)(1 << 60)),
                dict(states=(0, 64, 64, 64)), dict(states=(64, 0, 64, 64)),
                dict(states=(64, 64, 0, 64)), dict(states=(64, 64, 64, 0)),
                dict(states=(66, 64, 64, 64)), dict(states=(64, 66, 64, 64))):
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
