"""Sizes at the ends of what the operators take, refused without a GPU."""
from __future__ import annotations

import ctypes

import pytest

INVALID = 1  # hipErrorInvalidValue
NULL = ctypes.c_void_p(0)


@pytest.fixture(scope="module")
def L():
    from hyperkernels_amd import _lib

    return _lib.lib()


@pytest.mark.parametrize("size", [2 ** 63 - 1, 2 ** 63 - 256, 2 ** 62, (2 ** 31 - 1) * 256 + 1])
def test_adam8_sizes_past_the_blocks(L, size):
    one = lambda x: (ctypes.c_void_p * 1)(x)  # noqa: E731
    plan = ctypes.c_void_p(1)
    assert L.hk_adam8_plan_create(1, one(1 << 20), one(1 << 60), 0, NULL, (ctypes.c_int64 * 1)(size), 1 << 12,
                                  1 << 13, 1 << 14, 1 << 15, ctypes.byref(plan)) == INVALID
    assert plan.value is None
    assert L.hk_adam8_quantize(64, 64, size, 64, 64, 64, 64, NULL) == INVALID
    assert L.hk_adam8_dequantize(64, 64, 64, 64, size, 64, 64, NULL) == INVALID
