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


def test_front_end_sizes_past_int():
    """Extents and leading dimensions that the C entry's int does not hold are not cut to one that it does."""
    import torch
    from hyperkernels_amd import kernels as hk

    meta = lambda *s: torch.empty(*s, device="meta", dtype=torch.bfloat16)  # noqa: E731
    big = 2 ** 32 + 8
    for a, b, ta, tb in ((meta(big, 8), meta(8, 16), False, False), (meta(4, 8), meta(8, big), False, False),
                         (meta(4, big), meta(big, 8), False, False), (meta(8, big), meta(8, 16), True, False),
                         (meta(4, 8), meta(big, 8), False, True),
                         (meta(big, 1, 8), meta(big, 8, 16), False, False)):
        for f in (hk.bgemm_act, hk.bgemm_act_backward):
            with pytest.raises(ValueError, match="2\\^31"):
                f(a, b, trans_a=ta, trans_b=tb)
    for t in (meta(4, big)[:, :16], meta(2, 4, big)[:, :, :16]):
        with pytest.raises(ValueError, match="2\\^31"):
            hk._matrix("f", t, -1, 1 if t.dim() == 2 else 2, 4, 16)
    assert hk._matrix("f", meta(4, 2 ** 31 - 1)[:, :16], -1, 1, 4, 16)[1] == 2 ** 31 - 1
    assert hk._matrix("f", meta(1, big)[:, :16], -1, 1, 1, 16)[1] == 16  # one row: any leading dimension


@pytest.mark.parametrize("M,N,tb", [(2 ** 30 + 72, 8, 0), (8, 2 ** 30 + 72, 1)])
def test_plain_products_of_tiles_past_one_launch(L, M, N, tb):
    """Rows of 9 elements take the tiles for any alignment: 2^24 of them and two more, of 256 threads."""
    K = 9
    assert L.hk_bgemm_small_tile(0, tb, M, N, K, 1, 0) == 64
    assert L.hk_bgemm(0, tb, M, N, K, 0x3F80, 64, K, 0, 1 << 40, K if tb else N, 0, 0, 1 << 41, N, 0, 1,
                      NULL) == INVALID
