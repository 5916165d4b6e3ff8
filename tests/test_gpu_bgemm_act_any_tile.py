"""The GEMM with an epilogue on the 256 x 256 tiles for rows of any alignment, which large products with odd rows take,
against the formulas in 64 bits. Tolerances are test_gpu_bgemm_act.py's."""
from __future__ import annotations

import pytest
import torch
from test_gpu_bgemm_act import LAYOUTS, Data

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ta,tb", LAYOUTS)
@pytest.mark.parametrize("M,N,K,pad,off", [(3001, 3003, 577, 0, 0), (8191, 5119, 129, 0, 1), (3001, 3008, 640, 3, 0)])
def test_every_layout(hk, M, N, K, pad, off, ta, tb):
    lib = hk.lib()
    if N % 2:  # the planning queries take packed rows: here those are the call's own
        assert lib.hk_bgemm_small_tile(ta, tb, M, N, K, 1, 0) == 256
        assert lib.hk_bgemm_split_count(ta, tb, M, N, K, 1, 0) == 1
    print("act 256", M, N, K, ta, tb, pad, off, flush=True)
    d = Data(M, N, K, ta, tb, 800 + K, pad=pad, off=off)
    first = d.check_forward(hk, "gelu")
    assert torch.equal(first, d.check_forward(hk, "gelu"))
    d.check_forward(hk, "silu", inplace=True, preact=False, alpha=-0.5)
    d.check_forward(hk, "none", bias=False, residual=False, preact=False)
    one = d.check_backward(hk, "gelu")
    two = d.check_backward(hk, "gelu")
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    d.check_backward(hk, "relu", accumulate=False, alpha=2.0)
    d.untouched()
