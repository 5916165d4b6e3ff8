"""The gradients of rows that see few keys, in tiles of rows that see more: with a query or more fewer than keys the rows of
2 to 60 keys lie beside rows of more than 128. The norm's bound is that of test_gpu_attn_packed.py's test of it."""
from __future__ import annotations

import pytest
import torch
from test_gpu_attn_packed import BF, F16, check, cu_of, make, reference, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [BF, F16])
@pytest.mark.parametrize("lq,lk,H,Hk,d", [
    ([128] * 40, [129] * 40, 16, 16, 64), ([128] * 40, [140] * 40, 16, 16, 128), ([127] * 40, [129] * 40, 16, 16, 64),
    ([100] * 60, [131] * 60, 12, 6, 64), ([70] * 20, [133] * 20, 8, 4, 128), ([40] * 9, [129] * 9, 6, 2, 64),
])
def test_gradients_of_rows_of_few_keys(hk, lq, lk, H, Hk, d, t):
    # Where delta is formed from the o that was rounded (twice), over 65 keys and more, that adds at most 2 / 64 to the 2
    # under the root. A thirtieth for the chance in both.
    say(lq[0], lk[0], H, Hk, d, t)
    q, k, v, do = make(lq, lk, H, Hk, d, t)
    cq, ck = cu_of(lq), cu_of(lk)
    o, lse = hk.attn_packed_forward(q, k, v, cq, ck)
    dq, dk, dv = hk.attn_packed_backward(do, q, k, v, o, lse, cq, ck)
    ref = reference(q, k, v, lq, lk, True, d ** -0.5, do)
    check({"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}, ref)
    for name, got in (("dq", dq), ("dk", dk)):
        want = ref[name][0]
        least = float((want.to(t).double() - want).norm())
        off = float((got.double() - want).norm())
        print("   ", name, off / least, flush=True)
        assert off <= (2 + 1 / 32) ** 0.5 * (1 + 1 / 30) * least, (name, off / least)
