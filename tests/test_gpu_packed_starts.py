"""Packed attention whose queries' and keys' starts are one array over tensors of different lengths: starts past a tensor
count as its end, so the sequences have other numbers of queries than of keys. Values and tolerances as in
test_gpu_attn_packed.py."""
from __future__ import annotations

import math

import pytest
import torch
from test_gpu_attn_packed import BF, DEV, F16, check, make, reference, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,Hk,d,dt", [(4, 2, 64, BF), (2, 1, 128, F16), (8, 8, 128, BF)])
@pytest.mark.parametrize("starts,tq,tk", [
    ([0, 1000], 100, 1000), ([0, 500, 1000], 1000, 600), ([0, 300, 700, 1300, 1400], 900, 1400),
    ([10 * i for i in range(101)], 350, 1000), ([40 * i for i in range(71)], 2800, 1313),
    ([7 * i for i in range(69)] + [900, 1500], 700, 1500),
])
def test_one_array_of_starts_over_different_lengths(hk, starts, tq, tk, H, Hk, d, dt, causal):
    say(starts[:5], tq, tk, H, Hk, d, dt, causal)
    lens = lambda t: [min(b, t) - min(a, t) for a, b in zip(starts, starts[1:])]  # noqa: E731
    lq, lk = lens(tq), lens(tk)
    q, k, v, do = make(lq, lk, H, Hk, d, dt, seed=tq)
    cu = torch.tensor(starts, device=DEV, dtype=torch.int32)
    o, lse = hk.attn_packed_forward(q, k, v, cu, causal=causal)
    dk, dv = torch.full_like(k, math.nan), torch.full_like(k, math.nan)
    dq, dk, dv = hk.attn_packed_backward(do, q, k, v, o, lse, cu, causal=causal, dk=dk, dv=dv)
    torch.cuda.synchronize()
    got = {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    check(got, reference(q, k, v, lq, lk, causal, d ** -0.5, do))
    for n, t in zip(got, (*hk.attn_packed_forward(q, k, v, cu, cu.clone(), causal),
                          *hk.attn_packed_backward(do, q, k, v, o, lse, cu, cu.clone(), causal))):
        assert torch.equal(got[n], t), n
