"""Packed attention in fp16 at the ends of its range. Values and tolerances as in test_gpu_attn_packed.py."""
from __future__ import annotations

import pytest
import torch
from test_gpu_attn_packed import DEV, F16, check, cu_of, make, reference, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,Hk,d,lens", [(4, 2, 64, [300, 41]), (2, 2, 128, [129, 2, 700]), (8, 8, 64, [4097]),
                                         (16, 4, 128, [2048, 1001, 333]), (3, 1, 8, [50])])
def test_large_values_and_small_gradients(hk, H, Hk, d, lens):
    # dout of 2^-10 along values of up to 2^13 of the same signs: dS is some hundreds, but past fp16 for a dout of 1
    say(H, Hk, d, lens)
    q, k, v, do = make(lens, lens, H, Hk, d, F16)
    g = torch.Generator(device=DEV).manual_seed(1)
    sign = lambda *s: torch.randint(0, 2, s, generator=g, device=DEV) * 2.0 - 1  # noqa: E731
    u = sign(1, 1, d)
    large = torch.rand(v.shape[0], Hk, 1, generator=g, device=DEV) < 0.7  # and others of 1
    v = torch.where(large, 2.0 ** 13 * sign(v.shape[0], Hk, 1) * u, v.float()).to(F16)
    do = (2.0 ** -10 * sign(do.shape[0], H, 1) * u * (0.5 + 0.5 * torch.rand(do.shape, generator=g, device=DEV))).to(F16)
    do[5::7] = 0
    cq = cu_of(lens)
    o, lse = hk.attn_packed_forward(q, k, v, cq)
    dq, dk, dv = hk.attn_packed_backward(do, q, k, v, o, lse, cq)
    # dS is held for a dout of at most 2^14: half a step of fp16's smallest numbers times that, and the power of two
    # above the largest dout
    want = reference(q, k, v, lens, lens, True, d ** -0.5, do, 2.0 ** -25 * 2.0 ** 14 * 2 * float(do.abs().max()))
    assert all(torch.isfinite(t[0].to(F16)).all() for n, t in want.items() if n != "lse")
    check({"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}, want)


def test_values_at_the_end_of_fp16(hk):
    # the largest dS that finite inputs of few keys can have: the gradients' own range is the limit
    lens, d = [2, 3], 128
    q, k, v, do = make(lens, lens, 2, 2, d, F16, std=2.0 ** -6)
    v = torch.full_like(v, 65504.0)
    v[1::2] = -65504.0
    do = torch.full_like(do, 2.0 ** -8)
    do[:, :, ::2] *= -0.5
    cq = cu_of(lens)
    o, lse = hk.attn_packed_forward(q, k, v, cq)
    got = dict(zip(("dq", "dk", "dv"), hk.attn_packed_backward(do, q, k, v, o, lse, cq)))
    want = reference(q, k, v, lens, lens, True, d ** -0.5, do, 2.0 ** -25 * 2.0 ** 14 * 2 * 2.0 ** -8)
    del want["o"], want["lse"]
    assert all(torch.isfinite(t[0].to(F16)).all() for t in want.values())
    check(got, want)


@pytest.mark.parametrize("n,d,causal", [(208412, 64, False), (120000, 128, True)])
def test_flat_rows_over_many_keys(hk, n, d, causal):
    # Equal scores: p = 1 / n, which fp16's own steps of 2^-24 are off by one in 160. dv = p sum of dout, with P's rounding
    # and the result's, 2^-11 each. In fp32: the sum of n terms (n / 4096 additions one after the other: blocks of 64 keys, 16
    # of them a lane, in four sums), and the log-sum-exp (under 16), the exponential and 32 products, 2^-18 together.
    say(n, d, causal)
    m = 32
    q, k, v, do = make([m], [n], 1, 1, d, F16)
    q.zero_()
    do = (do * 1024).abs()
    cq, ck = cu_of([m]), cu_of([n])
    o, lse = hk.attn_packed_forward(q, k, v, cq, ck, causal)
    _, _, dv = hk.attn_packed_backward(do, q, k, v, o, lse, cq, ck, causal)
    i = torch.arange(m, device=DEV, dtype=torch.float64)
    p = 1 / (i + n - m + 1) if causal else torch.full_like(i, 1 / n)
    x = do.double()[:, 0] * p[:, None]
    want = x.sum(0).expand(n, d).clone()
    if causal:  # the last keys are seen by the last queries alone
        want[n - m:] = x.flip(0).cumsum(0).flip(0)
    off = (dv.double()[:, 0] - want).abs()
    tol = (2 * 2.0 ** -11 * 1.01 + n / 4096 * 2.0 ** -24 + 2.0 ** -18) * want + 2.0 ** -25
    assert bool((off <= tol).all()), float((off / want).max())


@pytest.mark.parametrize("H,Hk,d", [(4, 2, 64), (4, 4, 128)])
def test_not_finite_stays_in_its_sequence(hk, H, Hk, d):
    lens = [65, 130, 40]
    for bad in (float("nan"), float("inf")):
        for where in range(4):
            x = make(lens, lens, H, Hk, d, F16)
            want = reference(*x[:3], lens, lens, True, d ** -0.5, x[3])
            x[where][100, 1, 3] = bad
            q, k, v, do = x
            cq = cu_of(lens)
            o, lse = hk.attn_packed_forward(q, k, v, cq)
            got = dict(zip(("o", "lse", "dq", "dk", "dv"),
                           (o, lse.t(), *hk.attn_packed_backward(do, q, k, v, o, lse, cq))))
            want["lse"] = [t.t() for t in want["lse"]]
            for s in (slice(0, 65), slice(195, 235)):
                check({n: t[s] for n, t in got.items()}, {n: [t[s] for t in w] for n, w in want.items()})
            # the gradient of the query that it is in, or that sees the key (through its score, its dP or its delta)
            reader = 1 if where in (0, 3) else H // Hk  # the first query head of key head 1
            assert not torch.isfinite(got["dq"][100, reader]).all()
