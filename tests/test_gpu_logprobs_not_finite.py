"""Token log probabilities of rows with NaN, +inf or nothing above -inf in every type: NaN, with their alternatives'
indices as of any row, and no effect on the rows beside them."""
from __future__ import annotations

import math

import pytest
import torch
from test_gpu_token_logprobs import BF, DEV, F16, F32, check, make, order, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [F32, BF, F16])
@pytest.mark.parametrize("rows,vocab", [(8, 9), (8, 500), (600, 1500), (8, 30000), (300, 50257), (600, 3000)])
def test_rows_without_a_softmax(hk, rows, vocab, dt):
    say(rows, vocab, dt)
    x, t = make(rows, vocab, dt, seed=vocab)
    ends = [0, vocab // 3, vocab - 1]
    x[0, ends[0]] = x[1, ends[2]] = math.nan
    x[2, ends[1]] = x[3, ends[0]] = math.inf
    x[4] = -math.inf
    x[5, ends] = torch.tensor([math.nan, math.inf, -math.inf], device=DEV, dtype=dt)
    top = min(5, vocab)
    for n in (0, top):
        p = hk.token_logprobs(x, t, entropy=True, top=n)
        one = torch.ones(rows, device=DEV)
        dx = hk.token_logprobs_backward(x, t, p.lse, one, p.entropy, one)
        for v in (p.logp, p.entropy, dx):
            assert torch.isnan(v[:6]).all() and torch.isfinite(v[6:]).all()
    assert torch.isnan(p.top_logp[:6]).all()
    for r in (0, 1, 2, 3, 5):
        assert torch.equal(p.top_index[r], order(x[r:r + 1])[0, :top]), r
    assert p.top_index[4].tolist() == list(range(top))
    check(hk, x[6:], t[6:], top)


@pytest.mark.parametrize("dt", [F32, BF, F16])
def test_two_calls_at_once(hk, dt):
    cases = [make(16, 50257, dt, seed=1), make(3, 100003, dt, seed=2)]
    run = lambda x, t: hk.token_logprobs(x, t, entropy=True, top=20)  # noqa: E731
    want = [run(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(run(*c))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        for a, b in zip(g, want[i % 2]):
            assert torch.equal(a, b), i
