"""The gradient of token log probabilities for rows whose log-sum-exp is so far from 0 that one fp32 number has no room for
the logarithm of the sum beside the maximum: against the definition in 64 bits, with the maximum taken off first.

Tolerances as in test_gpu_token_logprobs.py, but of x - m and log s in the place of x and lse: p is off by
tl = 2^-16 + 2^-21 (A + log s + |x - m| + 4) of itself, with A = sum p |x - m|. Where p goes by lse (|lse| under 128 in fp32, 1024 in
fp16, 4096 in bf16) that adds half a step of lse: 2^-18 in fp32, 2^-15 for the 16-bit cases at 1000 here; 2^-16, the
other terms (2^-16 again for a log s over 9) and 1 % of the result's rounding have room for both."""
from __future__ import annotations

import math

import pytest
import torch
from test_gpu_token_logprobs import BF, DEV, F16, F32, make, say

pytestmark = pytest.mark.gpu


def check(hk, x, t, grad=None, entropy=True):
    rows, vocab = x.shape
    g, h = torch.randn(rows, device=DEV), torch.randn(rows, device=DEV) * entropy
    z = x.double() - x.double().amax(1, keepdim=True)
    log_s = z.exp().sum(1, keepdim=True).log()
    lp = z - log_s
    prob = lp.exp()
    info = torch.where(prob > 0, lp, 0.0)
    ent = -(prob * info).sum(1, keepdim=True)
    gd, hd = g.double()[:, None], h.double()[:, None]
    hot = torch.zeros_like(z)
    ok = (t >= 0) & (t < vocab)
    hot[ok.nonzero()[:, 0], t[ok].long()] = 1
    want = gd * (hot - prob) - hd * prob * (info + ent)
    zz = torch.where(prob > 0, z, 0.0).abs()
    A = (prob * zz).sum(1, keepdim=True)
    rel = 2.0 ** -16 + 2.0 ** -21 * (A + log_s + zz + 4)
    te = (1 + A) * (2.0 ** -16 + 2.0 ** -21 * (A + log_s))
    tol = prob * (gd.abs() + hd.abs() * (info + ent).abs()) * rel + prob * hd.abs() * (rel + te)
    tol = tol + gd.abs() * hot * 2.0 ** -22 + torch.finfo(x.dtype).eps / 2 * 1.01 * want.abs()
    tol = tol + 2.0 ** -126 * (1 + gd.abs() + hd.abs() * (info + ent).abs()) + (2.0 ** -25 if x.dtype is F16 else 0.0)
    p = hk.token_logprobs(x, t, entropy=True)
    got = hk.token_logprobs_backward(x, t, p.lse, g, p.entropy if entropy else None, h if entropy else None, grad=grad)
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("dt", [F32, BF, F16])
@pytest.mark.parametrize("rows,vocab", [(5, 20000), (600, 700), (300, 50257), (2, 3), (4, 1)])
@pytest.mark.parametrize("allowed", [0, 1, 7, 40])
def test_words_masked_by_the_lowest_value(hk, rows, vocab, allowed, dt):
    say(rows, vocab, allowed, dt)
    x, t = make(rows, vocab, dt)
    g = torch.Generator(device=DEV).manual_seed(2)
    keep = torch.randperm(vocab, generator=g, device=DEV)[:allowed]
    y = torch.full_like(x, torch.finfo(dt).min)
    y[:, keep] = x[:, keep]
    check(hk, y, t)
    check(hk, y, t, entropy=False)


@pytest.mark.parametrize("rows,vocab,stride", [(6, 50257, 50304), (700, 1000, 1000), (9, 4099, 4099)])
@pytest.mark.parametrize("at", [100.0, 127.9, 128.0, -1000.0, 1e5, -3e7])
def test_far_logits(hk, rows, vocab, stride, at):
    say(rows, vocab, at)
    x, t = make(rows, vocab, F32, stride)
    x += at
    x[::3] -= at  # and near ones between them
    t[1] = vocab
    check(hk, x, t)
    off = torch.empty(rows * (stride + 2) + 1, device=DEV)[1:].as_strided((rows, vocab), (stride + 2, 1))
    check(hk, x, t, grad=off)
    x.masked_fill_(torch.rand_like(x) < 0.5, -math.inf)
    x[:, vocab // 2] = at
    check(hk, x, t)
    check(hk, x, t, grad=x)


@pytest.mark.parametrize("dt,at", [(BF, 1000.0), (F16, 1000.0), (F16, 5000.0), (BF, -1e4), (BF, -1e9), (BF, 1e30)])
@pytest.mark.parametrize("rows,vocab", [(6, 20001), (700, 1000)])
def test_far_logits_in_16_bits(hk, rows, vocab, dt, at):
    # steps of 4 (bf16) and 0.5 (fp16) at 1000, or all words equal: the definition takes them as they are
    say(rows, vocab, dt, at)
    x, t = make(rows, vocab, F32)
    check(hk, (x + at).to(dt), t)


def test_far_rows_captured(hk):
    x, t = make(40, 9001, F32)
    x[::2] += 5000
    g = torch.randn(40, device=DEV)

    def run():
        p = hk.token_logprobs(x, t, entropy=True)
        return hk.token_logprobs_backward(x, t, p.lse, g, p.entropy, g)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(3):
        x.copy_(torch.randn_like(x) * 3)
        x[i::2] -= 700 * i
        want = run()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
