"""GPU parity of the embedding lookup and of its table's gradient against their definitions in 64 bits. The lookup rounds
scale * row (fp32), its sum with the residual (fp32), and the result; a gradient's sum of k fp32 terms has k additions,
then the scale, what it is added to, and the rounding of the result."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16


def say(*a):
    print("[case]", *a, flush=True)


def tokens(n, vocab, kind, seed=0, wide=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    if kind == "words":
        t = ((vocab + 1.0) ** u - 1).long().clamp_(0, vocab - 1)
    elif kind == "even":
        t = (u * vocab).long()
    elif kind == "one":
        t = torch.full((n,), vocab - 1, device=DEV)
    elif kind == "runs":  # rows that begin and end at the places where the work is cut
        t = (torch.arange(n, device=DEV) // 32 * 7) % vocab
    else:  # "outside": some of no row
        t = (u * 1.5 * vocab).long() - vocab // 4
    return t if wide else t.int()


def half(dt):
    return torch.finfo(dt).eps / 2 * 1.01


@pytest.mark.parametrize("tt,ot", [(F32, BF), (BF, BF), (BF, F32), (F16, F16), (F32, F32), (F16, BF)])
@pytest.mark.parametrize("n,vocab,d,pad", [(1, 1, 1, 0), (5, 9, 7, 3), (300, 1000, 768, 0), (33, 50, 131, 1),
                                           (1000, 77, 68, 4), (4097, 300, 96, 8), (2, 3, 5000, 0)])
def test_lookup(hk, n, vocab, d, pad, tt, ot):
    say(n, vocab, d, pad, tt, ot)
    table = torch.randn(vocab, d + pad, device=DEV).to(tt)[:, pad // 2:pad // 2 + d]
    res = torch.randn(n, d + 2 * pad, device=DEV).to(ot)[:, :d]
    t = tokens(n, vocab, "outside", wide=n % 2 == 0)
    ok = (t >= 0) & (t < vocab)
    want = table.double()[t.long().clamp(0, vocab - 1)] * 2.5
    y = hk.embedding_forward(table, t, scale=2.5, out_dtype=ot)
    z = hk.embedding_forward(table, t, scale=2.5, residual=res, out=torch.empty(n, d + pad, device=DEV, dtype=ot)[:, :d])
    tiny = 2.0 ** -25 if ot is F16 else 0.0
    for got, w, extra in ((y, want, 0.0), (z, want + res.double(), want.abs() * 2.0 ** -24)):
        assert torch.isnan(got[~ok]).all()
        tol = extra + (2.0 ** -23 + half(ot)) * w.abs() + tiny
        assert bool(((got.double() - w).abs() <= tol)[ok].all())
    assert torch.equal(hk.embedding_forward(table, t, scale=2.5, residual=res, out=res)[ok], z[ok])


@pytest.mark.parametrize("gt,tt", [(BF, F32), (F32, F32), (F16, F16), (BF, BF), (F32, BF)])
@pytest.mark.parametrize("kind", ["words", "even", "one", "runs", "outside"])
@pytest.mark.parametrize("n,vocab,d,pad", [(0, 10, 8, 0), (1, 3, 1, 0), (7, 1009, 131, 0), (512, 300, 64, 0),
                                           (513, 300, 64, 1), (2048, 50, 36, 2), (5000, 5003, 200, 0),
                                           (9000, 1, 16, 0), (20000, 70001, 24, 0), (1024, 700, 52, 0),
                                           (1025, 701, 52, 0), (2048, 3, 300, 0), (2048, 9001, 131, 1), (2048, 40000, 36, 0),
                                           (1500, 2049, 1100, 0), (2049, 2048, 64, 0), (6000, 65, 7, 1)])
def test_gradient(hk, n, vocab, d, pad, kind, gt, tt):
    say(n, vocab, d, pad, kind, gt, tt)
    grad = torch.randn(n, d + pad, device=DEV).to(gt)[:, :d]
    t = tokens(n, vocab, kind, wide=(n + d) % 2 == 0)
    ok = (t >= 0) & (t < vocab)
    at, rows = t.long()[ok], grad.double()[ok]
    want = torch.zeros(vocab, d, device=DEV, dtype=torch.float64).index_add_(0, at, rows) * 0.5
    size = torch.zeros(vocab, d, device=DEV, dtype=torch.float64).index_add_(0, at, rows.abs()) * 0.5
    count = torch.bincount(at, minlength=vocab)[:, None]
    tiny = 2.0 ** -25 if tt is F16 else 0.0
    whole = torch.randn(vocab, d + pad, device=DEV).to(tt)
    base = whole[:, :d]
    before = whole.clone()
    tol = size * count * 2.0 ** -24
    hk.embedding_backward(grad, t, base, scale=0.5)
    w = before[:, :d].double() + want
    assert bool(((base.double() - w).abs() <= tol + 2.0 ** -24 * want.abs() + half(tt) * w.abs() + tiny).all())
    none = (count == 0)[:, 0]
    assert torch.equal(base[none], before[none, :d])
    if pad:
        assert torch.equal(whole[:, d:], before[:, d:])
    out = torch.full((vocab, d), math.nan, device=DEV, dtype=tt)
    hk.embedding_backward(grad, t, out, scale=0.5, accumulate=False)
    assert bool(((out.double() - want).abs() <= tol + half(tt) * want.abs() + tiny).all())
    again = torch.full((vocab, d), math.nan, device=DEV, dtype=tt)
    hk.embedding_backward(grad, t, again, scale=0.5, accumulate=False)
    assert torch.equal(out, again)  # the same bits


def test_gradient_of_many_tokens(hk):
    # chunks of 64 and 128 positions, ranges of 256 and 512 table rows, one word on a tenth of all places
    for n, vocab, d in ((70000, 200003, 8), (300001, 400000, 4)):
        say(n, vocab, d)
        t = tokens(n, vocab, "words")
        t[::10] = 12345
        grad = torch.randint(-4, 5, (n, d), device=DEV).float()  # sums that fp32 holds exactly
        out = torch.full((vocab, d), math.nan, device=DEV)
        hk.embedding_backward(grad, t, out, accumulate=False)
        want = torch.zeros(vocab, d, device=DEV, dtype=torch.float64).index_add_(0, t, grad.double())
        assert torch.equal(out.double(), want)


def test_gradient_of_one_row_for_all(hk):
    # a gradient that was broadcast: one row for all tokens
    for n in (300, 3000):
        t = tokens(n, 40, "words")
        row = torch.randint(-3, 4, (1, 24), device=DEV).float()
        out = hk.embedding_backward(row.expand(n, 24), t, torch.full((40, 24), 5.0, device=DEV), accumulate=False)
        assert torch.equal(out, torch.bincount(t, minlength=40)[:, None] * row)


def test_gradient_is_the_lookup_s(hk):
    # <lookup(table), g> = <table, gradient(g)>
    for n in (200, 3000):
        t = tokens(n, 500, "words")
        table, g = torch.randn(500, 40, device=DEV), torch.randn(n, 40, device=DEV)
        y = hk.embedding_forward(table, t, scale=3.0)
        d = hk.embedding_backward(g, t, torch.zeros_like(table), scale=3.0)
        a, b = float((y.double() * g.double()).sum()), float((table.double() * d.double()).sum())
        # both sums are of products that are off by (count + 2) 2^-24
        size = float((y.double() * g.double()).abs().sum())
        assert abs(a - b) <= size * (n + 2) * 2.0 ** -24


def test_captured_and_other_stream(hk):
    t = tokens(3000, 5000, "words")
    few = tokens(100, 5000, "words")
    g = torch.randn(3000, 64, device=DEV)
    table = torch.randn(5000, 64, device=DEV)

    def run():
        a = hk.embedding_backward(g, t, torch.empty_like(table), accumulate=False)
        return a, hk.embedding_backward(g[:100], few, torch.empty_like(table), accumulate=False), hk.embedding_forward(
            table, t)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    side = torch.cuda.Stream()
    for _ in range(3):
        g.copy_(torch.randn_like(g))
        t.copy_(t[torch.randperm(3000, device=DEV)])
        want = run()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = run()
        graph.replay()
        torch.cuda.synchronize()
        for x, y, z in zip(want, out, again):
            assert torch.equal(x, y) and torch.equal(x, z)
