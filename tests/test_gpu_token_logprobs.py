"""GPU parity of token log probabilities, entropy, alternatives and the logits' gradient against their definitions in 64
bits, element by element.

Tolerances: a sum of positive fp32 terms has at most 128 additions a lane and 9 levels behind them, 2^-17 relative in
all; a term's exponent is off by 2^-23 (|m| + |t|) and its exponential by 2^-22. With A = sum p |x - m| that is
tl = 2^-16 + 2^-21 (|lse| + |m| + A) for lse and logp, te = (1 + A) tl for the entropy. The gradient carries p's relative
error, tl + 2^-21 (|x| + |lse|), and te, and is rounded once."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16


def say(*a):
    print("[case]", *a, flush=True)


def make(rows, vocab, dt, stride=None, offset=0, seed=0, std=2.5, masked=0.0, wide=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    stride = vocab if stride is None else stride
    whole = (torch.randn(rows * stride + offset, generator=g, device=DEV) * std).to(dt)
    x = whole[offset:].as_strided((rows, vocab), (stride, 1))
    if masked:
        off = torch.rand(rows, vocab, generator=g, device=DEV) < masked
        off[:, vocab // 2] = False
        x.masked_fill_(off, -math.inf)
    t = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    return x, t if wide else t.int()


def order(x):
    """Indices by falling value, of equal ones the lowest first, NaN last."""
    y = x.double()
    y = torch.where(torch.isnan(y), -math.inf, y)  # of no test beside a real -inf
    return torch.sort(y, dim=1, descending=True, stable=True).indices


def check(hk, x, t, top, entropy=True, grads=True):
    rows, vocab = x.shape
    p = hk.token_logprobs(x, t, entropy=entropy, top=top)
    xd, td = x.double(), t.long()
    m = xd.amax(1)
    lse = torch.logsumexp(xd, 1)
    lp = xd - lse[:, None]
    prob = lp.exp()
    info = torch.where(prob > 0, lp, 0.0)
    ent = -(prob * info).sum(1)
    A = torch.where(prob > 0, prob * (xd - m[:, None]).abs(), 0.0).sum(1)
    tl = 2.0 ** -16 + 2.0 ** -21 * (lse.abs() + m.abs() + A)
    te = (1 + A) * tl

    def near(name, got, want, tol):
        got = got.double()
        fine = torch.isfinite(want)
        assert torch.equal(got[~fine], want[~fine]), name
        off = (got - want).abs()[fine]
        assert bool((off <= tol.expand(want.shape)[fine]).all()), (name, float((off / tol.expand(want.shape)[fine]).max()))

    near("lse", p.lse, lse, tl)
    near("logp", p.logp, lp.gather(1, td[:, None])[:, 0], 2 * tl)
    if entropy:
        near("entropy", p.entropy, ent, te)
    if top:
        best = order(x)[:, :top]
        assert torch.equal(p.top_index, best)
        near("top", p.top_logp, lp.gather(1, best), 2 * tl[:, None])
    if not grads:
        return p
    g, h = torch.randn(rows, device=DEV), torch.randn(rows, device=DEV)
    dx = hk.token_logprobs_backward(x, t, p.lse, g, p.entropy, h if entropy else None)
    gd, hd = g.double()[:, None], h.double()[:, None] * entropy
    hot = torch.zeros_like(xd).scatter_(1, td[:, None], 1.0)
    want = gd * (hot - prob) - hd * prob * (info + ent[:, None])
    size = torch.where(prob > 0, xd.abs(), 0.0) + lse.abs()[:, None]
    rel = tl[:, None] + 2.0 ** -21 * (size + 4)
    tol = prob * (gd.abs() + hd.abs() * (info + ent[:, None]).abs()) * rel + prob * hd.abs() * (tl + te)[:, None]
    tol = tol + gd.abs() * hot * 2.0 ** -22 + torch.finfo(x.dtype).eps / 2 * 1.01 * want.abs()
    # a p under 2^-126 is 0 to the hardware's exp2, off by all of itself, and so is a product with it
    tol = tol + 2.0 ** -126 * (1 + gd.abs() + hd.abs() * (info + ent[:, None]).abs())
    tol = tol + (2.0 ** -25 if x.dtype is F16 else 0.0)
    near("dx", dx, want, tol)
    return p


@pytest.mark.parametrize("dt", [F32, BF, F16])
@pytest.mark.parametrize("rows,vocab,stride,offset,top", [
    (1, 1, 1, 0, 1), (3, 5, 7, 1, 5), (2, 64, 64, 0, 64), (5, 257, 257, 3, 20), (700, 300, 304, 0, 3),
    (600, 1023, 1023, 1, 64), (600, 1025, 1032, 0, 7), (33, 2049, 2049, 0, 20), (3, 8191, 8192, 5, 1),
    (16, 50257, 50257, 0, 20), (300, 50257, 50304, 0, 5), (1, 131072, 131072, 0, 64), (2, 100003, 100003, 1, 33),
    (260, 33001, 33001, 0, 20), (1, 70000, 70000, 0, 0),
])
def test_sizes(hk, rows, vocab, stride, offset, top, dt):
    say(rows, vocab, stride, offset, top, dt)
    x, t = make(rows, vocab, dt, stride, offset, seed=rows + vocab, wide=rows % 2 == 0)
    check(hk, x, t, top)


@pytest.mark.parametrize("std", [1e-3, 30.0])
@pytest.mark.parametrize("rows,vocab", [(4, 50257), (400, 1000)])
def test_ranges(hk, std, rows, vocab):
    x, t = make(rows, vocab, F32, std=std)
    check(hk, x, t, 20)
    check(hk, x + 1000, t, 20)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("rows,vocab", [(3, 700), (600, 1000), (5, 40000), (270, 9000)])
def test_masked(hk, rows, vocab, dt):
    say(rows, vocab, dt)
    for part in (0.3, 0.999):
        x, t = make(rows, vocab, dt, masked=part)
        check(hk, x, t, 20)
    x[:] = -math.inf  # three words allowed, fewer than are asked for
    x[:, [1, vocab // 2, vocab - 1]] = torch.tensor([0.5, -1.0, 0.5], device=DEV, dtype=dt)
    check(hk, x, torch.full((rows,), vocab - 1, device=DEV), 20)


@pytest.mark.parametrize("rows,vocab", [(3, 700), (600, 900), (5, 40000), (270, 9000)])
def test_equal_values(hk, rows, vocab):
    x, t = make(rows, vocab, BF)
    check(hk, x.mul(4).round().div(4), t, 64)  # many of each
    x[:] = 3.0
    check(hk, x, t, 64)
    x[:] = 0.0
    x[:, ::2] = -0.0
    check(hk, x, t, 20)
    x.copy_(torch.arange(vocab, device=DEV).to(BF))  # the largest all in one place, in runs
    check(hk, x, t, 20, grads=False)
    x[:, :vocab - 600] = x[:, 600:].clone()
    check(hk, x, t, 20, grads=False)


@pytest.mark.parametrize("rows,vocab,top", [(3000, 20000, 64), (2000, 1500, 64), (400, 50257, 50), (30, 200000, 64)])
def test_many_rows_and_alternatives(hk, rows, vocab, top):
    # in some of so many rows the first bound lets many more pass than are asked for
    say(rows, vocab, top)
    x, t = make(rows, vocab, F16 if vocab == 1500 else BF, seed=top)
    check(hk, x, t, top, grads=False)


@pytest.mark.parametrize("rows,vocab", [(5, 60000), (600, 1500), (300, 30000)])
@pytest.mark.parametrize("allowed", [0, 1, 3, 19, 20, 200])
def test_few_words_allowed(hk, rows, vocab, allowed):
    say(rows, vocab, allowed)
    x, t = make(rows, vocab, BF)
    g = torch.Generator(device=DEV).manual_seed(1)
    keep = torch.randperm(vocab, generator=g, device=DEV)[:allowed]
    y = torch.full_like(x, -math.inf)
    y[:, keep] = x[:, keep]
    if allowed == 0:
        p = hk.token_logprobs(y, t, top=20)
        assert torch.equal(p.top_index, torch.arange(20, device=DEV).expand(rows, 20))
        return
    t = keep[torch.arange(rows, device=DEV) % allowed]
    check(hk, y, t, 20)


@pytest.mark.parametrize("dt", [BF, F16, F32])
@pytest.mark.parametrize("rows,vocab", [(5, 20000), (600, 700), (300, 50257), (300, 9000)])
@pytest.mark.parametrize("allowed", [0, 1, 7, 19, 20, 21, 40])
def test_words_masked_by_the_lowest_value(hk, rows, vocab, allowed, dt):
    # all but a few words at the type's lowest value: equal ones rank by their index, behind the few
    say(rows, vocab, allowed, dt)
    x, t = make(rows, vocab, dt)
    g = torch.Generator(device=DEV).manual_seed(2)
    keep = torch.randperm(vocab, generator=g, device=DEV)[:allowed]
    y = torch.full_like(x, torch.finfo(dt).min)
    y[:, keep] = x[:, keep]
    p = hk.token_logprobs(y, t, entropy=True, top=20)
    q = hk.token_logprobs(y, t, entropy=True)
    few, order = torch.sort(y[:, keep].float(), dim=1, descending=True, stable=True)
    rest = torch.ones(vocab, device=DEV, dtype=torch.bool)
    rest[keep] = False
    first = rest.nonzero()[:20, 0]
    for i in range(min(allowed, 20)):
        assert torch.equal(y.gather(1, p.top_index[:, i:i + 1])[:, 0].float(), few[:, i])
    if allowed < 20:
        assert torch.equal(p.top_index[:, allowed:], first[:20 - allowed].expand(rows, -1))
    # less the maximum first: beside the lowest value lse has no room for log s
    z = y.double() - y.double().amax(1, keepdim=True)
    log_s = z.exp().sum(1, keepdim=True).log()
    lp = z - log_s
    prob = lp.exp()
    ent = -(prob * torch.where(prob > 0, lp, 0.0)).sum(1)
    tol = lambda want: 2.0 ** -16 + 2.0 ** -21 * (want.abs() + log_s.abs().max() + 8)  # noqa: E731  logits under 16
    for got, want in ((p.top_logp, lp.gather(1, p.top_index)), (p.logp, lp.gather(1, t[:, None])[:, 0]),
                      (q.logp, lp.gather(1, t[:, None])[:, 0])):
        assert bool(((got.double() - want).abs() <= tol(want)).logical_or(got.double() == want.float().double()).all())
    for r in (p, q):
        assert bool(((r.entropy.double() - ent).abs() <= 2 * tol(ent)).all())
        dx = hk.token_logprobs_backward(y, t, r.lse, torch.ones(rows, device=DEV), r.entropy, torch.ones(rows, device=DEV))
        assert torch.isfinite(dx).all()


def test_entropy_left_out(hk):
    x, t = make(5, 3001, BF)
    p = check(hk, x, t, 3, entropy=False)
    assert p.entropy is None
    x, t = make(300, 1000, F16)
    p = check(hk, x, t, 0, entropy=False)
    assert p.top_logp is None and p.top_index is None


@pytest.mark.parametrize("rows,vocab", [(6, 500), (6, 30000), (300, 1000)])
def test_rows_without_a_softmax(hk, rows, vocab):
    x, t = make(rows, vocab, F32)
    x[0, 7], x[1, 9], x[2] = math.nan, math.inf, -math.inf
    t[3], t[4] = vocab, -1
    keep = x.clone()
    p = hk.token_logprobs(x, t, entropy=True, top=4)
    dx = hk.token_logprobs_backward(x, t, p.lse, torch.ones(rows, device=DEV), p.entropy, torch.ones(rows, device=DEV))
    assert torch.isnan(p.logp[:5]).all() and torch.isnan(p.entropy[:3]).all() and torch.isnan(p.top_logp[:3]).all()
    assert torch.isnan(dx[:3]).all() and torch.isfinite(dx[3:]).all()
    assert torch.equal(p.top_index[0], order(keep)[0, :4])  # NaN under everything
    assert int(p.top_index[1, 0]) == 9
    assert p.top_index[2].tolist() == [0, 1, 2, 3]
    prob = (x[3:5].double() - torch.logsumexp(x[3:5].double(), 1, keepdim=True)).exp()
    ent = p.entropy[3:5].double()[:, None]
    want = -prob - prob * (prob.log() + ent)  # without a one-hot
    assert float((dx[3:5].double() - want).abs().max()) <= 2.0 ** -16 * float(prob.max()) * (1 + float(ent.max()))
    check(hk, x[5:], t[5:], 4)


@pytest.mark.parametrize("dt", [F32, BF])
def test_gradient_in_place_and_unaligned(hk, dt):
    for rows, vocab, stride, off in ((7, 3001, 3001, 0), (3, 999, 1003, 1)):
        x, t = make(rows, vocab, dt, stride, 0)
        p = hk.token_logprobs(x, t)
        g = torch.randn(rows, device=DEV)
        want = hk.token_logprobs_backward(x, t, p.lse, g)
        other = torch.full((rows * (stride + 2) + 8,), 5.0, device=DEV, dtype=dt)
        view = other[off:].as_strided((rows, vocab), (stride + 2, 1))
        hk.token_logprobs_backward(x, t, p.lse, g, grad=view)
        assert torch.equal(view, want)
        assert bool((other[off + vocab:off + stride + 2] == 5).all())  # a row's padding
        assert hk.token_logprobs_backward(x, t, p.lse, g, grad=x) is x
        assert torch.equal(x, want)


def test_gradient_against_differences(hk):
    # logp and the entropy along a direction; fp32, central differences in 64 bits on the kernel's outputs
    x, t = make(6, 2000, F32, std=1.5)
    g, h = torch.randn(6, device=DEV), torch.randn(6, device=DEV)
    p = hk.token_logprobs(x, t, entropy=True)
    dx = hk.token_logprobs_backward(x, t, p.lse, g, p.entropy, h).double()
    u = torch.randn_like(x)
    step = 2.0 ** -4
    ends = [hk.token_logprobs(x + s * u, t, entropy=True) for s in (step, -step)]
    change = sum(s * (e.logp.double() * g.double() + e.entropy.double() * h.double())
                 for s, e in zip((1, -1), ends)) / (2 * step)
    along = (dx * u.double()).sum(1)
    # both ends are off by tl and te (A is 3 to 5 here) over 2 step, and the third derivative of both is of order
    # E|u|^3 (1 + H), 1.6 * 10, times step^2 / 6
    tol = (2 * 2.0 ** -15 * (g.abs() + 6 * h.abs()) / (2 * step) + step ** 2 / 6 * 16 * (g.abs() + h.abs())).double()
    assert bool(((along - change).abs() <= tol).all()), (along, change, tol)


def test_no_rows(hk):
    x, t = torch.empty(0, 50, device=DEV), torch.empty(0, device=DEV, dtype=torch.int32)
    p = hk.token_logprobs(x, t, entropy=True, top=2)
    assert p.logp.shape == (0,) and p.top_index.shape == (0, 2)
    assert hk.token_logprobs_backward(x, t, p.lse, p.logp).shape == (0, 50)


def test_captured_and_other_stream(hk):
    x, t = make(5, 50257, BF)
    y, s = make(3, 30000, F32)

    def run():
        p, q = hk.token_logprobs(x, t, entropy=True, top=7), hk.token_logprobs(y, s, top=64)
        return *p, hk.token_logprobs_backward(x, t, p.lse, p.logp, p.entropy, p.logp), q.logp, q.top_index

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    side = torch.cuda.Stream()
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        y.copy_(torch.randn_like(y))
        want = run()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = run()
        graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(want, out, again):
            assert torch.equal(a, b) and torch.equal(a, c)
