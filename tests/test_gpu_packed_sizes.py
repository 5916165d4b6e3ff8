"""Tensors past 2^31 elements or 2^32 bytes through the packed attention, the token log probabilities and the embeddings:
the same bits as on small copies of the rows that count."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def say(*a):
    print("[case]", *a, flush=True)


def test_attention_over_a_cache_of_gigabytes(hk):
    # tokens 128 KiB apart: 70000 of them span 9 GB
    n, step = 70000, 1 << 16
    say("cache", n, step)
    whole = torch.empty(n * step, device=DEV, dtype=BF)
    k, v = (whole[o:].as_strided((n, 2, 64), (step, 64, 1)) for o in (0, 256))
    small = [torch.randn(n, 2, 64, device=DEV).to(BF) for _ in range(2)]
    k.copy_(small[0])
    v.copy_(small[1])
    for lq, lk in (([1], [n]), ([1, 30], [40000, 30000])):
        q, do = (torch.randn(sum(lq), 8, 64, device=DEV).to(BF) for _ in range(2))
        cq, ck = (torch.tensor([0, *torch.tensor(x).cumsum(0)], device=DEV, dtype=torch.int32) for x in (lq, lk))
        o, lse = hk.attn_packed_forward(q, k, v, cq, ck)
        want = hk.attn_packed_forward(q, *small, cq, ck)
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
        dk, dv = (whole[i:].as_strided((n, 2, 64), (step, 64, 1)) for i in (512, 768))
        got = hk.attn_packed_backward(do, q, k, v, o, lse, cq, ck, dk=dk, dv=dv)
        for x, y in zip(got, hk.attn_packed_backward(do, q, *small, o, lse, cq, ck)):
            assert torch.equal(x, y)


def test_queries_far_apart(hk):
    # heads 1 GiB apart and more: [heads, tokens, head_dim] of a buffer for many tokens
    T, far = 300, 1 << 29
    say("heads", far)
    whole = torch.empty(8 * far, device=DEV, dtype=BF)
    q = whole.as_strided((T, 8, 64), (64, far, 1))
    do = whole[64 * T:].as_strided((T, 8, 64), (64, far, 1))
    qs, dos, k, v = (torch.randn(T, h, 64, device=DEV).to(BF) for h in (8, 8, 2, 2))
    q.copy_(qs)
    do.copy_(dos)
    cu = torch.tensor([0, 170, T], device=DEV, dtype=torch.int32)
    dq = whole[128 * T:].as_strided((T, 8, 64), (64, far, 1))
    o, lse = hk.attn_packed_forward(q, k, v, cu)
    want = hk.attn_packed_forward(qs, k, v, cu)
    assert torch.equal(o, want[0])
    for x, y in zip(hk.attn_packed_backward(do, q, k, v, o, lse, cu, dq=dq),
                    hk.attn_packed_backward(dos, qs, k, v, o, lse, cu)):
        assert torch.equal(x, y)


def test_logits_past_2_to_31_elements(hk):
    rows, vocab, stride = 50000, 50257, 50304
    say("logits", rows, stride)
    x = torch.empty(rows, stride, device=DEV, dtype=BF)
    for r in range(0, rows, 5000):
        x[r:r + 5000] = torch.randn(5000, stride, device=DEV)
    x = x[:, :vocab]
    t = torch.randint(0, vocab, (rows,), device=DEV)
    g = torch.randn(rows, device=DEV)
    tail = slice(rows - 600, rows)
    last, lt = torch.empty(600, stride, device=DEV, dtype=BF)[:, :vocab], t[tail].clone()
    last.copy_(x[tail])  # rows begin as x's do within 16 bytes, so the sums have one order
    for top in (0, 3):
        p = hk.token_logprobs(x, t, entropy=True, top=top)
        want = hk.token_logprobs(last, lt, entropy=True, top=top)
        for a, b in zip(p, want):
            assert a is None or torch.equal(a[tail], b)
    dx = hk.token_logprobs_backward(x, t, p.lse, g, p.entropy, g, grad=x)
    # the gradient goes by elements
    assert torch.equal(dx[tail], hk.token_logprobs_backward(last, lt, want.lse, g[tail].clone(), want.entropy,
                                                            g[tail].clone()))


def test_a_table_past_2_to_31_elements(hk):
    vocab, d, n = 2200000, 1024, 3000
    say("table", vocab, d)
    table = torch.zeros(vocab, d, device=DEV, dtype=BF)
    rows = torch.randn(1000, d, device=DEV).to(BF)
    table[-1000:] = rows
    t = torch.randint(vocab - 1000, vocab, (n,), device=DEV)
    y = hk.embedding_forward(table, t)
    assert torch.equal(y, rows[t - (vocab - 1000)])
    for m in (n, 500):  # sorted, and few
        table.fill_(3.0)
        hk.embedding_backward(y[:m], t[:m].clone(), table, accumulate=False)
        small = hk.embedding_backward(y[:m], t[:m] - (vocab - 1000), torch.empty_like(rows), accumulate=False)
        assert torch.equal(table[-1000:], small)
        assert not table[:-1000].any()
