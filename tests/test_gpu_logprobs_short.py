"""The likeliest alternatives of rows, or of pieces of them, that are too short for every wave of a workgroup, or whose words
are masked a wave's worth at a time: the right ones, and without a pass over the row for each."""
from __future__ import annotations

import math

import pytest
import torch
from test_gpu_token_logprobs import BF, DEV, F16, F32, check, make, say

pytestmark = pytest.mark.gpu


def device_us(run):
    """Device time of one of 20 captured calls, the least of five replays."""
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(20):
            run()
    best = math.inf
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) * 50)
    return best


CASES = [(16, 50257, BF, 20), (3, 50257, F16, 64), (600, 3000, BF, 20), (600, 1700, F32, 20), (600, 2100, BF, 64)]


def blocked(rows, vocab, dt):
    """The words of the first 64 vectors of every 512 are masked: a wave's share, in all of its rounds."""
    x, t = make(rows, vocab, dt)
    e = 16 // x.element_size()
    word = torch.arange(vocab, device=DEV) // e % 512
    x[:, word < 64] = -math.inf
    x[:, vocab // 2] = 1.0
    return x, torch.full_like(t, vocab // 2)


@pytest.mark.parametrize("rows,vocab,dt,top", CASES)
def test_values(hk, rows, vocab, dt, top):
    say(rows, vocab, dt, top)
    check(hk, *make(rows, vocab, dt), top)
    check(hk, *blocked(rows, vocab, dt), top)


@pytest.mark.parametrize("rows,vocab,dt,top", CASES + [(600, 8192, BF, 20), (300, 50257, BF, 5)])
def test_no_pass_for_each(hk, rows, vocab, dt, top):
    # Against the call without alternatives: the selection is some steps within the workgroup and its alternatives'
    # ranks, where a pass over the row in memory for each of 20 or 64 alternatives would take 1 us and more each.
    for name, (x, t) in (("plain", make(rows, vocab, dt)), ("blocked", blocked(rows, vocab, dt))):
        least = device_us(lambda: hk.token_logprobs(x, t, entropy=True))
        took = device_us(lambda: hk.token_logprobs(x, t, entropy=True, top=top))
        say(rows, vocab, dt, top, name, took, least)
        assert took <= 2 * least + 0.25 * top + 10, (name, took, least)
