"""Packed attention over more sequences than a wave has lanes, with several tiles each; over caches with room behind each
sequence; and with groups of more heads than a tile has rows. Values and tolerances as in test_gpu_attn_packed.py."""
from __future__ import annotations

import random

import pytest
import torch
from test_gpu_attn_packed import BF, DEV, F16, both, check, cu_of, make, reference, say

pytestmark = pytest.mark.gpu


def lens(n, lo, hi, seed):
    r = random.Random(seed)
    return [r.choice([0, 1, r.randint(lo, hi), r.randint(lo, hi), r.randint(lo, hi)]) for _ in range(n)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,lo,hi,H,Hk,d,dt", [
    (66, 30, 700, 2, 1, 64, BF),        # 64 rows a workgroup
    (130, 100, 400, 12, 12, 64, BF),    # 128
    (90, 100, 500, 4, 4, 128, F16),
    (70, 20, 300, 3, 1, 40, BF),        # 32
    (200, 1, 150, 8, 2, 128, F16),
])
def test_more_than_64_sequences_of_several_tiles(hk, n, lo, hi, H, Hk, d, dt, causal):
    say(n, lo, hi, H, Hk, d, dt, causal)
    lq = lens(n, lo, hi, n)
    both(hk, lq, lq, H, Hk, d, dt, causal, seed=n)
    both(hk, lq, lens(n, lo, hi, n + 1), H, Hk, d, dt, causal, seed=n)


@pytest.mark.parametrize("n", [64, 65, 128, 129, 200])
def test_tokens_of_many_sequences_over_long_keys(hk, n):
    r = random.Random(n)
    lq = [r.choice([1, 1, 1, 3]) for _ in range(n)]
    lk = [r.choice([1, 17, 600, r.randint(1, 1500)]) for _ in range(n)]
    for H, Hk, d in ((4, 1, 64), (16, 4, 128)):
        say(n, H, Hk, d)
        both(hk, lq, lk, H, Hk, d, BF, True, seed=n)


def test_more_sequences_of_one_tile_than_tiles(hk):
    # what the sequences' numbers bound, and not their rows
    for n in (63, 64, 65, 300):
        both(hk, [1] * n, [1] * n, 2, 2, 64, BF, True, seed=n)
        both(hk, [0] * n + [3], [0] * n + [5], 2, 1, 64, F16, True, seed=n)


@pytest.mark.parametrize("n,room", [(5, 3000), (40, 300)])
def test_a_cache_with_room_behind_each_sequence(hk, n, room):
    # A sequence without queries between any two takes the room: its keys are read into no other, and have gradients of 0.
    say(n, room)
    r = random.Random(n)
    lens_q, lens_k = [r.choice([1, 2, 40]) for _ in range(n)], [r.randint(41, room) for _ in range(n)]
    lq = [x for m in lens_q for x in (m, 0)]
    lk = [x for k in lens_k for x in (k, room - k)]
    q, k, v, do = make(lq, lk, 8, 2, 64, BF, seed=n)
    cq, ck = cu_of(lq), cu_of(lk)
    free = torch.zeros(k.shape[0], device=DEV, dtype=torch.bool)
    for i, m in enumerate(lens_k):
        free[i * room + m:(i + 1) * room] = True
    keep = [t.clone() for t in (k, v)]
    for t in (k, v):
        t[free] = float("nan")
    o, lse = hk.attn_packed_forward(q, k, v, cq, ck)
    dq, dk, dv = hk.attn_packed_backward(do, q, k, v, o, lse, cq, ck)
    torch.cuda.synchronize()
    assert not dk[free].any() and not dv[free].any()
    check({"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}, reference(q, *keep, lq, lk, True, 0.125, do))


@pytest.mark.parametrize("H,Hk,d,dt", [(48, 1, 64, BF), (128, 1, 128, F16), (80, 2, 32, BF), (33, 1, 96, F16)])
def test_groups_of_more_heads_than_a_tile_has_rows(hk, H, Hk, d, dt):
    say(H, Hk, d, dt)
    both(hk, [1, 5, 33], [200, 5, 64], H, Hk, d, dt, True, seed=H)
    both(hk, [1], [3000], H, Hk, d, dt, True, seed=H)


def test_gradient_of_one_row_or_head_for_all(hk):
    # a gradient that was broadcast over tokens or heads
    ls = [70, 33]
    q, k, v, do = make(ls, ls, 4, 2, 64, BF)
    cq = cu_of(ls)
    o, lse = hk.attn_packed_forward(q, k, v, cq)
    for g in (do[:1].expand_as(do), do[:, :1].expand_as(do)):
        for x, y in zip(hk.attn_packed_backward(g, q, k, v, o, lse, cq),
                        hk.attn_packed_backward(g.contiguous(), q, k, v, o, lse, cq)):
            assert torch.equal(x, y)


def test_two_calls_at_once(hk):
    a = make([900, 33], [900, 33], 8, 2, 128, F16, seed=1)
    b = make([1, 3], [4000, 900], 8, 2, 128, F16, seed=2)
    starts = ((cu_of([900, 33]), None), (cu_of([1, 3]), cu_of([4000, 900])))

    def step(t, cu):
        o, lse = hk.attn_packed_forward(*t[:3], *cu)
        return o, lse, *hk.attn_packed_backward(t[3], *t[:3], o, lse, *cu)

    want = [step(t, cu) for t, cu in zip((a, b), starts)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for s, t, cu in zip(streams, (a, b), starts):
            with torch.cuda.stream(s):
                got.append(step(t, cu))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        for x, y in zip(g, want[i % 2]):
            assert torch.equal(x, y), i
