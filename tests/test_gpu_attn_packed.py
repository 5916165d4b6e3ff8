"""GPU parity of the 16-bit attention over packed sequences, forward and backward, against its definition in 64 bits.

Tolerances, element by element, from what is rounded where (e: half a step of the type, relative):
  s      sums of d exact products in fp32: ds = d 2^-23 scale sum |q| |k|, which P and the log-sum-exp carry on
  o      P rounded, then o: e (A + |o|), A = sum p |v|; A (2 ds + n 2^-23 + 2^-20) for the rest of P and the sum
  dv     the same with dout in the place of v
  delta  dout times o's error, td
  ds     p (td + d 2^-23 sum |dout| |v|) + |ds| (e + 2 ds + 2^-20), times |k| or |q| and summed, then rounded
fp16 values under its normal range have an absolute step: 2^-25 for each P or dS, 2^-25 for a result. The hardware's
exp2 and the products give 0 for fp32 and bf16 values under 2^-126 (a P of 2^-130 is no error of P's rounding: it is
off by all of itself, which is under 2^-126, and dS by that times |dp - delta|)."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16 = torch.bfloat16, torch.float16


def say(*a):
    print("[case]", *a, flush=True)


def cu_of(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, device=DEV, dtype=torch.int32)


def reference(q, k, v, lq, lk, causal, scale, do=None, step=None):
    """Per output its value and tolerance, in 64 bits: {name: (value, tolerance)}. step: the absolute one of dS."""
    H, Hk, d = q.shape[1], k.shape[1], q.shape[2]
    e = torch.finfo(q.dtype).eps / 2
    tiny = 2.0 ** -25 if q.dtype is F16 else 2.0 ** -126
    z = lambda t: torch.zeros(t.shape, device=DEV, dtype=torch.float64)  # noqa: E731
    out = {"o": [z(q), z(q)], "lse": [torch.full((H, q.shape[0]), -math.inf, device=DEV, dtype=torch.float64),
                                      torch.zeros(H, q.shape[0], device=DEV, dtype=torch.float64)]}
    if do is not None:
        out |= {"dq": [z(q), z(q)], "dk": [z(k), z(k)], "dv": [z(k), z(k)]}
    heads = lambda t: t.double().transpose(0, 1)  # noqa: E731
    a = b = 0
    for m, n in zip(lq, lk):
        qs, ks = slice(a, a + m), slice(b, b + n)
        a, b = a + m, b + n
        if m == 0 or n == 0:
            continue
        Q = heads(q[qs])
        K, V = (heads(t[ks]).repeat_interleave(H // Hk, 0) for t in (k, v))
        see = torch.ones(m, n, device=DEV, dtype=torch.bool)
        if causal:
            see = see.tril(n - m)
        x = (Q @ K.transpose(1, 2) * scale).masked_fill(~see, -math.inf)
        lse = torch.logsumexp(x, 2)
        p = torch.where(see, (x - lse.nan_to_num(neginf=0.0)[..., None]).exp(), 0.0)
        ds_ = d * 2.0 ** -23 * scale * (Q.abs() @ K.abs().transpose(1, 2)).amax(2, keepdim=True)
        rest = 2 * ds_ + n * 2.0 ** -23 + 2.0 ** -20
        o, A = p @ V, p @ V.abs()
        to = e * (A + o.abs()) * 1.01 + A * rest + n * tiny * V.abs().amax() + tiny
        out["o"][0][qs], out["o"][1][qs] = o.transpose(0, 1), to.transpose(0, 1)
        out["lse"][0][:, qs] = lse
        out["lse"][1][:, qs] = (rest[..., 0] + lse.nan_to_num(neginf=0.0).abs() * 2.0 ** -22)
        if do is None:
            continue
        G = heads(do[qs])
        fold = lambda t: t.view(Hk, H // Hk, n, d).sum(1).transpose(0, 1)  # noqa: E731
        pt = p.transpose(1, 2)
        dv, Ad = pt @ G, pt @ G.abs()
        tv = (p * (e * 1.01 + rest)).transpose(1, 2) @ G.abs() + tiny * G.abs().sum(1, keepdim=True)
        dp = G @ V.transpose(1, 2)
        delta = (G * o).sum(2, keepdim=True)
        td = (G.abs() * (to + d * 2.0 ** -23 * o.abs())).sum(2, keepdim=True)
        ds = p * (dp - delta)
        t = p * (td + d * 2.0 ** -23 * (G.abs() @ V.abs().transpose(1, 2))) + ds.abs() * (e * 1.01 + rest)
        t = torch.where(see, t + (tiny * (1 + (dp - delta).abs()) if step is None else step), 0.0)
        dq, tq = scale * ds @ K, scale * t @ K.abs()
        dk, tk = scale * ds.transpose(1, 2) @ Q, scale * t.transpose(1, 2) @ Q.abs()
        # n and m products are summed in fp32
        tq = tq + n * 2.0 ** -24 * scale * ds.abs() @ K.abs()
        rows = m * (H // Hk) * 2.0 ** -24
        tk = tk + rows * scale * ds.abs().transpose(1, 2) @ Q.abs()
        tv = tv + rows * Ad
        out["dq"][0][qs], out["dq"][1][qs] = dq.transpose(0, 1), tq.transpose(0, 1)
        for name, val, tol in (("dk", dk, tk), ("dv", dv, tv)):
            out[name][0][ks], out[name][1][ks] = fold(val), fold(tol)
    for name in ("dq", "dk", "dv"):
        if name in out:
            out[name][1] += e * 1.01 * out[name][0].abs() + tiny
    return out


def check(got, want):
    for name, (val, tol) in want.items():
        x = got[name].double()
        fine = torch.isfinite(val)
        assert torch.equal(torch.isfinite(x), fine), name
        assert torch.equal(x[~fine], val[~fine]), name
        off = (x - val).abs()[fine]
        bad = off > tol[fine]
        assert not bad.any(), (name, int(bad.sum()), float((off / tol[fine].clamp_min(1e-300)).max()), float(off[bad].max()))


def make(lq, lk, H, Hk, d, dt, seed=0, layout="plain", std=1.0, pad=(0, 0)):
    g = torch.Generator(device=DEV).manual_seed(seed)
    tq, tk = sum(lq) + sum(pad), sum(lk) + sum(pad)

    def rand(t, h):
        if layout == "heads":  # [heads, tokens, head_dim]
            return (torch.randn(h, t, d, generator=g, device=DEV) * std).to(dt).transpose(0, 1)
        return (torch.randn(t, h, d, generator=g, device=DEV) * std).to(dt)

    if layout == "projection" and tq == tk:
        x = rand(tq, H + 2 * Hk)
        return x[:, :H], x[:, H:H + Hk], x[:, H + Hk:], rand(tq, H)
    return rand(tq, H), rand(tk, Hk), rand(tk, Hk), rand(tq, H)


def both(hk, lq, lk, H, Hk, d, dt, causal, scale=None, seed=0, layout="plain", std=1.0):
    q, k, v, do = make(lq, lk, H, Hk, d, dt, seed, layout, std)
    cq, ck = cu_of(lq), None if lq == lk else cu_of(lk)
    o, lse = hk.attn_packed_forward(q, k, v, cq, ck, causal, scale)
    dq, dk, dv = hk.attn_packed_backward(do, q, k, v, o, lse, cq, ck, causal, scale)
    torch.cuda.synchronize()
    got = {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    check(got, reference(q, k, v, lq, lk, causal, d ** -0.5 if scale is None else scale, do))
    return got


LENS = {
    "one": ([1], [1]),
    "borders": ([31, 32, 33, 63, 64, 65, 127, 128, 129], None),
    "odd": ([17, 1, 250, 3, 77], None),
    "empty": ([5, 0, 40, 0, 0, 7], [5, 0, 40, 9, 0, 0]),
    "longer_keys": ([1, 7, 33, 64, 100], [300, 7, 160, 65, 511]),
    "longer_queries": ([40, 130, 65, 3], [33, 2, 64, 1]),
    "many": ([(7 * i) % 23 for i in range(150)], None),
}


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,Hk,d,dt", [(4, 4, 64, BF), (6, 2, 128, F16), (5, 1, 64, F16), (3, 3, 128, BF),
                                       (2, 1, 8, BF), (4, 2, 80, F16), (2, 2, 40, BF), (2, 1, 96, BF)])
@pytest.mark.parametrize("lens", list(LENS))
def test_small(hk, lens, H, Hk, d, dt, causal):
    lq, lk = LENS[lens]
    say(lens, H, Hk, d, dt, causal)
    both(hk, lq, lq if lk is None else lk, H, Hk, d, dt, causal, seed=H * d)


@pytest.mark.parametrize("lq,lk,H,Hk,d,dt,causal", [
    ([4097], None, 8, 8, 64, BF, True),             # 128 rows a workgroup
    ([2048, 1001, 333], None, 16, 4, 128, F16, True),
    ([1500, 700, 1900], None, 12, 3, 64, BF, False),
    ([2000, 2100], [1700, 2500], 12, 12, 96, BF, True),
    ([700, 1100], [1200, 650], 32, 1, 128, BF, True),
    ([1, 1, 1, 2, 5], [4000, 17, 1, 2049, 300], 16, 4, 128, BF, True),  # shares of keys
    ([1], [8191], 8, 1, 64, F16, True),
    ([3], [5000], 3, 3, 128, BF, False),
])
def test_larger(hk, lq, lk, H, Hk, d, dt, causal):
    say(lq, lk, H, Hk, d, dt, causal)
    both(hk, lq, lq if lk is None else lk, H, Hk, d, dt, causal, seed=1)


@pytest.mark.parametrize("layout", ["projection", "heads"])
@pytest.mark.parametrize("lens,H,Hk", [([100, 29], 4, 2), ([4100], 8, 8), ([1], 4, 1)])
def test_strides(hk, layout, lens, H, Hk):
    say(layout, lens)
    both(hk, lens, lens, H, Hk, 64, BF, True, layout=layout)


@pytest.mark.parametrize("std,scale", [(8.0, 1.0), (1e-3, 1.0), (3.0, 0.01), (30.0, 0.2)])
def test_ranges(hk, std, scale):
    # sharp softmaxes whose maximum moves from tile to tile, and flat ones
    say(std, scale)
    both(hk, [300, 41], [300, 41], 4, 2, 64, BF, True, scale=scale, std=std)


@pytest.mark.parametrize("size", [2.0 ** -12, 1.0, 2.0 ** 9])
@pytest.mark.parametrize("H,Hk,d,lens", [(4, 2, 64, [1500, 70]), (2, 2, 128, [900]), (16, 4, 128, [2048, 600])])
def test_small_and_large_gradients_in_fp16(hk, size, H, Hk, d, lens):
    # a dS of P times dout, 1e-3 * 2e-4, is no normal fp16 number: it is held for a dout of 1
    say(size, H, Hk, d, lens)
    q, k, v, do = make(lens, lens, H, Hk, d, F16, std=0.3)
    do = (do * (size / 0.3)).to(F16)
    do[::3] *= 0.125  # rows of different sizes, and of nothing, as a loss leaves out
    do[5::7] = 0
    cq = cu_of(lens)
    o, lse = hk.attn_packed_forward(q, k, v, cq)
    dq, dk, dv = hk.attn_packed_backward(do, q, k, v, o, lse, cq)
    # half a step of fp16's smallest numbers, times the power of two above the largest dout; a result's own is not scaled
    step = 2.0 ** -24 * float(do.abs().max())
    want = reference(q, k, v, lens, lens, True, d ** -0.5, do, step)
    check({"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}, want)


def test_rows_of_no_sequence_stay(hk):
    lens = [70, 0, 133]
    for H, Hk, lk in ((4, 2, lens), (4, 1, [900, 5, 700])):
        q, k, v, do = make(lens, lk, H, Hk, 64, BF, pad=(5, 9))
        cq, ck = cu_of(lens) + 5, cu_of(lk) + 5
        for t in (q, k, v, do):  # what lies there is not read into any sequence
            t[:5] = math.nan
            t[-9:] = math.nan
        o, dq = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
        dk, dv = torch.full_like(k, 7.0), torch.full_like(k, 7.0)
        lse = torch.full((H, q.shape[0]), 7.0, device=DEV)
        hk.attn_packed_forward(q, k, v, cq, ck, o=o, lse=lse)
        hk.attn_packed_backward(do, q, k, v, o, lse, cq, ck, dq=dq, dk=dk, dv=dv)
        torch.cuda.synchronize()
        for t in (o, dq, dk, dv, lse.t()):
            assert (t[:5] == 7).all() and (t[-9:] == 7).all()
        cut = lambda t: t[5:-9]  # noqa: E731
        got = {"o": cut(o), "lse": lse[:, 5:-9], "dq": cut(dq), "dk": cut(dk), "dv": cut(dv)}
        check(got, reference(cut(q), cut(k), cut(v), lens, lk, True, 0.125, cut(do)))


def test_not_finite_stays_in_its_sequence(hk):
    lens = [65, 130, 40]
    for bad in (math.nan, math.inf):
        q, k, v, do = make(lens, lens, 4, 2, 128, BF)
        want = reference(q, k, v, lens, lens, True, 128 ** -0.5, do)
        q[100, 1, 3] = k[70, 0, 5] = v[194, 1, 7] = bad
        cq = cu_of(lens)
        o, lse = hk.attn_packed_forward(q, k, v, cq)
        dq, dk, dv = hk.attn_packed_backward(do, q, k, v, o, lse, cq)
        for s in (slice(0, 65), slice(195, 235)):
            part = lambda name, x: x[:, s] if name == "lse" else x[s]  # noqa: E731
            check({n: part(n, t) for n, t in dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv).items()},
                  {n: [part(n, t) for t in w] for n, w in want.items()})
        assert not torch.isfinite(o[100, 1]).all() and not torch.isfinite(o[194, 3]).all()


def test_starts_past_the_tensors(hk):
    q, k, v, do = make([100], [100], 4, 2, 64, BF)
    good = torch.tensor([0, 50, 100, 100, 100], device=DEV, dtype=torch.int32)
    bad = torch.tensor([-7, 50, 2 ** 31 - 1, 2 ** 30, 12345], device=DEV, dtype=torch.int32)
    o, lse = hk.attn_packed_forward(q, k, v, good)
    p, lse2 = hk.attn_packed_forward(q, k, v, bad)
    assert torch.equal(o, p) and torch.equal(lse, lse2)
    for x, y in zip(hk.attn_packed_backward(do, q, k, v, o, lse, good),
                    hk.attn_packed_backward(do, q, k, v, o, lse, bad)):
        assert torch.equal(x, y)


def test_starts_that_fall_stay_inside(hk):
    # not what cu may hold: which rows are written is not said, but none outside the tensors is
    q, k, v, do = make([300], [300], 4, 2, 64, BF)
    for starts in ([0, 100, 0, 100, 0, 100], [300, 200, 100, 0], [-5, 400, -5, 400], [50, 50, 10, 90, 20, 290]):
        cu = torch.tensor(starts, device=DEV, dtype=torch.int32)
        held = [torch.full((t.shape[0] + 20, *t.shape[1:]), 7.0, device=DEV, dtype=BF) for t in (q, q, k, v)]
        lses = torch.full((4, 340), 7.0, device=DEV)
        o, dq, dk, dv = (t[10:-10] for t in held)
        lse = lses[:, 20:320]
        lse[:] = 0
        hk.attn_packed_forward(q, k, v, cu, o=o, lse=lse)
        hk.attn_packed_backward(do, q, k, v, o, lse, cu, dq=dq, dk=dk, dv=dv)
        torch.cuda.synchronize()
        for t in held:
            assert (t[:10] == 7).all() and (t[-10:] == 7).all(), starts
        assert (lses[:, :20] == 7).all() and (lses[:, 320:] == 7).all(), starts


def test_no_keys_and_no_queries(hk):
    for lq, lk in (([5], [0]), ([0], [7]), ([0, 0], [0, 0])):
        both(hk, lq, lk, 4, 2, 64, BF, True)
    # no sequence: nothing is written
    q, k, v, _ = make([3], [3], 2, 1, 64, F16)
    o = torch.full_like(q, 7.0)
    hk.attn_packed_forward(q, k, v, torch.zeros(1, device=DEV, dtype=torch.int32), o=o)
    assert (o == 7).all()


def test_same_bits_and_other_stream(hk):
    lens = [700, 33, 1000]
    a = both(hk, lens, lens, 8, 2, 128, BF, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = both(hk, lens, lens, 8, 2, 128, BF, True)
    torch.cuda.synchronize()
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_captured(hk):
    lq, lk = [1, 2, 64], [3000, 700, 64]
    q, k, v, do = make(lq, lk, 8, 2, 128, BF)
    cq, ck = cu_of(lq), cu_of(lk)
    run = lambda: (lambda o, lse: (o, lse, *hk.attn_packed_backward(do, q, k, v, o, lse, cq, ck)))(  # noqa: E731
        *hk.attn_packed_forward(q, k, v, cq, ck))
    run()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        graphs.append((g, out))
    for i in range(4):
        q.copy_(torch.randn_like(q))
        do.copy_(torch.randn_like(do))
        want = run()
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for x, y in zip(out, want):
                assert torch.equal(x, y), i


def test_gradients_against_differences(hk):
    # the gradient along a direction against the difference of the outputs, both in 64 bits from the kernel's outputs
    lens = [40, 25]
    q, k, v, do = make(lens, lens, 4, 2, 64, F16)
    cq = cu_of(lens)
    o, lse = hk.attn_packed_forward(q, k, v, cq)
    grads = hk.attn_packed_backward(do, q, k, v, o, lse, cq)
    step = 2.0 ** -4
    for i, x in enumerate((q, k, v)):
        u = torch.randn(x.shape, device=DEV).sign().to(F16)
        ends = []
        for s in (step, -step):
            args = [t.clone() for t in (q, k, v)]
            args[i] += s * u
            ends.append((args[i].double(), hk.attn_packed_forward(*args, cq)[0].double()))
        (x1, o1), (x0, o0) = ends
        along = float((grads[i].double() * (x1 - x0)).sum())
        change = float(((o1 - o0) * do.double()).sum())
        # both ends' outputs are off by their tolerance at random signs, and the third difference of a softmax over
        # scores that move by 2^-4 * sqrt(d) / sqrt(d) is under 2^-8 of the first in norm
        ref = [reference(*[t if j != i else e[0].to(F16) for j, t in enumerate((q, k, v))], lens, lens, True, 0.125)
               for e in ends]
        noise = sum(float((r["o"][1] * do.double()).square().sum()) for r in ref) ** 0.5 * 4
        size = float(grads[i].double().square().sum()) ** 0.5 * float((x1 - x0).square().sum()) ** 0.5
        assert abs(along - change) <= noise + 2.0 ** -6 * size, (i, along, change, noise, size)


@pytest.mark.parametrize("t", [BF, F16])
@pytest.mark.parametrize("H,Hk,d", [(4, 4, 64), (8, 2, 128)])
@pytest.mark.parametrize("lens", [[24, 117, 390, 5, 64], [1300], [16] * 40])
def test_gradients_are_off_by_little_more_than_their_rounding(hk, lens, H, Hk, d, t):
    # In the norm: dq and dk have the rounding of dS beside their own, both of the same relative size at random signs:
    # sqrt(2) of their own. Where delta is formed from the o that was rounded (twice), over 65 keys and more, that adds
    # at most 2 / 64 to the 2 under the root. A thirtieth for the chance in both.
    say(lens, H, Hk, d, t)
    q, k, v, do = make(lens, lens, H, Hk, d, t)
    cu = cu_of(lens)
    o, lse = hk.attn_packed_forward(q, k, v, cu)
    dq, dk, _ = hk.attn_packed_backward(do, q, k, v, o, lse, cu)
    ref = reference(q, k, v, lens, lens, True, d ** -0.5, do)
    for name, got in (("dq", dq), ("dk", dk)):
        want = ref[name][0]
        least = float((want.to(t).double() - want).norm())
        off = float((got.double() - want).norm())
        print("   ", name, off / least, flush=True)
        assert off <= (2 + 1 / 32) ** 0.5 * (1 + 1 / 30) * least, (name, off / least)
