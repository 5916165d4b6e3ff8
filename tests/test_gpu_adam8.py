"""AdamW with 8-bit moments (adamw8.hip) against its definition in 64 bits: the codes and scales have
to be the definition's own, the parameters within fp32 rounding."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BLOCK = 256
HYPER = dict(lr=3e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)
M_VALUES = np.arange(128.0) ** 2 / 127.0 ** 2
V_VALUES = np.arange(256.0) ** 4 / 255.0 ** 4
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def say(*a):
    print(*a, flush=True)


def _nearest(x, values, least):
    code = np.searchsorted((values[1:] + values[:-1]) / 2, x, side="right")
    return np.where(x > 0, np.maximum(code, least), code)


def _encode(m, v):
    """(m codes, v codes, m scales, v scales) of fp64 moments [blocks, 256]."""
    ms, vs = np.abs(m).max(1).astype(np.float32), v.max(1).astype(np.float32)
    rm = np.abs(m) / np.where(ms > 0, ms, 1).astype(np.float64)[:, None]
    rv = v / np.where(vs > 0, vs, 1).astype(np.float64)[:, None]
    return ((_nearest(rm, M_VALUES, 0) * np.sign(m)).astype(np.int8),
            _nearest(rv, V_VALUES, 1).astype(np.uint8), ms, vs)


def _decode(mc, vc, ms, vs):
    c = mc.astype(np.int64)
    return (np.sign(c) * M_VALUES[np.abs(c)] * ms.astype(np.float64)[:, None],
            V_VALUES[vc] * vs.astype(np.float64)[:, None])


def _blocks(x, fill=0):
    n = -(-x.size // BLOCK) * BLOCK
    return np.concatenate([x, np.full(n - x.size, fill, x.dtype)]).reshape(-1, BLOCK)


def _step(p, g, state, step, h=HYPER):
    """One step of one tensor in 64 bits: (p, state, the largest error that fp32 leaves in p)."""
    b1, b2, lr, eps, wd = (float(np.float32(h[k])) for k in ("beta1", "beta2", "lr", "eps",
                                                           "weight_decay"))
    bc1, bc2 = (float(np.float32(1 - h[k] ** step)) for k in ("beta1", "beta2"))
    m, v = _decode(*state)
    gb = _blocks(g.astype(np.float64))
    m, v = b1 * m + (1 - b1) * gb, b2 * v + (1 - b2) * gb * gb
    keep = _blocks(np.ones(g.size)) > 0
    m, v = m * keep, v * keep
    update = ((m / bc1) / (np.sqrt(v / bc2) + eps)).reshape(-1)[:p.size]
    p64 = p.astype(np.float64)
    new = p64 - lr * (update + wd * p64)
    # p's own last rounding and two of its products' (half a step each), and of the update: two
    # conversions, two constants and their products (half a step each), square root and reciprocal
    # (a step each), the sum and the quotient: under 8 whole steps of 2^-23
    tol = (np.abs(p64) + np.abs(new)) * 2.0 ** -23 + lr * (np.abs(update) * 2.0 ** -20 +
                                                         wd * np.abs(p64) * 2.0 ** -22)
    return new, _encode(m, v), tol


def _views(flat, sizes, offset):
    """Tensors of these sizes in one buffer, each `offset` elements behind a multiple of 64."""
    out, at = [], 0
    for n in sizes:
        out.append(flat[at + offset:at + offset + n])
        at += -(-(n + offset) // 64) * 64
    return out


def _buffer(sizes, offset, dtype=torch.float32, fill=7.0):
    n = sum(-(-(k + offset) // 64) * 64 for k in sizes)
    return torch.full((n + 64,), fill, device=DEV, dtype=dtype)


def _split(state, sizes):
    """The states of each tensor as numpy blocks."""
    m, v, ms, vs = (t.cpu().numpy() for t in state)
    m, v, at, out = m.reshape(-1, BLOCK), v.reshape(-1, BLOCK), 0, []
    for n in sizes:
        b = -(-n // BLOCK)
        out.append((m[at:at + b], v[at:at + b], ms[at:at + b], vs[at:at + b]))
        at += b
    return out


@pytest.mark.parametrize("sizes", [[1], [255, 256, 257], [513, 3, 70001, 0, 768, 1024],
                                   [2304 * 768]])
@pytest.mark.parametrize("grad", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_step_matches_its_definition(hk, sizes, grad, offset):
    say("adam8", sizes, grad, offset)
    rng = np.random.default_rng(11 + len(sizes) + offset)
    P, G = _buffer(sizes, offset), _buffer(sizes, offset, TYPES[grad])
    C = _buffer(sizes, offset, torch.bfloat16)
    ps, gs, cs = _views(P, sizes, offset), _views(G, sizes, offset), _views(C, sizes, offset)
    for p in ps:
        p.copy_(torch.from_numpy(rng.normal(0, 0.02, p.numel()).astype(np.float32)))
    copies = [c if i % 2 == 0 else None for i, c in enumerate(cs)]
    state = hk.adam8_states(sizes, DEV)
    plan = hk.Adam8Plan(ps, gs, *state, copies=copies)
    assert plan.num_blocks == sum(-(-n // BLOCK) for n in sizes)
    for step in (1, 2, 3):
        for g in gs:
            # elements of all magnitudes, some exactly zero
            x = rng.normal(0, 1e-2, g.numel()) * 10.0 ** rng.uniform(-4, 0, g.numel())
            g.copy_(torch.from_numpy((x * (rng.random(g.numel()) > 0.05)).astype(np.float32)))
        before = [p.cpu().numpy() for p in ps]
        old = _split(state, sizes)
        plan.step(HYPER["lr"], HYPER["beta1"], HYPER["beta2"], HYPER["eps"],
                  HYPER["weight_decay"], 1 - HYPER["beta1"] ** step, 1 - HYPER["beta2"] ** step)
        for p, p0, g, s0, s1, c in zip(ps, before, gs, old, _split(state, sizes), copies):
            want, s, tol = _step(p0, g.float().cpu().numpy(), s0, step)
            for got, ref in zip(s1, s):
                assert np.array_equal(got, ref)
            assert (np.abs(p.cpu().numpy() - want) <= tol).all()
            if c is not None:
                assert torch.equal(c, p.bfloat16())
    # nothing beside the tensors was written
    for buf, views in ((P, ps), (C, [c for c in copies if c is not None])):
        for t in views:
            t.fill_(7.0)
        assert bool((buf == 7.0).all())


def test_codes_at_the_borders(hk):
    """Moments on and beside every border between two codes, and every code's own value."""
    edges = (M_VALUES[1:] + M_VALUES[:-1]) / 2
    m = np.concatenate([M_VALUES, np.nextafter(np.float32(edges), np.float32(0)),
                        np.nextafter(np.float32(edges), np.float32(2))]).astype(np.float32)
    edges = (V_VALUES[1:] + V_VALUES[:-1]) / 2
    v = np.concatenate([V_VALUES, np.nextafter(np.float32(edges), np.float32(0)),
                        np.nextafter(np.float32(edges), np.float32(2))]).astype(np.float32)
    n = max(m.size, v.size)
    m, v = np.resize(m, n), np.resize(v, n)
    m[1::2] *= -1
    blocks = []
    for scale in (1.0, 3.7e-5, 2.9e-30, 5e7):
        # 255 values a block behind one that sets the scale
        for a in range(0, n, BLOCK - 1):
            mm, vv = m[a:a + BLOCK - 1], v[a:a + BLOCK - 1]
            one = np.ones(1, np.float32)
            blocks.append((_blocks(np.concatenate([one, mm]))[0] * np.float32(scale),
                           _blocks(np.concatenate([one, vv]))[0] * np.float32(scale)))
    m = np.stack([b[0] for b in blocks]).astype(np.float32)
    v = np.stack([b[1] for b in blocks]).astype(np.float32)
    dev = lambda a: torch.from_numpy(a.reshape(-1)).to(DEV)  # noqa: E731
    state = hk.adam8_quantize(dev(m), dev(v))
    want = _encode(m.astype(np.float64), v.astype(np.float64))
    got = _split(state, [m.size])[0]
    for a, b in zip(got, want):
        assert np.array_equal(a, b)
    mo, vo = hk.adam8_dequantize(*state)
    wm, wv = _decode(*want)
    # the value's product with the scale, rounded to fp32 once (in fp64 before, 2^-52)
    assert np.allclose(mo.cpu().numpy().reshape(m.shape), wm, rtol=2.0 ** -23, atol=1e-44)
    assert np.allclose(vo.cpu().numpy().reshape(m.shape), wv, rtol=2.0 ** -23, atol=1e-44)


@pytest.mark.parametrize("n", [1, 255, 256, 257, 5000])
def test_quantize_and_back(hk, n):
    rng = np.random.default_rng(n)
    m = rng.normal(0, 1e-3, n).astype(np.float32)
    v = (rng.normal(0, 1e-3, n).astype(np.float32)) ** 2
    buf = torch.full((n + 8,), 5.0, device=DEV)
    state = hk.adam8_quantize(torch.from_numpy(m).to(DEV), torch.from_numpy(v).to(DEV))
    mo, vo = hk.adam8_dequantize(*state, m_out=buf[3:n + 3], v_out=torch.empty(n, device=DEV))
    wm, wv = _decode(*_encode(_blocks(m.astype(np.float64)), _blocks(v.astype(np.float64))))
    assert np.allclose(mo.cpu().numpy(), wm.reshape(-1)[:n], rtol=2.0 ** -23, atol=0)
    assert np.allclose(vo.cpu().numpy(), wv.reshape(-1)[:n], rtol=2.0 ** -23, atol=0)
    assert bool((buf[:3] == 5).all()) and bool((buf[n + 3:] == 5).all())
    # quantizing what codes stand for gives the codes again
    again = hk.adam8_quantize(mo.clone(), vo)
    assert all(torch.equal(a, b) for a, b in zip(again, state))


def test_blocks_of_zero_and_of_what_is_not_finite(hk):
    """A block of zeros stays zero; NaN and infinity stay inside their own block."""
    n = 6 * BLOCK
    p = torch.full((n,), 0.5, device=DEV)
    g = torch.full((n,), 1e-2, device=DEV)
    g[:BLOCK] = 0
    g[BLOCK + 7] = float("nan")
    g[2 * BLOCK + 9] = float("inf")
    g[3 * BLOCK + 255] = -float("inf")
    g[4 * BLOCK] = 3e25  # its square passes fp32
    state = hk.adam8_states([n], DEV)
    plan = hk.Adam8Plan([p], [g], *state)
    plan.step(0.1, 0.9, 0.95, 1e-8, 0.0, 0.1, 0.05)
    m, v, ms, vs = (t.cpu().numpy() for t in state)
    assert ms[0] == 0 and vs[0] == 0 and not m[:BLOCK].any() and not v[:BLOCK].any()
    assert np.isnan(ms[1:5]).all() and np.isnan(vs[1:5]).all()
    assert ms[5] == np.float32((1 - float(np.float32(0.9))) * float(np.float32(1e-2)))
    got = p.cpu().numpy()
    assert (got[:BLOCK] == 0.5).all() and np.isfinite(got[5 * BLOCK:]).all()
    assert np.isnan(got[BLOCK + 7]) and np.isfinite(got[BLOCK:BLOCK + 7]).all()
    plan.step(0.1, 0.9, 0.95, 1e-8, 0.0, 0.1, 0.05)
    got = p.cpu().numpy()
    assert np.isnan(got[BLOCK:5 * BLOCK]).all() and np.isfinite(got[5 * BLOCK:]).all()
    assert (got[:BLOCK] == 0.5).all()


def test_captured_step_replays_as_it_ran(hk):
    sizes = [3000, 77, 768 * 5]
    rng = np.random.default_rng(3)

    def make():
        ps = [torch.from_numpy(rng.normal(0, 1, n).astype(np.float32)).to(DEV) for n in sizes]
        gs = [torch.from_numpy(rng.normal(0, 1, n).astype(np.float32)).to(DEV) for n in sizes]
        st = hk.adam8_states(sizes, DEV)
        return ps, gs, st, hk.Adam8Plan(ps, gs, *st)

    args = (1e-2, 0.9, 0.95, 1e-8, 0.1, 0.1, 0.05)
    ps, gs, st, plan = make()
    ps2 = [p.clone() for p in ps]
    st2 = hk.adam8_states(sizes, DEV)
    plan2 = hk.Adam8Plan(ps2, gs, *st2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        plan.step(*args)
    for _ in range(4):
        for g in gs:
            g.mul_(-0.7).add_(0.01)
        graph.replay()
        plan2.step(*args)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ps + list(st), ps2 + list(st2)))


def test_32_bit_plan_with_the_same_moments(hk):
    """The first step from zero moments uses the moments before they are rounded: AdamPlan's step."""
    rng = np.random.default_rng(5)
    n = 10_000
    p = torch.from_numpy(rng.normal(0, 0.02, n).astype(np.float32)).to(DEV)
    g = torch.from_numpy(rng.normal(0, 0.01, n).astype(np.float32)).to(DEV)
    q, m, v = p.clone(), torch.zeros_like(p), torch.zeros_like(p)
    args = (3e-4, 0.9, 0.95, 1e-8, 0.1, 1 - 0.9, 1 - 0.95)
    hk.AdamPlan([q], [g], [m], [v]).step(*args)
    hk.Adam8Plan([p], [g], *hk.adam8_states([n], DEV)).step(*args)
    # |update| is 1 here: lr times 8 steps of fp32 on each side, and p's own rounding
    tol = q.abs() * 2.0 ** -23 + 3e-4 * 2.0 ** -19
    assert bool(((p - q).abs() <= tol).all())
