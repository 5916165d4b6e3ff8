"""Calls whose work takes more threads than one launch has (2^32 a dimension), against 64 bits or a small call on
the same data."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16
ULP, HALF_STEP = 2.0 ** -24, 2.0 ** -8
FIRST = 2 ** 20  # elements at the start of a tensor that are compared


@pytest.fixture(autouse=True)
def memory():
    """Gives back what other tests have left with the allocator, before and behind."""
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def _room(gib):
    free = torch.cuda.mem_get_info()[0]
    if free < (gib + 4) << 30:
        pytest.skip(f"needs {gib + 4} GiB of device memory, {free >> 30} are free")


def _normal(gen, *shape, dtype=BF):
    return torch.empty(*shape, device=DEV, dtype=dtype).normal_(generator=gen)


def _gen(seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return gen


def _spans(n, *at):
    """Short ranges at the ends and around the given places."""
    return [slice(0, 70), slice(n - 90, n)] + [slice(a - 70, a + 70) for a in at]


@pytest.mark.parametrize("tb,N,K", [(1, 2 ** 26 + 44, 8), (0, 2 ** 29 + 72, 2)])
def test_one_row(hk, tb, N, K):
    _room(12)
    gen = _gen(1)
    x, w, b = _normal(gen, 1, K), _normal(gen, *((N, K) if tb else (K, N))), _normal(gen, N)
    r, z = _normal(gen, 1, N), torch.empty(1, N, device=DEV, dtype=BF)
    y = hk.bgemm_act(x, w, bias=b, activation="relu", residual=r, preact=z, trans_b=bool(tb))
    print("forward", flush=True)
    db = torch.full((N,), 0.5, device=DEV)
    d = hk.bgemm_act_backward(x, w, preact=z, activation="relu", dbias=db, trans_b=bool(tb))
    print("backward", flush=True)
    for s in _spans(N, N // 2, 2 ** 25, 2 ** 26 - 30, N - N // 3):
        ws = (w[s].t() if tb else w[:, s]).double().contiguous()
        prod, mag = x.double() @ ws, x.double().abs() @ ws.abs()
        want = prod + b[s].double()
        tol = (K + 4) * ULP * (mag + b[s].double().abs())
        assert bool(((z[:, s].double() - want).abs() <= tol + HALF_STEP * want.abs()).all())
        want = want.clamp_min(0) + r[:, s].double()
        assert bool(((y[:, s].double() - want).abs() <= tol + (ULP + HALF_STEP) * want.abs() + 1e-37).all())
        want = prod * (z[:, s] > 0)
        assert bool(((d[:, s].double() - want).abs() <= tol + HALF_STEP * want.abs()).all())
        assert bool(((db[s].double() - want[0] - 0.5).abs() <= tol[0] + ULP * (want[0].abs() + 1)).all())


def test_products_without_k(hk):
    """The plain kernel: 16 GiB of outputs."""
    M, N = 2 ** 17 + 40, 2 ** 16 + 8
    _room(36)
    gen = _gen(2)
    x, w = torch.empty(M, 0, device=DEV, dtype=BF), torch.empty(0, N, device=DEV, dtype=BF)
    b = _normal(gen, N)
    y = torch.full((M, N), 7.0, device=DEV, dtype=BF)
    hk.bgemm_act(x, w, bias=b, activation="relu", out=y)
    for at in range(0, M, 2 ** 13):
        assert bool((y[at:at + 2 ** 13] == b.clamp_min(0)).all()), at
    print("forward", flush=True)
    db = torch.full((N,), 3.0, device=DEV)
    hk.bgemm_act_backward(x, w, preact=y, activation="relu", dbias=db, out=y, accumulate=False)
    for at in range(0, M, 2 ** 13):
        assert bool((y[at:at + 2 ** 13] == 0).all()), at
    assert bool((db == 0).all())


def test_no_rows(hk):
    """A bias gradient of zero in more columns than one launch has."""
    N, K = 2 ** 29 + 72, 2
    _room(6)
    empty, w = torch.empty(0, K, device=DEV, dtype=BF), torch.empty(K, N, device=DEV, dtype=BF)
    db = torch.full((N,), 2.0, device=DEV)
    hk.bgemm_act_backward(empty, w, dbias=db)
    assert bool((db == 2).all())
    hk.bgemm_act_backward(empty, w, dbias=db, accumulate=False)
    assert bool((db == 0).all())


@pytest.mark.parametrize("K", [8, 9])
def test_rows_past_the_tiles(hk, K):
    """Small tiles over more than 2^30 rows; of 9 elements, unaligned."""
    M, N = 2 ** 30 + 72, 8
    _room(68)
    gen = _gen(3)
    x, w, b = _normal(gen, M, K), _normal(gen, K, N), _normal(gen, N)
    z = torch.empty(M, N, device=DEV, dtype=BF)
    y = hk.bgemm_act(x, w, bias=b, activation="relu", preact=z)
    print("forward, tile", hk.lib().hk_bgemm_small_tile(0, 0, M, N, K, 1, 0), flush=True)
    wd = w.double()
    for s in _spans(M, 2 ** 25, M // 2, 2 ** 30):
        xd = x[s].double()
        want = xd @ wd + b.double()
        tol = (K + 4) * ULP * (xd.abs() @ wd.abs() + b.double().abs())
        assert bool(((z[s].double() - want).abs() <= tol + HALF_STEP * want.abs()).all())
        want = want.clamp_min(0)
        assert bool(((y[s].double() - want).abs() <= tol + HALF_STEP * want.abs()).all())
    del y
    db = torch.full((N,), 5.0, device=DEV)
    d = hk.bgemm_act_backward(x, w, preact=z, activation="relu", dbias=db, accumulate=False)
    print("backward", flush=True)
    total, size, tol = (torch.zeros(N, device=DEV, dtype=torch.float64) for _ in range(3))
    for at in range(0, M, 2 ** 24):
        s = slice(at, min(M, at + 2 ** 24))
        xd = x[s].double()
        want = xd @ wd * (z[s] > 0)
        t = (K + 4) * ULP * (xd.abs() @ wd.abs())
        assert bool(((d[s].double() - want).abs() <= t + HALF_STEP * want.abs()).all()), at
        total += want.sum(0)
        size += want.abs().sum(0)
        tol += t.sum(0)
    # a chain of at most 48 + M / 128 additions of values of either sign, and one for each call that adds to it
    tol += (48 + M / 128) * ULP * size
    assert bool(((db.double() - total).abs() <= tol).all())


def test_query_norms_of_64_lanes_a_row(hk):
    """Two rotated elements of 128: a row takes 64 lanes, so 2^26 of them are 2^32."""
    B, H, T, d = 1, 64, 2 ** 20 + 3, 128
    _room(20)
    q = _normal(_gen(4), B, T, H, d).transpose(1, 2)
    ang = torch.randn(T, 1, generator=_gen(5), device=DEV)
    cos, sin = ang.cos(), ang.sin()
    parts = [slice(0, 5), slice(T // 2, T // 2 + 5), slice(T - 5, T)]
    x = [q[:, :, s].double() for s in parts]
    hk.qk_norm_rope_forward(q, None, cos, sin, q_out=q)
    for s, t in zip(parts, x):
        n = t * (t.square().mean(-1, keepdim=True) + 1e-6) ** -0.5
        c, sn = cos[s, 0].double(), sin[s, 0].double()
        want, spread = n.clone(), n.abs()
        want[..., 0], want[..., 1] = n[..., 0] * c - n[..., 1] * sn, n[..., 1] * c + n[..., 0] * sn
        spread[..., :2] = n[..., :2].abs().sum(-1, keepdim=True)
        tol = 24 * ULP * spread + HALF_STEP * want.abs()
        assert bool(((q[:, :, s].double() - want).abs() <= tol).all()), s


def test_8_bit_adamw(hk):
    """17.2 G parameters of bf16 gradients: 2^26 blocks and two more."""
    n = 2 ** 34 + 300
    cut = n - 300 - 2 ** 20
    _room(200)
    gen = _gen(6)
    p, g = _normal(gen, n, dtype=torch.float32), _normal(gen, n)
    states = hk.adam8_states([n])
    small = [p[cut:].clone(), g[cut:].clone()]
    small_states = hk.adam8_states([n - cut])
    first = [p[:FIRST].clone(), g[:FIRST].clone()]
    first_states = hk.adam8_states([FIRST])
    hyper = (1e-3, 0.9, 0.99, 1e-8, 0.01, 0.1, 0.01)
    plans = [hk.Adam8Plan([p], [g], *states), hk.Adam8Plan([small[0]], [small[1]], *small_states),
             hk.Adam8Plan([first[0]], [first[1]], *first_states)]
    for plan in plans:
        plan.step(*hyper)
    print("step", flush=True)

    def same(whole, a, b):
        return torch.equal(whole[:a.numel()], a) and torch.equal(whole[-b.numel():], b)

    assert same(p, first[0], small[0])
    for t, a, b in zip(states, first_states, small_states):
        assert same(t, a, b)
    for plan in plans:
        plan.close()
    del p, g, plans, plan
    torch.cuda.empty_cache()
    m, v = torch.empty(n, device=DEV), torch.empty(n, device=DEV)
    hk.adam8_dequantize(*states, m_out=m, v_out=v)
    print("dequantize", flush=True)
    rest = hk.adam8_dequantize(*small_states, m_out=torch.empty(n - cut, device=DEV),
                               v_out=torch.empty(n - cut, device=DEV))
    head = hk.adam8_dequantize(*first_states)
    assert same(m, head[0], rest[0]) and same(v, head[1], rest[1])
    again = hk.adam8_quantize(m, v)
    print("quantize", flush=True)
    # what codes stand for has the same codes again
    assert all(torch.equal(a, b) for a, b in zip(again, states))
