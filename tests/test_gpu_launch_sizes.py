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
