"""Tensors of more than 2^31 elements through the GEMM with an epilogue, the query/key norms and the 8-bit AdamW:
what lies behind the 32-bit offsets, against 64 bits or a small call on the same data.

Tolerances count roundings as in test_gpu_bgemm_act.py and test_gpu_qk_norm_rope.py."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16
ULP, HALF_STEP = 2.0 ** -24, 2.0 ** -8


def _normal(gen, *shape, dtype=BF):
    return torch.empty(*shape, device=DEV, dtype=dtype).normal_(generator=gen)


def _gen(seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return gen


def test_gemm_with_an_epilogue(hk):
    M, N, K = 66000, 33000, 64
    assert M * N > 2 ** 31
    gen = _gen(1)
    x, w, b = _normal(gen, M, K), _normal(gen, K, N), _normal(gen, N)
    r, z = _normal(gen, M, N), torch.empty(M, N, device=DEV, dtype=BF)
    y = hk.bgemm_act(x, w, bias=b, activation="relu", residual=r, preact=z)
    print("forward", flush=True)
    rows, cols = slice(M - 70, M), slice(N - 70, N)
    prod = x[rows].double() @ w[:, cols].double()
    mag = x[rows].double().abs() @ w[:, cols].double().abs() + b[cols].double().abs()
    want = prod + b[cols].double()
    tol = (K + 4) * ULP * mag
    assert bool(((z[rows, cols].double() - want).abs() <= tol + HALF_STEP * want.abs()).all())
    want = want.clamp_min(0) + r[rows, cols].double()
    err = (y[rows, cols].double() - want).abs()
    assert bool((err <= tol + ULP * want.abs() + HALF_STEP * want.abs() + 1e-37).all())
    del y, r
    db = torch.empty(N, device=DEV)
    d = hk.bgemm_act_backward(x, w, preact=z, activation="relu", dbias=db, accumulate=False)
    print("backward", flush=True)
    want = x.double() @ w[:, cols].double() * (z[:, cols] > 0)
    tol = (K + 4) * ULP * (x.double().abs() @ w[:, cols].double().abs())
    assert bool(((d[:, cols].double() - want).abs() <= tol + HALF_STEP * want.abs()).all())
    tol = tol.sum(0) + (48 + M / 128) * ULP * want.abs().sum(0)
    assert bool(((db[cols].double() - want.sum(0)).abs() <= tol).all())


def test_query_and_key_norms(hk):
    B, T, H, d = 2, 70000, 120, 128
    assert B * T * H * d > 2 ** 31
    gen = _gen(2)
    q = _normal(gen, B, T, H, d).transpose(1, 2)
    ang = torch.randn(T, d // 2, generator=gen, device=DEV)
    cos, sin = ang.cos(), ang.sin()
    y = hk._by_token(q)
    hk.qk_norm_rope_forward(q, None, cos, sin, q_out=y)
    print("forward", flush=True)
    part = (slice(B - 1, B), slice(0, H), slice(T - 5, T))

    def pairs(t):
        t = t[part].double()
        return t[..., :d // 2], t[..., d // 2:]

    c, s = cos[T - 5:].double(), sin[T - 5:].double()
    x = q[part].double()
    r = (x.square().mean(-1, keepdim=True) + 1e-6) ** -0.5
    a, b = (t * r for t in pairs(q))
    want = torch.cat([a * c - b * s, b * c + a * s], -1)
    tol = torch.cat([a.abs() + b.abs()] * 2, -1) * 24 * ULP + HALF_STEP * want.abs()
    assert bool(((y[part].double() - want).abs() <= tol).all())
    # y as the gradient of the outputs, its own as the gradient of q: in place
    g = torch.cat([pairs(y)[0] * c + pairs(y)[1] * s, pairs(y)[1] * c - pairs(y)[0] * s], -1)
    ga = torch.cat([pairs(y)[0].abs() + pairs(y)[1].abs()] * 2, -1)
    n = x * r
    want = r * (g - n * (g * n).mean(-1, keepdim=True))
    tol = ULP * r * (24 * ga + 64 * n.abs() * (ga * n.abs()).mean(-1, keepdim=True)) + HALF_STEP * want.abs()
    hk.qk_norm_rope_backward(y, None, q, None, cos, sin, dq=y)
    print("backward", flush=True)
    assert bool(((y[part].double() - want).abs() <= tol).all())


def test_8_bit_adamw(hk):
    n, cut = 2 ** 31 + 300, 2 ** 31 - 512
    gen = _gen(3)
    p, g = _normal(gen, n, dtype=torch.float32), _normal(gen, n)
    copy = torch.empty(n, device=DEV, dtype=BF)
    states = hk.adam8_states([n])
    small = [t[cut:].clone() for t in (p, g, copy)]
    small_states = hk.adam8_states([n - cut])
    hyper = (1e-3, 0.9, 0.99, 1e-8, 0.01, 0.1, 0.01)
    whole = hk.Adam8Plan([p], [g], *states, copies=[copy])
    part = hk.Adam8Plan([small[0]], [small[1]], *small_states, copies=[small[2]])
    for _ in range(2):
        whole.step(*hyper)
        part.step(*hyper)
    print("steps", flush=True)
    assert torch.equal(p[cut:], small[0]) and torch.equal(copy[cut:], small[2])
    for a, b in zip(states, small_states):
        assert torch.equal(a[-b.numel():], b)
    m, v = hk.adam8_dequantize(*states, m_out=torch.empty(n, device=DEV), v_out=torch.empty(n, device=DEV))
    rest = hk.adam8_dequantize(*small_states, m_out=torch.empty(n - cut, device=DEV),
                               v_out=torch.empty(n - cut, device=DEV))
    assert torch.equal(m[cut:], rest[0]) and torch.equal(v[cut:], rest[1])
