"""One training step of a transformer block through the kernels as a program strings them together -
LayerNorm, projection, query / key norms with rotation, attention, projection onto the residual stream,
feed-forward block, their backward passes, 8-bit AdamW with the bf16 weights of the next step - against
the same block by autograd in 64 bits, on the same bf16 weights."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
B, T, H, D = 2, 96, 2, 64
C, F = H * D, 5 * H * D
EPS, QK_EPS = 1e-5, 1e-6


def say(*a):
    print(*a, flush=True)


SHAPES = {"g1": (C,), "c1": (C,), "wqkv": (C, 3 * C), "bqkv": (3 * C,), "qw": (D,), "kw": (D,),
          "wo": (C, C), "bo": (C,), "g2": (C,), "c2": (C,), "w1": (C, F), "b1": (F,), "w2": (F, C),
          "b2": (C,)}


def _weights(gen):
    out = {}
    for n, s in SHAPES.items():
        t = torch.randn(*s, generator=gen, device=DEV)
        out[n] = 1 + 0.1 * t if n in ("g1", "g2", "qw", "kw") else 0.1 * t if len(s) == 1 else (
            t * s[0] ** -0.5)
    return out


def _reference(w, x, dy, cos, sin):
    """(y, gradients of x and of every weight) in 64 bits."""
    w = {n: t.double().requires_grad_() for n, t in w.items()}
    x = x.double().requires_grad_()

    def norm(t, g, c):
        m = t.mean(-1, keepdim=True)
        return (t - m) * ((t - m).square().mean(-1, keepdim=True) + EPS) ** -0.5 * g + c

    def turned(t, weight):
        t = t * (t.square().mean(-1, keepdim=True) + QK_EPS) ** -0.5 * weight
        a, b = t[..., :D // 2], t[..., D // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    qkv = (norm(x, w["g1"], w["c1"]) @ w["wqkv"] + w["bqkv"]).view(B, T, 3, H, D)
    q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    s = turned(q, w["qw"]) @ turned(k, w["kw"]).transpose(-1, -2) * D ** -0.5
    s = s.masked_fill(torch.ones(T, T, device=DEV, dtype=torch.bool).triu(1), float("-inf"))
    o = (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B * T, C)
    x2 = o @ w["wo"] + w["bo"] + x
    z = norm(x2, w["g2"], w["c2"]) @ w["w1"] + w["b1"]
    h = 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z ** 3)))
    y = h @ w["w2"] + w["b2"] + x2
    y.backward(dy.double())
    return y.detach(), x.grad, {n: t.grad for n, t in w.items()}


def _column_sums(hk, t):
    """fp32 sums over the rows of a bf16 gradient."""
    t = t.float().contiguous()
    n, c = t.shape
    return hk.unified_reduce_sum(t, hk.ReductionLayout(hk.REDUCE_OUTER, c, n, 0, c, c))


def _step(hk, w, x, dy, cos, sin):
    """(y, gradient of x, gradients of the weights) through the kernels."""
    g = {n: torch.zeros(*s, device=DEV) for n, s in SHAPES.items()}
    n1, m1, r1 = hk.layer_norm_forward(x, w["g1"], w["c1"], EPS)
    qkv = hk.bgemm_act(n1, w["wqkv"], bias=w["bqkv"]).view(B, T, 3, H, D)
    q0, k0, v0 = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    rope = dict(cos=cos, sin=sin, q_weight=w["qw"], k_weight=w["kw"], eps=QK_EPS)
    q, k = hk.qk_norm_rope_forward(q0, k0, out_dtype=torch.float32, **rope)
    v = v0.float()
    o, lse = hk.fused_attn_forward(q, k, v, True)
    ob = o.transpose(1, 2).reshape(B * T, C).to(BF)
    x2 = hk.bgemm_act(ob, w["wo"], bias=w["bo"], residual=x)
    n2, m2, r2 = hk.layer_norm_forward(x2, w["g2"], w["c2"], EPS)
    pre = torch.empty(B * T, F, device=DEV, dtype=BF)
    h = hk.bgemm_act(n2, w["w1"], bias=w["b1"], activation="gelu", preact=pre)
    y = hk.bgemm_act(h, w["w2"], bias=w["b2"], residual=x2)
    # backward
    g["b2"] = _column_sums(hk, dy)
    g["w2"] = hk.bgemm_act(h, dy, trans_a=True)
    dz = hk.bgemm_act_backward(dy, w["w2"], preact=pre, activation="gelu", dbias=g["b1"], trans_b=True)
    g["w1"] = hk.bgemm_act(n2, dz, trans_a=True)
    dn2 = hk.bgemm_act(dz, w["w1"], trans_b=True)
    dx2 = hk.layer_norm_backward(dn2, x2, m2, r2, w["g2"], g["g2"], g["c2"]) + dy
    g["bo"] = _column_sums(hk, dx2)
    g["wo"] = hk.bgemm_act(ob, dx2, trans_a=True)
    do = hk.bgemm_act(dx2, w["wo"], trans_b=True).view(B, T, H, D).transpose(1, 2).float()
    dq, dk, dv = hk.attn_backward(q, k, v, do, lse, hk.attn_bwd_precompute_D(do, o), True)
    dqkv = torch.empty(B, T, 3, H, D, device=DEV, dtype=BF)
    hk.qk_norm_rope_backward(dq, dk, q0, k0, grad_q_weight=g["qw"], grad_k_weight=g["kw"],
                             dq=dqkv[:, :, 0].transpose(1, 2), dk=dqkv[:, :, 1].transpose(1, 2),
                             **rope)
    dqkv[:, :, 2] = dv.transpose(1, 2)
    dqkv = dqkv.view(B * T, 3 * C)
    g["bqkv"] = _column_sums(hk, dqkv)
    g["wqkv"] = hk.bgemm_act(n1, dqkv, trans_a=True)
    dn1 = hk.bgemm_act(dqkv, w["wqkv"], trans_b=True)
    dx = hk.layer_norm_backward(dn1, x, m1, r1, w["g1"], g["g1"], g["c1"]) + dx2
    return y, dx, g


def _off(got, want):
    d = got.double() - want
    return float(d.norm() / want.norm())


def test_two_steps_of_a_block(hk):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(23)
    master = _weights(gen)
    x = torch.randn(B * T, C, generator=gen, device=DEV).to(BF)
    dy = (torch.randn(B * T, C, generator=gen, device=DEV) * 1e-2).to(BF)
    a = torch.arange(T, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    cos, sin = a.cos(), a.sin()
    copies = {n: t.to(BF) for n, t in master.items()}
    names = list(SHAPES)
    grads = {n: torch.zeros(*SHAPES[n], device=DEV, dtype=BF) for n in names}
    state = hk.adam8_states([master[n].numel() for n in names], DEV)
    plan = hk.Adam8Plan([master[n] for n in names], [grads[n] for n in names], *state,
                        copies=[copies[n] for n in names])
    for step in (1, 2):
        y, dx, g = _step(hk, copies, x, dy, cos.float(), sin.float())
        ry, rdx, rg = _reference(copies, x, dy, cos, sin)
        # A value passes at most 12 bf16 roundings on its way (norm, projection, attention's output,
        # projection, norm, hidden layer, output, and as many back for a gradient: 24), each at most
        # 2^-8 of it and 2^-8 / sqrt(3) in the mean square, and adding up like independent ones:
        # sqrt(24) 2^-8 / sqrt(3) = 1.1e-2 of the result's norm; the norms and the softmax can pass an
        # error on up to twice.
        tol = 2.2e-2
        off = {"y": _off(y, ry), "dx": _off(dx, rdx), **{n: _off(g[n], rg[n]) for n in names}}
        say("block step", step, {n: "%.1e" % v for n, v in off.items()})
        assert max(off.values()) <= tol, off
        before = {n: master[n].clone() for n in names}
        for n in names:
            grads[n].copy_(g[n])
        plan.step(1e-2, 0.9, 0.95, 1e-8, 0.01, 1 - 0.9 ** step, 1 - 0.95 ** step)
        for n in names:
            assert torch.equal(copies[n], master[n].to(BF)) and not torch.equal(before[n], master[n])
            if step == 1:
                # from zero moments every element steps lr against its gradient's sign
                move = (master[n] - before[n] * (1 - 1e-2 * 0.01)).double()
                some = grads[n] != 0
                want = -1e-2 * torch.sign(grads[n].double())
                # eps beside sqrt(v): relative eps / |g|; p's rounding; the fp32 constants
                tol_p = 1e-2 * (1e-8 / grads[n].double().abs().clamp_min(1e-30) + 2.0 ** -18) + (
                    before[n].abs() + 1) * 2.0 ** -22
                assert bool(((move - want).abs() <= tol_p)[some].all()), n
    m, v = hk.adam8_dequantize(*state)
    assert bool(torch.isfinite(m).all()) and bool((v >= 0).all())
