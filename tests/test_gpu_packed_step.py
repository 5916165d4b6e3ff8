"""One training step of a small model on packed sequences, as a program strings the kernels together - token and
position embeddings, LayerNorm, projection, query / key norms with rotation, packed attention with shared key heads,
projection onto the residual stream, logits by the tied table, log probabilities with an entropy bonus, and all the way
back to the table's gradient - against the same by autograd in 64 bits; then the same step captured and replayed."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
LENS, PAD = [37, 1, 90, 0, 64], 8  # sequences, and rows behind the last
N = sum(LENS)
H, HK, D = 4, 2, 32
C, V, STRIDE = H * D, 503, 512
EPS, QK_EPS, SCALE = 1e-5, 1e-6, 2.0


def _inputs(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s, std=1.0: torch.randn(*s, generator=g, device=DEV) * std  # noqa: E731
    w = {"wte": r(V, C, std=C ** -0.5), "wpe": r(128, C, std=0.5), "g1": 1 + r(C, std=0.1), "c1": r(C, std=0.1),
         "wqkv": r(C, (H + 2 * HK) * D, std=C ** -0.5), "qw": 1 + r(D, std=0.1), "kw": 1 + r(D, std=0.1),
         "wo": r(C, C, std=C ** -0.5)}
    w = {n: t.to(BF) for n, t in w.items()}
    rows = N + PAD
    tok = torch.randint(0, V, (rows,), generator=g, device=DEV)
    pos = torch.zeros(rows, device=DEV, dtype=torch.long)
    pos[:N] = torch.cat([torch.arange(n, device=DEV) for n in LENS])
    cu = torch.tensor([0] + list(torch.tensor(LENS).cumsum(0)), device=DEV, dtype=torch.int32)
    loss_g, loss_h = r(rows, std=0.1), r(rows, std=0.02)
    loss_g[N:] = 0  # rows behind the last sequence have no loss
    loss_h[N:] = 0
    return w, dict(tok=tok, pos=pos, cu=cu, next=torch.randint(0, V, (rows,), generator=g, device=DEV), g=loss_g,
                   h=loss_h)


def _angles():
    a = torch.arange(128, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    return a.cos(), a.sin()


def _step(hk, w, s):
    """{name: value} through the kernels."""
    cos, sin = (t.float() for t in _angles())
    rows = N + PAD
    e = hk.embedding_forward(w["wpe"], s["pos"])
    x = hk.embedding_forward(w["wte"], s["tok"], scale=SCALE, residual=e, out=e)
    n1, m1, r1 = hk.layer_norm_forward(x, w["g1"], w["c1"], EPS)
    qkv = hk.bgemm_act(n1, w["wqkv"]).view(rows, H + 2 * HK, D)
    rope = dict(cos=cos, sin=sin, positions=s["pos"], q_weight=w["qw"], k_weight=w["kw"], eps=QK_EPS)
    q0, k0 = (t.transpose(0, 1)[None] for t in (qkv[:, :H], qkv[:, H:H + HK]))
    q, k = (t[0].transpose(0, 1) for t in hk.qk_norm_rope_forward(q0, k0, **rope))
    v = qkv[:, H + HK:]
    o = torch.zeros(rows, H, D, device=DEV, dtype=BF)  # rows of no sequence are not written
    o, lse = hk.attn_packed_forward(q, k, v, s["cu"], o=o)
    x2 = hk.bgemm_act(o.view(rows, C), w["wo"], residual=x)
    logits = hk.bgemm_act(x2, w["wte"], trans_b=True,
                          out=torch.empty(rows, STRIDE, device=DEV, dtype=BF)[:, :V])
    p = hk.token_logprobs(logits, s["next"], entropy=True, top=3)
    # backward
    dlog = hk.token_logprobs_backward(logits, s["next"], p.lse, s["g"], p.entropy, s["h"], grad=logits)
    dx2 = hk.bgemm_act(dlog, w["wte"])
    dtable = hk.bgemm_act(dlog, x2, trans_a=True).float()
    dwo = hk.bgemm_act(o.view(rows, C), dx2, trans_a=True)
    do = hk.bgemm_act(dx2, w["wo"], trans_b=True).view(rows, H, D)
    dqkv = torch.zeros(rows, H + 2 * HK, D, device=DEV, dtype=BF)
    dq, dk = torch.zeros_like(q), torch.zeros_like(k)
    hk.attn_packed_backward(do, q, k, v, o, lse, s["cu"], dq=dq, dk=dk, dv=dqkv[:, H + HK:])
    dqw, dkw = torch.empty(D, device=DEV), torch.empty(D, device=DEV)
    hk.qk_norm_rope_backward(dq.transpose(0, 1)[None], dk.transpose(0, 1)[None], q0, k0, grad_q_weight=dqw,
                             grad_k_weight=dkw, accumulate=False, dq=dqkv[:, :H].transpose(0, 1)[None],
                             dk=dqkv[:, H:H + HK].transpose(0, 1)[None], **rope)
    dqkv = dqkv.view(rows, -1)
    dwqkv = hk.bgemm_act(n1, dqkv, trans_a=True)
    dg, dc = torch.zeros(C, device=DEV), torch.zeros(C, device=DEV)
    dx = hk.layer_norm_backward(hk.bgemm_act(dqkv, w["wqkv"], trans_b=True), x, m1, r1, w["g1"], dg, dc) + dx2
    hk.embedding_backward(dx, s["tok"], dtable, scale=SCALE)  # onto the logits' part
    dwpe = hk.embedding_backward(dx, s["pos"], torch.empty(128, C, device=DEV), accumulate=False)
    return {"logp": p.logp[:N], "entropy": p.entropy[:N], "top": p.top_logp[:N], "wte": dtable, "wpe": dwpe,
            "wqkv": dwqkv, "wo": dwo, "qw": dqw, "kw": dkw, "g1": dg, "c1": dc}


def _reference(w, s):
    w = {n: t.double().requires_grad_() for n, t in w.items()}
    cos, sin = _angles()
    pos = s["pos"][:N]
    x = SCALE * w["wte"][s["tok"][:N]] + w["wpe"][pos]
    m = x.mean(-1, keepdim=True)
    n1 = (x - m) * ((x - m).square().mean(-1, keepdim=True) + EPS) ** -0.5 * w["g1"] + w["c1"]
    qkv = (n1 @ w["wqkv"]).view(N, H + 2 * HK, D)

    def turned(t, weight):
        t = t * (t.square().mean(-1, keepdim=True) + QK_EPS) ** -0.5 * weight
        a, b, c, z = t[..., :D // 2], t[..., D // 2:], cos[pos][:, None], sin[pos][:, None]
        return torch.cat([a * c - b * z, b * c + a * z], -1)

    q, k, v = turned(qkv[:, :H], w["qw"]), turned(qkv[:, H:H + HK], w["kw"]), qkv[:, H + HK:]
    outs, a = [], 0
    for n in LENS:
        Q, K, U = (t[a:a + n].transpose(0, 1) for t in (q, k, v))
        K, U = K.repeat_interleave(H // HK, 0), U.repeat_interleave(H // HK, 0)
        z = Q @ K.transpose(1, 2) * D ** -0.5
        z = z.masked_fill(torch.ones(n, n, device=DEV, dtype=torch.bool).triu(1), float("-inf"))
        outs.append((torch.softmax(z, -1) @ U).transpose(0, 1))
        a += n
    x2 = torch.cat(outs).reshape(N, C) @ w["wo"] + x
    lp = torch.log_softmax(x2 @ w["wte"].t(), 1)
    logp = lp.gather(1, s["next"][:N, None])[:, 0]
    ent = -(lp.exp() * lp).sum(1)
    (logp * s["g"][:N] + ent * s["h"][:N]).sum().backward()
    return {"logp": logp.detach(), "entropy": ent.detach(), "top": lp.detach().topk(3, 1).values,
            **{n: t.grad for n, t in w.items()}}


def test_a_step_on_packed_sequences(hk):
    w, s = _inputs(5)
    got, want = _step(hk, w, s), _reference(w, s)
    # A value passes 8 bf16 roundings up to the logits (embedding, norm, projection, norm of heads, P, attention's
    # output, projection, logits) and 9 on its way back (of logits, dx2, dout, dS, dq, through the norm of heads, dn1,
    # dx, and the product with it), each at most 2^-8 of it and 2^-8 / sqrt(3) in the mean square, adding up like
    # independent ones: sqrt(17) 2^-8 / sqrt(3) = 9.3e-3; norms and both softmaxes can pass an error on up to twice.
    tol = 1.9e-2
    off = {n: float((got[n].double() - want[n]).norm() / want[n].norm()) for n in want}
    print("[case] packed step", {n: "%.1e" % v for n, v in off.items()}, flush=True)
    assert max(off.values()) <= tol, off
    untouched = torch.ones(128, device=DEV, dtype=torch.bool)
    untouched[s["pos"]] = False
    assert not got["wpe"][untouched].any()


def test_the_step_captured(hk):
    w, s = _inputs(6)
    _step(hk, w, s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(hk, w, s)
    for seed in (7, 8, 9):
        w2, s2 = _inputs(seed)
        for old, new in ((w, w2), (s, s2)):
            for n in old:
                old[n].copy_(new[n])
        want = _step(hk, w, s)
        graph.replay()
        torch.cuda.synchronize()
        for n in want:
            assert torch.equal(out[n], want[n]), (seed, n)


def test_front_ends_refuse(hk):
    q = torch.zeros(8, 4, 64, device=DEV, dtype=BF)
    k = torch.zeros(8, 3, 64, device=DEV, dtype=BF)
    cu = torch.tensor([0, 8], device=DEV, dtype=torch.int32)
    x, t = torch.zeros(4, 10, device=DEV), torch.zeros(4, device=DEV, dtype=torch.long)
    f = torch.zeros(4, device=DEV)
    lse = torch.zeros(4, 8, device=DEV)
    for call in (lambda: hk.attn_packed_forward(q, k, k, cu),  # 3 key heads for 4
                 lambda: hk.attn_packed_forward(q, q, q[:7], cu), lambda: hk.attn_packed_forward(q, q, q, cu.long()),
                 lambda: hk.attn_packed_forward(q, q, q, cu, cu[:1]), lambda: hk.attn_packed_forward(q, q, q.half(), cu),
                 lambda: hk.attn_packed_forward(q, q, q.transpose(1, 2), cu),
                 lambda: hk.attn_packed_forward(q[..., :60], q[..., :60], q[..., :60], cu),
                 lambda: hk.attn_packed_forward(q, q, q, cu, lse=lse[:3]),
                 lambda: hk.attn_packed_forward(q, q, q, cu[:0]), lambda: hk.attn_packed_forward(q, q, q, cu[None]),
                 lambda: hk.attn_packed_backward(q.half(), q, q, q, q, lse, cu),
                 lambda: hk.token_logprobs(x, t[:3]), lambda: hk.token_logprobs(x, t.float()),
                 lambda: hk.token_logprobs(x.t(), torch.zeros(10, device=DEV, dtype=torch.long)),
                 lambda: hk.token_logprobs(x, t, top=11), lambda: hk.token_logprobs(x, t, entropy=f.double()),
                 lambda: hk.token_logprobs(x, t, top_logp=x[:, :2]), lambda: hk.token_logprobs(x[:, :0], t),
                 lambda: hk.token_logprobs_backward(x, t, f, f, None, f),
                 lambda: hk.token_logprobs_backward(x, t, f, f, grad=x.bfloat16()),
                 lambda: hk.embedding_forward(x, t.float()), lambda: hk.embedding_forward(x, t, out=x[:3]),
                 lambda: hk.embedding_forward(x, t, residual=x.bfloat16()),
                 lambda: hk.embedding_backward(x, t, x[:, :9].contiguous()),
                 lambda: hk.embedding_backward(x, t[:2], x.clone())):
        with pytest.raises(ValueError):
            call()
    # what only the library sees
    for call in (lambda: hk.attn_packed_forward(q, q, q, cu, scale=-1.0), lambda: hk.attn_packed_forward(q, q, q, cu, o=q),
                 lambda: hk.attn_packed_forward(
                     torch.zeros(3000, device=DEV, dtype=BF).as_strided((8, 4, 64), (260, 65, 1)), q, q, cu),
                 lambda: hk.embedding_backward(x, t, x), lambda: hk.embedding_forward(x, t, out=x[:4]),
                 lambda: hk.token_logprobs(x, t, logp=x.view(-1)[:4])):
        with pytest.raises(hk.HKError):
            call()
