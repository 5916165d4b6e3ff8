"""Operands that are parts of one buffer and lie in and out of each other without sharing an element: the same bits as
from tensors of their own, and nothing beside the outputs written."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


def _gen(seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return gen


@pytest.mark.parametrize("M,N,K", [(70, 72, 64), (1, 72, 64), (300, 65, 33)])
@pytest.mark.parametrize("batch", [None, 3])
def test_gemm_in_one_buffer(hk, M, N, K, batch):
    """Input, residual, pre-activation and output as columns of one buffer, its batches row by row."""
    n, gen = batch or 1, _gen(1)
    width = 3 * N + K + 5
    buf = torch.randn(M, n, width, generator=gen, device=DEV).to(BF)
    at = [0, N, 2 * N, 2 * N + K]
    r, y, x, z = (buf[:, :, a:a + (K if a == 2 * N else N)].transpose(0, 1) for a in at)
    if batch is None:
        r, y, x, z = (t[0] for t in (r, y, x, z))
    w = torch.randn(*((n,) if batch else ()), K, N, generator=gen, device=DEV).to(BF)
    b = torch.randn(N, generator=gen, device=DEV).to(BF)
    before = buf.clone()
    own = [t.contiguous() for t in (x, r)]
    pre = torch.empty_like(own[1])
    want = hk.bgemm_act(own[0], w, bias=b, activation="gelu", residual=own[1], preact=pre)
    hk.bgemm_act(x, w, bias=b, activation="gelu", residual=r, preact=z, out=y)
    # the two take other stores, and row kernels or tiles of the same sums: the same roundings
    assert torch.equal(y, want) and torch.equal(z, pre)
    y.copy_(r)
    hk.bgemm_act(x, w, bias=b, activation="gelu", residual=y, out=y)
    assert torch.equal(y, want)
    db = torch.zeros(2, N, device=DEV)
    want = hk.bgemm_act_backward(own[0], w, preact=pre, activation="gelu", dbias=db[0])
    hk.bgemm_act_backward(x, w, preact=z, activation="gelu", dbias=db[1], out=y)
    assert torch.equal(y, want)
    # sums of the same values in two orders, chains of at most 48 + rows / 128 additions; want is rounded to bf16
    size = want.double().abs().reshape(-1, N).sum(0) * (1 + 2.0 ** -8)
    assert bool(((db[0] - db[1]).abs() <= 2 * (48 + M * n / 128) * 2.0 ** -24 * size).all())
    hk.bgemm_act_backward(x, w, preact=z, activation="gelu", out=z)
    assert torch.equal(z, want)
    for a in (0, 2 * N):
        assert torch.equal(buf[:, :, a:a + N if a == 0 else a + K], before[:, :, a:a + N if a == 0 else a + K])
    assert torch.equal(buf[:, :, 3 * N + K:], before[:, :, 3 * N + K:])


@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("H,K,d,rot", [(4, 4, 64, 64), (6, 2, 70, 50), (4, 1, 33, 32)])
def test_queries_and_keys_of_one_projection(hk, dtype, H, K, d, rot):
    """q, k and v as the projection has them: turned in place, and gradients into a buffer like it or in place."""
    B, T, gen = 2, 37, _gen(2)
    heads = (slice(0, H), slice(H, H + K), slice(H + K, H + 2 * K))

    def packed():
        buf = torch.randn(B, T, H + 2 * K, d, generator=gen, device=DEV).to(dtype)
        return buf, *(buf[:, :, h].transpose(1, 2) for h in heads)

    ang = torch.randn(T, rot // 2, generator=gen, device=DEV)
    cs = (ang.cos(), ang.sin())
    w = (torch.rand(2, d, generator=gen, device=DEV) + 0.5).to(dtype)
    kw = dict(q_weight=w[0], k_weight=w[1])
    buf, q, k, v = packed()
    grad, gq, gk, _ = packed()
    keep = [t.clone() for t in (q, k, v, gq, gk)]
    want = hk.qk_norm_rope_forward(q, k, *cs, **kw)
    dw = torch.zeros(4, d, device=DEV)
    dwant = hk.qk_norm_rope_backward(gq, gk, q, k, *cs, grad_q_weight=dw[0], grad_k_weight=dw[1], **kw)
    # into the parts of another projection's gradient, and over the gradients and the inputs themselves
    dbuf, dq, dk, dv = packed()
    held = dv.clone()
    hk.qk_norm_rope_backward(gq, gk, q, k, *cs, grad_q_weight=dw[2], grad_k_weight=dw[3], dq=dq, dk=dk, **kw)
    assert torch.equal(dq, dwant[0]) and torch.equal(dk, dwant[1]) and torch.equal(dv, held)
    assert torch.equal(dw[:2], dw[2:])
    hk.qk_norm_rope_backward(gq, gk, q, k, *cs, dq=gq, dk=gk, **kw)
    assert torch.equal(gq, dwant[0]) and torch.equal(gk, dwant[1])
    gq.copy_(keep[3]), gk.copy_(keep[4])
    hk.qk_norm_rope_forward(q, k, *cs, q_out=q, k_out=k, **kw)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, keep[2])
    q.copy_(keep[0]), k.copy_(keep[1])
    hk.qk_norm_rope_backward(gq, gk, q, k, *cs, dq=q, dk=k, **kw)
    assert torch.equal(q, dwant[0]) and torch.equal(k, dwant[1]) and torch.equal(v, keep[2])
