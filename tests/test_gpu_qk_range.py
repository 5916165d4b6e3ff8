"""Query/key norms of rows whose squares leave fp32's range: the formulas hold for every finite row.

Tolerances are test_gpu_qk_norm_rope.py's: the rows are turned by powers of two, which round nothing."""
from __future__ import annotations

import pytest
import torch
from test_gpu_qk_norm_rope import DEV, TYPES, _close, _reference, _table

pytestmark = pytest.mark.gpu

# sizes of the rows, whose mean squares are 1e-68 .. 1e-40 (fp32 holds whole digits from 1e-38 on), ordinary,
# and 1e40 .. 1e74 (fp32 ends at 3e38)
SMALL = (1e-34, 1e-28, 3e-23, 1e-20, 1e-19, 1e-12, 1.0)
LARGE = (1.0, 1e12, 1.5e19, 1e20, 1e30, 1e37)


@pytest.mark.parametrize("io", ["f32", "bf16", "bf16-f32"])
@pytest.mark.parametrize("d,rot,inter", [(64, 64, False), (128, 32, True), (63, 62, False), (256, 2, False),
                                         (70, 64, True), (32, 0, False)])
@pytest.mark.parametrize("sizes,eps", [(SMALL, 0.0), (SMALL, 1e-40), (LARGE, 1e-6), (LARGE, 0.0)])
def test_rows_of_any_size(hk, d, rot, inter, io, sizes, eps):
    print("qk range", d, rot, inter, io, sizes[0], eps, flush=True)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(d + rot)
    dt, out = TYPES[io.split("-")[0]], TYPES[io.split("-")[-1]]
    eps = float(torch.tensor(eps))  # as the call takes it
    B, H, T = 2, 3, 2 * len(sizes)
    size = torch.tensor(sizes * 2, device=DEV)[:, None]
    q = (torch.randn(B, H, T, d, generator=gen, device=DEV).clamp(-3, 3) * size).to(dt)
    # gradients of dx ~ 1
    dy = (torch.randn(B, H, T, d, generator=gen, device=DEV) * size.clamp(1e-18, 1e18)).to(out)
    w = (torch.rand(d, generator=gen, device=DEV) + 0.5).to(dt)
    cos, sin = _table(T, rot) if rot else (None, None)
    kw = dict(cos=cos, sin=sin, q_weight=w, eps=eps, interleaved=inter)
    y, _ = hk.qk_norm_rope_forward(q, None, out_dtype=out, **kw)
    gw = torch.zeros(d, device=DEV)
    dq, _ = hk.qk_norm_rope_backward(dy, None, q, None, grad_q_weight=gw, **kw)
    ry, ty, rx, tx, rw, tw = _reference(q, w, cos, sin, None, rot, inter, eps, dy)
    _close(y, ry, ty, "y")
    _close(dq, rx, tx, "dq")
    _close(gw, rw, tw, "dw")
