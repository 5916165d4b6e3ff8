"""RMS norm of query and key heads with the position rotation (qk_norm_rope.hip) against the formulas in
64 bits, and its gradients against differences too.

Tolerances count roundings of 2^-24: the sum of squares adds at most 22 numbers in a chain, half of
which reaches r, with the reciprocal root (2) and two products; the weight, the rotation's product and
sum make it 24 of |a| + |b| for an output pair (a, b), before the rounding of 16-bit outputs. The
gradients' are counted beside them."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
ULP = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def say(*a):
    print(*a, flush=True)


def _half_step(t, x):
    """Half a step of a 16-bit type at |x| (fp32: nothing beside the counted roundings)."""
    if t == torch.float32:
        return torch.zeros_like(x)
    return x.abs() * torch.finfo(t).eps / 2 + torch.finfo(t).smallest_normal * torch.finfo(t).eps


def _pairs(x, rot, interleaved):
    h = rot // 2
    return (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :h], x[..., h:rot])


def _join(a, b, rest, interleaved):
    y = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([y, rest], -1)


def _rotate(x, c, s, rot, interleaved):
    a, b = _pairs(x, rot, interleaved)
    return _join(a * c - b * s, b * c + a * s, x[..., rot:], interleaved)


def _spread(x, rot, interleaved):
    """|a| + |b| of each element's pair, |x| behind the rotated part."""
    a, b = (t.abs() for t in _pairs(x, rot, interleaved))
    return _join(a + b, a + b, x[..., rot:].abs(), interleaved)


def _reference(x, w, cos, sin, pos, rot, interleaved, eps, dy=None):
    """(y, tol, dx, tol, dw, tol) in 64 bits on the CPU."""
    x = x.double().cpu()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double().cpu()
    B, H, T, d = x.shape
    if rot:
        pos = torch.arange(T).expand(B, T) if pos is None else pos.cpu().expand(B, T)
        c, s = (t.double().cpu()[pos][:, None] for t in (cos, sin))
    else:
        c = s = torch.zeros(B, 1, T, 0, dtype=torch.float64)
    r = (x.square().mean(-1, keepdim=True) + eps) ** -0.5
    n = x * r
    y = _rotate(n * w, c, s, rot, interleaved)
    tol = 24 * ULP * _spread(n * w, rot, interleaved)
    if dy is None:
        return y, tol
    dy = dy.double().cpu()
    g = _rotate(dy, c, -s, rot, interleaved)
    ga = _spread(dy, rot, interleaved)
    gw = g * w
    dx = r * (gw - n * (gw * n).mean(-1, keepdim=True))
    # g w: 3 roundings of |dy|'s spread, w, r and the difference; the mean: the chain of 22, its
    # factors (8), r twice (15 each)
    dx_tol = ULP * r * (24 * ga * w.abs() + 64 * n.abs() * (ga * w.abs() * n.abs()).mean(-1, keepdim=True))
    dw = (g * n).sum((0, 1, 2))
    # n and g (20), and the longest chain of additions: rows of a lane group, butterfly, workgroups
    dw_tol = 128 * ULP * (ga * n.abs()).sum((0, 1, 2))
    return y, tol, dx, dx_tol, dw, dw_tol


def _table(rows, rot, pad=0):
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    a = torch.arange(rows, dtype=torch.float64)[:, None] * freq
    wide = lambda t: torch.nn.functional.pad(t.float(), (0, pad)).to(DEV)[:, :rot // 2]  # noqa: E731
    return wide(a.cos()), wide(a.sin())


def _heads(gen, B, H, T, d, dtype, layout, scale=1.0):
    """A [B, H, T, d] tensor: dense, by token, inside a wider buffer, or one element off alignment."""
    r = lambda *s: (torch.randn(*s, generator=gen, device=DEV) * scale).to(dtype)  # noqa: E731
    if layout == "dense":
        return r(B, H, T, d)
    if layout == "token":
        return r(B, T, H, d).transpose(1, 2)
    if layout == "wide":
        return r(B, T, H + 3, d + 5)[:, :, 1:H + 1, 2:d + 2].transpose(1, 2)
    return r(B * H * T * d + 1)[1:].view(B, H, T, d)


def _close(got, want, tol, what):
    err = (got.double().cpu() - want).abs()
    bad = err > tol + _half_step(got.dtype, want)
    assert not bool(bad.any()), (what, float((err / (tol + 1e-300)).max()), int(bad.sum()))


CASES = [
    # d, rot, interleaved, q heads, k heads, B, T, positions, layout
    (64, 64, False, 12, 12, 2, 37, False, "token"),
    (64, 64, True, 12, 4, 2, 37, True, "wide"),
    (128, 64, False, 16, 2, 1, 65, True, "dense"),
    (128, 128, True, 3, 1, 3, 19, False, "odd"),
    (80, 80, False, 5, 5, 2, 33, True, "token"),
    (96, 48, True, 4, 2, 2, 21, False, "wide"),
    (256, 256, False, 2, 1, 1, 17, True, "dense"),
    (256, 2, True, 2, 3, 1, 9, False, "odd"),
    (255, 254, False, 2, 1, 2, 11, True, "token"),
    (130, 130, True, 1, 2, 1, 13, False, "dense"),
    (34, 10, False, 3, 3, 2, 7, True, "wide"),
    (63, 62, True, 3, 1, 1, 5, False, "odd"),
    (72, 24, False, 2, 2, 1, 40, True, "token"),
    (64, 0, False, 4, 2, 2, 6, False, "token"),
    (33, 0, False, 4, 2, 2, 6, False, "dense"),
    (2, 2, False, 7, 1, 5, 3, True, "wide"),
    (1, 0, False, 3, 1, 1, 4, False, "dense"),
    (64, 64, False, 12, 12, 16, 1, True, "token"),
    (64, 64, False, 12, 1, 1, 700, False, "token"),
]


@pytest.mark.parametrize("io", ["f32", "bf16", "f16", "bf16-f32", "f16-f32"])
@pytest.mark.parametrize("d,rot,inter,Hq,Hk,B,T,use_pos,layout", CASES)
def test_forward_and_backward(hk, d, rot, inter, Hq, Hk, B, T, use_pos, layout, io):
    say("qk", d, rot, inter, Hq, Hk, B, T, use_pos, layout, io)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(d * 1000 + rot + T)
    dt = TYPES[io.split("-")[0]]
    out = TYPES[io.split("-")[-1]]
    q, k = _heads(gen, B, Hq, T, d, dt, layout), _heads(gen, B, Hk, T, d, dt, layout, 3.0)
    dq, dk = _heads(gen, B, Hq, T, d, out, layout), _heads(gen, B, Hk, T, d, out, "dense", 1e-3)
    wq = (torch.rand(d, generator=gen, device=DEV) + 0.5).to(dt)
    wk = None if rot == 10 else (torch.randn(d, generator=gen, device=DEV)).to(dt)
    cos, sin = _table(T + 50, rot, pad=3) if rot else (None, None)
    pos = torch.randint(0, T + 50, (B, T), generator=gen, device=DEV) if use_pos else None
    args = dict(cos=cos, sin=sin, positions=pos, q_weight=wq, k_weight=wk, eps=1e-5,
                interleaved=inter)
    yq, yk = hk.qk_norm_rope_forward(q, k, out_dtype=out, **args)
    gw = torch.full((2, d), 0.25, device=DEV)
    gq, gk = hk.qk_norm_rope_backward(dq, dk, q, k, grad_q_weight=gw[0], grad_k_weight=gw[1], **args)
    set_w = torch.full((2, d), float("nan"), device=DEV)
    again = hk.qk_norm_rope_backward(dq, dk, q, k, grad_q_weight=set_w[0], grad_k_weight=set_w[1],
                                     accumulate=False, **args)
    assert torch.equal(again[0], gq) and torch.equal(again[1], gk)
    for x, w, y, dy, dx, g0, g1, n in ((q, wq, yq, dq, gq, gw[0], set_w[0], "q"),
                                       (k, wk, yk, dk, gk, gw[1], set_w[1], "k")):
        assert y.dtype == out and dx.dtype == dt
        ry, ty, rx, tx, rw, tw = _reference(x, w, cos, sin, pos, rot, inter, 1e-5, dy)
        _close(y, ry, ty, n)
        _close(dx, rx, tx, "d" + n)
        _close(g1, rw, tw, "dw" + n)
        _close(g0, rw + 0.25, tw + ULP * (rw.abs() + 0.25), "dw added " + n)


def test_table_rows_in_a_wider_buffer_do_not_leak(hk):
    """Only a call's own outputs are written, whatever lies between their rows."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(3)
    q = _heads(gen, 2, 3, 9, 64, torch.bfloat16, "wide")
    cos, sin = _table(9, 64)
    buf = torch.full((2, 9, 3 + 2, 64 + 7), 9.0, device=DEV)
    out = buf[:, :, 1:4, 3:67].transpose(1, 2)
    y, none = hk.qk_norm_rope_forward(q, None, cos, sin, q_out=out)
    assert none is None and y is out
    ry, ty = _reference(q, None, cos, sin, None, 64, False, 1e-6)
    _close(out, ry, ty, "q")
    out.fill_(9.0)
    assert bool((buf == 9.0).all())


@pytest.mark.parametrize("side", ["q", "k"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_in_place_and_one_side_alone(hk, side, dt):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(5)
    x = _heads(gen, 2, 5, 33, 96, TYPES[dt], "token")
    dy = _heads(gen, 2, 5, 33, 96, TYPES[dt], "token")
    w = torch.rand(96, generator=gen, device=DEV).to(TYPES[dt])
    cos, sin = _table(64, 32)
    pos = torch.randint(0, 64, (33,), generator=gen, device=DEV)
    one = lambda a, b=None: (a, b) if side == "q" else (b, a)  # noqa: E731
    kw = dict(cos=cos, sin=sin, positions=pos, **{f"{side}_weight": w})
    i = 0 if side == "q" else 1
    y = hk.qk_norm_rope_forward(*one(x), **kw)[i]
    g = torch.zeros(96, device=DEV)
    dx = hk.qk_norm_rope_backward(*one(dy), *one(x), **{f"grad_{side}_weight": g}, **kw)[i]
    no_w = hk.qk_norm_rope_backward(*one(dy), *one(x), **kw)[i]
    assert torch.equal(dx, no_w)
    ry, ty, rx, tx, rw, tw = _reference(x, w, cos, sin, pos, 32, False, 1e-6, dy)
    _close(y, ry, ty, "y")
    _close(dx, rx, tx, "dx")
    _close(g, rw, tw, "dw")
    x2, dy2 = x.clone(), dy.clone()
    hk.qk_norm_rope_backward(*one(dy2), *one(x), **{f"d{side}": dy2}, **kw)
    assert torch.equal(dy2, dx)
    hk.qk_norm_rope_backward(*one(dy), *one(x2), **{f"d{side}": x2}, **kw)
    assert torch.equal(x2, dx)
    x2 = x.clone()
    hk.qk_norm_rope_forward(*one(x2), **{f"{side}_out": x2}, **kw)
    assert torch.equal(x2, y)


@pytest.mark.parametrize("io", ["f32", "bf16", "f16-f32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 20), (64, 6), (70, 64), (66, 50), (90, 90), (17, 8), (22, 14),
                                   (256, 6), (250, 8), (10, 0), (9, 4), (127, 118)])
def test_parts_that_are_no_whole_vectors(hk, d, rot, inter, io):
    """Rotated parts and rests of every remainder; into a wider buffer, and in place."""
    say("qk parts", d, rot, inter, io)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(d * 300 + rot)
    dt, out = TYPES[io.split("-")[0]], TYPES[io.split("-")[-1]]
    B, H, T = 2, 3, 21
    q, dy = _heads(gen, B, H, T, d, dt, "wide"), _heads(gen, B, H, T, d, out, "token")
    w = torch.randn(d, generator=gen, device=DEV).to(dt)
    cos, sin = _table(T, rot, pad=1) if rot else (None, None)
    kw = dict(cos=cos, sin=sin, q_weight=w, interleaved=inter)
    buf = torch.full((B, T, H + 2, d + 7), 9.0, device=DEV, dtype=out)
    y = buf[:, :, 1:H + 1, 3:d + 3].transpose(1, 2)
    hk.qk_norm_rope_forward(q, None, q_out=y, **kw)
    gw = torch.zeros(d, device=DEV)
    dq, _ = hk.qk_norm_rope_backward(dy, None, q, None, grad_q_weight=gw, **kw)
    ry, ty, rx, tx, rw, tw = _reference(q, w, cos, sin, None, rot, inter, 1e-6, dy)
    _close(y, ry, ty, "y")
    _close(dq, rx, tx, "dq")
    _close(gw, rw, tw, "dw")
    if dt == out:
        q2 = q.clone()
        hk.qk_norm_rope_forward(q2, None, q_out=q2, **kw)
        assert torch.equal(q2, y)
        q2.copy_(q)
        hk.qk_norm_rope_backward(dy, None, q2, None, dq=q2, **kw)
        assert torch.equal(q2, dq)
        d2 = dy.clone()
        hk.qk_norm_rope_backward(d2, None, q, None, dq=d2, **kw)
        assert torch.equal(d2, dq)
    y.fill_(9.0)
    assert bool((buf == 9.0).all())


def test_positions_outside_the_table_give_nan_for_their_tokens(hk):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(7)
    q = _heads(gen, 1, 2, 6, 64, torch.float32, "token")
    cos, sin = _table(10, 32)
    pos = torch.tensor([[0, 9, 10, -1, 1 << 40, 3]], device=DEV)
    y, _ = hk.qk_norm_rope_forward(q, None, cos, sin, pos)
    ok = torch.tensor([True, True, False, False, False, True], device=DEV)
    assert bool(torch.isfinite(y[:, :, ok]).all()) and bool(torch.isnan(y[:, :, ~ok]).all())
    dx, _ = hk.qk_norm_rope_backward(y.clone().nan_to_num(), None, q, None, cos, sin, pos)
    assert bool(torch.isfinite(dx[:, :, ok]).all()) and bool(torch.isnan(dx[:, :, ~ok]).all())


def test_rows_of_zero_and_of_what_is_not_finite(hk):
    q = torch.zeros(1, 4, 1, 64, device=DEV)
    q[0, 1, 0, 5] = float("inf")
    q[0, 2, 0, 5] = float("nan")
    q[0, 3] = 1.0
    cos, sin = _table(4, 64)
    y, _ = hk.qk_norm_rope_forward(q, None, cos, sin)
    assert bool((y[0, 0] == 0).all()) and bool(torch.isnan(y[0, 2]).all())
    assert bool(torch.isnan(y[0, 1, 0, 5])) and bool(torch.isfinite(y[0, 3]).all())
    dx, _ = hk.qk_norm_rope_backward(torch.ones_like(q), None, q, None, cos, sin)
    ry, ty, rx, tx, _, _ = _reference(q[:, :1], None, cos, sin, None, 64, False, 1e-6,
                                      torch.ones_like(q[:, :1]))
    _close(dx[:, :1], rx, tx, "dx of zeros")


@pytest.mark.parametrize("B,T,Hq,Hk", [(0, 5, 2, 1), (2, 0, 2, 1), (2, 5, 0, 0)])
def test_empty(hk, B, T, Hq, Hk):
    q, k = torch.zeros(B, Hq, T, 64, device=DEV), torch.zeros(B, Hk, T, 64, device=DEV)
    cos, sin = _table(8, 64)
    yq, yk = hk.qk_norm_rope_forward(q, k, cos, sin)
    assert yq.shape == q.shape and yk.shape == k.shape
    g = torch.full((2, 64), 3.0, device=DEV)
    hk.qk_norm_rope_backward(yq, yk, q, k, cos, sin, grad_q_weight=g[0], grad_k_weight=g[1])
    assert bool((g == 3).all())
    hk.qk_norm_rope_backward(yq, yk, q, k, cos, sin, grad_q_weight=g[0], grad_k_weight=g[1],
                             accumulate=False)
    # a side without heads has no gradient to write
    assert bool((g == (3 if Hq == 0 else 0)).all())


def test_gradients_against_differences(hk):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(9)
    q = _heads(gen, 1, 2, 3, 32, torch.float32, "token").contiguous()
    w = torch.rand(32, generator=gen, device=DEV) + 0.5
    cos, sin = _table(3, 32)
    dy = torch.randn(q.shape, generator=gen, device=DEV)
    f = lambda x, v: float((hk.qk_norm_rope_forward(  # noqa: E731
        x, None, cos, sin, q_weight=v)[0].double() * dy.double()).sum())
    gw = torch.zeros(32, device=DEV)
    dx, _ = hk.qk_norm_rope_backward(dy, None, q, None, cos, sin, q_weight=w, grad_q_weight=gw)
    h = 2.0 ** -7
    for seed in range(4):
        gen.manual_seed(100 + seed)
        u, z = torch.randn(q.shape, generator=gen, device=DEV), torch.randn(32, generator=gen, device=DEV)
        # central differences: h^2 / 6 of a third derivative (|u|^3 of order 1 an element) and the
        # outputs' 24 roundings over 2 h
        scale = float((dy.abs() * 4).sum())
        tol = scale * (h * h + 24 * ULP / h)
        assert abs((f(q + h * u, w) - f(q - h * u, w)) / (2 * h) - float((dx * u).sum())) <= tol
        assert abs((f(q, w + h * z) - f(q, w - h * z)) / (2 * h) - float((gw * z).sum())) <= tol


def test_large_enough_for_every_workgroup_and_repeatable(hk):
    """More rows than the backward pass has lane groups: the same bits twice, and on another stream."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(13)
    B, H, T, d = 4, 24, 1024, 128
    q = _heads(gen, B, H, T, d, torch.bfloat16, "token")
    dy = torch.randn(B, H, T, d, generator=gen, device=DEV)
    w = torch.rand(d, generator=gen, device=DEV).bfloat16()
    cos, sin = _table(T, d)
    g = torch.zeros(3, d, device=DEV)
    dx, _ = hk.qk_norm_rope_backward(dy, None, q, None, cos, sin, q_weight=w, grad_q_weight=g[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        d2, _ = hk.qk_norm_rope_backward(dy, None, q, None, cos, sin, q_weight=w, grad_q_weight=g[1])
    hk.qk_norm_rope_backward(dy, None, q, None, cos, sin, q_weight=w, grad_q_weight=g[2])
    torch.cuda.synchronize()
    assert torch.equal(g[0], g[1]) and torch.equal(g[0], g[2]) and torch.equal(dx, d2)
    x = q.double()
    n = x * (x.square().mean(-1, keepdim=True) + 1e-6) ** -0.5
    c, sn = cos.double(), sin.double()
    gg = _rotate(dy.double(), c, -sn, d, False)
    rows = B * H * T
    # the chain: rows / (1024 workgroups x 32 groups), 6 + 4 levels, 64 of the second kernel
    tol = (20 + rows / 32768 + 10 + 80) * ULP * (_spread(dy.double(), d, False) * n.abs()).sum((0, 1, 2))
    assert bool(((g[0].double() - (gg * n).sum((0, 1, 2))).abs() <= tol).all())


def test_captured_calls_replay_as_they_ran(hk):
    """Two graphs captured on one stream, replayed in turn with eager calls between them."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(17)
    cos, sin = _table(64, 64)
    s = torch.cuda.Stream()
    sets = []
    for T in (64, 40):
        q = _heads(gen, 2, 6, T, 64, torch.bfloat16, "token")
        dy = torch.randn(2, 6, T, 64, generator=gen, device=DEV)
        w = torch.rand(64, generator=gen, device=DEV).bfloat16()
        gw = torch.zeros(64, device=DEV)
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            y, _ = hk.qk_norm_rope_forward(q, None, cos, sin, q_weight=w, out_dtype=torch.float32)
            dx, _ = hk.qk_norm_rope_backward(dy, None, q, None, cos, sin, q_weight=w,
                                             grad_q_weight=gw, accumulate=False)
        sets.append((graph, q, dy, w, y, dx, gw))
    for _ in range(3):
        for graph, q, dy, w, y, dx, gw in sets:
            q.mul_(-0.5).add_(0.1)
            graph.replay()
        torch.cuda.synchronize()
        for graph, q, dy, w, y, dx, gw in sets:
            g2 = torch.zeros(64, device=DEV)
            y2, _ = hk.qk_norm_rope_forward(q, None, cos, sin, q_weight=w, out_dtype=torch.float32)
            d2, _ = hk.qk_norm_rope_backward(dy, None, q, None, cos, sin, q_weight=w,
                                             grad_q_weight=g2, accumulate=False)
            assert torch.equal(y, y2) and torch.equal(dx, d2) and torch.equal(gw, g2)


def test_library_workspace_where_none_is_passed(hk):
    """The C entry with no workspace: the stream's own, the same bits."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(19)
    q, dy = _heads(gen, 2, 6, 50, 64, torch.float32, "token"), torch.randn(2, 6, 50, 64, generator=gen, device=DEV)
    cos, sin = _table(50, 64)
    g = torch.zeros(2, 64, device=DEV)
    dx, _ = hk.qk_norm_rope_backward(dy, None, q, None, cos, sin, grad_q_weight=g[0], accumulate=False)
    d2 = torch.empty_like(dx)
    p = hk._qk_params("t", q, None, cos, sin, None, None, None, 1e-6, False, dy, None, True, d2, None,
                      g[1], None, False)
    assert hk.lib().hk_qk_norm_rope_workspace(p, 0) > 0
    hk.call("hk_qk_norm_rope_backward", p, 0, None, 0, hk._stream())
    assert torch.equal(dx, d2) and torch.equal(g[0], g[1])
    # one that is too small is refused
    small = torch.empty(4, device=DEV, dtype=torch.uint8)
    with pytest.raises(hk.HKError):
        hk.call("hk_qk_norm_rope_backward", p, 0, small.data_ptr(), 4, hk._stream())
