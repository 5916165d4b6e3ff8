"""8-bit AdamW at the ends of fp32's range, against the definition in 64 bits: blocks with scales whose reciprocal
fp32 does not hold, or whose sum, and squares of gradients that fp32 does not hold.

The codes and scales have to be the definition's own; the parameters' tolerance is test_gpu_adam8.py's."""
from __future__ import annotations

import numpy as np
import pytest
import torch
from test_gpu_adam8 import BLOCK, DEV, HYPER, M_VALUES, V_VALUES, _decode, _encode, _split, _step

pytestmark = pytest.mark.gpu


def _quantized(hk, m, v):
    state = hk.adam8_quantize(*(torch.from_numpy(a.reshape(-1)).to(DEV) for a in (m, v)))
    return state, _split(state, [m.size])[0]


@pytest.mark.parametrize("m_scale,v_scale", [(1e38, 1.0), (1.0, 1e38), (3.4e38, 1e-3), (1e-3, 3.4e38),
                                             (9e37, 9e37), (1.0, 2.0 ** 126), (2.0 ** 126, 1.0)])
def test_codes_of_large_scales(hk, m_scale, v_scale):
    """Every code's own value, and values beside the borders, in blocks whose largest is near fp32's."""
    print("adam8 scales", m_scale, v_scale, flush=True)
    rng = np.random.default_rng(int(np.log2(m_scale) * 7 + np.log2(v_scale)) + 1000)
    edges = (V_VALUES[1:] + V_VALUES[:-1]) / 2
    m = np.stack([np.resize(M_VALUES, BLOCK), rng.uniform(0, 1, BLOCK), np.resize(M_VALUES[::-1], BLOCK)])
    v = np.stack([V_VALUES, np.append(edges, 1.0) * (1 + 2.0 ** -20), rng.uniform(0, 1, BLOCK) ** 4])
    m[:, 0] = v[:, 0] = 1.0  # the scale
    m[:, 1::2] *= -1
    m, v = (m * m_scale).astype(np.float32), (v * v_scale).astype(np.float32)
    state, got = _quantized(hk, m, v)
    want = _encode(m.astype(np.float64), v.astype(np.float64))
    for a, b in zip(got, want):
        assert np.array_equal(a, b)
    mo, vo = hk.adam8_dequantize(*state)
    wm, wv = _decode(*want)
    assert np.allclose(mo.cpu().numpy().reshape(m.shape), wm, rtol=2.0 ** -23, atol=1e-44)
    assert np.allclose(vo.cpu().numpy().reshape(m.shape), wv, rtol=2.0 ** -23, atol=1e-44)


def test_finite_scales_whose_sum_is_not(hk):
    rng = np.random.default_rng(3)
    m = (rng.uniform(-1, 1, (2, BLOCK)) * 3e38).astype(np.float32)
    v = (rng.uniform(0, 1, (2, BLOCK)) * 3e38).astype(np.float32)
    m[1, 5] = np.inf  # this block only
    _, got = _quantized(hk, m, v)
    want = _encode(m[:1].astype(np.float64), v[:1].astype(np.float64))
    for a, b in zip(got, want):
        assert np.array_equal(a[:1], b)
    assert np.isnan(got[2][1]) and np.isnan(got[3][1])


@pytest.mark.parametrize("size", [5e19, 5.5e19])
def test_steps_of_large_gradients(hk, size):
    """v past 2^126, finite: three steps, the last with an ordinary gradient."""
    rng = np.random.default_rng(5)
    n = 2 * BLOCK + 77
    p = rng.normal(0, 0.02, n).astype(np.float32)
    g = torch.zeros(n, device=DEV)
    dev = torch.from_numpy(p).to(DEV)
    state = hk.adam8_states([n], DEV)
    plan = hk.Adam8Plan([dev], [g], *state)
    for step in (1, 2, 3):
        x = (rng.normal(0, 0.25, n).clip(-1, 1) * (size if step < 3 else 1e-2)).astype(np.float32)
        if step < 3:
            x[::97] = np.float32(size) * 0.99
        g.copy_(torch.from_numpy(x))
        before, old = dev.cpu().numpy(), _split(state, [n])[0]
        plan.step(HYPER["lr"], HYPER["beta1"], HYPER["beta2"], HYPER["eps"], HYPER["weight_decay"],
                  1 - HYPER["beta1"] ** step, 1 - HYPER["beta2"] ** step)
        want, s, tol = _step(before, x, old, step)
        assert np.isfinite(want).all() and np.isfinite(s[3]).all() and (step > 1 or s[3].max() > 2.0 ** 126)
        for a, b in zip(_split(state, [n])[0], s):
            assert np.array_equal(a, b), step
        assert (np.abs(dev.cpu().numpy() - want) <= tol).all(), step


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-20, 1e-12])
@pytest.mark.parametrize("grad", ["f32", "bf16"])
def test_steps_of_gradients_whose_squares_fp32_does_not_hold(hk, eps, grad):
    """Subnormal v, and v that fp32 rounds to 0, under an eps that does not hide them."""
    h = dict(HYPER, eps=eps)
    rng = np.random.default_rng(9)
    n = 3 * BLOCK + 5
    p = rng.normal(0, 0.02, n).astype(np.float32)
    g = torch.zeros(n, device=DEV, dtype=torch.float32 if grad == "f32" else torch.bfloat16)
    dev = torch.from_numpy(p).to(DEV)
    state = hk.adam8_states([n], DEV)
    plan = hk.Adam8Plan([dev], [g], *state)
    for step in (1, 2):
        sign = np.where(rng.random(n) < 0.5, -1.0, 1.0)
        # squares of 1e-60 .. 1e-36; fp32 holds 1e-45, whole digits from 1e-38 on
        x = sign * 10.0 ** rng.uniform(-30, -18, n)
        g.copy_(torch.from_numpy(x.astype(np.float32)))
        before, old = dev.cpu().numpy(), _split(state, [n])[0]
        plan.step(h["lr"], h["beta1"], h["beta2"], eps, h["weight_decay"], 1 - h["beta1"] ** step,
                  1 - h["beta2"] ** step)
        want, s, tol = _step(before, g.float().cpu().numpy(), old, step, h)
        assert np.isfinite(want).all()
        for a, b in zip(_split(state, [n])[0], s):
            assert np.array_equal(a, b), step
        assert (np.abs(dev.cpu().numpy() - want) <= tol).all(), step
