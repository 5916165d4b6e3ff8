"""Operators of a transformer block's training step whose speed is measured: the linear layer whose
product applies bias, activation and residual itself, with its backward product; the norms of queries
and keys with the position rotation, forward and backward; and the AdamW step whose states are held in
8 bits. Each in its plain form (elementary torch operations) and, where `own` is true, through the
public entry points of hyperkernels_amd.

Sizes are those of this repository's benchmark and configurations (a 124M-parameter model of width 768
in 12 heads of 64, a context of 1024, a batch of 8192 tokens, an 1280 -> 5120 linear layer) and generic
small, odd and ragged ones. `draw` spreads sizes over the same ranges.

The operators, from their formulas:

  linear       z = x W + b,  y = act(z) + r;  z is kept in 16 bits for the backward pass where asked.
  linear_grad  dz = (dy W^T) act'(z),  db = the column sums of dz before it is rounded.
  qk           per token and head: n = x rsqrt(mean(x^2) + eps) w, then each pair of its first `rot`
               elements turned by its angle, whose cosine and sine come from a table row chosen by the
               token's position. Backward: gradients of x and, summed over tokens and heads, of w.
  adam8        AdamW over many tensors; m and v in blocks of 256 elements, each block with one fp32
               scale: m stands for scale c |c| / 127^2 (c of -127 .. 127), v for scale (c / 255)^4
               (c of 0 .. 255). After the update the scale of m is the largest |m| of the block (that of
               v the largest v) in fp32, and each code the one whose value is nearest (a v > 0 keeps at
               least code 1). The step uses m and v before they are rounded to codes.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF = torch.bfloat16
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 256  # elements of one block of 8-bit states
# lr, beta1, beta2, eps, weight decay, and the step that the bias corrections are of
ADAM = dict(lr=3e-4, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)
STEP = 10
QK_EPS = 1e-6


def listed():
    return [
        # One token through the first half of a feed-forward block, as in decoding: the weights are
        # read once, and the launch counts.
        {"name": "linear_one_token", "kind": "linear", "tokens": 1, "n_in": 1280, "n_out": 5120,
         "act": "gelu", "residual": False, "preact": False, "trans_w": False},
        # The projection behind the attention of a small batch, added to the residual stream.
        {"name": "linear_residual", "kind": "linear", "tokens": 512, "n_in": 768, "n_out": 768,
         "act": "none", "residual": True, "preact": False, "trans_w": False},
        # The first half of the feed-forward block in a training step: GELU in the product's
        # epilogue, its input kept for the backward pass.
        {"name": "linear_gelu", "kind": "linear", "tokens": 8192, "n_in": 1280, "n_out": 5120,
         "act": "gelu", "residual": False, "preact": True, "trans_w": False},
        # Odd sizes everywhere: rows of every alignment, the weights stored by output.
        {"name": "linear_ragged", "kind": "linear", "tokens": 1021, "n_in": 1001, "n_out": 1537,
         "act": "relu", "residual": True, "preact": False, "trans_w": True},
        # The backward product through the second half of the feed-forward block of the same step.
        {"name": "linear_grad", "kind": "linear_grad", "tokens": 8192, "n_in": 1280, "n_out": 5120,
         "act": "gelu", "trans_w": True},
        # The same of a small last batch.
        {"name": "linear_grad_small", "kind": "linear_grad", "tokens": 333, "n_in": 768,
         "n_out": 2304, "act": "silu", "trans_w": False},
        # Decoding: the new token of each of 16 sequences, at positions of their own.
        {"name": "qk_one_token", "kind": "qk", "B": 16, "T": 1, "q_heads": 12, "k_heads": 12,
         "d": 64, "rot": 64, "interleaved": False, "dtype": "bf16", "f32_out": True,
         "train": False, "positions": True, "table": 1024},
        # The benchmark's batch in mixed precision: a 16-bit projection in, fp32 queries and keys out
        # for the attention, and the fp32 gradients that it returns.
        {"name": "qk_train", "kind": "qk", "B": 8, "T": 1024, "q_heads": 12, "k_heads": 12,
         "d": 64, "rot": 64, "interleaved": False, "dtype": "bf16", "f32_out": True,
         "train": True, "positions": False, "table": 1024},
        # Keys shared by groups of queries, half of each head rotated, a ragged length.
        {"name": "qk_grouped", "kind": "qk", "B": 3, "T": 333, "q_heads": 16, "k_heads": 4,
         "d": 128, "rot": 64, "interleaved": True, "dtype": "f16", "f32_out": False,
         "train": True, "positions": True, "table": 2048},
        # The optimizer step of a small model: few, odd tensors.
        {"name": "adam8_small", "kind": "adam8", "tensors": 20, "scale": 0.011, "grad": "f32",
         "copy": False},
        # One step over the 148 tensors of the 124M-parameter model.
        {"name": "adam8", "kind": "adam8", "tensors": 148, "scale": 1.0, "grad": "f32",
         "copy": False},
        # The same of a smaller model in mixed precision: 16-bit gradients in, and a 16-bit copy of
        # the parameters out for the next forward pass.
        {"name": "adam8_mixed", "kind": "adam8", "tensors": 74, "scale": 0.43, "grad": "bf16",
         "copy": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A feature size: a multiple of 64 usually, any number sometimes."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.3 else max(64, n // 64 * 64)


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear_grad", "linear_grad", "qk", "qk", "adam8"])
    if kind in ("linear", "linear_grad"):
        c = {"kind": kind, "tokens": 1 if rng.random() < 0.1 else _log_int(rng, 2, 8192),
             "n_in": _width(rng, 64, 4096), "n_out": _width(rng, 64, 5120),
             "act": rng.choice(["none", "relu", "gelu", "silu"]), "trans_w": rng.random() < 0.5}
        most = 8192 * 1280 * 5120
        c["tokens"] = max(1, min(c["tokens"], most // (c["n_in"] * c["n_out"])))
        if kind == "linear":
            c |= {"residual": rng.random() < 0.5, "preact": rng.random() < 0.5}
        return c
    if kind == "qk":
        d = rng.choice([32, 64, 64, 80, 96, 128, 128, 2 * rng.randint(8, 64)])
        H = rng.choice([4, 8, 12, 16])
        train = rng.random() < 0.7
        T = _log_int(rng, 1, 2048)
        most = 8 * 1024 * 12 * 64 // (T * H * d)
        table = 2048 if rng.random() < 0.7 else 8192
        return {"kind": kind, "B": max(1, min(16, _log_int(rng, 1, max(1.01, most)))), "T": T,
                "q_heads": H, "k_heads": rng.choice([1, H // 4, H // 2, H, H]), "d": d,
                "rot": d if rng.random() < 0.6 else 2 * rng.randint(1, d // 2),
                "interleaved": rng.random() < 0.4, "dtype": rng.choice(["f32", "bf16", "f16"]),
                "f32_out": rng.random() < 0.5, "train": train,
                "positions": rng.random() < 0.5, "table": table}
    return {"kind": kind, "tensors": rng.randint(2, 148),
            "scale": math.exp(rng.uniform(math.log(0.005), math.log(0.9))),
            "grad": rng.choice(["f32", "bf16", "f16"]), "copy": rng.random() < 0.5}


# ---- inputs --------------------------------------------------------------------------------------
class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed))

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=self.g, device=DEV) * std).to(dtype)

    def uniform(self, *shape, lo=0.0, hi=1.0, dtype=torch.float32):
        return (torch.rand(*shape, generator=self.g, device=DEV) * (hi - lo) + lo).to(dtype)


def _param_sizes(case):
    """The parameter tensors of a decoder of width 768, 12 layers and 50257 words; a smaller model has
    evenly chosen ones of them, each a fraction of its size (odd lengths among them)."""
    C = 768
    layer = [C, C, 3 * C * C, 3 * C, C * C, C, C, C, 4 * C * C, 4 * C, 4 * C * C, C]
    sizes = [50257 * C, 1024 * C] + 12 * layer + [C, C]
    n = case["tensors"]
    if n == len(sizes) and case["scale"] == 1.0:
        return sizes
    return [max(1, int(sizes[i * len(sizes) // n] * case["scale"])) for i in range(n)]


def _spans(case):
    """(start, size) of each tensor in one flat buffer, each from a block's first element on, and the
    buffer's length."""
    spans, total = [], 0
    for n in _param_sizes(case):
        spans.append((total, n))
        total += -(-n // BLOCK) * BLOCK
    return spans, total


def _inputs(case, seed):
    r = _Rand(seed)
    k = case["kind"]
    if k in ("linear", "linear_grad"):
        M, I, O = case["tokens"], case["n_in"], case["n_out"]
        w = r.normal(*((O, I) if case["trans_w"] else (I, O)), std=I ** -0.5, dtype=BF)
        s = {"x": r.normal(M, I, dtype=BF), "w": w}
        if k == "linear":
            s["b"] = r.normal(O, std=0.1, dtype=BF)
            s["r"] = r.normal(M, O, dtype=BF) if case["residual"] else None
            s["y"] = torch.empty(M, O, device=DEV, dtype=BF)
        else:
            s["z"] = r.normal(M, O, dtype=BF)
        return s
    if k == "qk":
        B, T, Hq, Hk, d, rot = (case[n] for n in ("B", "T", "q_heads", "k_heads", "d", "rot"))
        dt = DTYPES[case["dtype"]]
        out = torch.float32 if case["f32_out"] else dt
        # queries, keys and values as one projection leaves them, viewed by head
        qkv = r.normal(B, T, Hq + 2 * Hk, d, dtype=dt)
        angle = (torch.arange(case["table"], device=DEV, dtype=torch.float64)[:, None]
                 * 10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot))
        s = {"q": qkv[:, :, :Hq].transpose(1, 2), "k": qkv[:, :, Hq:Hq + Hk].transpose(1, 2),
             "cos": angle.cos().float(), "sin": angle.sin().float(),
             "wq": r.uniform(d, lo=0.5, hi=1.5, dtype=dt),
             "wk": r.uniform(d, lo=0.5, hi=1.5, dtype=dt), "positions": None}
        if case["positions"] or T > case["table"]:
            s["positions"] = torch.randint(0, case["table"], (B, T), generator=r.g, device=DEV)
        if case["train"]:
            s["dq"] = r.normal(B, Hq, T, d, dtype=out)
            s["dk"] = r.normal(B, Hk, T, d, dtype=out)
        else:
            s["q_out"] = torch.empty(B, Hq, T, d, device=DEV, dtype=out)
            s["k_out"] = torch.empty(B, Hk, T, d, device=DEV, dtype=out)
        return s
    spans, total = _spans(case)
    keep = torch.zeros(total, device=DEV, dtype=torch.bool)
    for a, n in spans:
        keep[a:a + n] = True
    m = r.normal(total, std=1e-3).masked_fill_(~keep, 0).view(-1, BLOCK)
    v = r.uniform(total, lo=1e-7, hi=1e-4).masked_fill_(~keep, 0).view(-1, BLOCK)
    ms, vs = m.abs().amax(1), v.amax(1)
    # codes such as an earlier step left them
    mc = ((m.abs() / ms[:, None]).sqrt_().mul_(127).round_() * m.sign()).to(torch.int8)
    vc = (v / vs[:, None]).sqrt_().sqrt_().mul_(255).round_().to(torch.uint8)
    dt = DTYPES[case["grad"]]
    return {"p": r.normal(total, std=0.02).masked_fill_(~keep, 0),
            "g": r.normal(total, std=1e-2).masked_fill_(~keep, 0).to(dt),
            "copy": torch.zeros(total, device=DEV, dtype=BF) if case["copy"] else None,
            "m": mc.view(-1), "v": vc.view(-1), "m_scale": ms, "v_scale": vs}


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    if case["kind"] == "adam8" and own:
        # the plan that a program builds once for its parameters
        from hyperkernels_amd import kernels as hk
        views = lambda t: None if t is None else [t[a:a + n] for a, n in _spans(case)[0]]  # noqa: E731
        s["plan"] = hk.Adam8Plan(views(s["p"]), views(s["g"]), s["m"], s["v"], s["m_scale"],
                                 s["v_scale"], copies=views(s["copy"]))
    return s


# ---- one pass ------------------------------------------------------------------------------------
def _bias_corrections():
    return 1 - ADAM["beta1"] ** STEP, 1 - ADAM["beta2"] ** STEP


def _run_own(s):
    from hyperkernels_amd import kernels as hk
    case = s["case"]
    k = case["kind"]
    if k == "linear":
        z = torch.empty_like(s["y"]) if case["preact"] else None
        y = hk.bgemm_act(s["x"], s["w"], bias=s["b"], activation=case["act"], residual=s["r"],
                         preact=z, out=s["y"], trans_b=case["trans_w"])
        return {"y": y, "z": z}
    if k == "linear_grad":
        db = torch.empty(case["n_out"], device=DEV)
        dz = hk.bgemm_act_backward(s["x"], s["w"], preact=s["z"], activation=case["act"], dbias=db,
                                   accumulate=False, trans_b=case["trans_w"])
        return {"dz": dz, "db": db}
    if k == "qk":
        shared = dict(cos=s["cos"], sin=s["sin"], positions=s["positions"], q_weight=s["wq"],
                      k_weight=s["wk"], eps=QK_EPS, interleaved=case["interleaved"])
        if not case["train"]:
            q, kk = hk.qk_norm_rope_forward(s["q"], s["k"], q_out=s["q_out"], k_out=s["k_out"],
                                            **shared)
            return {"q": q, "k": kk}
        q, kk = hk.qk_norm_rope_forward(s["q"], s["k"], out_dtype=s["dq"].dtype, **shared)
        dw = torch.empty(2, case["d"], device=DEV)
        dq, dk = hk.qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], grad_q_weight=dw[0],
                                          grad_k_weight=dw[1], accumulate=False, **shared)
        return {"q": q, "k": kk, "dq": dq, "dk": dk, "dw": dw}
    a = ADAM
    s["plan"].step(a["lr"], a["beta1"], a["beta2"], a["eps"], a["weight_decay"],
                   *_bias_corrections())
    m, v = hk.adam8_dequantize(s["m"], s["v"], s["m_scale"], s["v_scale"])
    return {"p": s["p"], "copy": s["copy"], "m": m, "v": v}


# The plain forms.
_C0, _C1 = math.sqrt(2 / math.pi), 0.044715


def _act(z, name):
    if name == "relu":
        return z.clamp_min(0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.tanh(_C0 * (z + _C1 * z * z * z)))
    return z * torch.sigmoid(z) if name == "silu" else z


def _act_grad(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        t = torch.tanh(_C0 * (z + _C1 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * _C0 * (1 + 3 * _C1 * z * z)
    if name == "silu":
        t = torch.sigmoid(z)
        return t * (1 + z * (1 - t))
    return torch.ones_like(z)


def _turned(x, cos, sin, interleaved):
    """x [B, H, T, d] with its first 2 cos.shape[-1] elements turned, pair by pair."""
    h = cos.shape[-1]
    a, b = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if interleaved else (x[..., :h], x[..., h:2 * h])
    a, b = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([y, x[..., 2 * h:]], -1)


def _qk_plain(x, w, cos, sin, dy, interleaved, out):
    """(y, dx, dw) of one of queries and keys; the last two None without a gradient dy."""
    x, w = x.float(), w.float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + QK_EPS)
    n = x * r
    y = _turned(n * w, cos, sin, interleaved).to(out)
    if dy is None:
        return y, None, None
    g = _turned(dy.float(), cos, -sin, interleaved)  # back by the same angles
    gw = g * w
    dx = r * (gw - n * (gw * n).mean(-1, keepdim=True))
    return y, dx, (g * n).sum((0, 1, 2))


def _nearest(ratio, values, lowest):
    """The index of the value that is nearest to each ratio, `lowest` at least where it is over 0."""
    borders = (values[1:] + values[:-1]) / 2
    code = torch.bucketize(ratio, borders, right=True)
    return torch.where(ratio > 0, code.clamp_min(lowest), code)


def _adam8_plain(s):
    # in 64 bits: a value next to the border between two codes has to fall on the right side
    a = {n: float(torch.tensor(x, dtype=torch.float32)) for n, x in ADAM.items()}
    bc1, bc2 = _bias_corrections()
    p, g = s["p"].view(-1, BLOCK), s["g"].view(-1, BLOCK).double()
    steps_m = torch.arange(128, device=DEV, dtype=torch.float64).square() / 127 ** 2
    steps_v = (torch.arange(256, device=DEV, dtype=torch.float64) / 255) ** 4

    c = s["m"].view(-1, BLOCK).double()
    m = c * c.abs() * (s["m_scale"].double() / 127 ** 2)[:, None]
    m = a["beta1"] * m + (1 - a["beta1"]) * g
    del c
    v = steps_v[s["v"].view(-1, BLOCK).long()] * s["v_scale"].double()[:, None]
    v = a["beta2"] * v + (1 - a["beta2"]) * g * g
    del g
    update = (m / bc1) / ((v / bc2).sqrt() + a["eps"])
    p.copy_(p.double() - a["lr"] * (update + a["weight_decay"] * p.double()))
    del update
    if s["copy"] is not None:
        s["copy"].copy_(s["p"])

    s["m_scale"].copy_(m.abs().amax(1))
    s["v_scale"].copy_(v.amax(1))
    ms, vs = s["m_scale"].double()[:, None], s["v_scale"].double()[:, None]
    code = _nearest(torch.where(ms > 0, m.abs() / ms, 0.0), steps_m, 0)
    s["m"].view(-1, BLOCK).copy_(code * m.sign())
    m_out = (steps_m[code] * m.sign() * ms).float()
    del m
    code = _nearest(torch.where(vs > 0, v / vs, 0.0), steps_v, 1)
    s["v"].view(-1, BLOCK).copy_(code)
    v_out = (steps_v[code] * vs).float()
    return {"p": s["p"], "copy": s["copy"], "m": m_out.view(-1), "v": v_out.view(-1)}


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    k = case["kind"]
    if k in ("linear", "linear_grad"):
        w = s["w"].float()
        z = torch.mm(s["x"].float(), w.t() if case["trans_w"] else w)
        if k == "linear":
            z += s["b"].float()
            y = _act(z, case["act"])
            y = y + s["r"].float() if case["residual"] else y
            return {"y": s["y"].copy_(y), "z": z.to(BF) if case["preact"] else None}
        dz = z * _act_grad(s["z"].float(), case["act"])
        return {"dz": dz.to(BF), "db": dz.sum(0)}
    if k == "qk":
        at = slice(case["T"]) if s["positions"] is None else s["positions"]
        cos, sin = s["cos"][at], s["sin"][at]
        if s["positions"] is not None:
            cos, sin = cos[:, None], sin[:, None]
        out = s["dq"].dtype if case["train"] else s["q_out"].dtype
        q, dq, dwq = _qk_plain(s["q"], s["wq"], cos, sin, s.get("dq"), case["interleaved"], out)
        kk, dk, dwk = _qk_plain(s["k"], s["wk"], cos, sin, s.get("dk"), case["interleaved"], out)
        if not case["train"]:
            return {"q": s["q_out"].copy_(q), "k": s["k_out"].copy_(kk)}
        dt = s["q"].dtype
        return {"q": q, "k": kk, "dq": dq.to(dt), "dk": dk.to(dt), "dw": torch.stack([dwq, dwk])}
    return _adam8_plain(s)


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    k = case["kind"]
    if k in ("linear", "linear_grad"):
        M, I, O = case["tokens"], case["n_in"], case["n_out"]
        outputs = 2 if k == "linear_grad" else 1 + case["residual"] + case["preact"]
        return {"bytes": 2 * (M * I + I * O + M * O * outputs) + (2 if k == "linear" else 4) * O,
                "flops": 2 * M * I * O + 20 * M * O}
    if k == "qk":
        B, T, d, rot = case["B"], case["T"], case["d"], case["rot"]
        n = B * T * (case["q_heads"] + case["k_heads"]) * d
        e = 4 if case["dtype"] == "f32" else 2
        o = 4 if case["f32_out"] else e
        rows = B * T if case["positions"] else T
        table = min(rows, case["table"]) * rot * 4 + (8 * rows if case["positions"] else 0)
        train = case["train"]
        return {"bytes": n * (2 if train else 1) * (e + o) + table + 2 * d * (e + 4 * train),
                "flops": n * (24 if train else 8)}
    n = sum(_param_sizes(case))
    g = 4 if case["grad"] == "f32" else 2
    # p, its gradient and the codes in; p, the codes and the values of m and v out
    return {"bytes": n * (8 + g + 4 + 8 + 2 * case["copy"]) + 16 * (n // BLOCK), "flops": 40 * n}


# ---- the same in 64 bits, from the definitions ----------------------------------------------------
def _exact_linear(case, s):
    x, w = s["x"].double(), s["w"].double()
    z = torch.mm(x, w.t().contiguous()) if case["trans_w"] else torch.mm(x, w)
    name = case["act"]
    if case["kind"] == "linear":
        z = z + s["b"].double()
        u = z * (1.5957691216057308 * (1 + 0.044715 * z * z))  # twice tanh's argument
        y = {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, 0.0),
             "gelu": lambda: z / (1 + torch.exp(-u)), "silu": lambda: z / (1 + torch.exp(-z))}[name]()
        return {"y": y + s["r"].double() if case["residual"] else y,
                "z": z if case["preact"] else None}
    h = s["z"].double()
    if name == "gelu":
        f = 1 / (1 + torch.exp(-h * (1.5957691216057308 * (1 + 0.044715 * h * h))))
        z *= f + h * f * (1 - f) * 1.5957691216057308 * (1 + 0.134145 * h * h)
    elif name == "silu":
        f = 1 / (1 + torch.exp(-h))
        z *= f + h * f * (1 - f)
    elif name == "relu":
        z = torch.where(h > 0, z, 0.0)
    return {"dz": z, "db": z.sum(0)}


def _exact_qk(case, s):
    rot, d = case["rot"], case["d"]
    pos = s["positions"]
    if pos is None:
        pos = torch.arange(case["T"], device=DEV).expand(case["B"], -1)
    # one complex factor a pair; the two elements of pair i
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None]
    i = torch.arange(rot // 2, device=DEV)
    one, two = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)

    def rotate(x, by):
        c = torch.complex(x[..., one], x[..., two]) * by
        y = x.clone()
        y[..., one], y[..., two] = c.real, c.imag
        return y

    out = {}
    for n, dw in (("q", "wq"), ("k", "wk")):
        x, w = s[n].double(), s[dw].double()
        norm = (x.pow(2).sum(-1, keepdim=True) / d + QK_EPS).sqrt()
        out[n] = rotate(x / norm * w, turn)
        if case["train"]:
            g = rotate(s["d" + n].double(), turn.conj())
            out["d" + n] = g * w / norm - x * (g * w * x).sum(-1, keepdim=True) / (d * norm ** 3)
            out[dw] = (g * x / norm).sum((0, 1, 2))
    if case["train"]:
        out["dw"] = torch.stack([out.pop("wq"), out.pop("wk")])
    return out


def _exact_adam8(s):
    b1, b2, lr, eps, wd = (float(torch.tensor(ADAM[n], dtype=torch.float32))
                           for n in ("beta1", "beta2", "lr", "eps", "weight_decay"))

    def value(code, scale, top, power):
        c = code.double().div_(top)
        return (c.abs().pow_(power) * c.sign()).view(-1, BLOCK).mul_(scale.double()[:, None])

    def held(x, top, power, least):
        """The values that the 8-bit codes of x stand for."""
        scale = x.abs().amax(1, keepdim=True).float().double()  # held in fp32
        r = torch.where(scale > 0, x.abs() / scale, 0.0)
        low = (r.pow(1 / power) * top).floor_().clamp_(0, top - 1)  # the two codes beside r
        a, b = (low / top) ** power, ((low + 1) / top) ** power
        c = torch.where(r - a < b - r, low, low + 1)
        c = torch.where(r > 0, c.clamp_min_(least), c)
        return ((c / top) ** power * scale * x.sign()).view(-1)

    g = s["g"].double().view(-1, BLOCK)
    m = value(s["m"], s["m_scale"], 127, 2).mul_(b1).add_(g * (1 - b1))
    v = value(s["v"], s["v_scale"], 255, 4).mul_(b2).add_(g.square_() * (1 - b2))
    p = s["p"].double().view(-1, BLOCK)
    bc1, bc2 = _bias_corrections()
    p = (p * (1 - lr * wd) - lr / bc1 * m / ((v / bc2).sqrt() + eps)).view(-1)
    return {"p": p, "copy": None if s["copy"] is None else p, "m": held(m, 127, 2, 0),
            "v": held(v, 255, 4, 1)}


def exact(case, seed):
    s = _inputs(case, seed)
    k = case["kind"]
    if k == "qk":
        return _exact_qk(case, s)
    return _exact_adam8(s) if k == "adam8" else _exact_linear(case, s)
