"""Operators of a model on packed sequences whose speed is measured: the lookup of its tokens' embeddings
and that table's gradient, causal attention in 16 bits over sequences of different lengths that lie one
behind the other (with heads that share keys, and its backward pass), and the log probabilities of given
tokens with the entropy and the likeliest alternatives, and their gradient. Each in its plain form
(elementary torch operations) and, where `own` is true, through the public entry points of hyperkernels_amd.

Sizes are those of this repository's benchmark and configurations (a vocabulary of 50257 in rows of 50304,
width 768 in 12 heads of 64, a batch of 8192 tokens, 16 query heads on 4 key heads of 128) and generic small,
odd and ragged ones. `draw` spreads sizes over the same ranges.

The operators, from their formulas:

  attn       sequence s has queries cu_q[s] .. cu_q[s + 1] and keys cu_k[s] .. cu_k[s + 1]; query i of m sees
             key j of n where j <= i + n - m (causal) or all n; head h of the queries goes with head
             h // (q_heads / k_heads) of the keys: o = softmax(scale q k^T) v, and the log of the softmax's
             denominator. A query that sees no key has o = 0 and -inf.
  attn_train the same and, from the gradient of o, those of q, k and v.
  logprobs   per row of logits: logp = x[token] - lse, the entropy -sum p log p, and the `top` largest log
             probabilities with their indices (of equal ones the lowest index first).
  logprobs_train  logp and entropy, and from the gradients of both that of the logits.
  embed      out = scale table[token] + residual.
  embed_grad grad_table[v] = scale times the sum of grad over the tokens that are v, for all v.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

# lengths of documents that fill a batch of 8192 tokens as a packer leaves them
PACKED = "1024,1024,713,311,1024,1000,24,517,390,117,1024,641,383"


def listed():
    return [
        # Four short turns of a chat that arrived together: the launch counts.
        {"name": "attn_turns", "kind": "attn", "lens": "17,1,64,33", "q_heads": 12, "k_heads": 12, "d": 64,
         "dtype": "bf16", "causal": True},
        # Decoding: the new token of each of 16 sequences over all of its keys, one row a head.
        {"name": "attn_decode", "kind": "attn", "q_heads": 16, "k_heads": 4, "d": 128,
         "lens": "1:4000,1:17,1:2048,1:1,1:999,1:3001,1:512,1:64,1:1500,1:2777,1:333,1:128,1:3500,1:720,"
                 "1:1024,1:2222", "dtype": "bf16", "causal": True},
        # One long prompt.
        {"name": "attn_prompt", "kind": "attn", "lens": "8192", "q_heads": 16, "k_heads": 4, "d": 128,
         "dtype": "bf16", "causal": True},
        # A training step of the 124M-parameter model over documents packed into its batch.
        {"name": "attn_train", "kind": "attn_train", "lens": PACKED, "q_heads": 12, "k_heads": 12, "d": 64,
         "dtype": "bf16", "causal": True},
        # Fewer, longer documents, keys shared by groups of queries.
        {"name": "attn_train_grouped", "kind": "attn_train", "lens": "2048,1001,333", "q_heads": 16,
         "k_heads": 4, "d": 128, "dtype": "f16", "causal": True},
        # What a server returns beside the sampled token of each of 16 sequences.
        {"name": "logprobs_decode", "kind": "logprobs", "rows": 16, "vocab": 50257, "stride": 50257,
         "dtype": "f32", "top": 20, "masked": False},
        # Scoring prompts: every token's log probability and the 5 likeliest others.
        {"name": "logprobs_prompt", "kind": "logprobs", "rows": 4096, "vocab": 50257, "stride": 50304,
         "dtype": "bf16", "top": 5, "masked": False},
        # A policy-gradient step with an entropy bonus over the benchmark's batch.
        {"name": "logprobs_train", "kind": "logprobs_train", "rows": 8192, "vocab": 50257, "stride": 50304,
         "dtype": "bf16", "masked": False},
        # The same of a small batch, rows of every alignment.
        {"name": "logprobs_train_odd", "kind": "logprobs_train", "rows": 333, "vocab": 8191, "stride": 8191,
         "dtype": "f16", "masked": True},
        # The batch's first activations: token rows of an fp32 table added to the positions' rows.
        {"name": "embed", "kind": "embed", "tokens": 8192, "vocab": 50257, "d": 768, "scale": 1.0,
         "dtype": "f32", "out": "bf16", "residual": True},
        # The table's gradient for the optimizer, all rows written.
        {"name": "embed_grad", "kind": "embed_grad", "tokens": 8192, "vocab": 50257, "d": 768, "scale": 1.0,
         "dtype": "bf16"},
        # The same of a small model, odd everywhere, with scaled embeddings.
        {"name": "embed_grad_small", "kind": "embed_grad", "tokens": 333, "vocab": 1009, "d": 131,
         "scale": 11.4, "dtype": "f32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn_train", "attn_train", "logprobs", "logprobs_train", "embed",
                       "embed_grad"])
    if kind in ("attn", "attn_train"):
        d = rng.choice([32, 64, 64, 64, 80, 96, 128, 128, 128, 8 * rng.randint(1, 16)])
        H = rng.choice([4, 8, 12, 16])
        Hk = rng.choice([1, H // 4, H // 2, H, H])
        n = _log_int(rng, 1, 64)
        decode = kind == "attn" and rng.random() < 0.3
        top = rng.choice([64, 512, 2048, 4096])
        most = 2 ** 32 // (H * d)  # pairs of a query and a key
        lens, pairs = [], 0
        for _ in range(n):
            q = k = _log_int(rng, 1 if lens else 16, top)
            if decode:  # a token, or a few drafted ones, over a longer cache
                q = min(k, rng.choice([1, 1, 1, 2, 5]))
            elif rng.random() < 0.15:  # a chunk of a prompt, or more queries than keys
                q = _log_int(rng, 1, top)
            elif lens and rng.random() < 0.05:  # a place in the batch that nothing fills
                q = k = 0
            if pairs + q * k > most and lens:
                break
            pairs += q * k
            lens.append(f"{q}:{k}" if q != k else str(q))
        return {"kind": kind, "lens": ",".join(lens), "q_heads": H, "k_heads": Hk, "d": d,
                "dtype": rng.choice(["bf16", "bf16", "f16"]), "causal": rng.random() < 0.85}
    if kind in ("logprobs", "logprobs_train"):
        vocab = _log_int(rng, 64, 131072)
        rows = min(_log_int(rng, 1, 8192), max(1, 2 ** 27 // vocab))
        c = {"kind": kind, "rows": rows, "vocab": vocab,
             "stride": vocab if rng.random() < 0.5 else -(-vocab // 64) * 64,
             "dtype": rng.choice(["f32", "bf16", "f16"]), "masked": rng.random() < 0.25}
        return c if kind == "logprobs_train" else c | {"top": rng.choice([0, 1, 5, 20, rng.randint(0, 64)])}
    d = _log_int(rng, 32, 4096)
    d = d if rng.random() < 0.3 else -(-d // 64) * 64
    vocab = min(_log_int(rng, 256, 131072), 2 ** 26 // d)
    c = {"kind": kind, "tokens": min(_log_int(rng, 1, 32768), 2 ** 25 // d), "vocab": vocab, "d": d,
         "scale": 1.0 if rng.random() < 0.5 else math.sqrt(d), "dtype": rng.choice(["f32", "bf16", "f16"])}
    if kind == "embed":
        c |= {"out": rng.choice([c["dtype"], "f32", "bf16"]), "residual": rng.random() < 0.5}
    return c


# ---- inputs --------------------------------------------------------------------------------------
class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed))

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=self.g, device=DEV) * std).to(dtype)

    def tokens(self, n, vocab):
        """Tokens as texts have them: the frequency of the i-th falls as 1 / (i + 1)."""
        u = torch.rand(n, generator=self.g, device=DEV, dtype=torch.float64)
        return ((vocab + 1.0) ** u - 1).long().clamp_(0, vocab - 1)


def _lens(case):
    pairs = [p.split(":") for p in case["lens"].split(",")]
    return [int(p[0]) for p in pairs], [int(p[-1]) for p in pairs]


def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _inputs(case, seed):
    r = _Rand(seed)
    k, dt = case["kind"], DTYPES[case["dtype"]]
    if k in ("attn", "attn_train"):
        lq, lk = _lens(case)
        H, Hk, d = case["q_heads"], case["k_heads"], case["d"]
        cu = lambda lens: torch.tensor(_starts(lens), device=DEV, dtype=torch.int32)  # noqa: E731
        s = {"cu_q": cu(lq), "cu_k": cu(lk)}
        if lq == lk:  # queries, keys and values as one projection leaves them
            qkv = r.normal(sum(lq), H + 2 * Hk, d, dtype=dt)
            s |= {"q": qkv[:, :H], "k": qkv[:, H:H + Hk], "v": qkv[:, H + Hk:]}
        else:
            s |= {"q": r.normal(sum(lq), H, d, dtype=dt), "k": r.normal(sum(lk), Hk, d, dtype=dt),
                  "v": r.normal(sum(lk), Hk, d, dtype=dt)}
        if k == "attn_train":
            s["do"] = r.normal(sum(lq), H, d, dtype=dt)
        return s
    if k in ("logprobs", "logprobs_train"):
        rows, vocab = case["rows"], case["vocab"]
        whole = r.normal(rows, case["stride"], std=2.5)
        x = whole[:, :vocab]
        t = r.tokens(rows, vocab)
        x[torch.arange(rows, device=DEV), t] += 6  # the model has learnt something
        if case["masked"]:  # what a grammar does not allow here
            off = torch.rand(rows, vocab, generator=r.g, device=DEV) < 0.3
            off[:, 0] = False
            x.masked_fill_(off, -math.inf)
        s = {"x": whole.to(dt)[:, :vocab], "t": t}
        if k == "logprobs_train":
            s["g"], s["h"] = r.normal(rows, std=1 / rows), r.normal(rows, std=0.01 / rows)
            # gradients in fp16 are scaled as its range asks
            if case["dtype"] == "f16":
                s["g"], s["h"] = s["g"] * 4096, s["h"] * 4096
            s["dx"] = torch.zeros_like(whole, dtype=dt)[:, :vocab]
        return s
    n, d = case["tokens"], case["d"]
    s = {"t": r.tokens(n, case["vocab"])}
    if k == "embed":
        s["table"] = r.normal(case["vocab"], d, std=0.02, dtype=dt)
        s["r"] = r.normal(n, d, std=0.02, dtype=DTYPES[case["out"]]) if case["residual"] else None
        s["out"] = torch.empty(n, d, device=DEV, dtype=DTYPES[case["out"]])
    else:
        s["g"] = r.normal(n, d, std=1e-2, dtype=dt)
        s["dtable"] = torch.empty(case["vocab"], d, device=DEV)
    return s


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


# ---- one pass ------------------------------------------------------------------------------------
def _run_own(s):
    from hyperkernels_amd import kernels as hk
    case = s["case"]
    k = case["kind"]
    if k in ("attn", "attn_train"):
        seqs = dict(cu_q=s["cu_q"], cu_k=s["cu_k"], causal=case["causal"])
        o, lse = hk.attn_packed_forward(s["q"], s["k"], s["v"], **seqs)
        if k == "attn":
            return {"o": o, "lse": lse}
        dq, dk, dv = hk.attn_packed_backward(s["do"], s["q"], s["k"], s["v"], o, lse, **seqs)
        return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    if k == "logprobs":
        p = hk.token_logprobs(s["x"], s["t"], entropy=True, top=case["top"])
        return {"logp": p.logp, "lse": p.lse, "entropy": p.entropy, "top": p.top_logp, "index": p.top_index}
    if k == "logprobs_train":
        p = hk.token_logprobs(s["x"], s["t"], entropy=True)
        dx = hk.token_logprobs_backward(s["x"], s["t"], p.lse, s["g"], p.entropy, s["h"], grad=s["dx"])
        return {"logp": p.logp, "entropy": p.entropy, "dx": dx}
    if k == "embed":
        return hk.embedding_forward(s["table"], s["t"], scale=case["scale"], residual=s["r"], out=s["out"])
    return hk.embedding_backward(s["g"], s["t"], s["dtable"], scale=case["scale"], accumulate=False)


# The plain forms.
def _visible(m, n, causal):
    """Whether query i of m sees key j of n."""
    if not causal:
        return torch.ones(m, n, device=DEV, dtype=torch.bool)
    i, j = torch.arange(m, device=DEV)[:, None], torch.arange(n, device=DEV)
    return j <= i + (n - m)


def _attn_plain(s):
    case = s["case"]
    lq, lk = _lens(case)
    H, Hk, d = case["q_heads"], case["k_heads"], case["d"]
    scale, dt, train = d ** -0.5, s["q"].dtype, case["kind"] == "attn_train"
    out = {"o": torch.zeros(sum(lq), H, d, device=DEV, dtype=dt),
           "lse": torch.full((H, sum(lq)), -math.inf, device=DEV)}
    if train:
        out |= {"dq": torch.zeros_like(out["o"])}
        out |= {n: torch.zeros(sum(lk), Hk, d, device=DEV, dtype=dt) for n in ("dk", "dv")}
    heads = lambda t: t.float().transpose(0, 1).contiguous()  # noqa: E731
    spread = lambda t: heads(t).repeat_interleave(H // Hk, 0)  # noqa: E731
    gather = lambda t: t.view(Hk, H // Hk, -1, d).sum(1).transpose(0, 1)  # noqa: E731
    for m, n, a, b in zip(lq, lk, _starts(lq), _starts(lk)):
        if m == 0 or n == 0:
            continue
        q, k, v = heads(s["q"][a:a + m]), spread(s["k"][b:b + n]), spread(s["v"][b:b + n])
        x = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(scale)
        x.masked_fill_(~_visible(m, n, case["causal"]), -math.inf)
        top = x.amax(2, keepdim=True)
        top = torch.where(top == -math.inf, 0.0, top)
        p = x.sub_(top).exp_()
        z = p.sum(2, keepdim=True)
        p /= torch.where(z == 0, 1.0, z)
        o = torch.matmul(p, v)
        out["o"][a:a + m] = o.transpose(0, 1)
        out["lse"][:, a:a + m] = (z.log() + top)[..., 0]
        if train:
            do = heads(s["do"][a:a + m])
            out["dv"][b:b + n] = gather(torch.matmul(p.transpose(1, 2).contiguous(), do))
            ds = torch.matmul(do, v.transpose(1, 2).contiguous())
            ds = ds.sub_((do * o).sum(2, keepdim=True)).mul_(p).mul_(scale)
            out["dq"][a:a + m] = torch.matmul(ds, k).transpose(0, 1)
            out["dk"][b:b + n] = gather(torch.matmul(ds.transpose(1, 2).contiguous(), q))
    return out


def _softmax_plain(x, t):
    """(logp of t, lse, entropy, log probabilities, probabilities) of fp32 rows."""
    m = x.amax(1, keepdim=True)
    y = x - m
    p = y.exp()
    z = p.sum(1, keepdim=True)
    p /= z
    y -= z.log()
    ent = -torch.where(p > 0, p * y, 0.0).sum(1)
    return y.gather(1, t[:, None])[:, 0], (m + z.log())[:, 0], ent, y, p


def _largest(x, n):
    """Indices of the n largest of each row, of equal ones the lowest index first."""
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, bits ^ 0x7fffffff, bits)  # ordered as the values are
    key = (key << 32) + torch.arange(x.shape[1] - 1, -1, -1, device=DEV)
    return key.topk(n, 1).indices


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    k = case["kind"]
    if k in ("attn", "attn_train"):
        return _attn_plain(s)
    if k in ("logprobs", "logprobs_train"):
        x = s["x"].float()
        logp, lse, ent, y, p = _softmax_plain(x, s["t"])
        if k == "logprobs":
            top = index = None
            if case["top"]:
                index = _largest(x, case["top"])
                top = y.gather(1, index)
            return {"logp": logp, "lse": lse, "entropy": ent, "top": top, "index": index}
        bonus = torch.where(p > 0, y + ent[:, None], 0.0).mul_(s["h"][:, None])
        dx = p.mul_(-(bonus.add_(s["g"][:, None])))
        dx.scatter_add_(1, s["t"][:, None], s["g"][:, None])
        return {"logp": logp, "entropy": ent, "dx": s["dx"].copy_(dx)}
    if k == "embed":
        y = s["table"][s["t"]].float() * case["scale"]
        return s["out"].copy_(y if s["r"] is None else y + s["r"].float())
    s["dtable"].zero_()
    return s["dtable"].index_add_(0, s["t"], s["g"].float() * case["scale"])


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    k, e = case["kind"], 4 if case["dtype"] == "f32" else 2
    if k in ("attn", "attn_train"):
        lq, lk = _lens(case)
        H, Hk, d = case["q_heads"], case["k_heads"], case["d"]
        pairs = 0
        for m, n in zip(lq, lk):
            first = max(1, n - m + 1) if case["causal"] else n  # keys of the first query that sees any
            rows = min(m, n) if case["causal"] else m
            pairs += rows * (first + n) // 2
        q, kv = 2 * sum(lq) * H * d, 2 * sum(lk) * Hk * d
        lse = 4 * sum(lq) * H
        if k == "attn":  # q, k, v in, o and lse out; two products
            return {"bytes": 2 * q + 2 * kv + lse, "flops": 4 * d * H * pairs}
        # and do in, dq, dk, dv out; five more products
        return {"bytes": 4 * q + 4 * kv + lse, "flops": 14 * d * H * pairs}
    if k in ("logprobs", "logprobs_train"):
        n = case["rows"] * case["vocab"]
        if k == "logprobs":
            return {"bytes": n * e + case["rows"] * (20 + 12 * case["top"]), "flops": 6 * n}
        return {"bytes": 2 * n * e + case["rows"] * 24, "flops": 14 * n}
    n, d, vocab = case["tokens"], case["d"], case["vocab"]
    if k == "embed":
        o = 4 if case["out"] == "f32" else 2
        # words fall as 1 / (i + 1): about this many different rows are read
        rows = sum(1 - (1 - 1 / ((i + 1) * math.log(vocab + 1))) ** n for i in range(vocab))
        return {"bytes": int(rows * d * e) + n * (8 + d * o * (1 + case["residual"])), "flops": 2 * n * d}
    return {"bytes": n * (8 + d * e) + vocab * d * 4, "flops": 2 * n * d}


# ---- the same in 64 bits, from the definitions ----------------------------------------------------
def _exact_attn(case, s):
    lq, lk = _lens(case)
    H, Hk, d = case["q_heads"], case["k_heads"], case["d"]
    train = case["kind"] == "attn_train"
    q, k, v = (s[n].double().requires_grad_(train) for n in ("q", "k", "v"))
    o = torch.zeros(sum(lq), H, d, device=DEV, dtype=torch.float64)
    lse = torch.full((H, sum(lq)), -math.inf, device=DEV, dtype=torch.float64)
    grads = [torch.zeros_like(t) for t in (q, k, v)] if train else []
    for i in range(len(lq)):
        qs, ks = slice(sum(lq[:i]), sum(lq[:i + 1])), slice(sum(lk[:i]), sum(lk[:i + 1]))
        m, n = lq[i], lk[i]
        if m == 0 or n == 0:
            continue
        # the last query is level with the last key
        off = torch.ones(m, n, device=DEV).triu(n - m + 1).bool() if case["causal"] else None
        some = max(0, m - n) if case["causal"] else 0  # queries before the first that sees a key
        for h in range(H):
            parts = [t.detach().clone().requires_grad_(train)
                     for t in (q[qs, h], k[ks, h * Hk // H], v[ks, h * Hk // H])]
            x = torch.mm(parts[0], parts[1].t()) / math.sqrt(d)
            x = x if off is None else x.masked_fill(off, -math.inf)
            x = x[some:]
            z = torch.logsumexp(x, 1)
            y = torch.mm(torch.exp(x - z[:, None]), parts[2])
            o[qs, h][some:] = y.detach()
            lse[h, qs][some:] = z.detach()
            if train:
                got = torch.autograd.grad(y, parts, s["do"][qs, h][some:].double())
                grads[0][qs, h] = got[0]
                grads[1][ks, h * Hk // H] += got[1]
                grads[2][ks, h * Hk // H] += got[2]
    out = {"o": o, "lse": lse}
    return out | dict(zip(("dq", "dk", "dv"), grads)) if train else out


def _exact_logprobs(case, s):
    train = case["kind"] == "logprobs_train"
    out = {n: [] for n in (("logp", "entropy", "dx") if train else ("logp", "lse", "entropy", "top", "index"))}
    step = max(1, 2 ** 26 // case["vocab"])
    for a in range(0, case["rows"], step):
        x, t = s["x"][a:a + step].double(), s["t"][a:a + step]
        lse = torch.logsumexp(x, 1, keepdim=True)
        lp = x - lse
        p = torch.exp(lp)
        info = torch.where(p > 0, lp, 0.0)
        ent = -(p * info).sum(1)
        out["logp"].append(lp[torch.arange(len(t), device=DEV), t])
        out["entropy"].append(ent)
        if train:
            g, h = (s[n][a:a + step].double()[:, None] for n in ("g", "h"))
            hot = torch.zeros_like(x)
            hot[torch.arange(len(t), device=DEV), t] = 1
            out["dx"].append(g * (hot - p) - h * p * (info + ent[:, None]))
            continue
        out["lse"].append(lse[:, 0])
        if case["top"]:
            best = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
            out["index"].append(best)
            out["top"].append(torch.gather(lp, 1, best))
    return {n: torch.cat(v) if v else None for n, v in out.items()}


def exact(case, seed):
    s = _inputs(case, seed)
    k = case["kind"]
    if k in ("attn", "attn_train"):
        return _exact_attn(case, s)
    if k in ("logprobs", "logprobs_train"):
        return _exact_logprobs(case, s)
    if k == "embed":
        y = case["scale"] * s["table"].double()[s["t"]]
        return y if s["r"] is None else y + s["r"].double()
    d = torch.zeros(case["vocab"], case["d"], device=DEV, dtype=torch.float64)
    return d.index_add_(0, s["t"], s["g"].double()).mul_(case["scale"])
