"""What the packed attention, the token log probabilities and the embeddings refuse, checked without a GPU: the C ABI
rejects bad arguments before any device work, and the torch front end what is no device tensor."""
from __future__ import annotations

import ctypes
import math
import pathlib
import subprocess

import pytest
import torch

ROOT = pathlib.Path(__file__).resolve().parents[1]
INVALID = 1  # hipErrorInvalidValue
F32, BF16, F16 = 0, 1, 2
M = 1 << 20


@pytest.fixture(scope="module")
def L():
    from hyperkernels_amd import _lib

    return _lib.lib()


# ---- packed attention ------------------------------------------------------------------------------
GOOD = dict(q=16 * M, k=32 * M, v=48 * M, o=64 * M, lse=80 * M, dout=96 * M, dq=112 * M, dk=128 * M, dv=144 * M,
            cu_q=160 * M, cu_k=161 * M, num_seqs=3, q_heads=4, k_heads=2, head_dim=64, scale=0.125, is_causal=True,
            q_tokens=100, k_tokens=100, q_strideM=256, q_strideH=64, k_strideM=128, k_strideH=64, v_strideM=128,
            v_strideH=64, o_strideM=256, o_strideH=64, do_strideM=256, do_strideH=64, dq_strideM=256, dq_strideH=64,
            dk_strideM=128, dk_strideH=64, dv_strideM=128, dv_strideH=64, lse_strideH=100)


def packed(**change):
    from hyperkernels_amd.kernels import AttnPackedParams

    p = AttnPackedParams()
    for n, v in {**GOOD, **change}.items():
        setattr(p, n, v)
    return ctypes.byref(p)


def test_packed_struct_layout(tmp_path):
    from hyperkernels_amd.kernels import AttnPackedParams

    names = [n for n, _ in AttnPackedParams._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "hk.h"\nint main(void) {\n'
                   '  printf("%zu", sizeof(hk_attn_packed_params));\n' +
                   "".join(f'  printf(" %zu", offsetof(hk_attn_packed_params, {n}));\n' for n in names) +
                   "  return 0;\n}\n")
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-D__HIP_PLATFORM_AMD__", f"-I{ROOT / 'include'}", "-I/opt/rocm/include", str(src), "-o",
                    str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    assert got == [ctypes.sizeof(AttnPackedParams)] + [getattr(AttnPackedParams, n).offset for n in names]
    # the front end packs the same block in one go
    from hyperkernels_amd import kernels

    block = kernels._PACKED_PACK(*range(1, 12), 13, 14, 15, 16, 0.5, True, *range(20, 39))
    assert len(block) == got[0]
    p = AttnPackedParams.from_buffer_copy(block)
    assert p.q == 1 and p.cu_k == 11 and p.head_dim == 16 and p.scale == 0.5 and p.is_causal
    assert (p.q_tokens, p.k_tokens, p.q_strideM, p.lse_strideH) == (20, 21, 22, 38)


@pytest.mark.parametrize("backward", [0, 1])
def test_packed_attention_refuses(L, backward):
    fn = (L.hk_attn_packed_forward, L.hk_attn_packed_backward)[backward]
    both = [
        dict(num_seqs=-1), dict(q_tokens=-1), dict(k_tokens=-1), dict(k_heads=0), dict(q_heads=0), dict(q_heads=3),
        dict(head_dim=0), dict(head_dim=4), dict(head_dim=60), dict(head_dim=136), dict(scale=0.0),
        dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(q=0), dict(k=0), dict(v=0), dict(o=0),
        dict(cu_q=0), dict(cu_k=0), dict(cu_q=160 * M + 2), dict(cu_k=161 * M + 1), dict(q=16 * M + 8),
        dict(k=32 * M + 2), dict(v=48 * M + 4), dict(o=64 * M + 8), dict(lse=80 * M + 2), dict(q_strideM=260),
        dict(q_strideH=68), dict(k_strideM=132), dict(k_strideM=(1 << 23) + 8), dict(v_strideM=(1 << 23) + 8),
        dict(k_strideM=-128), dict(o_strideH=-64), dict(lse_strideH=-1), dict(q_tokens=1 << 31),
        dict(q_tokens=1 << 29), dict(k_tokens=1 << 31), dict(num_seqs=1 << 23), dict(q_strideH=1 << 41),
    ]
    one = [[  # outputs on each other and on what is read
        dict(o=16 * M), dict(o=32 * M + 1024), dict(o=160 * M - 1024), dict(lse=64 * M), dict(o_strideM=64),
        dict(o_strideM=0), dict(lse_strideH=99), dict(lse=48 * M), dict(o_strideH=32),
    ], [
        dict(dq=16 * M), dict(dq=96 * M), dict(dk=32 * M), dict(dv=48 * M), dict(dk=144 * M), dict(dq=64 * M),
        dict(dv=80 * M), dict(dk=161 * M - 512), dict(dq=128 * M), dict(dk_strideM=64), dict(dq=0), dict(dk=0),
        dict(dv=0), dict(dout=0), dict(lse=0), dict(dq_strideM=0), dict(dv_strideH=0), dict(dout=96 * M + 8),
        dict(dk=128 * M + 8), dict(dv_strideM=100),
    ]][backward]
    for bad in both + one:
        assert fn(packed(**bad), BF16, None, 0, None) == INVALID, bad
    for kind in (F32, 3, -1):
        assert fn(packed(), kind, None, 0, None) == INVALID
    assert fn(None, BF16, None, 0, None) == INVALID
    # nothing to do
    assert fn(packed(num_seqs=0), BF16, None, 0, None) == 0
    if not backward:
        assert fn(packed(q_tokens=0), F16, None, 0, None) == 0
    assert fn(packed(q_tokens=0, k_tokens=0), F16, None, 0, None) == 0


def test_packed_attention_workspace(L):
    ws = L.hk_attn_packed_workspace
    assert ws(packed(head_dim=7), BF16, 0) == -1 and ws(packed(), F32, 0) == -1 and ws(packed(dq=0), BF16, 1) == -1
    assert ws(packed(num_seqs=0), BF16, 1) == 0 and ws(packed(q_tokens=0), BF16, 0) == 0
    assert ws(packed(), BF16, 1) >= 12 * 100 * 4  # delta, log-sum-exp and exponent of each query and head
    # one token over a long cache: its keys are shared, so partial results are needed
    long = dict(q_tokens=1, num_seqs=1, k_tokens=100000)
    need = ws(packed(**long), BF16, 0)
    assert need > 0 and need % 16 == 0
    # too little of it, or unaligned, is refused before anything is launched
    assert L.hk_attn_packed_forward(packed(**long), BF16, 256 * M, need - 1, None) == INVALID
    assert L.hk_attn_packed_forward(packed(**long), BF16, 256 * M + 8, need, None) == INVALID
    need = ws(packed(), BF16, 1)
    assert L.hk_attn_packed_backward(packed(), BF16, 256 * M, need - 1, None) == INVALID


# ---- token log probabilities -------------------------------------------------------------------------
def test_token_logprobs_refuses(L):
    good = dict(logits=16 * M, type=BF16, rows=10, vocab=1000, stride=1000, tokens=32 * M, wide=1, logp=48 * M,
                lse=49 * M, entropy=50 * M, top=5, top_logp=51 * M, top_index=52 * M)

    def go(**c):
        g = {**good, **c}
        return L.hk_token_logprobs(g["logits"], g["type"], g["rows"], g["vocab"], g["stride"], g["tokens"], g["wide"],
                                   g["logp"], g["lse"], g["entropy"], g["top"], g["top_logp"], g["top_index"], None, 0,
                                   None)

    for bad in (dict(type=3), dict(type=-1), dict(rows=-1), dict(rows=1 << 31), dict(vocab=0), dict(vocab=(1 << 20) + 1),
                dict(stride=-1), dict(logits=0), dict(tokens=0), dict(logp=0), dict(top=65), dict(top=-1),
                dict(vocab=4), dict(top_logp=0), dict(top_index=0), dict(logits=16 * M + 1), dict(tokens=32 * M + 4),
                dict(type=F32, logits=16 * M + 2), dict(logp=48 * M + 2), dict(lse=49 * M + 1), dict(entropy=50 * M + 2),
                dict(top_index=52 * M + 4), dict(lse=48 * M), dict(entropy=48 * M + 36), dict(logp=16 * M + 2000),
                dict(logp=32 * M), dict(top_logp=52 * M), dict(top_index=16 * M + 19000)):
        assert go(**bad) == INVALID, bad
    assert go(rows=0, logits=0, tokens=0, logp=0) == 0
    ws = L.hk_token_logprobs_workspace
    assert ws(3, 1, 10, 0) == -1 and ws(F32, 1, 10, 11) == -1 and ws(F32, 1, 0, 0) == -1
    assert ws(BF16, 10000, 1000, 5) == 0 and ws(F32, 10000, 100000, 5) > 0
    need = ws(BF16, 1, 100000, 5)
    assert need > 0
    assert L.hk_token_logprobs(16 * M, BF16, 1, 100000, 100000, 32 * M, 1, 48 * M, 49 * M, 50 * M, 5, 51 * M, 52 * M,
                               64 * M, need - 1, None) == INVALID


def test_token_logprobs_backward_refuses(L):
    good = dict(logits=16 * M, type=F16, rows=10, vocab=1000, stride=1000, tokens=32 * M, wide=0, lse=49 * M,
                entropy=50 * M, g=51 * M, h=52 * M, grad=64 * M, gstride=1000)

    def go(**c):
        g = {**good, **c}
        return L.hk_token_logprobs_backward(g["logits"], g["type"], g["rows"], g["vocab"], g["stride"], g["tokens"],
                                            g["wide"], g["lse"], g["entropy"], g["g"], g["h"], g["grad"], g["gstride"],
                                            None)

    for bad in (dict(type=4), dict(rows=-2), dict(vocab=0), dict(stride=-8), dict(gstride=-8), dict(gstride=999),
                dict(gstride=0), dict(logits=0), dict(tokens=0), dict(lse=0), dict(grad=0), dict(entropy=0),
                dict(grad=64 * M + 1), dict(tokens=32 * M + 2), dict(g=51 * M + 1), dict(grad=16 * M + 2),
                dict(grad=16 * M, gstride=1008), dict(grad=49 * M - 19998), dict(grad=32 * M), dict(grad=51 * M)):
        assert go(**bad) == INVALID, bad
    assert go(rows=0, logits=0, grad=0, tokens=0, lse=0) == 0


# ---- embeddings ----------------------------------------------------------------------------------------
def test_embedding_refuses(L):
    good = dict(table=16 * M, type=F32, vocab=1000, d=64, ts=64, tokens=32 * M, wide=1, n=10, residual=48 * M, rs=64,
                out=64 * M, ot=BF16, os=64)

    def go(**c):
        g = {**good, **c}
        return L.hk_embedding_forward(g["table"], g["type"], g["vocab"], g["d"], g["ts"], g["tokens"], g["wide"], g["n"],
                                      1.0, g["residual"], g["rs"], g["out"], g["ot"], g["os"], None)

    for bad in (dict(type=3), dict(ot=-1), dict(vocab=0), dict(d=0), dict(n=-1), dict(n=1 << 31), dict(d=1 << 31),
                dict(vocab=1 << 31), dict(ts=-1), dict(os=1 << 41), dict(table=0), dict(tokens=0), dict(out=0),
                dict(table=16 * M + 2), dict(tokens=32 * M + 4), dict(out=64 * M + 1), dict(residual=48 * M + 1),
                dict(os=63), dict(os=0), dict(out=16 * M + 1000), dict(out=32 * M), dict(out=48 * M + 2),
                dict(residual=64 * M, rs=72)):
        assert go(**bad) == INVALID, bad
    assert go(n=0, table=0, tokens=0, out=0) == 0


def test_embedding_backward_refuses(L):
    good = dict(grad=16 * M, type=BF16, n=3000, d=64, gs=64, tokens=32 * M, wide=1, table=64 * M, tt=F32, vocab=1000,
                ts=64, acc=0, ws=128 * M, bytes=1 << 30)

    def go(**c):
        g = {**good, **c}
        return L.hk_embedding_backward(g["grad"], g["type"], g["n"], g["d"], g["gs"], g["tokens"], g["wide"], 1.0,
                                       g["table"], g["tt"], g["vocab"], g["ts"], g["acc"], g["ws"], g["bytes"], None)

    for bad in (dict(type=3), dict(tt=3), dict(n=-1), dict(n=1 << 30), dict(d=0), dict(vocab=0), dict(gs=-1),
                dict(ts=63), dict(ts=0), dict(table=0), dict(grad=0), dict(tokens=0), dict(table=64 * M + 2),
                dict(grad=16 * M + 1), dict(tokens=32 * M + 4), dict(table=16 * M + 4), dict(table=32 * M),
                dict(bytes=1000), dict(ws=128 * M + 8), dict(n=1 << 29, d=1 << 20)):
        assert go(**bad) == INVALID, bad
    assert go(n=0, acc=1, table=0) == 0
    ws = L.hk_embedding_workspace
    assert ws(-1, 10, 4) == -1 and ws(10, 0, 4) == -1 and ws(10, 10, 0) == -1
    assert ws(1024, 1000, 64) == 0 and ws(2048, 1000, 64) == 0 and ws(2049, 1000, 64) >= 8 * 2049 + 128
    assert ws(2048, 32769, 64) > 0


# ---- the torch front end ---------------------------------------------------------------------------------
def test_front_ends_refuse_host_tensors():
    from hyperkernels_amd import kernels as hk

    q = torch.zeros(8, 4, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 8], dtype=torch.int32)
    x, t = torch.zeros(4, 10), torch.zeros(4, dtype=torch.long)
    for call in (lambda: hk.attn_packed_forward(q, q, q, cu),
                 lambda: hk.attn_packed_forward(q.float(), q, q, cu),
                 lambda: hk.attn_packed_forward(q[0], q, q, cu),
                 lambda: hk.attn_packed_backward(q, q, q, q, q, None, cu),
                 lambda: hk.token_logprobs(x, t), lambda: hk.token_logprobs(x[0], t),
                 lambda: hk.token_logprobs(x.long(), t),
                 lambda: hk.token_logprobs_backward(x, t, x[:, 0]),
                 lambda: hk.embedding_forward(x, t), lambda: hk.embedding_forward(x[0], t),
                 lambda: hk.embedding_backward(x, t, x), lambda: hk.embedding_backward(x[0], t, x)):
        with pytest.raises(ValueError):
            call()
