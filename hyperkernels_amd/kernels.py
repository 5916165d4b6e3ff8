"""Host-side mirror of the reference kernel surface over torch device tensors.

Each function wraps one C-ABI entry point of ``include/hk.h`` and keeps the argument meaning of
the reference kernel it replaces (cited per function). Tensors must be HIP device tensors;
outputs may be passed in (as the reference caller does) or are allocated here. Launches go on
torch's current stream. Errors from the library raise ``HKError``; nothing falls back to a CPU
path.
"""
from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple, Sequence

import torch

from ._lib import HKError, _fns, call, lib  # noqa: F401

__all__ = [
    "HKError", "gelu_forward", "gelu_backward", "bgemm_act", "bgemm_act_backward", "layer_norm_forward", "ln_backward_input",
    "ln_backward_gamma_beta", "layer_norm_backward", "sparse_ce_forward", "sparse_ce_backward",
    "AdamLaunchMetadata", "multi_tensor_adam", "AdamPlan", "Adam8Plan", "ADAM8_BLOCK",
    "adam8_states", "adam8_quantize", "adam8_dequantize", "qk_norm_rope_forward",
    "qk_norm_rope_backward", "attn_packed_forward", "attn_packed_backward",
    "TokenLogprobs", "token_logprobs", "token_logprobs_backward", "embedding_forward", "embedding_backward",
    "ReductionLayout",
    "unified_reduce_sum", "reduce_generic", "REDUCE_INNER", "REDUCE_OUTER", "REDUCE_GENERIC",
]


# A small call is bound by this file, not by its kernel (LayerNorm over 64 x 768: 13 us of host time
# against 3 us on the device). So the current stream is read as a raw handle (0.2 us; building
# torch's Stream object takes 2.8), pointers and scalars go to ctypes as plain numbers, which the
# bound argument types convert, and the attention parameter blocks are filled in one go.
def _stream() -> int:
    """The handle of torch's current stream on the current device."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _dev(*ts: torch.Tensor | None) -> None:
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("hyperkernels_amd kernels take device tensors only")
        if not t.is_contiguous():
            raise ValueError("hyperkernels_amd kernels take contiguous tensors")


_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # HK_TYPE_*


_BF16, _F32 = torch.bfloat16, torch.float32


def _device(fn: str, t: torch.Tensor) -> int:
    """The device of a call's first tensor: the current one, whose stream the launch goes to."""
    d = t.get_device()  # -1: a host tensor
    if d < 0 or d != torch._C._cuda_getDevice():
        raise ValueError(f"{fn}: tensors of the current device only")
    return d


# ----------------------------------------------------------------------------------------------
# GELU: gelu_forward_sm89_kernel<T> (kernels/gelu/gelu_forward_sm89_kernel.cu:35-37),
#       gelu_backward_sm89_kernel<T> (kernels/gelu/gelu_backward_sm89_kernel.cu:44-47)
# ----------------------------------------------------------------------------------------------
# storage dtype -> entry-point suffix (the reference's float / __nv_bfloat16 / __half
# instantiations of the GELU and LayerNorm kernels)
_SUFFIX = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}


def gelu_forward(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    _dev(x, out)
    out = torch.empty_like(x) if out is None else out
    if x.dtype not in _SUFFIX or out.dtype != x.dtype or out.numel() != x.numel():
        raise ValueError("gelu_forward: fp32, bf16 or fp16 tensors of equal size")
    call(f"hk_gelu_forward_{_SUFFIX[x.dtype]}", _ptr(x), _ptr(out), x.numel(), _stream())
    return out


def gelu_backward(grad: torch.Tensor, x: torch.Tensor,
                  grad_in: torch.Tensor | None = None) -> torch.Tensor:
    _dev(grad, x, grad_in)
    grad_in = torch.empty_like(x) if grad_in is None else grad_in
    if x.dtype not in _SUFFIX or not (grad.dtype == x.dtype == grad_in.dtype) or not (
            grad.numel() == x.numel() == grad_in.numel()):
        raise ValueError("gelu_backward: fp32, bf16 or fp16 tensors of equal size")
    call(f"hk_gelu_backward_{_SUFFIX[x.dtype]}", _ptr(grad), _ptr(x), _ptr(grad_in),
         x.numel(), _stream())
    return grad_in


# ----------------------------------------------------------------------------------------------
# LayerNorm (kernels/layernorm/*.cu)
# ----------------------------------------------------------------------------------------------
def _rows_cols(x: torch.Tensor) -> tuple[int, int]:
    if x.dim() < 1:
        raise ValueError("layer norm needs at least one dimension")
    cols = x.shape[-1]
    return (x.numel() // cols if cols else 0), cols


def _ln_suffix(data, stats) -> str:
    """Entry-point suffix for LayerNorm: `data` tensors (x, gamma, beta, y, dy, dx) share one
    storage dtype; `stats` tensors (mean, rstd, grad_gamma, grad_beta) are fp32."""
    dt = data[0].dtype
    sfx = _SUFFIX.get(dt)
    for t in data:
        if sfx is None or (t is not None and t.dtype != dt):
            raise ValueError("layer norm: x, gamma, beta, y, dy and dx must share one dtype "
                             "(fp32, bf16 or fp16)")
    for t in stats:
        if t is not None and t.dtype != torch.float32:
            raise ValueError("layer norm: mean, rstd, grad_gamma and grad_beta are fp32")
    return sfx


def layer_norm_forward(x, gamma=None, beta=None, eps: float = 1e-5, y=None, mean=None, rstd=None):
    """layer_norm_forward_sm89_kernel<T,float> (layer_norm_forward_sm89_kernel.cu:27-32).

    Returns (y, mean, rstd); mean/rstd are [rows] fp32."""
    _dev(x, gamma, beta, y, mean, rstd)
    rows, cols = _rows_cols(x)
    y = torch.empty_like(x) if y is None else y
    mean = torch.empty(rows, device=x.device, dtype=torch.float32) if mean is None else mean
    rstd = torch.empty(rows, device=x.device, dtype=torch.float32) if rstd is None else rstd
    sfx = _ln_suffix([x, gamma, beta, y], [mean, rstd])
    call(f"hk_layer_norm_forward_{sfx}", _ptr(x), _ptr(gamma), _ptr(beta), _ptr(y), _ptr(mean),
         _ptr(rstd), rows, cols, eps, _stream())
    return y, mean, rstd


def ln_backward_input(grad_y, x, mean, rstd, gamma=None, grad_x=None):
    """OwnTensor::cuda::ln_backward_input_sm89_kernel<T> (ln_backward_input_sm89_kernel.cu:33-38)."""
    _dev(grad_y, x, mean, rstd, gamma, grad_x)
    rows, cols = _rows_cols(x)
    grad_x = torch.empty_like(x) if grad_x is None else grad_x
    sfx = _ln_suffix([x, grad_y, gamma, grad_x], [mean, rstd])
    call(f"hk_ln_backward_input_{sfx}", _ptr(grad_y), _ptr(x), _ptr(mean), _ptr(rstd),
         _ptr(gamma), _ptr(grad_x), rows, cols, _stream())
    return grad_x


def ln_backward_gamma_beta(grad_y, x, mean, rstd, grad_gamma, grad_beta):
    """ln_backward_gamma_beta_sm89_kernel<T> (ln_backward_gamma_beta_sm89_kernel.cu:15-21).

    ADDS the column sums into grad_gamma / grad_beta (the reference's atomics into caller-zeroed
    buffers), in a fixed order."""
    _dev(grad_y, x, mean, rstd, grad_gamma, grad_beta)
    rows, cols = _rows_cols(x)
    sfx = _ln_suffix([x, grad_y], [mean, rstd, grad_gamma, grad_beta])
    call(f"hk_ln_backward_gamma_beta_{sfx}", _ptr(grad_y), _ptr(x), _ptr(mean), _ptr(rstd),
         _ptr(grad_gamma), _ptr(grad_beta), rows, cols, _stream())
    return grad_gamma, grad_beta


def layer_norm_backward(grad_y, x, mean, rstd, gamma, grad_gamma, grad_beta, grad_x=None):
    """Fused backward: grad_x written (grad_y or x itself, too), grad_gamma / grad_beta added into."""
    _dev(grad_y, x, mean, rstd, gamma, grad_gamma, grad_beta, grad_x)
    rows, cols = _rows_cols(x)
    grad_x = torch.empty_like(x) if grad_x is None else grad_x
    sfx = _ln_suffix([x, grad_y, gamma, grad_x], [mean, rstd, grad_gamma, grad_beta])
    call(f"hk_layer_norm_backward_{sfx}", _ptr(grad_y), _ptr(x), _ptr(mean), _ptr(rstd),
         _ptr(gamma), _ptr(grad_x), _ptr(grad_gamma), _ptr(grad_beta), rows, cols, _stream())
    return grad_x


# ----------------------------------------------------------------------------------------------
# Sparse cross-entropy (kernels/loss/*.cu)
# ----------------------------------------------------------------------------------------------
# target dtype -> entry-point suffix: the reference's <float, int32_t | int64_t | uint16_t>
# instantiations (sparse_ce_forward_...cu:108-113; sparseCENormalize_from_stats.cu:52-60)
_CE_INDEX = {torch.int32: "i32", torch.int64: "i64", torch.uint16: "u16"}


def sparse_ce_forward(logits, targets, losses=None, saved_max=None, saved_sum=None):
    """sparse_ce_forward_kernel_vec_save_stats<float,TIdx> (sparse_ce_forward_...cu:14-23).

    Returns (losses, saved_max, saved_sum), each [rows] fp32."""
    _dev(logits, targets, losses, saved_max, saved_sum)
    if logits.dtype != torch.float32 or targets.dtype not in _CE_INDEX or logits.dim() != 2:
        raise ValueError("sparse_ce_forward: fp32 logits [rows, vocab] and int32/int64/uint16 "
                         "targets")
    rows, vocab = logits.shape
    mk = lambda: torch.empty(rows, device=logits.device, dtype=torch.float32)  # noqa: E731
    losses = mk() if losses is None else losses
    saved_max = mk() if saved_max is None else saved_max
    saved_sum = mk() if saved_sum is None else saved_sum
    call("hk_sparse_ce_forward_f32_" + _CE_INDEX[targets.dtype], _ptr(logits), _ptr(targets),
         _ptr(losses), _ptr(saved_max), _ptr(saved_sum), rows, vocab, _stream())
    return losses, saved_max, saved_sum


def sparse_ce_backward(logits, targets, saved_max, saved_sum, grad_output=None,
                       host_scale: float = 1.0, grad=None):
    """sparseCENormalize_from_stats<float,TIdx> (sparseCENormalize_from_stats.cu:7-17).

    grad_output is a 1-element device tensor (or None for 1.0)."""
    _dev(logits, targets, saved_max, saved_sum, grad_output, grad)
    if logits.dtype != torch.float32 or targets.dtype not in _CE_INDEX or logits.dim() != 2:
        raise ValueError("sparse_ce_backward: fp32 logits [rows, vocab] and int32/int64/uint16 "
                         "targets")
    rows, vocab = logits.shape
    grad = torch.empty_like(logits) if grad is None else grad
    call("hk_sparse_ce_backward_f32_" + _CE_INDEX[targets.dtype], _ptr(logits), _ptr(targets),
         _ptr(grad), _ptr(saved_max), _ptr(saved_sum), rows, vocab, _ptr(grad_output),
         host_scale, _stream())
    return grad


# ----------------------------------------------------------------------------------------------
# Multi-tensor AdamW (kernels/optimizer/multi_tensor_adam_sm89_kernel.cu)
# ----------------------------------------------------------------------------------------------
ADAM_CHUNK_SIZE = 32768
ADAM_MAX_BLOCKS = 320
ADAM_MAX_TENSORS = 48


class AdamLaunchMetadata(ctypes.Structure):
    """Byte-for-byte the reference's AdamLaunchMetadata (multi_tensor_adam_sm89_kernel.cu:13-21)."""

    _fields_ = [
        ("params", ctypes.c_void_p * ADAM_MAX_TENSORS),
        ("grads", ctypes.c_void_p * ADAM_MAX_TENSORS),
        ("ms", ctypes.c_void_p * ADAM_MAX_TENSORS),
        ("vs", ctypes.c_void_p * ADAM_MAX_TENSORS),
        ("sizes", ctypes.c_int64 * ADAM_MAX_TENSORS),
        ("block_to_tensor", ctypes.c_ubyte * ADAM_MAX_BLOCKS),
        ("block_to_chunk", ctypes.c_int * ADAM_MAX_BLOCKS),
    ]


def multi_tensor_adam(params: Sequence[torch.Tensor], grads, ms, vs, lr, beta1, beta2, eps,
                      weight_decay, bias_correction1, bias_correction2) -> None:
    """One launch of the reference ABI: <= 48 tensors, <= 320 chunks of 32768 elements."""
    if not (len(params) == len(grads) == len(ms) == len(vs)) or len(params) > ADAM_MAX_TENSORS:
        raise ValueError("multi_tensor_adam: at most 48 tensors, equal list lengths")
    meta = AdamLaunchMetadata()
    blk = 0
    for t, (p, g, m, v) in enumerate(zip(params, grads, ms, vs)):
        _dev(p, g, m, v)
        meta.params[t], meta.grads[t] = p.data_ptr(), g.data_ptr()
        meta.ms[t], meta.vs[t] = m.data_ptr(), v.data_ptr()
        meta.sizes[t] = p.numel()
        for c in range((p.numel() + ADAM_CHUNK_SIZE - 1) // ADAM_CHUNK_SIZE):
            if blk >= ADAM_MAX_BLOCKS:
                raise ValueError("multi_tensor_adam: more than 320 chunks")
            meta.block_to_tensor[blk], meta.block_to_chunk[blk] = t, c
            blk += 1
    call("hk_multi_tensor_adam", ctypes.byref(meta), blk, lr, beta1, beta2, eps, weight_decay,
         bias_correction1, bias_correction2, _stream())


class AdamPlan:
    """Device-resident tensor/chunk table: one launch per step over any number of tensors."""

    def __init__(self, params, grads, ms, vs):
        n = len(params)
        if not (n == len(grads) == len(ms) == len(vs)):
            raise ValueError("AdamPlan: equal list lengths")
        for ts in zip(params, grads, ms, vs):
            _dev(*ts)
            if len({t.numel() for t in ts}) != 1 or any(t.dtype != torch.float32 for t in ts):
                raise ValueError("AdamPlan: p, g, m, v of one tensor are fp32 of equal size")
        arr = lambda ts: (ctypes.c_void_p * n)(*[t.data_ptr() for t in ts])  # noqa: E731
        self._keep = (list(params), list(grads), list(ms), list(vs))
        sizes = (ctypes.c_int64 * n)(*[p.numel() for p in params])
        self._plan = ctypes.c_void_p()
        call("hk_adam_plan_create", n, arr(params), arr(grads), arr(ms), arr(vs), sizes,
             ctypes.byref(self._plan))
        self.num_chunks = lib().hk_adam_plan_num_chunks(self._plan)

    def step(self, lr, beta1, beta2, eps, weight_decay, bias_correction1, bias_correction2):
        call("hk_adam_plan_step", self._plan, lr, beta1, beta2, eps, weight_decay,
             bias_correction1, bias_correction2, _stream())

    def close(self):
        if self._plan:
            call("hk_adam_plan_destroy", self._plan)
            self._plan = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ----------------------------------------------------------------------------------------------
# Multi-tensor AdamW with both moments in 8 bits (no counterpart in the reference)
# ----------------------------------------------------------------------------------------------
ADAM8_BLOCK = 256


def _adam8_check(fn: str, m, v, m_scale, v_scale, blocks: int) -> None:
    if m.dtype is not torch.int8 or v.dtype is not torch.uint8 or (
            m_scale.dtype is not torch.float32) or v_scale.dtype is not torch.float32:
        raise ValueError(f"{fn}: m int8, v uint8, m_scale and v_scale fp32")
    n = blocks * ADAM8_BLOCK
    if m.numel() != n or v.numel() != n or m_scale.numel() != blocks or (
            v_scale.numel() != blocks):
        raise ValueError(f"{fn}: {blocks} blocks need {n} codes and {blocks} scales of each moment")


def _flat(fn: str, *ts: torch.Tensor | None) -> None:
    """Contiguous tensors of the current device."""
    cur = None
    for t in ts:
        if t is not None:
            if cur is None:
                cur = _device(fn, t)
            if t.get_device() != cur or not t.is_contiguous():
                raise ValueError(f"{fn}: contiguous tensors of the current device only")


def adam8_states(sizes: Sequence[int], device="cuda"):
    """(m, v, m_scale, v_scale), moments of zero for tensors of these sizes: the codes of all tensors
    one behind the other, each tensor from a block's first element on."""
    blocks = sum(-(-int(n) // ADAM8_BLOCK) for n in sizes)
    z = lambda n, dt: torch.zeros(n, device=device, dtype=dt)  # noqa: E731
    return (z(blocks * ADAM8_BLOCK, torch.int8), z(blocks * ADAM8_BLOCK, torch.uint8),
            z(blocks, torch.float32), z(blocks, torch.float32))


def adam8_quantize(m, v, states=None):
    """8-bit states (m, v, m_scale, v_scale) of fp32 moments of one tensor (or of several that each
    begin on a block)."""
    n = m.numel()
    if m.dtype is not torch.float32 or v.dtype is not torch.float32 or v.numel() != n:
        raise ValueError("adam8_quantize: fp32 moments of equal size")
    states = adam8_states([n], m.device) if states is None else states
    _flat("adam8_quantize", m, v, *states)
    _adam8_check("adam8_quantize", *states, -(-n // ADAM8_BLOCK))
    call("hk_adam8_quantize", m.data_ptr(), v.data_ptr(), n, *map(_ptr, states), _stream())
    return tuple(states)


def adam8_dequantize(m, v, m_scale, v_scale, m_out=None, v_out=None):
    """The fp32 moments (m, v) that 8-bit states stand for, of all their elements or of as many as
    m_out and v_out hold."""
    n = m.numel() if m_out is None else m_out.numel()
    _adam8_check("adam8_dequantize", m, v, m_scale, v_scale, -(-n // ADAM8_BLOCK))
    m_out = m_scale.new_empty(n) if m_out is None else m_out
    v_out = m_scale.new_empty(n) if v_out is None else v_out
    _flat("adam8_dequantize", m, v, m_scale, v_scale, m_out, v_out)
    if m_out.dtype is not torch.float32 or v_out.dtype is not torch.float32 or v_out.numel() != n:
        raise ValueError("adam8_dequantize: fp32 outputs of equal size")
    call("hk_adam8_dequantize", m.data_ptr(), v.data_ptr(), m_scale.data_ptr(), v_scale.data_ptr(), n,
         m_out.data_ptr(), v_out.data_ptr(), _stream())
    return m_out, v_out


class Adam8Plan:
    """AdamPlan with both moments in 8 bits: fp32 parameters, gradients of one type (fp32, bf16 or
    fp16), states as adam8_states lays them out, and optionally bf16 copies of the updated parameters
    (one tensor or None for each)."""

    def __init__(self, params, grads, m, v, m_scale, v_scale, copies=None):
        n = len(params)
        copies = [None] * n if copies is None else list(copies)
        if not (n == len(grads) == len(copies)):
            raise ValueError("Adam8Plan: equal list lengths")
        types = {g.dtype for g in grads} or {torch.float32}
        if len(types) != 1 or not types <= set(_TYPE):
            raise ValueError("Adam8Plan: the gradients share one type (fp32, bf16 or fp16)")
        _flat("Adam8Plan", m, v, m_scale, v_scale)
        for p, g, c in zip(params, grads, copies):
            _flat("Adam8Plan", p, g, c)
            if p.dtype != torch.float32 or g.numel() != p.numel():
                raise ValueError("Adam8Plan: fp32 parameters, gradients of equal size")
            if c is not None and (c.dtype != torch.bfloat16 or c.numel() != p.numel()):
                raise ValueError("Adam8Plan: copies are bf16 of the parameters' size")
        _adam8_check("Adam8Plan", m, v, m_scale, v_scale,
                     sum(-(-p.numel() // ADAM8_BLOCK) for p in params))
        arr = lambda ts: (ctypes.c_void_p * n)(*[_ptr(t) for t in ts])  # noqa: E731
        self._keep = (list(params), list(grads), copies, m, v, m_scale, v_scale)
        sizes = (ctypes.c_int64 * n)(*[p.numel() for p in params])
        self._plan = ctypes.c_void_p()
        call("hk_adam8_plan_create", n, arr(params), arr(grads), _TYPE[types.pop()], arr(copies),
             sizes, _ptr(m), _ptr(v), _ptr(m_scale), _ptr(v_scale), ctypes.byref(self._plan))
        self.num_blocks = lib().hk_adam8_plan_num_blocks(self._plan)

    def step(self, lr, beta1, beta2, eps, weight_decay, bias_correction1, bias_correction2):
        call("hk_adam8_plan_step", self._plan, lr, beta1, beta2, eps, weight_decay,
             bias_correction1, bias_correction2, _stream())

    def close(self):
        if self._plan:
            call("hk_adam8_plan_destroy", self._plan)
            self._plan = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ----------------------------------------------------------------------------------------------
# Attention (kernels/attention/*.cu), fp32, head_dim 64, tensors [B, nh, T, d] (any strides
# with a unit last dimension), LSE / D [B, nh, T]
# ----------------------------------------------------------------------------------------------
_I64 = ctypes.c_int64


class AttnFwdParams(ctypes.Structure):
    """MemEfficientFwdParams (fused_attn_forward_kernel_tc_sm89.cu:8-29), field for field."""

    _fields_ = [("Q", ctypes.c_void_p), ("K", ctypes.c_void_p), ("V", ctypes.c_void_p),
                ("O", ctypes.c_void_p), ("LSE", ctypes.c_void_p), ("B", ctypes.c_int),
                ("nh", ctypes.c_int), ("T", _I64), ("scale", ctypes.c_float),
                ("is_causal", ctypes.c_bool), ("dropout_p", ctypes.c_float),
                ("dropout_mask", ctypes.c_void_p)] + [
        (f"{t}_stride{s}", _I64) for t in ("q", "k", "v", "o") for s in ("B", "M", "H")] + [
        ("lse_strideB", _I64), ("lse_strideH", _I64)]


class AttnBwdParams(ctypes.Structure):
    """MemEfficientBwdParams (mem_efficient_bwd_precompute_D_sm89.cu:7-33), field for field."""

    _fields_ = [(n, ctypes.c_void_p) for n in ("Q", "K", "V", "O", "dO", "LSE", "D", "dQ", "dK",
                                               "dV")] + [
        ("B", ctypes.c_int), ("nh", ctypes.c_int), ("T", ctypes.c_int), ("scale", ctypes.c_float),
        ("is_causal", ctypes.c_bool)] + [
        (f"{t}_stride{s}", _I64) for t in ("q", "k", "v", "o", "do", "dq", "dk", "dv")
        for s in ("B", "M", "H")] + [
        ("lse_strideB", _I64), ("lse_strideH", _I64), ("d_strideB", _I64), ("d_strideH", _I64)]


def _strides(t: torch.Tensor | None) -> tuple[int, int, int]:
    """(batch, row, head) strides of a [B, nh, T, d] tensor."""
    if t is None:
        return 0, 0, 0
    st = t.stride()
    if len(st) != 4 or st[3] != 1:
        raise ValueError("attention tensors are [B, nh, T, d] with a unit last-dim stride")
    return st[0], st[2], st[1]


def fused_attn_forward(q, k, v, causal: bool, scale: float | None = None, o=None, lse=None,
                       dropout_p: float = 0.0, dropout_mask=None):
    """fused_attn_forward_kernel_tc_sm89<64,64,64,1>: returns (O, LSE).

    With dropout_p > 0 and a dropout_mask (contiguous fp32 [B, nh, T, T], the factor of each
    score, e.g. 0 or 1 / (1 - p)), the exp terms are multiplied by the mask and normalised by
    their post-dropout sum, as the reference kernel does (fused_attn_forward...:316-334)."""
    for t in (q, k, v):
        if not t.is_cuda or t.dtype != torch.float32:
            raise ValueError("fused_attn_forward: fp32 device tensors")
    B, H, T, D = q.shape
    if dropout_mask is not None and (
            not dropout_mask.is_cuda or dropout_mask.dtype != torch.float32
            or tuple(dropout_mask.shape) != (B, H, T, T) or not dropout_mask.is_contiguous()):
        raise ValueError("fused_attn_forward: dropout_mask is a contiguous fp32 [B, nh, T, T] "
                         "device tensor")
    scale = D ** -0.5 if scale is None else scale
    o = torch.empty_like(q) if o is None else o
    lse = torch.empty(B, H, T, device=q.device, dtype=torch.float32) if lse is None else lse
    p = AttnFwdParams(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), B, H, T, scale,
        bool(causal), dropout_p, _ptr(dropout_mask), *_strides(q), *_strides(k), *_strides(v),
        *_strides(o), lse.stride(0), lse.stride(1))
    call("hk_fused_attn_forward", ctypes.byref(p), D, _stream())
    return o, lse


def _bwd_params(q, k, v, o, do, lse, D, dq, dk, dv, causal, scale):
    B, H, T, _ = q.shape
    ls = (0, 0) if lse is None else (lse.stride(0), lse.stride(1))
    return AttnBwdParams(
        _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(do), _ptr(lse), _ptr(D), _ptr(dq), _ptr(dk),
        _ptr(dv), B, H, T, scale, bool(causal), *_strides(q), *_strides(k), *_strides(v),
        *_strides(o), *_strides(do), *_strides(dq), *_strides(dk), *_strides(dv), *ls,
        D.stride(0), D.stride(1))


def attn_bwd_precompute_D(do, o, D=None):
    """mem_efficient_bwd_precompute_D_sm89<HD>: D = rowsum(dO * O), [B, nh, T]."""
    B, H, T, Dh = o.shape
    D = torch.empty(B, H, T, device=o.device, dtype=torch.float32) if D is None else D
    p = _bwd_params(o, None, None, o, do, None, D, None, None, None, False, 1.0)
    p.Q = None
    call("hk_attn_bwd_precompute_D", ctypes.byref(p), Dh, _stream())
    return D


def attn_backward(q, k, v, do, lse, D, causal: bool, scale: float | None = None, dq=None, dk=None,
                  dv=None, o=None):
    """OwnTensor::mem_efficient_bwd_unified_kernel_exp12<64, Causal>: returns (dQ, dK, dV).

    dK and dV are written; dQ is ADDED into, as in the reference where the caller zeroes dQ before
    the launch, or written when it is not passed in."""
    B, H, T, Dh = q.shape
    scale = Dh ** -0.5 if scale is None else scale
    fn = "hk_attn_backward"
    if dq is None:
        dq, fn = torch.empty_like(q), "hk_attn_backward_set"
    dk = torch.empty_like(k) if dk is None else dk
    dv = torch.empty_like(v) if dv is None else dv
    p = _bwd_params(q, k, v, o, do, lse, D, dq, dk, dv, causal, scale)
    call(fn, ctypes.byref(p), Dh, _stream())
    return dq, dk, dv


# ----------------------------------------------------------------------------------------------
# BF16 GEMM with bias, activation and residual in its epilogue, and its backward product (no
# counterpart in the reference)
# ----------------------------------------------------------------------------------------------
_ACT = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}  # HK_ACT_*
_INT_MAX = 2 ** 31 - 1  # ctypes cuts a larger one to its low 32 bits


def _matrix(fn: str, t: torch.Tensor, dev: int, batch: int, rows: int,
            cols: int) -> tuple[int, int, int]:
    """(address, leading dimension, batch stride) of a bf16 matrix [rows, cols], or
    [batch, rows, cols]."""
    sh, st, step = t.shape, t.stride(), 0
    if batch != 1 or len(sh) != 2:
        if sh != (batch, rows, cols):
            raise ValueError(f"{fn}: [{batch}, {rows}, {cols}] expected, {tuple(sh)} given")
        step = st[0] if batch != 1 else 0
    elif sh != (rows, cols):
        raise ValueError(f"{fn}: [{rows}, {cols}] expected, {tuple(sh)} given")
    if t.dtype is not _BF16 or t.get_device() != dev or (st[-1] != 1 and cols > 1):
        raise ValueError(f"{fn}: bf16 matrices of one device with a unit last-dim stride")
    ld = st[-2]
    if rows == 1 and not cols <= ld <= _INT_MAX:
        ld = cols
    if ld > _INT_MAX:
        raise ValueError(f"{fn}: leading dimensions below 2^31 only")
    return t.data_ptr(), ld, step


def _vector(fn: str, t: torch.Tensor, dtype, dev: int, batch: int, n: int) -> tuple[int, int]:
    """(address, batch stride) of a vector [n], or [batch, n]."""
    sh, st = t.shape, t.stride()
    if t.dtype is not dtype or t.get_device() != dev or (sh != (n,) and sh != (batch, n)) or (
            st[-1] != 1 and n > 1):
        raise ValueError(f"{fn}: {dtype} vectors [{n}], or [{batch}, {n}]; {tuple(sh)} given")
    return t.data_ptr(), st[0] if len(sh) == 2 and batch != 1 else 0


_NO_MATRIX, _NO_VECTOR = (None, 0, 0), (None, 0)


def _product(fn: str, a, b, trans_a: bool, trans_b: bool, activation: str):
    """(batch, M, N, K, activation, device) of op(a) op(b)."""
    ash, bsh = a.shape, b.shape
    act = _ACT.get(activation)
    if act is None or len(ash) != len(bsh) or not 2 <= len(ash) <= 3:
        raise ValueError(f"{fn}: matrices or batches of them, and one of {', '.join(_ACT)}")
    if trans_a:
        K, M = ash[-2], ash[-1]
    else:
        M, K = ash[-2], ash[-1]
    batch, N = ash[0] if len(ash) == 3 else 1, bsh[-2] if trans_b else bsh[-1]
    if max(M, N, K, batch) > _INT_MAX:
        raise ValueError(f"{fn}: extents below 2^31 only")
    return batch, M, N, K, act, _device(fn, a)


def _call_captured(name: str, need, *args) -> None:
    """Calls an entry point whose arguments end in (workspace, bytes, stream), with the library's own
    workspace; where the call is captured into a graph and needs one, with need() bytes of the graph's."""
    f = _fns.get(name)
    if f is None:
        f = _fns[name] = getattr(lib(), name)
    stream = _stream()
    status = f(*args, None, 0, stream)
    if status == 900:  # hipErrorStreamCaptureUnsupported
        n = need()
        ws = torch.empty(n, device="cuda", dtype=torch.uint8)
        status = f(*args, ws.data_ptr(), n, stream)
    if status != 0:
        raise HKError(name, status)


def _bf16_bits(x: float) -> int:
    return int(torch.tensor(x, dtype=torch.bfloat16).view(torch.int16)) & 0xFFFF


def bgemm_act(a, b, bias=None, activation: str = "none", residual=None, preact=None, out=None,
              trans_a: bool = False, trans_b: bool = False, alpha: float = 1.0):
    """act(alpha op(a) op(b) + bias) + residual for bf16 matrices [rows, cols] or batches of them; what
    goes into the activation ("none", "relu", "gelu" or "silu") is stored in `preact` where that is
    passed. bias is [N], or [batch, N]; residual may be `out` itself; alpha is rounded to bf16."""
    fn = "bgemm_act"
    batch, M, N, K, act, dev = _product(fn, a, b, trans_a, trans_b, activation)
    if out is None:
        out = a.new_empty((M, N) if a.dim() == 2 else (batch, M, N))
    A = _matrix(fn, a, dev, batch, K, M) if trans_a else _matrix(fn, a, dev, batch, M, K)
    B = _matrix(fn, b, dev, batch, N, K) if trans_b else _matrix(fn, b, dev, batch, K, N)
    C = _matrix(fn, out, dev, batch, M, N)
    R = _NO_MATRIX if residual is None else _matrix(fn, residual, dev, batch, M, N)
    Z = _NO_MATRIX if preact is None else _matrix(fn, preact, dev, batch, M, N)
    v = _NO_VECTOR if bias is None else _vector(fn, bias, _BF16, dev, batch, N)
    _call_captured("hk_bgemm_act",
                   lambda: lib().hk_bgemm_act_workspace(trans_a, trans_b, M, N, K, batch, 0),
                   trans_a, trans_b, M, N, K, 0x3F80 if alpha == 1.0 else _bf16_bits(alpha), *A, *B,
                   *v, act, *R, *Z, *C, batch)
    return out


def bgemm_act_backward(a, b, preact=None, activation: str = "none", dbias=None, out=None,
                       trans_a: bool = False, trans_b: bool = False, alpha: float = 1.0,
                       accumulate: bool = True):
    """d = alpha op(a) op(b) * act'(preact) in bf16: the gradient of a layer's pre-activation, from the
    gradient behind the next layer and that layer's weights; out may be `preact` itself. dbias (fp32 [N], or [batch, N]; None: not
    wanted) is added to, or written where accumulate is False: the sums of d over rows (and, [N],
    batches) before it is rounded. alpha is rounded to bf16."""
    fn = "bgemm_act_backward"
    batch, M, N, K, act, dev = _product(fn, a, b, trans_a, trans_b, activation)
    if out is None:
        out = a.new_empty((M, N) if a.dim() == 2 else (batch, M, N))
    A = _matrix(fn, a, dev, batch, K, M) if trans_a else _matrix(fn, a, dev, batch, M, K)
    B = _matrix(fn, b, dev, batch, N, K) if trans_b else _matrix(fn, b, dev, batch, K, N)
    C = _matrix(fn, out, dev, batch, M, N)
    if preact is None and act:
        raise ValueError(f"{fn}: the activation's derivative needs preact")
    Z = _NO_MATRIX if preact is None else _matrix(fn, preact, dev, batch, M, N)
    v = _NO_VECTOR if dbias is None else _vector(fn, dbias, _F32, dev, batch, N)
    if v[1] < N and dbias is not None and dbias.dim() == 2 and batch != 1:
        raise ValueError(f"{fn}: the rows of dbias overlap")
    _call_captured("hk_bgemm_act_backward",
                   lambda: lib().hk_bgemm_act_workspace(trans_a, trans_b, M, N, K, batch,
                                                        dbias is not None),
                   trans_a, trans_b, M, N, K, 0x3F80 if alpha == 1.0 else _bf16_bits(alpha), *A, *B,
                   act, *Z, *C, *v, accumulate, batch)
    return out


# ----------------------------------------------------------------------------------------------
# RMS norm of query and key heads with the position rotation (no counterpart in the reference)
# ----------------------------------------------------------------------------------------------
class QkNormRopeParams(ctypes.Structure):
    """hk_qk_norm_rope_params (hk.h), field for field."""

    _fields_ = [(n, ctypes.c_void_p) for n in (
        "q", "k", "q_weight", "k_weight", "cos", "sin", "positions", "q_out", "k_out", "dq_out",
        "dk_out", "dq", "dk", "dq_weight", "dk_weight")] + [
        (n, ctypes.c_int) for n in ("B", "T", "q_heads", "k_heads", "head_dim", "rotary_dim")] + [
        ("eps", ctypes.c_float)] + [
        (n, ctypes.c_bool) for n in ("interleaved", "f32_io", "accumulate")] + [
        (n, _I64) for n in ("table_rows", "table_stride", "pos_strideB")] + [
        (f"{t}_stride{s}", _I64) for t in ("q", "k", "qo", "ko", "dq", "dk")
        for s in ("B", "M", "H")]


# the same block, packed in one go (2 us; the ctypes structure takes 6)
_QK_PACK = struct.Struct("@15P6if3?21q").pack
_NO_SIDE = (0,) * 15  # x, weight, output, gradients of x and weight; strides; heads


def _qk_side(fn, x, w, o, g, gw, dev, B, T, d, dt, out, backward):
    """(pointers, strides, heads) of q or of k; o: the output, or in the backward pass its gradient."""
    if x is None:
        if o is not None or g is not None or gw is not None:
            raise ValueError(f"{fn}: outputs and gradients of a tensor that is not passed")
        return _NO_SIDE
    sh = x.shape
    H = sh[1]
    if sh != (B, H, T, d) or x.dtype is not dt or x.get_device() != dev:
        raise ValueError(f"{fn}: q and k share type, device, batch, length and head_dim")
    if o is None or o.shape != sh or o.dtype is not out or o.get_device() != dev:
        raise ValueError(f"{fn}: outputs have their input's shape, and its type or fp32")
    xB, xH, xM, x1 = x.stride()
    oB, oH, oM, o1 = o.stride()
    if x1 != 1 or o1 != 1:
        raise ValueError(f"{fn}: tensors are [B, heads, T, head_dim] with a unit last-dim stride")
    wp = gp = gwp = gB = gM = gH = 0
    if w is not None:
        if w.dtype is not dt or w.shape != (d,) or w.get_device() != dev or (
                d > 1 and w.stride(0) != 1):
            raise ValueError(f"{fn}: weights are [head_dim] of the inputs' type")
        wp = w.data_ptr()
    if backward:
        if g is None or g.shape != sh or g.dtype is not dt or g.get_device() != dev:
            raise ValueError(f"{fn}: gradients have their input's shape and type")
        gB, gH, gM, g1 = g.stride()
        if g1 != 1:
            raise ValueError(f"{fn}: tensors are [B, heads, T, head_dim] with a unit last-dim stride")
        gp = g.data_ptr()
        if gw is not None:
            if gw.dtype is not _F32 or gw.shape != (d,) or gw.get_device() != dev or (
                    d > 1 and gw.stride(0) != 1):
                raise ValueError(f"{fn}: gradients of the weights are fp32 [head_dim]")
            gwp = gw.data_ptr()
    return (x.data_ptr(), wp, o.data_ptr(), gp, gwp, xB, xM, xH, oB, oM, oH, gB, gM, gH, H)


def _qk_params(fn, q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved, qo, ko,
               backward=False, dq=None, dk=None, dqw=None, dkw=None, accumulate=False) -> bytes:
    """The parameter block; qo, ko: the outputs, or in the backward pass their gradients."""
    x, o = (q, qo) if q is not None else (k, ko)
    if x is None or x.dim() != 4 or x.dtype not in _TYPE:
        raise ValueError(f"{fn}: q or k, [B, heads, T, head_dim], fp32, bf16 or fp16")
    dev = _device(fn, x)
    (B, _, T, d), dt, out = x.shape, x.dtype, None if o is None else o.dtype
    if out is not dt and out is not _F32:
        raise ValueError(f"{fn}: outputs have their input's type, or fp32")
    qp, qw, qy, qg, qgw, qB, qM, qH, qoB, qoM, qoH, qgB, qgM, qgH, hq = _qk_side(
        fn, q, q_weight, qo, dq, dqw, dev, B, T, d, dt, out, backward)
    kp, kw, ky, kg, kgw, kB, kM, kH, koB, koM, koH, kgB, kgM, kgH, nk = _qk_side(
        fn, k, k_weight, ko, dk, dkw, dev, B, T, d, dt, out, backward)
    cp = sp = pp = rows = stride = rot = pos_stride = 0
    if cos is not None or sin is not None:
        if cos is None or sin is None or cos.dim() != 2 or cos.shape != sin.shape or (
                cos.dtype is not _F32) or sin.dtype is not _F32 or cos.stride() != sin.stride() or (
                cos.get_device() != dev) or sin.get_device() != dev:
            raise ValueError(f"{fn}: cos and sin are fp32 [rows, rotary_dim / 2], laid out alike")
        rows, half = cos.shape
        stride, one = cos.stride()
        if one != 1 and half > 1:
            raise ValueError(f"{fn}: cos and sin have a unit last-dim stride")
        rot = 2 * half
        if rows == 1 and stride < half:
            stride = half
        cp, sp = cos.data_ptr(), sin.data_ptr()
    if positions is not None:
        sh, st = positions.shape, positions.stride()
        if positions.dtype is not torch.int64 or (sh != (B, T) and sh != (T,)) or (
                st[-1] != 1 and T > 1) or positions.get_device() != dev:
            raise ValueError(f"{fn}: positions are int64 [B, T] or [T]")
        pp = positions.data_ptr()
        pos_stride = st[0] if len(sh) == 2 else 0
    if backward:
        outs, grads = (0, 0), (qy, ky)
    else:
        outs, grads = (qy, ky), (0, 0)
    return _QK_PACK(qp, kp, qw, kw, cp, sp, pp, *outs, *grads, qg, kg, qgw, kgw, B, T, hq, nk, d, rot,
                    eps, interleaved, out is not dt, accumulate, rows, stride, pos_stride, qB, qM, qH,
                    kB, kM, kH, qoB, qoM, qoH, koB, koM, koH, qgB, qgM, qgH, kgB, kgM, kgH)


def qk_norm_rope_forward(q, k, cos=None, sin=None, positions=None, q_weight=None, k_weight=None,
                         eps: float = 1e-6, interleaved: bool = False, q_out=None, k_out=None,
                         out_dtype=None):
    """RMS norm of each head of q and k (either may be None) over its last dimension, times its weight,
    then the rotation of its first 2 * cos.shape[1] elements by the table rows of the tokens'
    positions (None: token t at position t). Returns (q_out, k_out) of q's type or out_dtype, which
    may be fp32 for 16-bit inputs. q_out and k_out may be q and k themselves."""
    if q_out is None and q is not None:
        q_out = q.new_empty(q.shape, dtype=out_dtype)
    if k_out is None and k is not None:
        k_out = k.new_empty(k.shape, dtype=out_dtype)
    p = _qk_params("qk_norm_rope_forward", q, k, cos, sin, positions, q_weight, k_weight, eps,
                   interleaved, q_out, k_out)
    call("hk_qk_norm_rope_forward", p, _TYPE[(q if q is not None else k).dtype], _stream())
    return q_out, k_out


def _by_token(t):
    """An empty [B, heads, T, d] tensor with the heads of a token together, as a projection has them."""
    B, H, T, d = t.shape
    return t.new_empty_strided((B, H, T, d), (T * H * d, d, H * d, 1))


def qk_norm_rope_backward(dq_out, dk_out, q, k, cos=None, sin=None, positions=None, q_weight=None,
                          k_weight=None, eps: float = 1e-6, interleaved: bool = False,
                          grad_q_weight=None, grad_k_weight=None, dq=None, dk=None,
                          accumulate: bool = True):
    """Gradients of qk_norm_rope_forward's inputs from those of its outputs: returns (dq, dk), which
    may be q, k or gradients of the same type passed in. grad_q_weight and grad_k_weight (fp32
    [head_dim]) are added to, or written where accumulate is False; None: not wanted."""
    dq = _by_token(q) if dq is None and q is not None else dq
    dk = _by_token(k) if dk is None and k is not None else dk
    p = _qk_params("qk_norm_rope_backward", q, k, cos, sin, positions, q_weight, k_weight, eps,
                   interleaved, dq_out, dk_out, True, dq, dk, grad_q_weight, grad_k_weight,
                   accumulate)
    kind = _TYPE[(q if q is not None else k).dtype]
    _call_captured("hk_qk_norm_rope_backward", lambda: lib().hk_qk_norm_rope_workspace(p, kind), p,
                   kind)
    return dq, dk


# ----------------------------------------------------------------------------------------------
# 16-bit attention over packed sequences (no counterpart in the reference)
# ----------------------------------------------------------------------------------------------
class AttnPackedParams(ctypes.Structure):
    """hk_attn_packed_params (hk.h), field for field."""

    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "k", "v", "o", "dout", "dq", "dk", "dv", "lse", "cu_q",
                                               "cu_k")] + [
        (n, ctypes.c_int) for n in ("num_seqs", "q_heads", "k_heads", "head_dim")] + [
        ("scale", ctypes.c_float), ("is_causal", ctypes.c_bool), ("q_tokens", _I64), ("k_tokens", _I64)] + [
        (f"{t}_stride{s}", _I64) for t in ("q", "k", "v", "o", "do", "dq", "dk", "dv") for s in ("M", "H")] + [
        ("lse_strideH", _I64)]


_PACKED_PACK = struct.Struct("@11P4if?19q").pack


def _heads(fn: str, t: torch.Tensor, shape, dt, dev: int) -> tuple[int, int, int]:
    """(address, token stride, head stride) of a [tokens, heads, head_dim] tensor."""
    if t.shape != shape or t.dtype is not dt or t.get_device() != dev:
        raise ValueError(f"{fn}: {dt} {list(shape)} of one device expected, {t.dtype} {list(t.shape)} given")
    m, h, one = t.stride()
    if one != 1:
        raise ValueError(f"{fn}: tensors are [tokens, heads, head_dim] with a unit last-dim stride")
    # the stride of a single token or head is never used, whatever it is
    return t.data_ptr(), m if shape[0] > 1 else 0, h if shape[1] > 1 else 0


_NO_HEADS = (0, 0, 0)


def _like(fn, t, x, sh, dt, dev):
    """An output of x's shape: the one passed in, checked, or a new contiguous one. (tensor, address, strides)"""
    if t is not None:
        return t, _heads(fn, t, sh, dt, dev)
    t = x.new_empty(sh)
    return t, (t.data_ptr(), sh[1] * sh[2], sh[2])


def _packed(fn, q, k, v, cu_q, cu_k, causal, scale, o, lse, backward=False, do=None, dq=None, dk=None, dv=None):
    """(parameter block, type, outputs)"""
    dt, qs, ks = q.dtype, q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3 or (dt is not _BF16 and dt is not torch.float16):
        raise ValueError(f"{fn}: bf16 or fp16 tensors [tokens, heads, head_dim]")
    dev = _device(fn, q)
    (tq, hq, d), (tk, hk, _) = qs, ks
    if hk == 0 or hq == 0 or hq % hk or d % 8 or not 8 <= d <= 128:
        raise ValueError(f"{fn}: key heads divide the query heads; head_dim is a multiple of 8, at most 128")
    n = cu_q.numel() - 1
    cq = ck = _starts(fn, cu_q, n, dev)
    if cu_k is not None:
        ck = _starts(fn, cu_k, n, dev)
    Q = _heads(fn, q, qs, dt, dev)
    ks = (tk, hk, d)
    K, V = _heads(fn, k, ks, dt, dev), _heads(fn, v, ks, dt, dev)
    if lse is None:
        if backward:
            raise ValueError(f"{fn}: the forward's o and lse are needed")
        lse = q.new_empty((hq, tq), dtype=_F32)
        L = lse.data_ptr(), tq
    else:
        if lse.dtype is not _F32 or lse.shape != (hq, tq) or lse.get_device() != dev or (
                lse.stride(1) != 1 and tq > 1):
            raise ValueError(f"{fn}: lse is fp32 [heads, tokens] with a unit last-dim stride")
        L = lse.data_ptr(), lse.stride(0) if hq > 1 else 0
    if backward:
        O, G = _heads(fn, o, qs, dt, dev), _heads(fn, do, qs, dt, dev)  # noqa: E741
        dq, DQ = _like(fn, dq, q, qs, dt, dev)
        dk, DK = _like(fn, dk, q, ks, dt, dev)
        dv, DV = _like(fn, dv, q, ks, dt, dev)
        outs = dq, dk, dv
    else:
        o, O = _like(fn, o, q, qs, dt, dev)  # noqa: E741
        G = DQ = DK = DV = _NO_HEADS
        outs = o, lse
    return _PACKED_PACK(Q[0], K[0], V[0], O[0], G[0], DQ[0], DK[0], DV[0], L[0], cq, ck, n, hq, hk, d,
                        d ** -0.5 if scale is None else scale, causal, tq, tk, Q[1], Q[2], K[1], K[2], V[1], V[2],
                        O[1], O[2], G[1], G[2], DQ[1], DQ[2], DK[1], DK[2], DV[1], DV[2], L[1]), _TYPE[dt], outs


def _starts(fn: str, cu: torch.Tensor, n: int, dev: int) -> int:
    """The address of the sequences' first rows, and the end of the last."""
    if cu.dtype is not torch.int32 or cu.dim() != 1 or cu.numel() != n + 1 or n < 0 or (
            cu.get_device() != dev or not cu.is_contiguous()):
        raise ValueError(f"{fn}: cu_q and cu_k are int32 [sequences + 1], contiguous, on the device")
    return cu.data_ptr()


def attn_packed_forward(q, k, v, cu_q, cu_k=None, causal: bool = True, scale: float | None = None, o=None,
                        lse=None):
    """Attention over packed sequences: q [tokens, q_heads, head_dim], k and v [key tokens, k_heads, head_dim],
    bf16 or fp16; sequence s has the queries cu_q[s] .. cu_q[s + 1] - 1 and the keys cu_k[s] .. (int32 on the device;
    None: as cu_q), and query i of m sees key j of n where j <= i + n - m, or all keys. Query head h goes with key
    head h // (q_heads / k_heads). Returns (o, lse): o like q, lse fp32 [q_heads, tokens], 0 and -inf where a
    query sees no key; rows of no sequence are not written."""
    p, kind, outs = _packed("attn_packed_forward", q, k, v, cu_q, cu_k, causal, scale, o, lse)
    _call_captured("hk_attn_packed_forward", lambda: lib().hk_attn_packed_workspace(p, kind, 0), p, kind)
    return outs


def attn_packed_backward(do, q, k, v, o, lse, cu_q, cu_k=None, causal: bool = True, scale: float | None = None,
                         dq=None, dk=None, dv=None):
    """Gradients (dq, dk, dv) of attn_packed_forward's inputs from that of its output, all of q's type. Written, not
    added to; those of rows of no sequence are not written."""
    p, kind, outs = _packed("attn_packed_backward", q, k, v, cu_q, cu_k, causal, scale, o, lse, True, do, dq, dk, dv)
    _call_captured("hk_attn_packed_backward", lambda: lib().hk_attn_packed_workspace(p, kind, 1), p, kind)
    return outs


# ----------------------------------------------------------------------------------------------
# Log probabilities of given tokens (no counterpart in the reference)
# ----------------------------------------------------------------------------------------------
class TokenLogprobs(NamedTuple):
    """What token_logprobs returns; None for what was not asked for."""

    logp: torch.Tensor
    lse: torch.Tensor
    entropy: torch.Tensor | None
    top_logp: torch.Tensor | None
    top_index: torch.Tensor | None


_WIDE = {torch.int32: 0, torch.int64: 1}


def _logits(fn: str, x: torch.Tensor, tokens: torch.Tensor) -> tuple[int, int, int, int]:
    """(device, rows, vocabulary, row stride) of logits [rows, vocabulary] and their tokens."""
    if x.dim() != 2 or x.dtype not in _TYPE or (x.shape[1] > 1 and x.stride(1) != 1):
        raise ValueError(f"{fn}: fp32, bf16 or fp16 logits [rows, vocabulary] with a unit last-dim stride")
    dev, (rows, vocab) = _device(fn, x), x.shape
    if vocab == 0:
        raise ValueError(f"{fn}: a vocabulary of one word at least")
    _tokens(fn, tokens, dev, rows)
    return dev, rows, vocab, x.stride(0) if rows > 1 else vocab


def _tokens(fn: str, t: torch.Tensor, dev: int, n: int) -> None:
    if t.dtype not in _WIDE or t.shape != (n,) or t.get_device() != dev or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{fn}: tokens are int32 or int64 [{n}], contiguous, on the device")


def _row_values(fn: str, name: str, t: torch.Tensor | None, dev: int, shape, dtype=_F32) -> int | None:
    """The address of one value (or `top` of them) a row."""
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{fn}: {name} is {dtype} {list(shape)}, contiguous, on the device")
    return t.data_ptr()


def token_logprobs(logits, tokens, entropy=False, top: int = 0, logp=None, lse=None, top_logp=None,
                   top_index=None) -> TokenLogprobs:
    """Per row of logits (fp32, bf16 or fp16 [rows, vocabulary], any row stride): the log probability of the row's
    token, the log-sum-exp, and where asked for the entropy (True, or an output) and the `top` largest log
    probabilities with their indices, falling, of equal ones the lowest index first. All fp32, indices int64."""
    fn = "token_logprobs"
    dev, rows, vocab, stride = _logits(fn, logits, tokens)
    if not 0 <= top <= min(64, vocab):
        raise ValueError(f"{fn}: top is 64 at most, and the vocabulary")
    entropy = False if entropy is None else entropy
    ent = None if entropy is True or entropy is False else entropy
    if logp is None and lse is None and ent is None:  # one allocation for all
        own = logits.new_empty((2 + entropy, rows), dtype=_F32)
        logp, lse, *more = own.unbind(0)
        ent = more[0] if more else None
        p = own.data_ptr()
        ptrs = p, p + 4 * rows, p + 8 * rows if more else None
    else:
        logp = logits.new_empty((rows,), dtype=_F32) if logp is None else logp
        lse = logits.new_empty((rows,), dtype=_F32) if lse is None else lse
        ent = logits.new_empty((rows,), dtype=_F32) if entropy is True else ent
        ptrs = (_row_values(fn, "logp", logp, dev, (rows,)), _row_values(fn, "lse", lse, dev, (rows,)),
                _row_values(fn, "entropy", ent, dev, (rows,)))
    vp = ip = None
    if top:
        top_logp = logits.new_empty((rows, top), dtype=_F32) if top_logp is None else top_logp
        top_index = logits.new_empty((rows, top), dtype=torch.int64) if top_index is None else top_index
        vp = _row_values(fn, "top_logp", top_logp, dev, (rows, top))
        ip = _row_values(fn, "top_index", top_index, dev, (rows, top), torch.int64)
    elif top_logp is not None or top_index is not None:
        raise ValueError(f"{fn}: outputs of alternatives that are not asked for")
    kind = _TYPE[logits.dtype]
    _call_captured("hk_token_logprobs", lambda: lib().hk_token_logprobs_workspace(kind, rows, vocab, top),
                   logits.data_ptr(), kind, rows, vocab, stride, tokens.data_ptr(), _WIDE[tokens.dtype], *ptrs, top, vp,
                   ip)
    return TokenLogprobs(logp, lse, ent, top_logp, top_index)


def token_logprobs_backward(logits, tokens, lse, grad_logp=None, entropy=None, grad_entropy=None, grad=None):
    """The gradient of the logits, of their type, from those of logp and of the entropy (fp32 [rows]; None: zero) and
    token_logprobs' lse and entropy. grad may be the logits themselves."""
    fn = "token_logprobs_backward"
    dev, rows, vocab, stride = _logits(fn, logits, tokens)
    grad = torch.empty((rows, vocab), device=logits.device, dtype=logits.dtype) if grad is None else grad
    if grad.dtype is not logits.dtype or grad.shape != logits.shape or grad.get_device() != dev or (
            vocab > 1 and grad.stride(1) != 1):
        raise ValueError(f"{fn}: grad has the logits' type and shape, with a unit last-dim stride")
    if lse is None or (grad_entropy is not None and entropy is None):
        raise ValueError(f"{fn}: lse, and for its gradient the entropy, are needed")
    call("hk_token_logprobs_backward", logits.data_ptr(), _TYPE[logits.dtype], rows, vocab, stride,
         tokens.data_ptr(), _WIDE[tokens.dtype], _row_values(fn, "lse", lse, dev, (rows,)),
         _row_values(fn, "entropy", entropy, dev, (rows,)), _row_values(fn, "grad_logp", grad_logp, dev, (rows,)),
         _row_values(fn, "grad_entropy", grad_entropy, dev, (rows,)), grad.data_ptr(),
         grad.stride(0) if rows > 1 else vocab, _stream())
    return grad


# ----------------------------------------------------------------------------------------------
# Embedding lookup and the table's gradient (no counterpart in the reference)
# ----------------------------------------------------------------------------------------------
def _rows_of(fn: str, name: str, t: torch.Tensor, dev: int, shape) -> tuple[int, int, int]:
    """(address, type, row stride) of a matrix."""
    if t.dtype not in _TYPE or t.shape != shape or t.get_device() != dev or (shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{fn}: {name} is fp32, bf16 or fp16 {list(shape)} with a unit last-dim stride, on the device")
    return t.data_ptr(), _TYPE[t.dtype], t.stride(0) if shape[0] > 1 else shape[1]


def embedding_forward(table, tokens, scale: float = 1.0, residual=None, out=None, out_dtype=None):
    """scale * table[tokens] + residual: table [vocabulary, d], tokens [n], residual and out [n, d]; each of fp32, bf16
    or fp16, residual of out's type (it may be out). out_dtype: of an out that is not passed (None: the table's). A
    token outside the table gives a row of NaN."""
    fn = "embedding_forward"
    if table.dim() != 2 or tokens.dim() != 1:
        raise ValueError(f"{fn}: a table [vocabulary, d] and tokens [n]")
    dev, (vocab, d), n = _device(fn, table), table.shape, tokens.shape[0]
    _tokens(fn, tokens, dev, n)
    out = torch.empty((n, d), device=table.device, dtype=out_dtype or table.dtype) if out is None else out
    tp, tt, ts = _rows_of(fn, "table", table, dev, (vocab, d))
    op, ot, os_ = _rows_of(fn, "out", out, dev, (n, d))
    rp = rs = 0
    if residual is not None:
        rp, rt, rs = _rows_of(fn, "residual", residual, dev, (n, d))
        if rt != ot:
            raise ValueError(f"{fn}: residual has out's type")
    call("hk_embedding_forward", tp, tt, vocab, d, ts, tokens.data_ptr(), _WIDE[tokens.dtype], n, scale, rp, rs, op, ot,
         os_, _stream())
    return out


def embedding_backward(grad, tokens, grad_table, scale: float = 1.0, accumulate: bool = True):
    """The table's gradient from that of embedding_forward's output: scale times the sum of grad's rows [n, d] over the
    tokens of each row of grad_table [vocabulary, d], added to it, or, where accumulate is False, written, zero for
    rows without a token. Each of fp32, bf16 or fp16; sums in fp32 and a fixed order. Returns grad_table."""
    fn = "embedding_backward"
    if grad.dim() != 2 or grad_table.dim() != 2:
        raise ValueError(f"{fn}: grad [n, d] and grad_table [vocabulary, d]")
    dev, (n, d), vocab = _device(fn, grad), grad.shape, grad_table.shape[0]
    _tokens(fn, tokens, dev, n)
    gp, gt, gs = _rows_of(fn, "grad", grad, dev, (n, d))
    tp, tt, ts = _rows_of(fn, "grad_table", grad_table, dev, (vocab, d))
    _call_captured("hk_embedding_backward", lambda: lib().hk_embedding_workspace(n, vocab, d), gp, gt, n, d, gs,
                   tokens.data_ptr(), _WIDE[tokens.dtype], scale, tp, tt, vocab, ts, accumulate)
    return grad_table


# ----------------------------------------------------------------------------------------------
# Unified reduce (kernels/reduction/unified_reduce_standalone.cu)
# ----------------------------------------------------------------------------------------------
REDUCE_INNER, REDUCE_OUTER, REDUCE_GENERIC = 0, 1, 2


class ReductionLayout(ctypes.Structure):
    """detail::ReductionLayout (unified_reduce_standalone.cu:46-56), path as int32."""

    _fields_ = [
        ("path", ctypes.c_int32),
        ("num_outputs", ctypes.c_int64),
        ("reduced_count", ctypes.c_int64),
        ("input_outer_stride", ctypes.c_int64),
        ("inner_count", ctypes.c_int64),
        ("input_row_stride", ctypes.c_int64),
    ]


def unified_reduce_sum(src: torch.Tensor, layout: ReductionLayout,
                       dst: torch.Tensor | None = None) -> torch.Tensor:
    _dev(src, dst)
    dst = torch.empty(layout.num_outputs, device=src.device, dtype=torch.float32) if dst is None else dst
    call("hk_unified_reduce_sum_f32", ctypes.byref(layout), _ptr(src), _ptr(dst), _stream())
    return dst


def reduce_generic(src: torch.Tensor, out_sizes, out_strides, red_sizes, red_strides,
                   dst: torch.Tensor | None = None) -> torch.Tensor:
    """Sum with explicit strided offset maps (the reference's OffsetCalculator pair)."""
    _dev(dst)
    if not src.is_cuda:
        raise ValueError("reduce_generic: device tensor")
    nout = 1
    for s in out_sizes:
        nout *= s
    dst = torch.empty(nout, device=src.device, dtype=torch.float32) if dst is None else dst
    a = lambda xs: (ctypes.c_int64 * max(len(xs), 1))(*xs)  # noqa: E731
    call("hk_reduce_generic_f32", _ptr(src), _ptr(dst), len(out_sizes), a(out_sizes),
         a(out_strides), len(red_sizes), a(red_sizes), a(red_strides), _stream())
    return dst
