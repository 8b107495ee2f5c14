"""Linear attention with a decay per head: host side of the gfx950 HIP path.

Where attention keeps every key and value of a sequence, linear attention keeps a state of one matrix
per KV head: with ``a`` its log decay,

    S_t = e^a S_{t-1} + k_t v_t^T        (fp32 [D, D], rows are the dims of k)
    o_t = sm_scale * q_t S_t             for every query head of the group

``linear_attention_varlen`` takes packed sequences -- prompts, chunks of prompts, single tokens -- from
their states to the states behind them, ``linear_attention_decode`` one token per sequence.  The
states of all sequences lie in one tensor of slots, updated in place.  Forward only.

Work is queued on the current stream; argument errors raise ``ArgumentError`` before any launch.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib
from .gqa import _aligned, _cu_count, _dtype_code, _require

HEAD_DIMS = (64, 128, 256)


def _check_rows(q, k, v):
    """(tokens, h_q, h_kv, d, dtype code) of a call's rows."""
    _require(q.dim() == 3 and k.dim() == 3, "q, k, v must be [tokens, heads, head_dim]")
    _require(v.shape == k.shape, "k and v shapes differ")
    total, h_q, d = q.shape
    _require(k.shape[0] == total, "q and k must have the same tokens")
    h_kv = k.shape[1]
    _require(k.shape[2] == d, "feature size of q, k, v should be equal")
    _require(d in HEAD_DIMS, f"head dim {d} not in {HEAD_DIMS}")
    _require(h_kv >= 1 and h_q >= 1 and h_q % h_kv == 0,
             "number of heads in q must be a multiple of that in k & v")
    _require(h_q * d < 1 << 23, "too many heads")
    code = _dtype_code(q.dtype)
    _require(k.dtype == q.dtype and v.dtype == q.dtype, "q, k, v dtypes differ")
    return total, h_q, h_kv, d, code


def _check_decay(log_decay, h_kv):
    _require(log_decay.dtype == torch.float32 and log_decay.shape == (h_kv,)
             and log_decay.is_contiguous(), "log_decay must be contiguous float32 [num_kv_heads]")


def _check_state(state, state_indices, num_seqs, h_kv, d):
    _require(state.dtype == torch.float32 and state.dim() == 4
             and tuple(state.shape[1:]) == (h_kv, d, d),
             "state must be float32 [num_slots, num_kv_heads, head_dim, head_dim]")
    _require(state.stride(3) == 1 and state.stride(2) == d and state.stride(0) % 4 == 0
             and state.stride(1) % 4 == 0 and state.data_ptr() % 16 == 0,
             "a head's state must be contiguous and 16-byte aligned")
    a, b = sorted((state.stride(i), state.shape[i]) for i in (0, 1))
    _require((a[1] <= 1 or a[0] >= d * d) and (b[1] <= 1 or b[0] >= d * d + max(a[1] - 1, 0) * a[0]),
             "states must not overlap")
    _require(state.shape[0] < 1 << 31, "too many slots")
    if state_indices is None:
        _require(state.shape[0] >= num_seqs, "fewer slots than sequences")
    else:
        _require(state_indices.dtype == torch.int32 and state_indices.shape == (num_seqs,)
                 and state_indices.is_contiguous(),
                 "state_indices must be contiguous int32 [num_seqs]")


def _scale(sm_scale, d):
    if sm_scale is None:
        return 1.0 / math.sqrt(d)
    _require(math.isfinite(sm_scale), "sm_scale must be finite")
    return float(sm_scale)


def _rows(q, k, v):
    """Rows that the kernels cannot read as they lie are copied (`contiguous` would keep a misaligned
    base, and any stride of a dimension of one)."""
    return (t if t.stride(2) == 1 and _aligned(t, (0, 1)) and t.stride(0) < 1 << 23
            else t.clone(memory_format=torch.contiguous_format) for t in (q, k, v))


def _args(q, k, v, log_decay, state, state_indices, out, num_seqs, scale, code):
    total, h_q, d = q.shape
    return _lib.LinearArgs(
        q=q.data_ptr(), q_stride_t=q.stride(0), q_stride_h=q.stride(1), k=k.data_ptr(),
        v=v.data_ptr(), k_stride_t=k.stride(0), k_stride_h=k.stride(1), v_stride_t=v.stride(0),
        v_stride_h=v.stride(1), log_decay=log_decay.data_ptr(), cu_seqlens=None,
        state=None if state is None else state.data_ptr(),
        state_stride_s=0 if state is None else state.stride(0),
        state_stride_h=0 if state is None else state.stride(1),
        state_indices=None if state_indices is None else state_indices.data_ptr(), has_state=None,
        out=out.data_ptr(), part=None, num_slots=0 if state is None else state.shape[0], num_seqs=num_seqs,
        total=total, h_q=h_q, h_kv=k.shape[1], d=d, segment=0, scale=scale,
        dtype=code)


def _one_device(*tensors):
    there = [t for t in tensors if t is not None]
    _require(all(t.is_cuda and t.device == there[0].device for t in there),
             "all tensors must be CUDA (HIP) tensors on one device")


def linear_attention_varlen(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    cu_seqlens: torch.Tensor,
    max_seqlen: int,
    state: Optional[torch.Tensor] = None,
    state_indices: Optional[torch.Tensor] = None,
    has_state: Optional[torch.Tensor] = None,
    sm_scale: Optional[float] = None,
) -> torch.Tensor:
    """Linear attention of packed sequences (grouped heads, fp16 or bf16, head dim 64, 128 or 256).

    q           [total, H, D]; k, v [total, H_kv, D], H a multiple of H_kv
    log_decay   fp32 [H_kv]: natural log of what a token leaves of the state before it, 0 or less
                (-inf: nothing); the query heads of a group share a state
    cu_seqlens  int32 [num_seqs + 1], up to 65535 sequences: rows cu_seqlens[s] ..
                cu_seqlens[s + 1] - 1 are the tokens of sequence s
    max_seqlen  an upper bound of the lengths; it chooses the launch, not what is computed
    state       fp32 [num_slots, H_kv, D, D], updated in place; None: every sequence starts from zeros
                and no state is kept
    state_indices
                int32 [num_seqs], the slot of each sequence; None: sequence s has slot s.  A sequence
                whose index lies outside the slots starts from zeros and its state is not kept.
                The slots of one call must differ: a state that two sequences write is undefined
    has_state   bool or uint8 [num_seqs]: sequences where it is 0 start from zeros whatever their slot
                holds; None: all start from their slots
    sm_scale    1 / sqrt(D) if None

    Returns ``o`` shaped and typed like ``q``.  States are float32 throughout.  Scores, and the copy of
    a state that meets q, are rounded to q's type for their products with v and q, so that an output is
    off by that beside its own rounding (in all 2.1e-3 of its size in bf16, 2.5e-4 to 2.9e-4 in fp16,
    for 1.7e-3 and 2.1e-4); ``linear_attention_decode`` keeps both in float32.  What a decay leaves below
    2^-126, and in fp16 weighted values below 2^-39 of the largest of their 32 tokens and dim, count as 0.

    Rows of q that belong to no sequence get 0, a
    sequence without tokens leaves its slot as it is.  An infinity or a NaN in k or v makes the
    outputs that it reaches and the state not finite (not always the infinity that the sums
    would have) while its weight is above 0 in float32, past which it may be forgotten; tokens before
    it are not touched.
    """
    fast = _lib.native()
    if fast is not None:
        o = fast.linear_varlen(q, k, v, log_decay, cu_seqlens, max_seqlen, state, state_indices,
                               has_state, sm_scale)
        if o is not None:
            return o
    total, h_q, h_kv, d, code = _check_rows(q, k, v)
    _check_decay(log_decay, h_kv)
    _require(cu_seqlens.dtype == torch.int32 and cu_seqlens.dim() == 1 and cu_seqlens.shape[0] >= 1
             and cu_seqlens.is_contiguous(), "cu_seqlens must be contiguous int32 [num_seqs + 1]")
    num_seqs = cu_seqlens.shape[0] - 1
    _require(isinstance(max_seqlen, int) and max_seqlen >= 0, "max_seqlen must be an int >= 0")
    _require(total <= (1 << 31) - 257, "too many tokens")
    _require(num_seqs <= 65535 and num_seqs * h_kv < 1 << 22, "too many sequences or heads")
    if state is not None:
        _check_state(state, state_indices, num_seqs, h_kv, d)
    else:
        _require(state_indices is None and has_state is None,
                 "state_indices and has_state need a state")
    if has_state is not None:
        _require(has_state.dtype in (torch.bool, torch.uint8) and has_state.shape == (num_seqs,)
                 and has_state.is_contiguous(), "has_state must be contiguous bool [num_seqs]")
    scale = _scale(sm_scale, d)
    _one_device(q, k, v, log_decay, cu_seqlens, state, state_indices, has_state)
    q, k, v = _rows(q, k, v)
    o = torch.empty((total, h_q, d), dtype=q.dtype, device=q.device)
    if total > 0:
        args = _args(q, k, v, log_decay, state, state_indices, o, num_seqs, scale, code)
        args.cu_seqlens = cu_seqlens.data_ptr()
        args.has_state = None if has_state is None else has_state.data_ptr()
        lib = _lib.load()
        floats = lib.fa_linear_plan(ctypes.byref(args), min(max_seqlen, total), _cu_count(q.device))
        _lib.check(min(floats, 0))
        with torch.cuda.device(q.device):
            part = torch.empty(floats, dtype=torch.float32, device=q.device) if floats > 0 else None
            args.part = None if part is None else part.data_ptr()
            _lib.check(lib.fa_linear_prompt(ctypes.byref(args),
                                            torch.cuda.current_stream(q.device).cuda_stream))
    return o


def linear_attention_decode(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    state: torch.Tensor,
    state_indices: Optional[torch.Tensor] = None,
    sm_scale: Optional[float] = None,
) -> torch.Tensor:
    """One token of linear attention per sequence (as ``linear_attention_varlen`` with lengths of one).

    q              fp16 or bf16 [num_seqs, H, D]; k, v [num_seqs, H_kv, D]
    log_decay      fp32 [H_kv]
    state          fp32 [num_slots, H_kv, D, D], updated in place
    state_indices  int32 [num_seqs], the slot of each sequence; None: sequence s has slot s.  A row
                   whose index lies outside the slots (the padding of a captured step) gets 0 and
                   touches no state.  The slots of one call must differ

    Returns ``o`` shaped and typed like ``q``.
    """
    fast = _lib.native()
    if fast is not None:
        o = fast.linear_decode(q, k, v, log_decay, state, state_indices, sm_scale)
        if o is not None:
            return o
    num_seqs, h_q, h_kv, d, code = _check_rows(q, k, v)
    _check_decay(log_decay, h_kv)
    _require(num_seqs <= 65535 and num_seqs * h_kv < 1 << 22, "too many sequences or heads")
    _check_state(state, state_indices, num_seqs, h_kv, d)
    scale = _scale(sm_scale, d)
    _one_device(q, k, v, log_decay, state, state_indices)
    q, k, v = _rows(q, k, v)
    if state.shape[0] == 0:
        return torch.zeros((num_seqs, h_q, d), dtype=q.dtype, device=q.device)
    o = torch.empty((num_seqs, h_q, d), dtype=q.dtype, device=q.device)
    if num_seqs > 0:
        args = _args(q, k, v, log_decay, state, state_indices, o, num_seqs, scale, code)
        lib = _lib.load()
        with torch.cuda.device(q.device):
            _lib.check(lib.fa_linear_token(ctypes.byref(args),
                                           torch.cuda.current_stream(q.device).cuda_stream))
    return o
