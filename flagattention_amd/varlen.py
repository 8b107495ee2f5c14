"""Prompt attention over packed sequences: host side of the gfx950 HIP path.

``flash_attention_varlen`` is ``flash_attention`` for sequences of different lengths without
padding: the tokens of all sequences lie one after the other in ``q [total_q, H, D]`` and
``k, v [total_k, H_kv, D]``, and ``cu_seqlens_q`` / ``cu_seqlens_k`` hold where each begins.  A
sequence may bring fewer new tokens than it has keys (a chunk of a prompt behind its prefix, a
single token), and causal masking is bottom-right aligned in each, as in ``flash_attention``.

The starts live on the device and are not read by the host, so the host plans with bounds: a
work-group finds its sequence itself.  Work is queued on the current stream; argument errors raise
``ArgumentError`` before any launch.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib
from .gqa import _aligned, _cu_count, _dtype_code, _require

HEAD_DIMS = (64, 128, 256)


def flash_attention_varlen(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: torch.Tensor,
    max_seqlen_q: int,
    max_seqlen_k: int,
    causal: bool = False,
    sm_scale: Optional[float] = None,
    return_log_normalizer: bool = False,
):
    """Attention of packed sequences (grouped heads, fp16 or bf16, head dim 64, 128 or 256).

    q             [total_q, H, D]; k, v [total_k, H_kv, D], H a multiple of H_kv
    cu_seqlens_q  int32 [num_seqs + 1], up to 65535 sequences: rows cu_seqlens_q[s] ..
                  cu_seqlens_q[s + 1] - 1 of q are the tokens of sequence s; cu_seqlens_k likewise
                  for the keys
    max_seqlen_q, max_seqlen_k
                  upper bounds of the lengths; they choose the launch, not the result.  One split
                  count holds for the whole launch, 1 where its rows fill the CUs: a single token of
                  a very long context beside a large chunk is then one work-group's walk (131,072
                  keys 1.46 ms, 0.11 in a call of its own)
    causal        token i of m sees keys <= n - m + i of its n

    Returns ``o`` shaped and typed like ``q``, with ``return_log_normalizer`` the pair ``(o, L)``,
    ``L`` the fp32 natural-log normaliser ``[H, total_q]``.  Tokens that see no key, and rows of
    q that belong to no sequence, get o = 0, L = -inf.
    """
    fast = _lib.native()
    if fast is not None:
        done = fast.varlen(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, causal,
                           sm_scale, return_log_normalizer)
        if done is not None:
            return done
    _require(q.dim() == 3 and k.dim() == 3, "q, k, v must be [tokens, heads, head_dim]")
    _require(v.shape == k.shape, "k and v shapes differ")
    total_q, h_q, d = q.shape
    total_k, h_kv, d_k = k.shape
    _require(d == d_k, "feature size of q, k, v should be equal")
    _require(d in HEAD_DIMS, f"head dim {d} not in {HEAD_DIMS}")
    _require(h_kv >= 1 and h_q >= 1 and h_q % h_kv == 0,
             "number of heads in q must be a multiple of that in k & v")
    _require(h_q * d < 1 << 23, "too many heads")
    code = _dtype_code(q.dtype)
    _require(k.dtype == q.dtype and v.dtype == q.dtype, "q, k, v dtypes differ")
    _require(cu_seqlens_q.dtype == torch.int32 and cu_seqlens_q.dim() == 1
             and cu_seqlens_q.shape[0] >= 1 and cu_seqlens_q.is_contiguous(),
             "cu_seqlens_q must be contiguous int32 [num_seqs + 1]")
    _require(cu_seqlens_k.dtype == torch.int32 and cu_seqlens_k.shape == cu_seqlens_q.shape
             and cu_seqlens_k.is_contiguous(),
             "cu_seqlens_k must be contiguous int32 [num_seqs + 1]")
    num_seqs = cu_seqlens_q.shape[0] - 1
    _require(isinstance(max_seqlen_q, int) and isinstance(max_seqlen_k, int)
             and max_seqlen_q >= 0 and max_seqlen_k >= 0,
             "max_seqlen_q and max_seqlen_k must be ints >= 0")
    _require(total_q * (h_q // h_kv) < 1 << 30 and total_k <= (1 << 31) - 257,
             "too many tokens")
    # the work-groups of a launch, 128 rows of a KV head each: every sequence, and the rows of none,
    # round up once
    _require(num_seqs <= 65535 and (total_q * (h_q // h_kv) // 128 + num_seqs + 2)
             * h_kv < 1 << 24, "too many query rows or sequences")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(d)
    _require(math.isfinite(sm_scale), "sm_scale must be finite")
    _require(all(t.is_cuda and t.device == q.device for t in (q, k, v, cu_seqlens_q,
                                                              cu_seqlens_k)),
             "all tensors must be CUDA (HIP) tensors on one device")
    # rows that the kernel cannot read as they lie are copied: past 32-bit offsets inside a tile of
    # keys and inside a block of rows (and its heads), or not 16-byte aligned (`contiguous` would keep
    # a misaligned base, and any stride of a dimension of one)
    q, k, v = (t if t.stride(2) == 1 and _aligned(t, (0, 1)) and t.stride(0) < 1 << 23
               and h_q // h_kv * t.stride(1) < 1 << 29
               else t.clone(memory_format=torch.contiguous_format) for t in (q, k, v))
    device = q.device
    o = torch.empty((total_q, h_q, d), dtype=q.dtype, device=device)
    lse = (torch.empty((h_q, total_q), dtype=torch.float32, device=device)
           if return_log_normalizer else None)
    if total_q > 0:
        args = _lib.VarlenArgs(
            q=q.data_ptr(), q_stride_t=q.stride(0), q_stride_h=q.stride(1), k=k.data_ptr(),
            v=v.data_ptr(), k_stride_t=k.stride(0), k_stride_h=k.stride(1),
            v_stride_t=v.stride(0), v_stride_h=v.stride(1),
            cu_seqlens_q=cu_seqlens_q.data_ptr(), cu_seqlens_k=cu_seqlens_k.data_ptr(),
            out=o.data_ptr(), o_stride_t=o.stride(0), o_stride_h=o.stride(1),
            lse=None if lse is None else lse.data_ptr(), o_part=None, lse_part=None,
            num_seqs=num_seqs, total_q=total_q, total_k=total_k, h_q=h_q, h_kv=h_kv, d=d,
            num_splits=1, split_tokens=1, scale=float(sm_scale),
            causal=int(bool(causal)), dtype=code)
        lib = _lib.load()
        _lib.check(lib.fa_varlen_plan(ctypes.byref(args), min(max_seqlen_q, total_q),
                                      min(max_seqlen_k, total_k), _cu_count(device)))
        s = args.num_splits
        with torch.cuda.device(device):
            stream = torch.cuda.current_stream(device).cuda_stream
            if s > 1:
                part = torch.empty(h_q * total_q * s * (d + 1), dtype=torch.float32, device=device)
                args.o_part = part.data_ptr()
                args.lse_part = part.data_ptr() + 4 * h_q * total_q * s * d
            _lib.check(lib.fa_varlen_attention(ctypes.byref(args), stream))
            if s > 1:
                _lib.check(lib.fa_varlen_combine(ctypes.byref(args), stream))
    return (o, lse) if return_log_normalizer else o
