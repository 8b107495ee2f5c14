"""A paged K/V cache in 4 bits: host side of the gfx950 HIP path.

Four tensors make the cache, codes and scales of K and of V:

* ``key_cache``, ``value_cache``    uint8 ``[num_blocks, H_kv, block_size, D / 2]``: e2m1 codes (a
  sign bit over the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6), dim 2i in the low half of byte i;
* ``key_scales``, ``value_scales``  uint8 ``[num_blocks, H_kv, block_size, D / 32]``: byte e
  scales its 32 dims by 2^(e - 127); 255 makes them NaN.

``cache_kv_mxfp4`` writes new tokens, ``gather_kv_mxfp4`` reads whole contexts back (what
``flash_attention_varlen`` takes for the next chunk of a prompt), ``paged_attention_mxfp4`` is
``paged_attention`` over this cache.  Work is queued on the current stream; argument errors raise
``ArgumentError`` before any launch.
"""
from __future__ import annotations

import ctypes
import math
from typing import Tuple

import torch

from . import _lib
from .gqa import TILE_TOKENS, _aligned, _cu_count, _dtype_code, _next_pow2, _require

HEAD_DIMS = (64, 128, 256)
GROUP = 32
# a launch has fewer than 2^24 work-groups, of up to 16 tokens in the writer and the reader
MAX_TOKENS = (1 << 28) - 16


def _check_cache(key_cache, key_scales, value_cache, value_scales):
    """(num_blocks, h_kv, block_size, d) of a cache."""
    _require(key_cache.dim() == 4 and value_cache.shape == key_cache.shape,
             "key_cache / value_cache must be [num_blocks, num_kv_heads, block_size, head_size / 2]")
    num_blocks, h_kv, block_size, half = key_cache.shape
    d = 2 * half
    _require(d in HEAD_DIMS, f"head_size={d} not in {HEAD_DIMS}")
    _require(key_scales.shape == (num_blocks, h_kv, block_size, d // GROUP)
             and value_scales.shape == key_scales.shape,
             "key_scales / value_scales must be [num_blocks, num_kv_heads, block_size, "
             "head_size / 32]")
    tensors = (key_cache, key_scales, value_cache, value_scales)
    _require(all(t.dtype == torch.uint8 for t in tensors), "the cache must be uint8")
    _require(1 <= num_blocks < 1 << 31 and 1 <= h_kv <= 65535,
             "the cache is empty or has too many blocks or heads")
    _require(16 <= block_size < 1 << 31 and block_size & (block_size - 1) == 0,
             "block_size must be a power of two of at least 16")
    _require(value_cache.stride() == key_cache.stride()
             and value_scales.stride() == key_scales.stride(),
             "the V cache must have the same strides as the K cache")
    _require(key_cache.stride(3) == 1 and key_scales.stride(3) == 1, "head dims must be contiguous")
    code_align, scale_align = min(16, d // 8), max(1, d // 128)
    _require(all(t.data_ptr() % n == 0 and all(t.stride(i) % n == 0 for i in range(3))
                 for t, n in ((key_cache, code_align), (value_cache, code_align),
                              (key_scales, scale_align), (value_scales, scale_align))),
             f"rows of codes must be {code_align}-byte aligned, rows of scales "
             f"{scale_align}-byte aligned")
    _require(key_cache.stride(2) < 1 << 27 and key_scales.stride(2) < 1 << 27,
             "the cache's rows are too far apart")
    return num_blocks, h_kv, block_size, d


def _check_device(*tensors):
    _require(all(t.is_cuda and t.device == tensors[0].device for t in tensors),
             "all tensors must be CUDA (HIP) tensors on one device")


def _cache_args(key_cache, key_scales, value_cache, value_scales) -> "_lib.Mxfp4Cache":
    num_blocks, h_kv, block_size, half = key_cache.shape
    return _lib.Mxfp4Cache(
        k_codes=key_cache.data_ptr(), k_scales=key_scales.data_ptr(),
        v_codes=value_cache.data_ptr(), v_scales=value_scales.data_ptr(),
        code_stride_0=key_cache.stride(0), code_stride_h=key_cache.stride(1),
        code_stride_t=key_cache.stride(2), scale_stride_0=key_scales.stride(0),
        scale_stride_h=key_scales.stride(1), scale_stride_t=key_scales.stride(2),
        num_blocks=num_blocks, block_size=block_size, h_kv=h_kv, d=2 * half)


def cache_kv_mxfp4(
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    key_scales: torch.Tensor,
    value_cache: torch.Tensor,
    value_scales: torch.Tensor,
    slot_mapping: torch.Tensor,
) -> None:
    """Write new tokens into the 4-bit cache (in place).

    key, value    fp16 or bf16 [T, H_kv, D]
    slot_mapping  int32 / int64 [T]: block * block_size + row of each token; negative slots
                  (padding tokens) and slots past the cache are skipped.  The slots of one call
                  must differ: rows that two tokens write are undefined

    Each group of 32 dims gets the smallest power of two with amax <= 7 * scale (at least 2^-127),
    so that no code is off by more than half of the widest step, and codes of x / scale rounded to
    nearest, ties to the even code.  A group with a NaN or an infinity becomes NaN as a whole.
    """
    fast = _lib.native()
    if fast is not None and fast.mxfp4_write(key, value, key_cache, key_scales, value_cache,
                                             value_scales, slot_mapping):
        return
    _require(key.dim() == 3 and value.shape == key.shape,
             "key / value must be [num_tokens, num_kv_heads, head_size]")
    code = _dtype_code(key.dtype)
    _require(value.dtype == key.dtype, "key / value dtypes differ")
    _, h_kv, _, d = _check_cache(key_cache, key_scales, value_cache, value_scales)
    t = key.shape[0]
    _require(tuple(key.shape[1:]) == (h_kv, d), "key / value heads or head size differ from the cache's")
    _require(slot_mapping.dim() == 1 and slot_mapping.shape[0] == t
             and slot_mapping.dtype in (torch.int32, torch.int64),
             "slot_mapping must be int32 / int64 [num_tokens]")
    _require(t * h_kv < 1 << 31 and t <= MAX_TOKENS, "too many tokens")
    _check_device(key, value, key_cache, key_scales, value_cache, value_scales, slot_mapping)
    if t == 0:
        return
    # not 16-byte aligned rows are copied (`contiguous` would keep a misaligned base)
    key, value = (x if x.stride(2) == 1 and _aligned(x, (0, 1))
                  else x.clone(memory_format=torch.contiguous_format) for x in (key, value))
    slots = slot_mapping.contiguous()
    args = _cache_args(key_cache, key_scales, value_cache, value_scales)
    lib = _lib.load()
    with torch.cuda.device(key.device):
        _lib.check(lib.fa_mxfp4_cache_write(
            ctypes.byref(args), key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(),
            value.stride(0), value.stride(1), slots.data_ptr(),
            int(slots.dtype == torch.int64), t, code,
            torch.cuda.current_stream(key.device).cuda_stream))


def gather_kv_mxfp4(
    key_cache: torch.Tensor,
    key_scales: torch.Tensor,
    value_cache: torch.Tensor,
    value_scales: torch.Tensor,
    block_tables: torch.Tensor,
    cu_seqlens: torch.Tensor,
    total_tokens: int,
    dtype: torch.dtype,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Read contexts back from the 4-bit cache as packed rows.

    block_tables  int32 [num_seqs, max_num_blocks_per_seq], as in ``paged_attention``
    cu_seqlens    int32 [num_seqs + 1], up to 65535 sequences: row cu_seqlens[s] + j of the result
                  is token j of sequence s
    total_tokens  rows of the result (cu_seqlens[-1], or more: rows behind it are zeros, as are
                  those of blocks outside the cache)

    Returns ``(key, value)``, each ``dtype`` (fp16 or bf16) ``[total_tokens, H_kv, D]``, the cache's
    values rounded to it: past fp16's range they are infinities (also what was written as more than
    57344, whose code is 4 * 2^14; ``paged_attention_mxfp4`` takes those as they are).  So are, here and
    there, those past bf16's (written as more than 1.75 * 2^127).
    """
    fast = _lib.native() if dtype in (torch.float16, torch.bfloat16) else None
    if fast is not None:
        done = fast.mxfp4_gather(key_cache, key_scales, value_cache, value_scales, block_tables,
                                 cu_seqlens, total_tokens, dtype == torch.bfloat16)
        if done is not None:
            return done
    code = _dtype_code(dtype)
    device = key_cache.device
    _, h_kv, _, d = _check_cache(key_cache, key_scales, value_cache, value_scales)
    _require(cu_seqlens.dtype == torch.int32 and cu_seqlens.dim() == 1 and cu_seqlens.shape[0] >= 1
             and cu_seqlens.is_contiguous(), "cu_seqlens must be contiguous int32 [num_seqs + 1]")
    num_seqs = cu_seqlens.shape[0] - 1
    _require(block_tables.dtype == torch.int32 and block_tables.dim() == 2
             and block_tables.shape[0] == num_seqs and block_tables.stride(1) == 1,
             "block_tables must be int32 [num_seqs, max_num_blocks_per_seq]")
    _require(isinstance(total_tokens, int) and total_tokens >= 0, "total_tokens must be an int >= 0")
    _require(total_tokens * h_kv < 1 << 31 and total_tokens <= MAX_TOKENS, "too many tokens")
    _require(num_seqs <= 65535, "too many sequences")
    _check_device(key_cache, key_scales, value_cache, value_scales, block_tables, cu_seqlens)
    k = torch.empty((total_tokens, h_kv, d), dtype=dtype, device=device)
    v = torch.empty_like(k)
    if total_tokens > 0:
        args = _cache_args(key_cache, key_scales, value_cache, value_scales)
        lib = _lib.load()
        with torch.cuda.device(device):
            _lib.check(lib.fa_mxfp4_gather(
                ctypes.byref(args), block_tables.data_ptr(), block_tables.stride(0),
                block_tables.shape[1], cu_seqlens.data_ptr(), num_seqs, total_tokens, k.data_ptr(),
                v.data_ptr(), code, torch.cuda.current_stream(device).cuda_stream))
    return k, v


def paged_attention_mxfp4(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    key_scales: torch.Tensor,
    value_cache: torch.Tensor,
    value_scales: torch.Tensor,
    context_lens: torch.Tensor,
    block_tables: torch.Tensor,
    attn_scale: float,
    max_context_len: int,
    num_splits: int = 0,
) -> torch.Tensor:
    """``paged_attention`` over the 4-bit cache: one query token per sequence.

    query         fp16 or bf16 [num_seqs, H, D], H a multiple of H_kv
    context_lens  int32 [num_seqs]; block_tables int32 [num_seqs, max_num_blocks_per_seq]: token
                  j of sequence s is row ``j % block_size`` of block
                  ``block_tables[s, j // block_size]``; a block outside the cache reads as masked
                  keys
    max_context_len
                  a bound of the lengths.  It chooses the launch, not the result, and is worth
                  keeping close: past it nothing is split any further, and under a loose one short
                  contexts lie in one split (20.7 us at the bound, 21.6 at twice that, 31.6 at 32 times
                  it, for 32 ragged contexts of up to 4,096 keys)
    num_splits    0 picks the split count, 1 disables splitting, s > 1 uses partitions of
                  ``next_pow2(cdiv(max_context_len, s))`` tokens, at least 32

    Returns ``out`` shaped and typed like ``query``; a sequence without keys gets 0.
    """
    fast = _lib.native()
    if fast is not None:
        done = fast.mxfp4_decode(query, key_cache, key_scales, value_cache, value_scales,
                                 context_lens, block_tables, attn_scale, max_context_len, num_splits)
        if done is not None:
            return done
    _require(query.dim() == 3, "query must be [num_seqs, num_heads, head_size]")
    num_seqs, h_q, d = query.shape
    code = _dtype_code(query.dtype)
    device = query.device
    _, h_kv, _, d_k = _check_cache(key_cache, key_scales, value_cache, value_scales)
    _require(d == d_k, f"query head_size {d} != cache head_size {d_k}")
    _require(h_q >= 1 and h_q % h_kv == 0, "num_heads must be a multiple of num_kv_heads")
    _require(query.stride(2) == 1 and _aligned(query, (0, 1)), "query rows must be 16-byte aligned")
    _require(context_lens.dtype == torch.int32 and context_lens.shape == (num_seqs,)
             and context_lens.is_contiguous(), "context_lens must be contiguous int32 [num_seqs]")
    _require(block_tables.dtype == torch.int32 and block_tables.dim() == 2
             and block_tables.shape[0] == num_seqs and block_tables.stride(1) == 1,
             "block_tables must be int32 [num_seqs, max_num_blocks_per_seq]")
    _require(num_seqs <= 65535 and h_kv * -(-(h_q // h_kv) // 16) <= 65535,
             "too many sequences or heads")
    _require(num_splits >= 0, "num_splits must be >= 0")
    _require(1 <= max_context_len <= 1 << 30, "max_context_len must be in [1, 2^30]")
    _require(math.isfinite(attn_scale), "attn_scale must be finite")
    _check_device(query, key_cache, key_scales, value_cache, value_scales, context_lens, block_tables)
    out = torch.empty((num_seqs, h_q, d), dtype=query.dtype, device=device)
    if num_seqs == 0:
        return out
    if block_tables.shape[1] == 0:
        return out.zero_()
    args = _lib.Mxfp4DecodeArgs(
        cache=_cache_args(key_cache, key_scales, value_cache, value_scales), q=query.data_ptr(),
        q_stride_b=query.stride(0), q_stride_h=query.stride(1),
        block_table=block_tables.data_ptr(), bt_stride_b=block_tables.stride(0),
        max_blocks_per_seq=block_tables.shape[1], seqlens=context_lens.data_ptr(),
        out=out.data_ptr(), o_stride_b=out.stride(0), o_stride_h=out.stride(1), o_part=None,
        lse_part=None, batch=num_seqs, h_q=h_q, num_splits=1, split_tokens=1,
        scale=float(attn_scale), dtype=code)
    lib = _lib.load()
    if num_splits == 0:
        _lib.check(lib.fa_mxfp4_decode_plan(num_seqs, h_q, h_kv, d, max_context_len,
                                            _cu_count(device), ctypes.byref(args)))
    elif num_splits > 1:
        args.split_tokens = max(TILE_TOKENS, _next_pow2(-(-max_context_len // num_splits)))
        args.num_splits = -(-max_context_len // args.split_tokens)
    s = args.num_splits
    _require(s == 1 or num_seqs * h_q < 1 << 24, "too many query rows for splits")
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream(device).cuda_stream
        if s > 1:
            part = torch.empty(num_seqs * h_q * s * (d + 1), dtype=torch.float32, device=device)
            args.o_part = part.data_ptr()
            args.lse_part = part.data_ptr() + 4 * num_seqs * h_q * s * d
        _lib.check(lib.fa_mxfp4_decode(ctypes.byref(args), stream))
        if s > 1:
            _lib.check(lib.fa_mxfp4_combine(ctypes.byref(args), stream))
    return out
