"""Rotary positions: host side of the gfx950 HIP path.

Pair i of a head -- dims ``i`` and ``i + R/2``, or ``2i`` and ``2i + 1`` -- turns by the angle
``position * inv_freq[i]``; the first ``R = 2 * len(inv_freq)`` dims turn, the others stay.  A token
has one position, or one on each of up to four axes (time, height, width of images and video): every
pair takes one axis, by the ``sections``.

``rotary_embedding`` turns q and k, for any of the attention operators here; ``rotary_cache_kv`` turns
q and writes the turned k and v into the paged 16-bit cache that ``paged_attention`` reads (and returns
the turned k for attention over a packed prompt).  Angles are worked out in 64 bits from
the positions as they are, so there is no table and no last position; with frequencies up to 1 they are
off by 2^-20 of a radian at most up to positions of 2^31, and twice as much for every doubling past
that.  Forward only.

Work is queued on the current stream; argument errors raise ``ArgumentError`` before any launch.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .gqa import _dtype_code, _require

MAX_AXES = 4
MAX_HEAD_DIM = 4096


def _check_turn(tokens, d, positions, inv_freq, sections, mixed_sections):
    """(pairs, sections) of a call."""
    _require(inv_freq.dtype == torch.float32 and inv_freq.dim() == 1 and inv_freq.is_contiguous(),
             "inv_freq must be contiguous float32 [pairs]")
    pairs = inv_freq.shape[0]
    _require(1 <= pairs and 2 * pairs <= d <= MAX_HEAD_DIM,
             f"{pairs} pairs do not fit head dim {d} (at most {MAX_HEAD_DIM})")
    _require(positions.dtype in (torch.int32, torch.int64), "positions must be int32 or int64")
    if sections is None:
        _require(positions.shape == (tokens,) and positions.is_contiguous(),
                 "positions must be contiguous [num_tokens]")
        _require(not mixed_sections, "mixed_sections needs sections")
        return pairs, (pairs,)
    sections = tuple(sections)
    _require(1 <= len(sections) <= MAX_AXES
             and all(isinstance(n, int) and n >= 0 for n in sections) and sum(sections) == pairs,
             f"sections must be 1 to {MAX_AXES} ints >= 0 that sum to {pairs}")
    _require(positions.shape == (len(sections), tokens)
             and (tokens <= 1 or positions.stride(1) == 1),
             "positions must be [len(sections), num_tokens], tokens contiguous")
    if mixed_sections:
        axes = len(sections)
        _require(all(n == 0 or (n - 1) * axes + a < pairs for a, n in enumerate(sections) if a > 0),
                 "sections do not fit when they are mixed")
    return pairs, sections


def _apart(x, row_dims) -> bool:
    """Whether no two rows of x share an element: every dimension steps past the ones inside it."""
    reach = x.shape[-1]
    for stride, size in sorted((x.stride(i), x.shape[i]) for i in row_dims):
        if size > 1:
            if stride < reach:
                return False
            reach += (size - 1) * stride
    return True


def _span(x):
    """The bytes from x's first element to its last."""
    first = x.data_ptr()
    last = sum((n - 1) * s for n, s in zip(x.shape, x.stride()))
    return (first, first + (last + 1) * x.element_size()) if x.numel() > 0 else (first, first)


def _reach_into(x, y) -> bool:
    a, b = _span(x), _span(y)
    return a[0] < b[1] and b[0] < a[1]


def _meet(x, y) -> bool:
    """Whether two views of one type may share an element: no where their spans lie apart, or their rows
    within every stride that they have in common (heads of one packed row, caches block by block).  Each
    view's own rows lie apart (_apart)."""
    if not _reach_into(x, y):
        return False
    delta, off = divmod(y.data_ptr() - x.data_ptr(), x.element_size())
    if off != 0:
        return True

    def reach(dims):
        return x.shape[-1] + sum((n - 1) * s for s, n in dims)

    def meet(delta, xs, ys):  # y starts delta elements behind x; (stride, size) of the rows, outermost first
        if delta >= reach(xs) or delta + reach(ys) <= 0:
            return False
        if not xs and not ys:
            return True
        step = max(d[0][0] for d in (xs, ys) if d)
        xs, ys = (d[1:] if d and d[0][0] == step else d for d in (xs, ys))
        if max(reach(xs), reach(ys)) > step:
            return True
        # what is left of each fits a step: only the copies next to each other can meet
        return meet(delta % step, xs, ys) or meet(delta % step - step, xs, ys)

    return meet(delta, *(sorted(((s, n) for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1),
                                reverse=True) for t in (x, y)))


def _one_device(*tensors):
    _require(all(t.is_cuda and t.device == tensors[0].device for t in tensors),
             "all tensors must be CUDA (HIP) tensors on one device")


def _dense(x):
    return x if x.stride(2) == 1 else x.contiguous()


def _args(q, k, q_out, positions, inv_freq, sections, mixed_sections, adjacent_pairs, code):
    return _lib.RotaryArgs(
        q=q.data_ptr(), q_stride_t=q.stride(0), q_stride_h=q.stride(1), k=k.data_ptr(),
        k_stride_t=k.stride(0), k_stride_h=k.stride(1), q_out=q_out.data_ptr(),
        q_out_stride_t=q_out.stride(0), q_out_stride_h=q_out.stride(1),
        positions=positions.data_ptr(),
        pos_stride_a=positions.stride(0) if positions.dim() == 2 else 0,
        inv_freq=inv_freq.data_ptr(), tokens=q.shape[0], h_q=q.shape[1], h_kv=k.shape[1],
        d=q.shape[2], pairs=inv_freq.shape[0], axes=len(sections),
        sections=(ctypes.c_int32 * MAX_AXES)(*sections), mixed=int(bool(mixed_sections)),
        adjacent=int(bool(adjacent_pairs)), pos64=int(positions.dtype == torch.int64), dtype=code)


def _check_heads(q, k, kv_rows=2):
    _require(q.dim() == 3 and k.dim() == 3 and k.shape[0] == q.shape[0]
             and k.shape[2] == q.shape[2], "q and k must be [num_tokens, heads, head_dim]")
    _require(1 <= q.shape[1] <= 65535 and 1 <= k.shape[1] <= 65535, "no heads or too many")
    code = _dtype_code(q.dtype)
    _require(k.dtype == q.dtype, "q and k dtypes differ")
    # a thread for at least a pair of four rows; what is taken 16 bytes at a time needs an eighth
    _require(q.shape[0] * -(-(q.shape[1] + kv_rows * k.shape[1] + 3) // 4) * (q.shape[2] // 2 + 1)
             < (1 << 31) - 1024, "too many tokens or heads")
    return code


def rotary_embedding(
    q: torch.Tensor,
    k: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    sections: Optional[Sequence[int]] = None,
    mixed_sections: bool = False,
    adjacent_pairs: bool = False,
    inplace: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Turn q and k by their tokens' positions.

    q          fp16 or bf16 [T, H, D]; k [T, H_kv, D]; any strides
    positions  int32 / int64 [T], or with ``sections`` [len(sections), T]
    inv_freq   fp32 [R/2], R <= D: the angle per position of each pair
    sections   pairs of each axis, up to four, which sum to R/2: the first ``sections[0]`` pairs take
               axis 0, the next ``sections[1]`` axis 1, ...; with ``mixed_sections`` pair i takes axis
               ``i % axes`` as long as that axis has its number, and axis 0 from there on
    adjacent_pairs
               pairs are dims 2i and 2i + 1 instead of i and i + R/2
    inplace    write into q and k themselves (their rows must not overlap, nor the two each other, which
               is refused: views of one packed projection are fine)

    Returns ``(q, k)``, turned.
    """
    fast = _lib.native()
    if fast is not None:
        both = fast.rotary(q, k, positions, inv_freq, sections, mixed_sections, adjacent_pairs,
                           inplace)
        if both is not None:
            return both
    code = _check_heads(q, k)
    _, sections = _check_turn(q.shape[0], q.shape[2], positions, inv_freq, sections, mixed_sections)
    if inplace:
        _require(all(x.stride(2) == 1 and _apart(x, (0, 1)) for x in (q, k)),
                 "q and k must have contiguous rows that do not overlap")
        _require(not _meet(q, k), "q and k overlap")
    _one_device(q, k, positions, inv_freq)
    if inplace:
        q_out, k_out = q, k
    else:
        q, k = _dense(q), _dense(k)
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    if q.shape[0] > 0:
        args = _args(q, k, q_out, positions, inv_freq, sections, mixed_sections, adjacent_pairs,
                     code)
        args.k_out, args.k_out_stride_t, args.k_out_stride_h = (k_out.data_ptr(), k_out.stride(0),
                                                                k_out.stride(1))
        lib = _lib.load()
        with torch.cuda.device(q.device):
            _lib.check(lib.fa_rotary(ctypes.byref(args),
                                     torch.cuda.current_stream(q.device).cuda_stream))
    return q_out, k_out


def rotary_cache_kv(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    sections: Optional[Sequence[int]] = None,
    mixed_sections: bool = False,
    adjacent_pairs: bool = False,
    return_key: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Turn q and k by their tokens' positions, and write k and v into the paged cache (in place).

    q, k, positions, inv_freq, sections, mixed_sections, adjacent_pairs
                  as in ``rotary_embedding``; v [T, H_kv, D]
    key_cache, value_cache
                  [num_blocks, H_kv, block_size, D] of q's type, as in ``paged_attention``; they share no
                  element with each other (views of one pool are fine), and no memory with q, k and v
    slot_mapping  int32 / int64 [T]: block * block_size + row of each token; negative slots (padding
                  tokens) and slots past the cache are skipped.  The slots of one call must differ:
                  rows that two tokens write are undefined
    return_key    return the turned k too, also of tokens without a slot

    Returns the turned ``q``, ready for ``paged_attention``; with ``return_key`` ``(q, k)``, both turned,
    as ``flash_attention_varlen`` takes them with the packed v of a prompt.
    """
    fast = _lib.native()
    if fast is not None:
        done = fast.rotary_cache(q, k, v, positions, inv_freq, key_cache, value_cache, slot_mapping,
                                 sections, mixed_sections, adjacent_pairs, return_key)
        if done is not None:
            return done
    code = _check_heads(q, k, 3 if return_key else 2)
    _require(v.shape == k.shape and v.dtype == k.dtype, "k and v shapes or dtypes differ")
    tokens, _, d = q.shape
    _, sections = _check_turn(tokens, d, positions, inv_freq, sections, mixed_sections)
    _require(key_cache.dim() == 4 and value_cache.shape == key_cache.shape
             and key_cache.shape[1] == k.shape[1] and key_cache.shape[3] == d,
             "key_cache / value_cache must be [num_blocks, num_kv_heads, block_size, head_size]")
    _require(key_cache.dtype == q.dtype and value_cache.dtype == q.dtype,
             "the cache's dtype differs from q's")
    _require(1 <= key_cache.shape[0] < 1 << 31 and 1 <= key_cache.shape[2] < 1 << 31,
             "the cache is empty or has too many blocks")
    _require(all(c.stride(3) == 1 and _apart(c, (0, 1, 2)) for c in (key_cache, value_cache)),
             "rows of the cache must be contiguous and not overlap")
    _require(not _meet(key_cache, value_cache), "key_cache and value_cache overlap")
    _require(not any(_reach_into(x, c) for x in (q, k, v) for c in (key_cache, value_cache)),
             "q, k and v must not lie in the caches")
    _require(slot_mapping.dim() == 1 and slot_mapping.shape[0] == tokens
             and slot_mapping.dtype in (torch.int32, torch.int64),
             "slot_mapping must be int32 / int64 [num_tokens]")
    _one_device(q, k, v, positions, inv_freq, key_cache, value_cache, slot_mapping)
    q, k, v = _dense(q), _dense(k), _dense(v)
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device) if return_key else None
    if tokens > 0:
        slots = slot_mapping.contiguous()
        args = _args(q, k, q_out, positions, inv_freq, sections, mixed_sections, adjacent_pairs,
                     code)
        if return_key:
            args.k_out, args.k_out_stride_t, args.k_out_stride_h = (k_out.data_ptr(), k_out.stride(0),
                                                                    k_out.stride(1))
        args.v, args.v_stride_t, args.v_stride_h = v.data_ptr(), v.stride(0), v.stride(1)
        args.key_cache, args.value_cache = key_cache.data_ptr(), value_cache.data_ptr()
        args.kc_stride_0, args.kc_stride_h, args.kc_stride_t = key_cache.stride()[:3]
        args.vc_stride_0, args.vc_stride_h, args.vc_stride_t = value_cache.stride()[:3]
        args.num_blocks, args.block_size = key_cache.shape[0], key_cache.shape[2]
        args.slots, args.slots64 = slots.data_ptr(), int(slots.dtype == torch.int64)
        lib = _lib.load()
        with torch.cuda.device(q.device):
            _lib.check(lib.fa_rotary(ctypes.byref(args),
                                     torch.cuda.current_stream(q.device).cuda_stream))
    return (q_out, k_out) if return_key else q_out
