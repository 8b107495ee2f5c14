"""Refusals of the packed-attention and 4-bit-cache operators, on the Python side and at the C ABI
-- CPU only: every check runs before any device work."""
import ctypes
import math

import pytest
import torch

import flag_attn
from flagattention_amd import ArgumentError, _lib, mxfp4, varlen
from oracle import packed_oracle as po
from tests._packed import varlen_splits


def _varlen(dtype=torch.float16):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return dict(q=torch.zeros((10, 4, 64), dtype=dtype), k=torch.zeros((12, 2, 64), dtype=dtype),
                v=torch.zeros((12, 2, 64), dtype=dtype), cu_seqlens_q=i32(0, 4, 10),
                cu_seqlens_k=i32(0, 6, 12), max_seqlen_q=6, max_seqlen_k=6)


@pytest.mark.parametrize("mutate,msg", [
    (lambda a: a.update(q=a["q"][0]), "tokens, heads, head_dim"),
    (lambda a: a.update(v=a["v"][:5]), "shapes differ"),
    (lambda a: a.update(q=torch.zeros((10, 4, 128)).half()), "feature size"),
    (lambda a: a.update(q=torch.zeros((10, 4, 96)).half(), k=torch.zeros((12, 2, 96)).half(),
                        v=torch.zeros((12, 2, 96)).half()), "head dim 96"),
    (lambda a: a.update(q=torch.zeros((10, 3, 64)).half()), "multiple"),
    (lambda a: a.update(q=torch.zeros((10, 0, 64)).half()), "multiple"),
    (lambda a: a.update(**{n: a[n].float() for n in "qkv"}), "float16 / bfloat16"),
    (lambda a: a.update(k=a["k"].bfloat16(), v=a["v"].bfloat16()), "dtypes differ"),
    (lambda a: a.update(cu_seqlens_q=a["cu_seqlens_q"].long()), "cu_seqlens_q"),
    (lambda a: a.update(cu_seqlens_q=a["cu_seqlens_q"][:0]), "cu_seqlens_q"),
    (lambda a: a.update(cu_seqlens_k=a["cu_seqlens_k"][:2]), "cu_seqlens_k"),
    (lambda a: a.update(max_seqlen_k=-1), "max_seqlen"),
    (lambda a: a.update(max_seqlen_q=2.0), "max_seqlen"),
    (lambda a: a.update(sm_scale=math.inf), "finite"),
    (lambda a: None, "CUDA"),  # valid, but CPU tensors
])
def test_varlen_rejects(mutate, msg):
    args = _varlen()
    mutate(args)
    with pytest.raises(ArgumentError, match=msg):
        flag_attn.flash_attention_varlen(**args)


def _cache(blocks=4, hk=2, block=16, d=64):
    return dict(key_cache=torch.zeros((blocks, hk, block, d // 2), dtype=torch.uint8),
                key_scales=torch.zeros((blocks, hk, block, d // 32), dtype=torch.uint8),
                value_cache=torch.zeros((blocks, hk, block, d // 2), dtype=torch.uint8),
                value_scales=torch.zeros((blocks, hk, block, d // 32), dtype=torch.uint8))


def _all(c, f):
    c.update({n: f(c[n]) for n in ("key_cache", "key_scales", "value_cache", "value_scales")})


CACHE_FAULTS = [
    (lambda c: c.update(key_cache=c["key_cache"][0]), "num_blocks, num_kv_heads"),
    (lambda c: c.update(value_cache=c["value_cache"][:3]), "num_blocks, num_kv_heads"),
    (lambda c: c.update(key_scales=c["key_scales"][..., :1]), "head_size / 32"),
    (lambda c: c.update(value_scales=c["value_scales"][:1]), "head_size / 32"),
    (lambda c: _all(c, lambda t: t.char()), "uint8"),
    (lambda c: _all(c, lambda t: t[:0]), "empty"),
    (lambda c: _all(c, lambda t: t[:, :, :8]), "power of two"),
    (lambda c: c.update(**_cache(d=96)), "head_size"),
    (lambda c: c.update(value_cache=c["value_cache"].transpose(0, 1).contiguous().transpose(0, 1)),
     "same strides"),
    (lambda c: _all(c, lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)), "contiguous"),
    (lambda c: c.update(key_cache=torch.zeros(4 * 2 * 16 * 32 + 1, dtype=torch.uint8)[1:].view(
        4, 2, 16, 32)), "aligned"),
    (lambda c: None, "CUDA"),
]


@pytest.mark.parametrize("mutate,msg", CACHE_FAULTS)
def test_every_cache_operator_rejects_a_bad_cache(mutate, msg):
    c = _cache()
    mutate(c)
    d = 2 * c["key_cache"].shape[-1]
    kv = torch.zeros((3, 2, d)).half()
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ArgumentError, match=msg):
        flag_attn.cache_kv_mxfp4(kv, kv, **c, slot_mapping=i32)
    with pytest.raises(ArgumentError, match=msg):
        flag_attn.gather_kv_mxfp4(**c, block_tables=i32.view(1, 3), cu_seqlens=i32[:2],
                                  total_tokens=5, dtype=torch.float16)
    with pytest.raises(ArgumentError, match=msg):
        flag_attn.paged_attention_mxfp4(kv, **c, context_lens=i32, block_tables=i32.view(3, 1),
                                        attn_scale=1.0, max_context_len=10)


@pytest.mark.parametrize("kw,msg", [
    (dict(key=torch.zeros((3, 64)).half()), "num_tokens"),
    (dict(value=torch.zeros((2, 2, 64)).half()), "num_tokens"),
    (dict(key=torch.zeros((3, 2, 64))), "float16"),
    (dict(value=torch.zeros((3, 2, 64)).bfloat16()), "dtypes differ"),
    (dict(key=torch.zeros((3, 4, 64)).half(), value=torch.zeros((3, 4, 64)).half()), "CUDA|differ"),
    (dict(slot_mapping=torch.zeros(2, dtype=torch.int32)), "slot_mapping|CUDA"),
    (dict(slot_mapping=torch.zeros(3)), "slot_mapping|CUDA"),
])
def test_write_rejects(kw, msg):
    args = dict(key=torch.zeros((3, 2, 64)).half(), value=torch.zeros((3, 2, 64)).half(), **_cache(),
                slot_mapping=torch.zeros(3, dtype=torch.int64))
    args.update(kw)
    with pytest.raises(ArgumentError, match=msg):
        flag_attn.cache_kv_mxfp4(**args)


def _write_args(**kw):
    return {**dict(key=torch.zeros((3, 2, 64)).half(), value=torch.zeros((3, 2, 64)).half(), **_cache(),
                   slot_mapping=torch.zeros(3, dtype=torch.int64)), **kw}


def _half(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("kw,msg", [
    (dict(key=_half(3, 4, 64), value=_half(3, 4, 64)), "heads or head size differ"),
    (dict(key=_half(3, 2, 128), value=_half(3, 2, 128)), "heads or head size differ"),
    (dict(slot_mapping=torch.zeros(2, dtype=torch.int64)), "slot_mapping must be"),
    (dict(slot_mapping=torch.zeros(4, dtype=torch.int32)), "slot_mapping must be"),
    (dict(slot_mapping=torch.zeros((3, 1), dtype=torch.int32)), "slot_mapping must be"),
    (dict(slot_mapping=torch.zeros(3)), "slot_mapping must be"),
    (dict(slot_mapping=torch.zeros(3, dtype=torch.int16)), "slot_mapping must be"),
    (dict(), "CUDA"),  # valid, but CPU tensors
])
def test_write_names_its_own_fault(kw, msg):
    with pytest.raises(ArgumentError, match=msg):
        flag_attn.cache_kv_mxfp4(**_write_args(**kw))


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=torch.float32), "float16 / bfloat16"),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int64)), "cu_seqlens must be"),
    (dict(cu_seqlens=_i32(3, 1)), "cu_seqlens must be"),
    (dict(cu_seqlens=_i32(0)), "cu_seqlens must be"),
    (dict(cu_seqlens=_i32(6)[::2]), "cu_seqlens must be"),
    (dict(block_tables=torch.zeros((2, 4), dtype=torch.int64)), "block_tables must be"),
    (dict(block_tables=_i32(8)), "block_tables must be"),
    (dict(block_tables=_i32(3, 4)), "block_tables must be"),
    (dict(block_tables=_i32(1, 4)), "block_tables must be"),
    (dict(block_tables=_i32(4, 2).t()), "block_tables must be"),
    (dict(total_tokens=-1), "total_tokens must be"),
    (dict(total_tokens=5.0), "total_tokens must be"),
    (dict(total_tokens=1 << 28), "too many tokens"),
    (dict(), "CUDA"),
])
def test_gather_names_its_own_fault(kw, msg):
    args = {**dict(**_cache(), block_tables=_i32(2, 4), cu_seqlens=_i32(3), total_tokens=5,
                   dtype=torch.float16), **kw}
    with pytest.raises(ArgumentError, match=msg):
        flag_attn.gather_kv_mxfp4(**args)


@pytest.mark.parametrize("kw,msg", [
    (dict(query=_half(2, 64)), "query must be"),
    (dict(query=torch.zeros((2, 4, 64))), "float16 / bfloat16"),
    (dict(query=_half(2, 4, 128)), "head_size 128"),
    (dict(query=_half(2, 3, 64)), "multiple"),
    (dict(query=_half(2, 0, 64)), "multiple"),
    (dict(query=_half(2, 4, 65)[..., 1:]), "16-byte aligned"),
    (dict(query=_half(513)[1:].view(2, 4, 64)), "16-byte aligned"),
    (dict(query=_half(2, 64, 4).transpose(1, 2)), "16-byte aligned"),
    (dict(context_lens=_i32(3)), "context_lens must be"),
    (dict(context_lens=_i32(2, 1)), "context_lens must be"),
    (dict(context_lens=_i32(4)[::2]), "context_lens must be"),
    (dict(context_lens=torch.zeros(2, dtype=torch.int64)), "context_lens must be"),
    (dict(block_tables=_i32(3, 4)), "block_tables must be"),
    (dict(block_tables=_i32(8)), "block_tables must be"),
    (dict(block_tables=torch.zeros((2, 4), dtype=torch.int64)), "block_tables must be"),
    (dict(block_tables=_i32(4, 2).t()), "block_tables must be"),
    (dict(num_splits=-1), "num_splits must be"),
    (dict(max_context_len=0), "max_context_len must be"),
    (dict(max_context_len=(1 << 30) + 1), "max_context_len must be"),
    (dict(attn_scale=math.nan), "attn_scale must be"),
    (dict(attn_scale=-math.inf), "attn_scale must be"),
    (dict(), "CUDA"),
])
def test_decode_names_its_own_fault(kw, msg):
    args = {**dict(query=_half(2, 4, 64), **_cache(), context_lens=_i32(2), block_tables=_i32(2, 4),
                   attn_scale=0.125, max_context_len=64), **kw}
    with pytest.raises(ArgumentError, match=msg):
        flag_attn.paged_attention_mxfp4(**args)


def test_sizes_past_a_launch_are_argument_errors():
    """What the library refuses for its size is an argument error before that.  (Large tensors are one
    row seen many times.)"""
    a = _varlen()
    a["q"] = a["q"][:1].expand((1 << 29) - 1, 4, 64)
    a["cu_seqlens_q"] = a["cu_seqlens_k"] = _i32(1 << 24)
    with pytest.raises(ArgumentError, match="too many query rows or sequences"):
        flag_attn.flash_attention_varlen(**a)
    a = _varlen()
    a.update({x: _half(1, 1, 64).expand(1 << 18, 1 << 14, 64) for x in "qkv"})
    with pytest.raises(ArgumentError, match="too many query rows or sequences"):
        flag_attn.flash_attention_varlen(**a)
    n = (1 << 28) - 15
    c = _cache(hk=1)
    kv = _half(1, 1, 64).expand(n, 1, 64)
    with pytest.raises(ArgumentError, match="too many tokens"):
        flag_attn.cache_kv_mxfp4(kv, kv, **c, slot_mapping=_i32(1).expand(n))
    with pytest.raises(ArgumentError, match="too many tokens"):
        flag_attn.gather_kv_mxfp4(**c, block_tables=_i32(2, 4), cu_seqlens=_i32(3), total_tokens=n,
                                  dtype=torch.float16)
    for seqs, h_q, hk in ((65536, 1, 1), (1, 65535 * 17, 65535)):
        c = {x: t.expand(4, hk, *t.shape[2:]) for x, t in _cache(hk=1).items()}
        with pytest.raises(ArgumentError, match="too many sequences or heads"):
            flag_attn.paged_attention_mxfp4(_half(1, 1, 64).expand(seqs, h_q, 64), **c,
                                            context_lens=_i32(seqs), block_tables=_i32(seqs, 1),
                                            attn_scale=1.0, max_context_len=1000)


def test_struct_mirrors_and_c_abi_refusals():
    lib = _lib.load()
    for name, mirror in (("fa_varlen_args", _lib.VarlenArgs), ("fa_mxfp4_cache", _lib.Mxfp4Cache),
                         ("fa_mxfp4_decode_args", _lib.Mxfp4DecodeArgs)):
        assert getattr(lib, name + "_size")() == ctypes.sizeof(mirror)

    def refused(rc, text):
        assert rc == -1 and text in lib.fa_last_error(), lib.fa_last_error()

    refused(lib.fa_varlen_attention(None, None), b"NULL")
    good = dict(q=4096, k=4096, v=4096, out=4096, cu_seqlens_q=4096, cu_seqlens_k=4096, num_seqs=1,
                total_q=4, total_k=4, h_q=2, h_kv=1, d=64, num_splits=1, split_tokens=1,
                q_stride_t=128, q_stride_h=64, k_stride_t=64, k_stride_h=64, v_stride_t=64,
                v_stride_h=64, o_stride_t=128, o_stride_h=64)
    for change, text in ((dict(total_q=0), b"total_q"), (dict(num_seqs=-1), b"num_seqs"),
                         (dict(h_q=3, h_kv=2), b"multiple"), (dict(d=32), b"head dim"),
                         (dict(dtype=2), b"dtype"), (dict(out=None), b"NULL"),
                         (dict(k=4104), b"aligned"), (dict(o_stride_h=60), b"aligned"),
                         (dict(k_stride_t=1 << 23), b"token strides"),
                         (dict(v_stride_t=-64), b"token strides"),
                         (dict(total_q=1 << 30), b"too many"),
                         (dict(num_seqs=1 << 24), b"too many"),
                         (dict(total_q=1 << 25, num_splits=2, o_part=4096, lse_part=4096),
                          b"too many"), (dict(num_splits=0), b"num_splits"),
                         (dict(num_splits=2), b"o_part"),
                         (dict(num_splits=9, split_tokens=1 << 29), b"num_splits")):
        refused(lib.fa_varlen_attention(ctypes.byref(_lib.VarlenArgs(**{**good, **change})), None), text)
    refused(lib.fa_varlen_combine(ctypes.byref(_lib.VarlenArgs(**good)), None), b"o_part")

    cache = dict(k_codes=4096, k_scales=4096, v_codes=4096, v_scales=4096, code_stride_0=1024,
                 code_stride_h=512, code_stride_t=32, scale_stride_0=64, scale_stride_h=32,
                 scale_stride_t=2, num_blocks=4, block_size=16, h_kv=2, d=64)
    for change, text in ((dict(d=32), b"head dim"), (dict(h_kv=0), b"h_kv"),
                         (dict(block_size=24), b"block_size"), (dict(num_blocks=0), b"num_blocks"),
                         (dict(num_blocks=1 << 31), b"num_blocks"), (dict(v_scales=None), b"NULL"),
                         (dict(k_codes=4100), b"codes"), (dict(code_stride_t=36), b"codes"),
                         (dict(d=256, scale_stride_h=33), b"scales")):
        c = _lib.Mxfp4Cache(**{**cache, **change})
        refused(lib.fa_mxfp4_cache_write(ctypes.byref(c), 4096, 128, 64, 4096, 128, 64, 4096, 1, 3, 0,
                                         None), text)
        refused(lib.fa_mxfp4_gather(ctypes.byref(c), 4096, 1, 1, 4096, 1, 3, 4096, 4096, 0, None), text)
        refused(lib.fa_mxfp4_decode(ctypes.byref(_lib.Mxfp4DecodeArgs(cache=c)), None), text)
    ok = _lib.Mxfp4Cache(**cache)
    refused(lib.fa_mxfp4_cache_write(ctypes.byref(ok), 4096, 128, 64, 4096, 128, 64, 4096, 1, -1, 0,
                                     None), b"num_tokens")
    refused(lib.fa_mxfp4_cache_write(ctypes.byref(ok), 4096, 128, 64, 4096, 128, 60, 4096, 1, 3, 0,
                                     None), b"aligned")
    refused(lib.fa_mxfp4_cache_write(ctypes.byref(ok), 4096, 128, 64, 4096, 128, 64, 4096, 1, 1 << 30, 0,
                                     None), b"2^31")
    refused(lib.fa_mxfp4_gather(ctypes.byref(ok), 4096, 1, 1, 4096, 1, 1 << 28, 4096, 4096, 0, None),
            b"2^28")
    refused(lib.fa_mxfp4_gather(ctypes.byref(ok), None, 1, 1, 4096, 1, 3, 4096, 4096, 0, None), b"NULL")
    decode = dict(cache=ok, q=4096, out=4096, block_table=4096, seqlens=4096, max_blocks_per_seq=1,
                  batch=1, h_q=4, num_splits=1, split_tokens=7, q_stride_b=256, q_stride_h=64)
    for change, text in ((dict(batch=0), b"batch"), (dict(batch=65536), b"batch"),
                         (dict(h_q=3), b"multiple"), (dict(dtype=5), b"dtype"),
                         (dict(num_splits=2, split_tokens=24), b"num_splits"),
                         (dict(num_splits=2, split_tokens=32), b"o_part"),
                         (dict(seqlens=None), b"NULL"), (dict(q=4098), b"aligned")):
        refused(lib.fa_mxfp4_decode(ctypes.byref(_lib.Mxfp4DecodeArgs(**{**decode, **change})), None),
                text)
    refused(lib.fa_mxfp4_combine(ctypes.byref(_lib.Mxfp4DecodeArgs(**decode)), None), b"o_part")


def test_grids_of_2_32_lanes_are_refused():
    """The largest sizes under each limit, one past it: a launch of 2^24 work-groups of 256 lanes has
    one lane too many for its counters."""
    lib = _lib.load()

    def refused(rc, text):
        assert rc == -1 and text in lib.fa_last_error(), (rc, lib.fa_last_error())

    cache = _lib.Mxfp4Cache(k_codes=4096, k_scales=4096, v_codes=4096, v_scales=4096, code_stride_0=512,
                            code_stride_h=512, code_stride_t=32, scale_stride_0=32, scale_stride_h=32,
                            scale_stride_t=2, num_blocks=4, block_size=16, h_kv=1, d=64)
    for n in ((1 << 28) - 15, (1 << 28) - 1):
        refused(lib.fa_mxfp4_cache_write(ctypes.byref(cache), 4096, 64, 64, 4096, 64, 64, 4096, 1, n, 0,
                                         None), b"2^28 - 16")
        refused(lib.fa_mxfp4_gather(ctypes.byref(cache), 4096, 1, 1, 4096, 1, n, 4096, 4096, 0, None),
                b"2^28 - 16")
    varlen_args = dict(q=4096, k=4096, v=4096, out=4096, cu_seqlens_q=4096, cu_seqlens_k=4096,
                       num_seqs=1, total_k=4, h_q=1, h_kv=1, d=64, num_splits=2, split_tokens=64,
                       q_stride_t=64, q_stride_h=64, k_stride_t=64, k_stride_h=64, v_stride_t=64,
                       v_stride_h=64, o_stride_t=64, o_stride_h=64, o_part=4096, lse_part=4096)
    for n in ((1 << 26) - 3, (1 << 26) - 1):
        args = _lib.VarlenArgs(**varlen_args, total_q=n)
        refused(lib.fa_varlen_attention(ctypes.byref(args), None), b"too many query rows")
        refused(lib.fa_varlen_combine(ctypes.byref(args), None), b"too many query rows")
    for batch, h_q in ((1 << 14, 1 << 10), (4097, 4096)):
        args = _lib.Mxfp4DecodeArgs(cache=cache, q=4096, out=4096, block_table=4096, seqlens=4096,
                                    max_blocks_per_seq=1, batch=batch, h_q=h_q, num_splits=2,
                                    split_tokens=32, q_stride_b=64, q_stride_h=64, o_part=4096,
                                    lse_part=4096)
        refused(lib.fa_mxfp4_decode(ctypes.byref(args), None), b"too many rows for splits")
        refused(lib.fa_mxfp4_combine(ctypes.byref(args), None), b"too many rows for splits")


@pytest.mark.parametrize("n", [2 ** 31 - 256, 2 ** 31 - 1])
def test_key_positions_stay_in_32_bits(n):
    """Packed keys may be one row seen many times (stride 0), so their count is bounded by its own
    check, not by memory: the walk over them adds up to 128 to the last position."""
    args = _lib.VarlenArgs(q=4096, k=4096, v=4096, out=4096, cu_seqlens_q=4096, cu_seqlens_k=4096,
                           num_seqs=1, total_q=1, total_k=n, h_q=1, h_kv=1, d=64, num_splits=1,
                           split_tokens=1, q_stride_t=64, q_stride_h=64, o_stride_t=64, o_stride_h=64)
    lib = _lib.load()
    assert lib.fa_varlen_attention(ctypes.byref(args), None) == -1 and b"total_k" in lib.fa_last_error()
    a = _varlen()
    a.update({x: a[x][:1].expand(n, 2, 64) for x in "kv"})
    with pytest.raises(ArgumentError, match="too many tokens"):
        flag_attn.flash_attention_varlen(**a)


def test_counts_of_sequences_that_a_launch_would_not_end_with_are_refused():
    """A wave finds its sequence by going through all starts, so that the work grows with the square of
    their number: as many sequences as one decode call takes."""
    lib = _lib.load()
    args = dict(q=4096, k=4096, v=4096, out=4096, cu_seqlens_q=4096, cu_seqlens_k=4096, total_q=4,
                total_k=4, h_q=1, h_kv=1, d=64, num_splits=1, split_tokens=1, q_stride_t=64,
                q_stride_h=64, k_stride_t=64, k_stride_h=64, v_stride_t=64, v_stride_h=64,
                o_stride_t=64, o_stride_h=64)
    cache = _lib.Mxfp4Cache(k_codes=4096, k_scales=4096, v_codes=4096, v_scales=4096, code_stride_0=512,
                            code_stride_h=512, code_stride_t=32, scale_stride_0=32, scale_stride_h=32,
                            scale_stride_t=2, num_blocks=4, block_size=16, h_kv=1, d=64)
    for n in (65536, 1 << 23):
        assert lib.fa_varlen_attention(ctypes.byref(_lib.VarlenArgs(num_seqs=n, **args)), None) == -1
        assert b"too many sequences" in lib.fa_last_error()
        assert lib.fa_mxfp4_gather(ctypes.byref(cache), 4096, 1, 1, 4096, n, 1, 4096, 4096, 0, None) == -1
        assert b"too many sequences" in lib.fa_last_error()
    a = _varlen()
    a["cu_seqlens_q"] = a["cu_seqlens_k"] = _i32(65537)
    with pytest.raises(ArgumentError, match="too many query rows or sequences"):
        flag_attn.flash_attention_varlen(**a)
    with pytest.raises(ArgumentError, match="too many sequences"):
        flag_attn.gather_kv_mxfp4(**_cache(), block_tables=_i32(65536, 1), cu_seqlens=_i32(65537),
                                  total_tokens=5, dtype=torch.float16)


def test_oracle_formats():
    """The oracle's writer keeps what a code can say exactly, and is never off by more than half of
    the widest step, which is the scale itself."""
    x = torch.tensor(po.MAGNITUDES + tuple(-m for m in po.MAGNITUDES)).repeat(2).view(1, 32) * 8.0
    codes, scales = po.quantise(x)
    assert int(scales) == 127 + 3 and torch.equal(po.values(codes, scales), x.double())
    gen = torch.Generator().manual_seed(0)
    x = torch.randn((200, 64), generator=gen) * torch.exp(torch.randn((200, 1), generator=gen) * 3)
    codes, scales = po.quantise(x)
    err = (po.values(codes, scales) - x.double()).abs().unflatten(-1, (-1, 32)).amax(-1)
    power = po.pow2(scales)
    assert bool((err <= power).all())
    top = x.double().abs().unflatten(-1, (-1, 32)).amax(-1)
    assert bool((top <= 7 * power).all()) and bool((top > 3.5 * power).all())


def test_split_rule():
    """The splits of packed prompts: none for one tile of keys or where the rows fill the CUs; they
    cover the keys, each with some."""
    for d in varlen.HEAD_DIMS:
        assert varlen_splits(1, 60, 1, 32, 8, d, True, 1, 60, 256)[0] == 1
        assert varlen_splits(100000, 100000, 4, 32, 8, d, True, 50000, 50000, 256)[0] == 1
        assert varlen_splits(5, 0, 1, 4, 4, d, True, 5, 0, 256)[0] == 1
        for total, seqs, h, hk, n in ((1, 1, 1, 1, 10000), (64, 1, 16, 2, 3000), (5, 4, 4, 1, 70000),
                                      (1, 1, 1, 1, 2 ** 31 - 1), (1, 1, 64, 1, 2 ** 31 - 100)):
            for causal in (True, False):
                s, each = varlen_splits(total, n, seqs, h, hk, d, causal, total, n, 256)
                assert 1 < s <= 128 and each % 64 == 0 and (s - 1) * each < n <= s * each
    for total in (1, 31, 500, 5000):
        for seqs in (1, 2, 64, 300):
            for h, hk in ((1, 1), (32, 8), (40, 40), (128, 1)):
                for n in (1, 64, 65, 127, 129, 513, 4097, 100000):
                    s, each = varlen_splits(total, n * seqs, seqs, h, hk, 128, True, total, n, 256)
                    assert s == 1 or (s - 1) * each < n <= s * each
    assert mxfp4.HEAD_DIMS == varlen.HEAD_DIMS == (64, 128, 256)
