"""Refusals of the rotary and linear-attention operators, on the Python side and at the C ABI, and what the
library plans -- CPU only: every check runs before any device work."""
import ctypes
import math

import pytest
import torch

import flag_attn
from flagattention_amd import ArgumentError, _lib, linear, rotary
from oracle import linear_oracle as lo


def half(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _rotary(**kw):
    return {**dict(q=half(5, 4, 64), k=half(5, 2, 64), positions=i32(5), inv_freq=torch.zeros(32)), **kw}


ROTARY_FAULTS = [
    (dict(q=half(4, 64)), "heads, head_dim"),
    (dict(k=half(4, 2, 64)), "heads, head_dim"),
    (dict(k=half(5, 2, 128)), "heads, head_dim"),
    (dict(k=half(5, 0, 64)), "no heads"),
    (dict(q=half(5, 4, 64).float(), k=half(5, 2, 64).float()), "float16 / bfloat16"),
    (dict(k=half(5, 2, 64).bfloat16()), "dtypes differ"),
    (dict(inv_freq=torch.zeros(32, dtype=torch.float64)), "inv_freq"),
    (dict(inv_freq=torch.zeros(2, 16)), "inv_freq"),
    (dict(inv_freq=torch.zeros(64)[::2]), "inv_freq"),
    (dict(inv_freq=torch.zeros(33)), "33 pairs"),
    (dict(inv_freq=torch.zeros(0)), "0 pairs"),
    (dict(q=half(5, 1, 4098), k=half(5, 1, 4098)), "4098"),
    (dict(positions=torch.zeros(5)), "int32 or int64"),
    (dict(positions=i32(4)), "num_tokens"),
    (dict(positions=i32(1, 5)), "num_tokens"),
    (dict(positions=i32(10)[::2]), "contiguous"),
    (dict(mixed_sections=True), "needs sections"),
    (dict(sections=(16, 16)), "len\\(sections\\)"),
    (dict(sections=(16, 8), positions=i32(2, 5)), "sum to 32"),
    (dict(sections=(40, -8), positions=i32(2, 5)), "sum to 32"),
    (dict(sections=(16.0, 16.0), positions=i32(2, 5)), "ints"),
    (dict(sections=(8, 8, 8, 4, 4), positions=i32(5, 5)), "1 to 4"),
    (dict(sections=(), positions=i32(0, 5)), "1 to 4"),
    (dict(sections=(16, 16), positions=i32(5, 2).t()), "tokens contiguous"),
    (dict(sections=(8, 24), positions=i32(2, 5), mixed_sections=True), "mixed"),
    (dict(), "CUDA"),
]


@pytest.mark.parametrize("kw,msg", ROTARY_FAULTS)
def test_rotary_rejects(kw, msg):
    with pytest.raises(ArgumentError, match=msg):
        flag_attn.rotary_embedding(**_rotary(**kw))
    args = _rotary(**kw)
    d = args["q"].shape[-1]
    with pytest.raises(ArgumentError, match=msg):
        flag_attn.rotary_cache_kv(**args, v=args["k"].clone(), key_cache=half(2, args["k"].shape[1], 16, d),
                                  value_cache=half(2, args["k"].shape[1], 16, d), slot_mapping=i32(5))


@pytest.mark.parametrize("kw", [
    dict(q=half(5, 1, 64).expand(5, 4, 64)), dict(k=half(1, 2, 64).expand(5, 2, 64)),
    dict(q=half(5, 4, 128)[..., ::2]), dict(k=half(5 * 64 + 64).as_strided((5, 2, 64), (64, 32, 1)))])
def test_in_place_needs_rows_of_their_own(kw):
    with pytest.raises(ArgumentError, match="overlap"):
        flag_attn.rotary_embedding(**_rotary(**kw), inplace=True)


def test_two_results_need_memory_of_their_own():
    x = half(5, 2, 64)
    with pytest.raises(ArgumentError, match="q and k overlap"):
        flag_attn.rotary_embedding(**_rotary(q=x, k=x), inplace=True)
    c = half(3, 2, 16, 64)
    with pytest.raises(ArgumentError, match="key_cache and value_cache overlap"):
        flag_attn.rotary_cache_kv(**_store(key_cache=c, value_cache=c))


def _store(**kw):
    return {**_rotary(), **dict(v=half(5, 2, 64), key_cache=half(3, 2, 16, 64),
                                value_cache=half(3, 2, 16, 64), slot_mapping=i32(5)), **kw}


@pytest.mark.parametrize("kw,msg", [
    (dict(v=half(5, 3, 64)), "k and v"),
    (dict(v=half(5, 2, 64).bfloat16()), "k and v"),
    (dict(key_cache=half(2, 16, 64)), "num_blocks"),
    (dict(value_cache=half(2, 2, 16, 64)), "num_blocks"),
    (dict(key_cache=half(3, 4, 16, 64), value_cache=half(3, 4, 16, 64)), "num_blocks"),
    (dict(key_cache=half(3, 2, 16, 32), value_cache=half(3, 2, 16, 32)), "num_blocks"),
    (dict(key_cache=half(3, 2, 16, 64).bfloat16()), "cache's dtype"),
    (dict(key_cache=half(0, 2, 16, 64), value_cache=half(0, 2, 16, 64)), "empty"),
    (dict(key_cache=half(1, 2, 16, 64).expand(3, 2, 16, 64)), "overlap"),
    (dict(value_cache=half(3, 2, 16, 128)[..., ::2]), "contiguous"),
    (dict(slot_mapping=i32(4)), "slot_mapping"),
    (dict(slot_mapping=torch.zeros(5)), "slot_mapping"),
    (dict(), "CUDA"),
])
def test_store_rejects(kw, msg):
    with pytest.raises(ArgumentError, match=msg):
        flag_attn.rotary_cache_kv(**_store(**kw))


@pytest.mark.parametrize("into", ["q", "k", "v"])
@pytest.mark.parametrize("cache", ["key_cache", "value_cache"])
def test_store_rejects_rows_of_the_caches(into, cache):
    whole = half(6 * 2 * 16 * 64)
    rows = whole[2047:2047 + 5 * 2 * 64].view(5, 2, 64)
    kw = _store(**{cache: whole[2048:2048 * 4].view(3, 2, 16, 64), into: rows, "q": half(5, 2, 64)}
                if into != "q" else {cache: whole[2048:2048 * 4].view(3, 2, 16, 64), "q": rows})
    with pytest.raises(ArgumentError, match="must not lie in the caches"):
        flag_attn.rotary_cache_kv(**kw)
    kw[into] = whole[2048 - 640:2048].view(5, 2, 64)  # up to the cache's first byte
    with pytest.raises(ArgumentError, match="CUDA"):
        flag_attn.rotary_cache_kv(**kw)


def _prompt(**kw):
    return {**dict(q=half(9, 4, 64), k=half(9, 2, 64), v=half(9, 2, 64), log_decay=torch.zeros(2),
                   cu_seqlens=i32(3), max_seqlen=9, state=torch.zeros(4, 2, 64, 64),
                   state_indices=i32(2), has_state=torch.zeros(2, dtype=torch.bool)), **kw}


ROWS = [
    (dict(q=half(9, 64)), "tokens, heads, head_dim"),
    (dict(v=half(9, 2, 128)), "shapes differ"),
    (dict(k=half(8, 2, 64), v=half(8, 2, 64)), "same tokens"),
    (dict(q=half(9, 4, 128)), "feature size"),
    (dict(q=half(9, 4, 96), k=half(9, 2, 96), v=half(9, 2, 96)), "head dim 96"),
    (dict(q=half(9, 3, 64)), "multiple"),
    (dict(q=half(9, 0, 64)), "multiple"),
    (dict(q=half(9, 4, 64).float()), "float16 / bfloat16"),
    (dict(v=half(9, 2, 64).bfloat16()), "dtypes differ"),
    (dict(log_decay=torch.zeros(4)), "log_decay"),
    (dict(log_decay=torch.zeros(2).double()), "log_decay"),
    (dict(log_decay=torch.zeros(4)[::2]), "log_decay"),
    (dict(state=torch.zeros(4, 2, 64, 128)), "state must be"),
    (dict(state=torch.zeros(4, 2, 64, 64).half()), "state must be"),
    (dict(state=torch.zeros(4, 2, 64, 64).transpose(2, 3)), "contiguous"),
    (dict(state=torch.zeros(4 * 2 * 4096 + 1)[1:].view(4, 2, 64, 64)), "aligned"),
    (dict(state=torch.zeros(1, 2, 64, 64).expand(4, 2, 64, 64)), "overlap"),
    (dict(state=torch.zeros(4, 1, 64, 64).expand(4, 2, 64, 64)), "overlap"),
    (dict(state=torch.zeros(6 * 4096).as_strided((4, 2, 64, 64), (4096, 4096, 64, 1))), "overlap"),
    (dict(state_indices=i32(3)), "state_indices"),
    (dict(state_indices=torch.zeros(2, dtype=torch.int64)), "state_indices"),
]


@pytest.mark.parametrize("kw,msg", ROWS + [
    (dict(cu_seqlens=i32(3).long()), "cu_seqlens"),
    (dict(cu_seqlens=i32(0)), "cu_seqlens"),
    (dict(max_seqlen=-1), "max_seqlen"),
    (dict(max_seqlen=2.0), "max_seqlen"),
    (dict(cu_seqlens=i32(65537), state_indices=None, has_state=None, state=None), "too many"),
    (dict(state=None), "need a state"),
    (dict(state=torch.zeros(1, 2, 64, 64), state_indices=None), "fewer slots"),
    (dict(has_state=torch.zeros(3, dtype=torch.bool)), "has_state"),
    (dict(has_state=torch.zeros(2)), "has_state"),
    (dict(sm_scale=math.inf), "finite"),
    (dict(), "CUDA"),
])
def test_prompt_rejects(kw, msg):
    with pytest.raises(ArgumentError, match=msg):
        flag_attn.linear_attention_varlen(**_prompt(**kw))


@pytest.mark.parametrize("kw,msg", ROWS + [(dict(sm_scale=math.nan), "finite"), (dict(), "CUDA"),
                                           (dict(state_indices=None, state=torch.zeros(3, 2, 64, 64)), "fewer slots")])
def test_decode_rejects(kw, msg):
    args = _prompt(**kw)
    for name in ("cu_seqlens", "max_seqlen", "has_state"):
        args.pop(name)
    if "state_indices" not in kw:
        args["state_indices"] = i32(args["q"].shape[0])
    with pytest.raises(ArgumentError, match=msg):
        flag_attn.linear_attention_decode(**args)


def _args(**kw):
    base = dict(q=64, q_stride_t=256, q_stride_h=64, k=64, v=64, k_stride_t=128, k_stride_h=64,
                v_stride_t=128, v_stride_h=64, log_decay=64, cu_seqlens=64, out=64, num_seqs=2, total=9,
                h_q=4, h_kv=2, d=64, scale=1.0, dtype=1)
    return _lib.LinearArgs(**{**base, **kw})


@pytest.mark.parametrize("kw,msg", [
    (dict(d=96), "head dim"), (dict(dtype=2), "dtype"), (dict(h_q=3), "multiple"), (dict(h_kv=0), "multiple"),
    (dict(h_q=1 << 17), "too many heads"), (dict(num_seqs=-1), "out of range"),
    (dict(num_seqs=65536), "out of range"), (dict(total=-1), "out of range"), (dict(q=None), "NULL"),
    (dict(log_decay=None), "NULL"), (dict(cu_seqlens=None), "NULL"), (dict(k=66), "aligned"),
    (dict(q_stride_h=60), "stride"), (dict(v_stride_t=1 << 23), "too far"),
    (dict(k_stride_t=-128), "stride"), (dict(state=66), "aligned"), (dict(state=64, num_slots=-1), "aligned"),
    (dict(state=64, num_slots=1, state_stride_h=2), "aligned"), (dict(segment=33), "segments"),
    (dict(segment=-32), "segments"), (dict(segment=32), "part"), (dict(segment=32, part=72), "part"),
    (dict(sorted=1, num_seqs=65), "sorted"), (dict(total=(1 << 31) - 1), "too many tokens"),
])
def test_prompt_abi_rejects(kw, msg):
    lib = _lib.load()
    assert lib.fa_linear_prompt(ctypes.byref(_args(**kw)), None) == -1
    assert msg in lib.fa_last_error().decode()


def test_other_abi_refusals():
    lib = _lib.load()

    def refused(rc, msg):
        assert rc == -1 and msg in lib.fa_last_error().decode()

    refused(lib.fa_linear_prompt(None, None), "NULL")
    refused(lib.fa_linear_plan(None, 1, 1), "NULL")
    refused(lib.fa_linear_plan(ctypes.byref(_args(d=32)), 1, 256), "head dim")
    refused(lib.fa_linear_plan(ctypes.byref(_args()), -1, 256), "max_seqlen")
    refused(lib.fa_linear_plan(ctypes.byref(_args()), 1, 0), "CUs")
    refused(lib.fa_linear_token(None, None), "NULL")
    refused(lib.fa_linear_token(ctypes.byref(_args(num_slots=9, state=64)), None), "sequences")
    refused(lib.fa_linear_token(ctypes.byref(_args(num_seqs=9)), None), "state is NULL")
    refused(lib.fa_linear_token(ctypes.byref(_args(num_seqs=65535, total=65535, h_q=512, h_kv=512, q_stride_t=1 << 15)), None),
            "too many")
    refused(lib.fa_rotary(None, None), "NULL")


@pytest.mark.parametrize("kw,msg", [
    (dict(tokens=-1), "out of range"), (dict(h_q=0, h_kv=0), "out of range"), (dict(h_q=65536), "out of range"),
    (dict(d=1), "head dim"), (dict(pairs=33), "head dim"), (dict(pairs=0), "head dim"), (dict(axes=0), "axes"),
    (dict(axes=5), "axes"), (dict(dtype=2), "dtype"), (dict(axes=2), "sections"),
    (dict(axes=2, sections=(ctypes.c_int32 * 4)(40, -8)), "negative"), (dict(q=None), "NULL"),
    (dict(q_out=None), "NULL"), (dict(positions=None), "NULL"), (dict(k_out=None), "NULL"),
    (dict(q_out=64), "in place"), (dict(key_cache=64), "NULL"),
    (dict(key_cache=64, value_cache=64, slots=64, v=64, num_blocks=0), "blocks"),
    (dict(tokens=1 << 28), "too many"),
])
def test_rotary_abi_rejects(kw, msg):
    lib = _lib.load()
    base = dict(q=64, k=64, q_out=128, k_out=128, positions=64, inv_freq=64, tokens=5, h_q=4, h_kv=2, d=64,
                pairs=32, axes=1, block_size=16)
    assert lib.fa_rotary(ctypes.byref(_lib.RotaryArgs(**{**base, **kw})), None) == -1
    assert msg in lib.fa_last_error().decode()


@pytest.mark.parametrize("d", linear.HEAD_DIMS)
@pytest.mark.parametrize("h,hk", [(8, 8), (8, 4), (56, 8)])
def test_plans(d, h, hk):
    """Segments are whole chunks and shorter than the longest sequence; the workspace holds a state for
    every piece; nothing is cut where the sequences fill the card or nothing is there."""
    lib = _lib.load()
    for seqs, total, most in ((1, 1, 1), (1, 64, 64), (3, 2000, 900), (1, 131001, 131001), (16, 30000, 8000),
                              (64, 65536, 1024), (200, 90000, 30000), (0, 50, 50), (5, 1 << 30, 1 << 30)):
        args = _lib.LinearArgs(num_seqs=seqs, total=total, h_q=h, h_kv=hk, d=d, dtype=1)
        floats = lib.fa_linear_plan(ctypes.byref(args), most, 256)
        assert args.segment % 32 == 0 and 0 <= args.segment < max(most, 1)
        assert floats == (0 if not args.segment else (total // args.segment + seqs) * hk * d * d)
        assert floats <= 1 << 30
        assert args.sorted == int(2 <= seqs <= 64 and most > 128)
        if most <= 64 or seqs == 0:
            assert args.segment == 0
        if seqs == 1 and most > 10000:
            assert args.segment > 0
        if seqs == 64 and hk == 8 and d == 256:
            assert args.segment == 0
    few = _lib.LinearArgs(num_seqs=0, total=0, h_q=h, h_kv=hk, d=d, dtype=0)
    assert lib.fa_linear_plan(ctypes.byref(few), 100, 256) == 0
    # nothing to do: no launch either
    assert lib.fa_linear_prompt(ctypes.byref(few), None) == 0
    assert lib.fa_linear_token(ctypes.byref(few), None) == 0


def test_the_oracle_is_the_recurrence():
    gen = torch.Generator().manual_seed(1)
    q, k, v, s0 = (torch.randn(s, generator=gen, dtype=torch.float64)
                   for s in ((11, 2, 4), (11, 4), (11, 4), (4, 4)))
    for a in (0.0, -0.3, -math.inf):
        o, _, end, _ = lo.attend(q, k, v, a, 0.5, s0)
        s = s0.clone()
        for t in range(11):
            s = math.exp(a) * s + k[t][:, None] * v[t]
            assert torch.allclose(o[t], 0.5 * q[t] @ s, rtol=1e-12, atol=1e-12)
        assert torch.allclose(end, s, rtol=1e-12, atol=1e-12)


def test_the_oracle_turns_by_the_axis():
    f = torch.tensor([1.0, 0.5, 0.25, 0.1])
    pos = torch.tensor([[3], [7], [11]])
    runs = lo.angles(pos, f, (2, 1, 1))
    assert torch.allclose(runs, torch.tensor([[3.0, 1.5, 1.75, 1.1]], dtype=torch.float64))
    mixed = lo.angles(pos, f, (2, 1, 1), True)
    assert torch.allclose(mixed, torch.tensor([[3.0, 3.5, 2.75, 0.3]], dtype=torch.float64))
    x = torch.randn((1, 1, 8), dtype=torch.float64)
    y, _ = lo.turn(x, runs)
    z, _ = lo.turn(x.view(1, 1, 2, 4).transpose(2, 3).reshape(1, 1, 8), runs, True)
    assert torch.allclose(z.view(1, 1, 4, 2).transpose(2, 3).reshape(1, 1, 8), y)


def test_calls_without_gpu_tensors_are_left_to_python():
    fast = _lib.native()
    a = _rotary()
    assert fast.rotary(a["q"], a["k"], a["positions"], a["inv_freq"], None, False, False, False) is None
    assert fast.rotary(a["q"]) is None
    s = _store()
    assert fast.rotary_cache(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["key_cache"],
                             s["value_cache"], s["slot_mapping"], None, False, False) is None
    p = _prompt()
    assert fast.linear_varlen(*p.values(), None) is None
    assert fast.linear_decode(p["q"], p["k"], p["v"], p["log_decay"], p["state"], i32(9), None) is None
    assert fast.linear_varlen(*[None] * 10) is None and fast.linear_decode(*[None] * 7) is None
    assert rotary.MAX_AXES == 4
