"""rotary_cache_kv with the turned k returned: what a prompt needs for its cache and its attention in one
call."""
import ctypes

import pytest
import torch

import flag_attn
from flagattention_amd import ArgumentError, _lib, rotary
from oracle import packed_oracle as po
from tests._helpers import DEV, need_gpu, say
from tests._packed import assert_rows
from tests.test_gpu_rotary import DTYPES, frequencies, positions, rows
from tests.test_native_host import _both, _same


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,h,hk,d,rot,block,sections,mixed,adjacent", [
    (1, 8, 2, 64, 64, 16, None, False, False), (300, 6, 3, 128, 128, 64, (16, 24, 24), False, False),
    (37, 4, 4, 256, 64, 16, (11, 11, 10), True, True), (50, 3, 1, 80, 30, 7, None, False, True),
    (2000, 32, 8, 128, 128, 16, None, False, False)])
def test_key_is_returned(monkeypatch, n, h, hk, d, rot, block, sections, mixed, adjacent, dtype):
    """q and k are those of rotary_embedding, also k of tokens without a slot; the caches those of the call
    without it; k a view of a packed projection."""
    need_gpu()
    say(f"rotary cache and key n={n} h={h} hk={hk} d={d} rot={rot} {sections} {dtype}")
    blocks = -(-n // block) + 2
    qkv = rows(n, h + 2 * hk, d, dtype, 1)
    q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    f, pos = frequencies(rot // 2), positions(n, 0 if sections is None else len(sections), 5000, 2)
    slots = torch.randperm(blocks * block, device=DEV)[:n]
    slots[n // 2] = -1
    want = flag_attn.rotary_embedding(q, k, pos, f, sections, mixed, adjacent)
    kept = torch.zeros((2, blocks, hk, block, d), dtype=dtype, device=DEV)
    flag_attn.rotary_cache_kv(q, k, v, pos, f, kept[0], kept[1], slots, sections, mixed, adjacent)

    def call():
        both = torch.zeros_like(kept)
        out = flag_attn.rotary_cache_kv(q, k, v, pos, f, both[0], both[1], slots, sections, mixed, adjacent,
                                        return_key=True)
        return out + (both,)

    got = call()
    torch.cuda.synchronize()
    for x, y in zip(got, want + (kept,)):
        assert torch.equal(x, y)
    assert _lib.native().rotary_cache(q, k, v, pos, f, kept[0], kept[1], slots, sections, mixed, adjacent,
                                      True) is not None
    _same(*_both(monkeypatch, call))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_prompt_from_one_call(dtype):
    """Two prompts: q and k of the call through flash_attention_varlen, against the formula."""
    need_gpu()
    say(f"rotary prompt {dtype}")
    h, hk, d, lens = 4, 2, 128, [70, 9]
    n, f = sum(lens), frequencies(d // 2)
    q, k, v = (rows(n, x, d, dtype, i) for i, x in enumerate((h, hk, hk)))
    kc, vc = (torch.zeros((8, hk, 16, d), dtype=dtype, device=DEV) for _ in range(2))
    pos = torch.cat([torch.arange(m, device=DEV) for m in lens])
    cu = torch.tensor([0, 70, 79], dtype=torch.int32, device=DEV)
    qr, kr = flag_attn.rotary_cache_kv(q, k, v, pos, f, kc, vc, torch.arange(n, device=DEV) + 5, return_key=True)
    o = flag_attn.flash_attention_varlen(qr, kr, v, cu, cu, 70, 70, causal=True)
    torch.cuda.synchronize()
    want_q, want_k = flag_attn.rotary_embedding(q, k, pos, f)
    for b, e in ((0, 70), (70, 79)):
        for j in range(h):
            args = want_q[b:e, j], want_k[b:e, j // 2], v[b:e, j // 2]
            ref, _, mag, ds = po.attend(*args, d ** -0.5, True)
            assert_rows(o[b:e, j], ref, mag, ds, e - b, float(v.abs().max()))


@pytest.mark.gpu
def test_no_tokens():
    need_gpu()
    q = rows(0, 2, 64, torch.float16, 1)
    kc = torch.zeros((1, 2, 16, 64), dtype=torch.float16, device=DEV)
    y, z = flag_attn.rotary_cache_kv(q, q, q, positions(0, 0, 5, 1), frequencies(32), kc, kc.clone(),
                                     torch.zeros(0, dtype=torch.int32, device=DEV), return_key=True)
    assert y.shape == z.shape == (0, 2, 64)


def test_too_many_rows_with_the_key():
    """A thread for at least a pair of four rows, k's twice: past 31 bits the call is refused on the host."""
    x = torch.zeros((1, 1, 2), dtype=torch.float16)
    n = (1 << 31) // 7  # 6 threads a token for 7 rows, 8 for 10
    q, k = x.expand(n, 1, 2), x.expand(n, 3, 2)
    assert rotary._check_heads(q, k) == 0
    with pytest.raises(ArgumentError, match="too many"):
        rotary._check_heads(q, k, 3)


def test_key_in_place_is_refused_at_the_abi():
    mem = 1 << 20
    args = _lib.RotaryArgs(q=mem, q_out=mem, k=mem, k_out=mem, v=mem, key_cache=mem, value_cache=mem, slots=mem,
                           positions=mem, inv_freq=mem, tokens=1, h_q=1, h_kv=1, d=64, pairs=32, axes=1,
                           num_blocks=1, block_size=16)
    assert _lib.load().fa_rotary(ctypes.byref(args), None) == -1
    assert b"in place" in _lib.load().fa_last_error()
