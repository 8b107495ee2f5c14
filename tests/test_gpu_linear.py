"""Linear attention with a decay per head (flag_attn.linear_attention_varlen, linear_attention_decode)
against the formula in 64 bits, with tolerances made of the roundings it makes (tests/_linear.py)."""
import math

import pytest
import torch

import flag_attn
from oracle import linear_oracle as lo
from tests._helpers import DEV, need_gpu, say
from tests._linear import assert_out, assert_state, small_out, small_state

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]
DIMS = (64, 128, 256)


def starts(lens, first=0):
    out = [first]
    for n in lens:
        out.append(out[-1] + n)
    return out


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def make(lens, h, hk, d, dtype, seed=0, first=0, behind=0, slots=None, gain=1.0):
    """Packed inputs with decays from fast to slow, and states in more slots than sequences."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    n = first + sum(lens) + behind
    slots = len(lens) + 2 if slots is None else slots

    def rows(heads):
        return (gain * torch.randn((n, heads, d), generator=gen, device=DEV)).to(dtype)

    q, k, v = rows(h), rows(hk), rows(hk)
    a = -torch.exp(torch.linspace(1.0, -7.0, hk, device=DEV))
    state = torch.randn((slots, hk, d, d), generator=gen, device=DEV) * (2.0 * gain * gain)
    ids = torch.randperm(slots, generator=gen, device=DEV)[:len(lens)].to(torch.int32)
    return q, k, v, a, starts(lens, first), state, ids


def check(q, k, v, a, cu, state=None, ids=None, has=None, scale=None):
    """One call against the oracle: rows, states, and every slot that no sequence has."""
    before = None if state is None else state.clone()
    most = max((e - b for b, e in zip(cu, cu[1:])), default=0)
    o = flag_attn.linear_attention_varlen(q, k, v, a, i32(cu), most, state, ids,
                                          None if has is None else torch.tensor(has, device=DEV), scale)
    torch.cuda.synchronize()
    assert o.shape == q.shape and o.dtype == q.dtype
    h, hk, d = q.shape[1], k.shape[1], q.shape[2]
    scale = d ** -0.5 if scale is None else scale
    if cu[0] > 0:
        assert not bool(o[:cu[0]].any())
    assert not bool(o[cu[-1]:].any()), "rows behind the last sequence"
    touched = set()
    for s, (b, e) in enumerate(zip(cu, cu[1:])):
        slot = None
        if state is not None:
            slot = s if ids is None else int(ids[s])
            slot = slot if 0 <= slot < state.shape[0] else None
        if e == b:
            continue
        touched.add(slot)
        for j in range(hk):
            heads = slice(j * (h // hk), (j + 1) * (h // hk))
            s0 = before[slot, j] if slot is not None and (has is None or has[s]) else None
            args = q[b:e, heads], k[b:e, j], v[b:e, j]
            ref, size, end, end_size = lo.attend(*args, float(a[j]), scale, s0)
            assert_out(o[b:e, heads], ref, size, e - b, small_out(*args, s0, scale))
            if slot is not None:
                assert_state(state[slot, j], end, end_size, e - b, q.dtype, small_state(k[b:e, j], v[b:e, j], q.dtype))
    if state is not None:
        for slot in set(range(state.shape[0])) - touched:
            assert torch.equal(state[slot], before[slot]), f"slot {slot} is nobody's"
    return o


LENS = [1, 31, 32, 33, 0, 64, 97, 2, 160, 7]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,hk,d", [(3, 3, 64), (8, 2, 64), (4, 4, 128), (7, 1, 128), (2, 2, 256),
                                    (6, 2, 256)])
def test_prompts_with_states(h, hk, d, dtype):
    """Lengths around the chunk, an empty sequence in the middle, rows before the first and behind the
    last sequence, states that are there for half of them."""
    need_gpu()
    say(f"linear prompts h={h} hk={hk} d={d} {dtype}")
    q, k, v, a, cu, state, ids = make(LENS, h, hk, d, dtype, seed=d + h, first=5, behind=40)
    for x in (q, k, v):
        x[:5] = x[-40:] = math.nan
    check(q, k, v, a, cu, state, ids, [s % 2 == 0 for s in range(len(LENS))])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", DIMS)
def test_prompts_without_states(d, dtype):
    need_gpu()
    say(f"linear without states d={d} {dtype}")
    q, k, v, a, cu, _, _ = make(LENS, 4, 2, d, dtype, seed=d)
    check(q, k, v, a, cu, scale=0.3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", DIMS)
def test_long_sequences(d, dtype):
    need_gpu()
    say(f"linear long d={d} {dtype}")
    q, k, v, a, cu, state, ids = make([1500, 3, 2049], 2, 2, d, dtype, seed=d)
    check(q, k, v, a, cu, state, ids)


@pytest.mark.parametrize("d", DIMS)
def test_slots_outside_and_default_slots(d):
    """A slot outside: from zeros, kept nowhere.  No indices: sequence s has slot s."""
    need_gpu()
    say(f"linear slots d={d}")
    q, k, v, a, cu, state, ids = make([40, 5, 70], 2, 1, d, torch.bfloat16, seed=1)
    ids[0], ids[2] = -1, state.shape[0]
    check(q, k, v, a, cu, state, ids)
    check(q, k, v, a, cu, state)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_sequences_and_no_tokens(dtype):
    need_gpu()
    say(f"linear nothing {dtype}")
    q, k, v, a, _, state, _ = make([40], 2, 2, 64, dtype)
    check(q, k, v, a, [0])
    check(q, k, v, a, [0, 0, 0], state)
    check(q[:0], k[:0], v[:0], a, [0, 0], state)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("a", [0.0, -1e-5, -0.02, -3.0, -40.0, -math.inf])
def test_decays(a, dtype):
    """None, slow, fast, and a decay to nothing (each token then sees itself alone)."""
    need_gpu()
    say(f"linear decay {a} {dtype}")
    q, k, v, _, cu, state, ids = make([200, 1, 33], 2, 1, 128, dtype, seed=2)
    check(q, k, v, torch.full((1,), a, device=DEV), cu, state, ids)


@pytest.mark.parametrize("gain", [2.0 ** -9, 2.0 ** -5, 64.0])
def test_fp16_outside_its_range(gain):
    """Scores and states past fp16's range, or far below it, between q, k and v inside it.  The scale
    brings the outputs back."""
    need_gpu()
    say(f"linear fp16 gain={gain}")
    q, k, v, a, cu, state, ids = make([120, 40], 2, 2, 128, torch.float16, seed=3, gain=gain)
    check(q, k, v, a, cu, state, ids, scale=0.05 * gain ** -3 if gain < 1 else 1e-5)


@pytest.mark.parametrize("h,hk,d", [(1, 1, 64), (3, 1, 128), (1, 1, 256)])
def test_fp16_columns_of_different_sizes(h, hk, d):
    """Dims of v from 2^-12 to 2^12, each within its own tolerance; and a state that is nothing for two
    chunks, then tiny, then large."""
    need_gpu()
    say(f"linear fp16 columns h={h} d={d}")
    q, k, v, a, cu, state, ids = make([150, 70], h, hk, d, torch.float16, seed=9)
    sizes = 2.0 ** torch.linspace(-12, 12, d, device=DEV)
    v = (v.float() * sizes[torch.randperm(d, device=DEV)]).half()
    check(q, k, v, a, cu, scale=2.0 ** -10)
    v2 = v.clone()
    v2[:70] = 0
    v2[70:110] *= 2.0 ** -8
    check(q, k, v2, torch.full_like(a, -0.001), [0, 220], scale=2.0 ** -10)


@pytest.mark.parametrize("d", DIMS)
def test_largest_finite_values(d):
    """One token of bf16's largest finite values behind slow decays: nothing on the way is larger."""
    need_gpu()
    say(f"linear largest values d={d}")
    top = float(torch.finfo(torch.bfloat16).max)
    q, k, v = (torch.zeros((200, 1, d), dtype=torch.bfloat16, device=DEV) for _ in range(3))
    q[:, 0, 5] = 1.0
    k[40, 0, 5], v[40] = 1.0, top
    v[40, 0, ::2] = -top
    for a in (-0.01, -0.08, 0.0):
        decay = torch.full((1,), a, device=DEV)
        state = torch.zeros((1, 1, d, d), device=DEV)
        o = flag_attn.linear_attention_varlen(q, k, v, decay, i32([0, 200]), 200, state, sm_scale=1.0)
        torch.cuda.synchronize()
        ref, size, end, end_size = lo.attend(q, k[:, 0], v[:, 0], float(decay[0]), 1.0)
        assert bool(torch.isfinite(o).all()) and bool(torch.isfinite(state).all())
        assert_out(o, ref, size, 200)
        assert_state(state[0, 0], end, end_size, 200, q.dtype)


@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16), (256, torch.bfloat16)])
def test_strides(d, dtype):
    """Rows that are views: interleaved q, k and v, heads outermost, off the alignment, one row seen by
    every token; states of every second slot."""
    need_gpu()
    say(f"linear strides d={d} {dtype}")
    lens, h = [50, 3, 90], 4
    n = sum(lens)
    gen = torch.Generator(device=DEV).manual_seed(5)
    a = torch.tensor([-0.5, -0.1, -0.01, -0.001], device=DEV)
    qkv = torch.randn((n, 3, h, d), generator=gen, device=DEV).to(dtype)
    heads = torch.randn((3, h, n, d), generator=gen, device=DEV).to(dtype)
    off = torch.randn((3, n, h, d + 1), generator=gen, device=DEV).to(dtype)[..., 1:]
    cu = starts(lens)
    big = torch.randn((8, h, d, d), generator=gen, device=DEV)
    ids = i32([2, 0, 3])
    for q, k, v in (qkv.unbind(1), heads.transpose(1, 2).unbind(0), off.unbind(0),
                    (qkv[:, 0], qkv[:1, 1].expand(n, h, d), qkv[:, 2])):
        check(q, k, v, a, cu, big[::2], ids)
    grouped = torch.randn((4, 3, 1, d, d), generator=gen, device=DEV)
    check(qkv[:, 0], qkv[:, 1, :1], qkv[:, 2, :1], a[:1], cu, grouped[:, 1], ids)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_what_is_not_finite_reaches_later_tokens_only(which, dtype, bad):
    """Token 41 of the middle sequence has one such dim in head 1."""
    need_gpu()
    say(f"linear {bad} in {which} {dtype}")
    lens, d = [40, 100, 40], 128
    q, k, v, a, cu, state, ids = make(lens, 4, 2, d, dtype, seed=6)
    a[:] = -0.05
    kept = state.clone()
    o = flag_attn.linear_attention_varlen(q, k, v, a, i32(cu), 100, state, ids)
    state2 = kept.clone()
    x = {"q": q, "k": k, "v": v}[which]
    t = cu[1] + 41
    head = 2 if which == "q" else 1
    x[t, head, 70] = bad
    o2 = flag_attn.linear_attention_varlen(q, k, v, a, i32(cu), 100, state2, ids)
    torch.cuda.synchronize()
    reached = torch.zeros(o.shape, dtype=torch.bool, device=DEV)
    if which == "q":
        reached[t, 2] = True
    elif which == "k":
        reached[t:cu[2], 2:4] = True
    else:
        reached[t:cu[2], 2:4, 70] = True
    assert torch.equal(o2[~reached], o[~reached])
    assert not bool(torch.isfinite(o2[reached]).any())
    rest = torch.ones(state.shape, dtype=torch.bool, device=DEV)
    slot = int(ids[1])
    if which == "k":
        rest[slot, 1, 70] = False
    elif which == "v":
        rest[slot, 1, :, 70] = False
    assert torch.equal(state2[rest], state[rest])
    assert not bool(torch.isfinite(state2[~rest]).any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,hk,d", [(2, 2, 64), (6, 2, 64), (2, 2, 128), (6, 2, 128), (2, 2, 256), (6, 2, 256)])
@pytest.mark.parametrize("which", ["q", "k", "v", "state"])
def test_what_is_not_finite_in_every_layout(which, h, hk, d, dtype):
    """An infinity in the second KV head (or its last query head) of token 41 of the middle sequence, or in
    its state: what it does not reach keeps its bits."""
    need_gpu()
    say(f"linear infinity in {which} h={h} hk={hk} d={d} {dtype}")
    lens, g = [40, 100, 40], h // hk
    q, k, v, a, cu, state, ids = make(lens, h, hk, d, dtype, seed=8)
    a[:] = -0.05
    state2, slot, col = state.clone(), int(ids[1]), d - 27
    o = flag_attn.linear_attention_varlen(q, k, v, a, i32(cu), 100, state, ids)
    t = cu[1] + 41
    reached = torch.zeros(o.shape, dtype=torch.bool, device=DEV)
    rest = torch.ones(state.shape, dtype=torch.bool, device=DEV)
    if which == "q":
        q[t, h - 1, col] = math.inf
        reached[t, h - 1] = True
    elif which == "k":
        k[t, 1, col] = math.inf
        reached[t:cu[2], g:] = True
        rest[slot, 1, col] = False
    elif which == "v":
        v[t, 1, col] = -math.inf
        reached[t:cu[2], g:, col] = True
        rest[slot, 1, :, col] = False
    else:
        state2[slot, 1, 5, col] = math.inf
        reached[cu[1]:cu[2], g:, col] = True
        rest[slot, 1, 5, col] = False
    o2 = flag_attn.linear_attention_varlen(q, k, v, a, i32(cu), 100, state2, ids)
    torch.cuda.synchronize()
    assert torch.equal(o2[~reached], o[~reached])
    assert not bool(torch.isfinite(o2[reached]).any())
    assert torch.equal(state2[rest], state[rest])
    assert not bool(torch.isfinite(state2[~rest]).any())


def test_a_last_token_that_is_not_finite():
    """Rows past the end of a chunk repeat no such value into the state's other dims."""
    need_gpu()
    say("linear last token")
    q, k, v, a, cu, state, ids = make([37], 1, 1, 64, torch.bfloat16, seed=7, slots=1)
    k[36, 0, 3] = math.inf
    o = flag_attn.linear_attention_varlen(q, k, v, a, i32(cu), 37, state, ids)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(o[:36]).all()) and not bool(torch.isfinite(o[36]).any())
    rows = torch.isfinite(state[0, 0]).all(1)
    assert not bool(rows[3]) and bool(rows[:3].all()) and bool(rows[4:].all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,hk,d", [(2, 2, 64), (16, 1, 64), (32, 32, 128), (21, 3, 128), (4, 4, 256),
                                    (8, 2, 256)])
@pytest.mark.parametrize("b", [1, 5, 70])
def test_decode(b, h, hk, d, dtype):
    """One token per sequence, some of them padding."""
    need_gpu()
    say(f"linear decode b={b} h={h} hk={hk} d={d} {dtype}")
    q, k, v, a, _, state, ids = make([1] * b, h, hk, d, dtype, seed=b)
    if b > 4:
        ids[1], ids[4] = -1, state.shape[0]
    before = state.clone()
    o = flag_attn.linear_attention_decode(q, k, v, a, state, ids)
    torch.cuda.synchronize()
    group = h // hk
    touched = []
    for s in range(b):
        slot = int(ids[s])
        if not 0 <= slot < state.shape[0]:
            assert not bool(o[s].any())
            continue
        touched.append(slot)
        s0 = before[slot].double()
        step = torch.exp(a.double())[:, None, None]
        kv = k[s].double()[:, :, None] * v[s].double()[:, None, :]
        end, size = step * s0 + kv, step * s0.abs() + kv.abs()
        qs = q[s].double().view(hk, group, d) * d ** -0.5
        assert_out(o[s].view(hk, group, d), qs @ end, qs.abs() @ size, 1)
        # fp32: a weight, a product, a sum
        assert bool(((state[slot] - end).abs() <= 8 * 2.0 ** -24 * size).all())
    rest = [s for s in range(state.shape[0]) if s not in touched]
    assert torch.equal(state[rest], before[rest])


@pytest.mark.parametrize("a", [0.0, -1e-6, -0.7, -20.0, -math.inf])
def test_decode_decays(a):
    need_gpu()
    say(f"linear decode decay {a}")
    q, k, v, _, _, state, _ = make([1] * 3, 2, 2, 64, torch.float16, seed=4)
    before = state.clone()
    flag_attn.linear_attention_decode(q, k, v, torch.full((2,), a, device=DEV), state)
    torch.cuda.synchronize()
    kv = k.double()[..., :, None] * v.double()[..., None, :]
    end, size = math.exp(a) * before[:3].double() + kv, math.exp(a) * before[:3].double().abs() + kv.abs()
    assert bool(((state[:3] - end).abs() <= 8 * 2.0 ** -24 * size).all())


def test_decode_of_nothing():
    need_gpu()
    q, k, v, a, _, state, _ = make([1], 2, 2, 64, torch.float16)
    before = state.clone()
    assert flag_attn.linear_attention_decode(q[:0], k[:0], v[:0], a, state).shape == (0, 2, 64)
    assert flag_attn.linear_attention_decode(q, k, v, a, state[:0], i32([0])).count_nonzero() == 0
    assert torch.equal(state, before)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", DIMS)
def test_prompt_then_tokens_is_one_sequence(d, dtype):
    """A prompt in two chunks, then tokens one at a time: the same as the whole sequence at once, each
    within its own tolerance of the formula over the whole."""
    need_gpu()
    say(f"linear prompt then tokens d={d} {dtype}")
    h, hk, n = 4, 2, 77
    q, k, v, a, _, state, _ = make([n], h, hk, d, dtype, seed=8, slots=3)
    slot = i32([2])
    parts = []
    for b, e, has in ((0, 40, False), (40, 70, True)):
        parts.append(flag_attn.linear_attention_varlen(
            q[b:e], k[b:e], v[b:e], a, i32([0, e - b]), e - b, state, slot,
            torch.tensor([has], device=DEV)))
    for t in range(70, n):
        parts.append(flag_attn.linear_attention_decode(q[t:t + 1], k[t:t + 1], v[t:t + 1], a, state, slot))
    torch.cuda.synchronize()
    o = torch.cat(parts)
    for j in range(hk):
        heads = slice(j * (h // hk), (j + 1) * (h // hk))
        args = q[:, heads], k[:, j], v[:, j]
        ref, size, end, end_size = lo.attend(*args, float(a[j]), d ** -0.5)
        # a state that is handed on is a term of the next call's tolerance: u^2 of it once more
        assert_out(o[:, heads], ref, size, 4 * n, small_out(*args, None, d ** -0.5))
        assert_state(state[2, j], end, 2 * end_size, 4 * n, dtype, small_state(k[:, j], v[:, j], dtype))
