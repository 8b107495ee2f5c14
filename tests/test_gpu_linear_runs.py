"""Linear attention cut into segments, in every way that a launch can be: segment lengths, states joined in
a launch of their own or added up where they are read, the longest runs first or in packed order --
through the C ABI, which takes any of them -- and what a serving program does around the operators:
graphs, streams, wrong bounds, starts that fall, states and rows past 32-bit offsets."""
import ctypes
import math

import pytest
import torch

import flag_attn
from flagattention_amd import _lib, linear
from oracle import linear_oracle as lo
from tests._helpers import DEV, need_gpu, say
from tests._linear import assert_out, assert_state, small_out, small_state
from tests.test_gpu_graph import _capture_and_replay
from tests.test_gpu_linear import check, i32, make, starts

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def launch(q, k, v, a, cu, state, ids, has, segment, joined, order):
    """fa_linear_prompt as asked for; the output."""
    num_seqs = cu.shape[0] - 1
    total, h, d = q.shape
    hk = k.shape[1]
    o = torch.full_like(q, math.nan)
    args = linear._args(q, k, v, a, state, ids, o, num_seqs, d ** -0.5,
                        int(q.dtype == torch.bfloat16))
    args.cu_seqlens, args.has_state = cu.data_ptr(), None if has is None else has.data_ptr()
    args.segment, args.joined, args.sorted = segment, int(joined), int(order)
    runs = total // segment + num_seqs if segment else 0
    part = torch.full((max(4, runs * hk * d * d),), math.nan, device=DEV)  # nothing is read unwritten
    args.part = part.data_ptr()
    _lib.check(_lib.load().fa_linear_prompt(ctypes.byref(args),
                                            torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    return o


@pytest.mark.parametrize("joined", [False, True])
@pytest.mark.parametrize("order", [False, True])
@pytest.mark.parametrize("h,hk,d,dtype", [(2, 2, 64, torch.bfloat16), (4, 2, 64, torch.float16),
                                          (6, 1, 64, torch.bfloat16), (2, 2, 128, torch.bfloat16),
                                          (2, 2, 128, torch.float16), (3, 1, 128, torch.bfloat16),
                                          (1, 1, 256, torch.float16), (2, 1, 256, torch.bfloat16)])
@pytest.mark.parametrize("segment", [0, 32, 64, 160])
def test_every_way_to_cut(segment, h, hk, d, dtype, order, joined):
    """Lengths around the segments, an empty sequence, rows of no sequence, decays from one that ends
    within a chunk to one that lasts."""
    need_gpu()
    say(f"linear segment={segment} h={h} hk={hk} d={d} {dtype} order={order} joined={joined}")
    lens = [1, 64, 0, 130, 320, 31, 161, 65]
    q, k, v, a, cu, state, ids = make(lens, h, hk, d, dtype, seed=segment + d, first=3, behind=20)
    for x in (q, k, v):
        x[:3] = x[-20:] = math.nan
    for decay in (a, torch.full_like(a, -0.3), torch.full_like(a, -12.0)):
        has = torch.tensor([s % 3 != 1 for s in range(len(lens))], device=DEV)
        before = state.clone()
        o = launch(q, k, v, decay, i32(cu), state, ids, has, segment, joined, order)
        assert not bool(o[:3].any()) and not bool(o[cu[-1]:].any())
        for s, (b, e) in enumerate(zip(cu, cu[1:])):
            slot = int(ids[s])
            if b == e:
                assert torch.equal(state[slot], before[slot])
                continue
            for j in range(hk):
                heads = slice(j * (h // hk), (j + 1) * (h // hk))
                s0 = before[slot, j] if bool(has[s]) else None
                rows = q[b:e, heads], k[b:e, j], v[b:e, j]
                ref, size, end, end_size = lo.attend(*rows, float(decay[j]), d ** -0.5, s0)
                # a segment's state is handed on in fp32: a chunk more for each
                n = 2 * (e - b) + 64
                assert_out(o[b:e, heads], ref, size, n, small_out(*rows, s0, d ** -0.5))
                assert_state(state[slot, j], end, end_size, n, dtype, small_state(k[b:e, j], v[b:e, j], dtype))


@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16), (256, torch.bfloat16)])
def test_more_sequences_than_lanes(d, dtype):
    """70 sequences, long and short, in packed order; and 1,000 of up to 3 tokens."""
    need_gpu()
    say(f"linear 70 sequences d={d} {dtype}")
    lens = [(37 * s) % 150 + (400 if s % 23 == 0 else 0) for s in range(70)]
    q, k, v, a, cu, state, ids = make(lens, 2, 1, d, dtype, seed=1)
    check(q, k, v, a, cu, state, ids)
    state2 = state.clone()
    o = launch(q, k, v, a, i32(cu), state, ids, None, 96, True, False)
    o2 = launch(q, k, v, a, i32(cu), state2, ids, None, 96, True, False)
    assert torch.equal(o, o2) and torch.equal(state, state2)
    lens = [s % 4 for s in range(1000)]
    q, k, v, a, cu, state, ids = make(lens, 1, 1, 64, dtype, seed=2)
    for s in range(1000):
        if s % 7 == 0:
            ids[s] = -1
    before = state.clone()
    o = flag_attn.linear_attention_varlen(q, k, v, a, i32(cu), 3, state, ids)
    torch.cuda.synchronize()
    for s in list(range(0, 1000, 97)) + [999]:
        b, e = cu[s], cu[s + 1]
        if b < e:
            s0 = before[int(ids[s]), 0] if int(ids[s]) >= 0 else None
            ref, size, _, _ = lo.attend(q[b:e], k[b:e, 0], v[b:e, 0], float(a[0]), 64 ** -0.5, s0)
            assert_out(o[b:e], ref, size, 3, small_out(q[b:e], k[b:e, 0], v[b:e, 0], s0, 64 ** -0.5))


@pytest.mark.parametrize("most", [0, 1, 100, 5000])
def test_a_wrong_bound_changes_the_launch_only(most):
    need_gpu()
    say(f"linear max_seqlen={most}")
    q, k, v, a, cu, state, ids = make([900, 30, 2, 511], 2, 2, 128, torch.bfloat16, seed=3)
    before = state.clone()
    o = flag_attn.linear_attention_varlen(q, k, v, a, i32(cu), most, state, ids)
    torch.cuda.synchronize()
    for s, (b, e) in enumerate(zip(cu, cu[1:])):
        for j in range(2):
            ref, size, end, end_size = lo.attend(q[b:e, j:j + 1], k[b:e, j], v[b:e, j], float(a[j]),
                                                 128 ** -0.5, before[int(ids[s]), j])
            assert_out(o[b:e, j:j + 1], ref, size, 2 * (e - b) + 64)
            assert_state(state[int(ids[s]), j], end, end_size, 2 * (e - b) + 64, q.dtype)


@pytest.mark.parametrize("joined", [False, True])
@pytest.mark.parametrize("steps", [(14, 0), (0, 14), (0, 7, 14, 3)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_fp16_segments_of_values_that_rise_and_fall(d, steps, joined):
    """Values of 2^-12 to 2 in their dims, up to 2^14 times larger from one part of a sequence to the next,
    behind states of nothing, tiny and large ones: the power that a segment's state is taken in follows."""
    need_gpu()
    say(f"linear fp16 segments d={d} {steps} joined={joined}")
    lens, dtype = [400, 350, 290], torch.float16
    q, k, v, a, cu, state, ids = make(lens, 2, 1, d, dtype, seed=d)
    q *= 2.0 ** -10
    gen = torch.Generator(device=DEV).manual_seed(3)
    v *= (2.0 ** torch.linspace(-12, 1, d, device=DEV))[torch.randperm(d, generator=gen, device=DEV)]
    for b, e in zip(cu, cu[1:]):
        for i, step in enumerate(steps):
            v[b + (e - b) * i // len(steps):b + (e - b) * (i + 1) // len(steps)] *= 2.0 ** (step - 7)
    state[int(ids[1])] *= 2.0 ** -24
    state[int(ids[2])] *= 2.0 ** 12
    for decay in (torch.full_like(a, -0.0005), torch.full_like(a, -0.2)):
        has, before, now = torch.tensor([0, 1, 1], device=DEV, dtype=torch.uint8), state.clone(), state.clone()
        o = launch(q, k, v, decay, i32(cu), now, ids, has, 96, joined, True)
        for s, (b, e) in enumerate(zip(cu, cu[1:])):
            s0 = before[int(ids[s]), 0] if s > 0 else None
            rows = q[b:e], k[b:e, 0], v[b:e, 0]
            ref, size, end, end_size = lo.attend(*rows, float(decay[0]), d ** -0.5, s0)
            n = 2 * (e - b) + 64
            assert_out(o[b:e], ref, size, n, small_out(*rows, s0, d ** -0.5))
            assert_state(now[int(ids[s]), 0], end, end_size, n, dtype, small_state(k[b:e, 0], v[b:e, 0], dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("h,hk,d", [(16, 16, 64), (24, 8, 64), (16, 16, 128), (24, 8, 128), (8, 8, 256), (24, 8, 256)])
def test_the_same_call_gives_the_same_bits(h, hk, d, dtype):
    """Of a full card, twenty times over: nothing depends on which wave or work-group comes first."""
    need_gpu()
    say(f"linear repeats h={h} hk={hk} d={d} {dtype}")
    lens = [1500, 3, 700, 33, 900, 0, 64, 1, 400, 1023]
    q, k, v, a, cu, state, ids = make(lens, h, hk, d, dtype, seed=d + h, behind=5)
    first = None
    for _ in range(20):
        end = state.clone()
        o = flag_attn.linear_attention_varlen(q, k, v, a, i32(cu), 1500, end, ids)
        if first is None:
            first = o, end
        else:
            assert torch.equal(o, first[0]) and torch.equal(end, first[1])


@pytest.mark.parametrize("segment", [0, 32])
@pytest.mark.parametrize("order", [False, True])
def test_starts_that_fall_or_leave_the_rows_stay_in_bounds(segment, order):
    """Such lists name no sequences; what lies around the outputs and the states is not touched."""
    need_gpu()
    say(f"linear bad starts segment={segment} order={order}")
    n, d = 100, 64
    rows = torch.randn((3, n, 2, d), device=DEV).half()
    a = torch.full((2,), -0.1, device=DEV)
    for cu in ([50, 20, 90, 10], [-5, 40, 1 << 30, 200], [100, 100, 0, 0], [-9, -8, -7, -6]):
        room = torch.full((7, 2, d, d), 7.0, device=DEV)
        state = room[2:5]
        launch(*rows.unbind(0), a, i32(cu), state, None, None, segment, True, order)
        assert bool((room[:2] == 7).all()) and bool((room[5:] == 7).all())


def test_offsets_past_32_bits():
    """Rows 2^16 apart (5.2 GB each), and a slot past 2^31 elements."""
    need_gpu()
    say("linear far rows and slots")
    n, d = 40000, 128
    big = torch.empty((n, 1 << 16), dtype=torch.bfloat16, device=DEV)
    rows = big[:, :3 * d].view(n, 3, d)
    tail = 300
    rows[n - tail:] = torch.randn((tail, 3, d), device=DEV).bfloat16()
    cu = [n - tail, n - 100, n]
    far = torch.empty((140000, 1, d, d), device=DEV)
    ids = i32([139999, 0])
    far[139999], far[0] = torch.randn((1, d, d), device=DEV), torch.randn((1, d, d), device=DEV)
    s0 = far[139999, 0].clone()
    q, k, v = (rows[:, i:i + 1] for i in range(3))
    a = torch.full((1,), -0.02, device=DEV)
    o = flag_attn.linear_attention_varlen(q, k, v, a, i32(cu), 200, far, ids)
    torch.cuda.synchronize()
    b, e = cu[:2]
    ref, size, end, end_size = lo.attend(q[b:e], k[b:e, 0], v[b:e, 0], float(a[0]), d ** -0.5, s0)
    assert_out(o[b:e], ref, size, 500)
    assert_state(far[139999, 0], end, end_size, 500, torch.bfloat16)
    assert not bool(o[:b].any())
    s1 = far[139999, 0].double()
    o1 = flag_attn.linear_attention_decode(q[-1:], k[-1:], v[-1:], a, far, ids[:1])
    torch.cuda.synchronize()
    end = math.exp(float(a[0])) * s1 + k[-1, 0].double()[:, None] * v[-1, 0].double()
    size = math.exp(float(a[0])) * s1.abs() + k[-1, 0].double().abs()[:, None] * v[-1, 0].double().abs()
    qs = q[-1].double() * d ** -0.5
    assert_out(o1, (qs @ end)[None], (qs.abs() @ size)[None], 1)


@pytest.mark.parametrize("d,lens", [(64, [5, 0, 33]), (128, [700, 20]), (256, [300])])
def test_graph_prompt_and_tokens(d, lens):
    """A prompt (cut into segments where it is long) and a decode step in one graph: the replays see new
    rows, states and lengths."""
    need_gpu()
    say(f"linear graph d={d} {lens}")
    q, k, v, a, cu, state, ids = make(lens, 4, 2, d, torch.bfloat16, seed=4, behind=8)
    cu = i32(cu)
    kept = state.clone()
    gen = torch.Generator(device=DEV).manual_seed(5)

    def eager():
        state.copy_(kept)
        o = flag_attn.linear_attention_varlen(q, k, v, a, cu, max(lens), state, ids)
        mid = state.clone()
        b = len(lens)
        o1 = flag_attn.linear_attention_decode(q[:b], k[:b], v[:b], a, state, ids)
        return o, mid, o1, state.clone()

    def update(rep):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=gen, device=DEV))
        kept.copy_(torch.randn(kept.shape, generator=gen, device=DEV))
        cu[1:] -= (cu[1:] > 3 * (rep + 1)) * (rep + 1)

    _capture_and_replay(eager, update, ("o", "state", "o1", "state after"))


def test_streams_of_their_own():
    """Calls on two other streams at once, each with its workspace: the same bits as one after the other."""
    need_gpu()
    say("linear streams")
    sets = [make([1500, 40], 4, 2, 128, torch.bfloat16, seed=s) for s in (1, 2)]
    want = []
    for q, k, v, a, cu, state, ids in sets:
        mine = state.clone()
        want.append((flag_attn.linear_attention_varlen(q, k, v, a, i32(cu), 1500, mine, ids), mine))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    cus = [i32(s[4]) for s in sets]
    torch.cuda.synchronize()
    got = []
    for (q, k, v, a, _, state, ids), cu, stream in zip(sets, cus, streams):
        with torch.cuda.stream(stream):
            got.append((flag_attn.linear_attention_varlen(q, k, v, a, cu, 1500, state, ids), state))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("segment,joined", [(0, False), (64, False), (64, True)])
def test_what_is_not_finite_across_segments(segment, joined, which):
    """Tokens before an infinity keep their bits; those after it, in its segment and the next ones, are
    not finite where it reaches them (its weight is above fp32's least here)."""
    need_gpu()
    say(f"linear infinity segment={segment} joined={joined} {which}")
    d, n, t = 64, 256, 70
    q, k, v, _, cu, state, ids = make([n], 1, 1, d, torch.bfloat16, seed=6, slots=1)
    a = torch.full((1,), -0.02, device=DEV)
    args = (a, i32(cu))
    o = launch(q, k, v, *args, state.clone(), ids, None, segment, joined, False)
    x = k if which == "k" else v
    x[t, 0, 9] = math.inf
    o2 = launch(q, k, v, *args, state, ids, None, segment, joined, False)
    assert torch.equal(o2[:t], o[:t])
    cols = slice(None) if which == "k" else slice(9, 10)
    assert not bool(torch.isfinite(o2[t:, 0, cols]).any())
    if which == "v":
        rest = torch.ones(d, dtype=torch.bool, device=DEV)
        rest[9] = False
        assert torch.equal(o2[:, :, rest], o[:, :, rest])
