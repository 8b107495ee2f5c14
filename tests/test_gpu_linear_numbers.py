"""Linear attention where its numbers are hard: fp16 states from tiny to large, states over many tokens
and segments, each against the formula in 64 bits."""
import ctypes
import math

import pytest
import torch

import flag_attn
from flagattention_amd import _lib, linear
from oracle import linear_oracle as lo
from tests._helpers import DEV, need_gpu, say
from tests._linear import assert_out, assert_state, small_out, small_state
from tests.test_gpu_linear import i32

pytestmark = pytest.mark.gpu


def rows(n, h, d, dtype, seed, gain=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (gain * torch.randn((n, h, d), generator=gen, device=DEV)).to(dtype)


def prompt(q, k, v, a, state, scale, segment, joined=True):
    """One sequence through fa_linear_prompt, in segments of so many tokens; the output."""
    n, _, d = q.shape
    hk = k.shape[1]
    o = torch.full_like(q, math.nan)
    cu = i32([0, n])
    args = linear._args(q, k, v, a, state, None, o, 1, scale, int(q.dtype == torch.bfloat16))
    args.cu_seqlens, args.segment, args.joined = cu.data_ptr(), segment, int(joined)
    part = torch.full(((n // segment + 1 if segment else 1) * hk * d * d,), math.nan, device=DEV)
    args.part = part.data_ptr()
    _lib.check(_lib.load().fa_linear_prompt(ctypes.byref(args),
                                            torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    return o


@pytest.mark.parametrize("segment", [0, 32, 96])
@pytest.mark.parametrize("h,d", [(1, 64), (4, 64), (1, 128), (2, 128), (1, 256), (2, 256)])
@pytest.mark.parametrize("a,first", [(-1.0, 1.0), (-0.65, 1.0), (-0.01, 1e-30), (-0.3, 0.0)])
def test_fp16_large_values_behind_next_to_nothing(a, first, h, d, segment):
    """A state that falls to nothing, that starts next to nothing, or that is nothing; 96 tokens without
    values in half of the columns; then one of 20,000 times 20,000, and ordinary ones."""
    need_gpu()
    say(f"linear fp16 from nothing a={a} first={first} h={h} d={d} segment={segment}")
    n, scale = 150, 2.0 ** -20  # brings outputs of 4e8 back into fp16
    q, k, v = (rows(n, x, d, torch.float16, i) for i, x in enumerate((h, 1, 1)))
    q *= 2.0 ** -10
    v[:96, :, ::2] = 0
    k[96], v[96] = 20000.0, 20000.0
    state = rows(1, d, d, torch.float32, 3, first)[None]
    decay = torch.full((1,), a, device=DEV)
    s0 = state[0, 0].clone()
    args = q, k[:, 0], v[:, 0]
    ref, size, end, end_size = lo.attend(*args, float(decay[0]), scale, s0)
    o = prompt(q, k, v, decay, state, scale, segment)
    assert bool(torch.isfinite(state).all()), "a state of 4e8 is finite"
    assert_out(o, ref, size, 2 * n + 64, small_out(*args, s0, scale))
    assert_state(state[0, 0], end, end_size, 2 * n + 64, q.dtype, small_state(k[:, 0], v[:, 0], q.dtype))


@pytest.mark.parametrize("segment", [0, 64, 96])
@pytest.mark.parametrize("a", [-0.05, -0.5])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_fp16_values_before_tokens_without_any(d, a, segment):
    """The last 90 tokens have no values in half of the columns: what the first 60 leave there is small, and
    as exact as any (the weighted values are held in 22 bits, the rest in fp32)."""
    need_gpu()
    say(f"linear fp16 before nothing d={d} a={a} segment={segment}")
    n = 150
    q, k, v = (rows(n, 1, d, torch.float16, i) for i in range(3))
    v[60:, :, ::2] = 0
    state = torch.zeros((1, 1, d, d), device=DEV)
    decay = torch.full((1,), a, device=DEV)
    ref, size, end, end_size = lo.attend(q, k[:, 0], v[:, 0], float(decay[0]), 0.1)
    o = prompt(q, k, v, decay, state, 0.1, segment)
    assert_out(o, ref, size, 2 * n + 64, small_out(q, k[:, 0], v[:, 0], None, 0.1))
    assert_state(state[0, 0], end, end_size, 2 * n + 64, q.dtype)


@pytest.mark.parametrize("segment", [0, 64])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_fp16_small_values_beside_large_ones(d, segment):
    """Values of 2^-8 between values of up to 2^15, the former with keys of their own: what they leave in the
    state is off by no more than 2^-36 of the largest value.  (The parts of a weighted value are off by
    2^-25 of a unit, which the largest is 2^11 of, at least.)"""
    need_gpu()
    say(f"linear fp16 small beside large d={d} segment={segment}")
    n = 150
    q, k, v = (rows(n, 1, d, torch.float16, i) for i in range(3))
    k[::2, :, ::2] = 0
    k[1::2, :, 1::2] = 0
    v[::2] *= 2.0 ** 12
    v[1::2] *= 2.0 ** -8
    state = torch.zeros((1, 1, d, d), device=DEV)
    decay = torch.full((1,), -0.02, device=DEV)
    _, _, end, end_size = lo.attend(q, k[:, 0], v[:, 0], float(decay[0]), 1e-4)
    prompt(q, k, v, decay, state, 1e-4, segment)
    assert_state(state[0, 0], end, end_size, 2 * n + 64, q.dtype,
                 2.0 ** -12 * small_state(k[:, 0], v[:, 0], q.dtype))


@pytest.mark.parametrize("h,d", [(1, 64), (1, 128), (3, 128), (1, 256)])
def test_fp16_small_scores_of_large_values(h, d):
    """Keys of 2^10 with values of 2^-10 between keys of 2^-14 with values of 2^13, which make most of the
    output: scores are off by 2^-11 of themselves, or by 2^-39 of the largest (2^-25 of a unit, which
    that is 2^14 of, at least)."""
    need_gpu()
    say(f"linear fp16 small scores h={h} d={d}")
    n = 64
    q, k, v = (rows(n, x, d, torch.float16, i) for i, x in enumerate((h, 1, 1)))
    k[::2] *= 2.0 ** 10
    v[::2] *= 2.0 ** -10
    k[1::2] *= 2.0 ** -14
    v[1::2] *= 2.0 ** 13
    decay = torch.full((1,), -0.02, device=DEV)
    # chunk after chunk from nothing, so that no state has a part
    for b in (0, 32):
        args = q[b:b + 32], k[b:b + 32], v[b:b + 32]
        ref, size, _, _ = lo.attend(args[0], args[1][:, 0], args[2][:, 0], float(decay[0]), 2.0 ** -3)
        o = prompt(*args, decay, None, 2.0 ** -3, 0)
        assert_out(o, ref, size, 32, 2.0 ** -14 * small_out(args[0], args[1][:, 0], args[2][:, 0], None, 2.0 ** -3))


@pytest.mark.parametrize("segment", [0, 64])
@pytest.mark.parametrize("h,d,used", [(2, 64, 48), (1, 128, 96), (4, 128, 80), (1, 256, 192)])
def test_fp16_heads_padded_with_zeros(h, d, used, segment):
    """Dims that have nothing keep nothing, and the others are what they are without them; one of them gets
    its first, tiny value late."""
    need_gpu()
    say(f"linear fp16 padded h={h} d={d} used={used} segment={segment}")
    n, scale = 300, used ** -0.5
    q, k, v = (rows(n, x, d, torch.float16, i) for i, x in enumerate((h, 1, 1)))
    for x in (q, k, v):
        x[..., used:] = 0
    v[200:, 0, used] = 2.0 ** -12 * v[200:, 0, 0]
    state = torch.zeros((1, 1, d, d), device=DEV)
    decay = torch.full((1,), -0.02, device=DEV)
    ref, size, end, end_size = lo.attend(q, k[:, 0], v[:, 0], float(decay[0]), scale)
    o = prompt(q, k, v, decay, state, scale, segment)
    assert_out(o, ref, size, 2 * n + 64, 2.0 ** -10 * small_out(q, k[:, 0], v[:, 0], None, scale))
    assert_state(state[0, 0], end, end_size, 2 * n + 64, q.dtype, 2.0 ** -12 * small_state(k[:, 0], v[:, 0], q.dtype))
    assert not bool(o[..., used + 1:].any()) and not bool(state[0, 0, :, used + 1:].any())
    assert not bool(o[:200, :, used].any()) and not bool(state[0, 0, used:].any())


def long_state(n, d, dtype, a, first, segment, joined):
    """(error, size) of the state that n tokens of one sign leave behind one of `first`, in 64 bits."""
    q, k, v = (rows(n, 1, d, dtype, i).abs() for i in range(3))
    state = rows(1, d, d, torch.float32, 3, first).abs()[None]
    decay = torch.full((1,), a, device=DEV)
    left = lo.powers(float(decay[0]), n - 1 - torch.arange(n, device=DEV))[:, None]
    fall = lo.powers(float(decay[0]), torch.full((1,), n, device=DEV))
    end = fall * state[0, 0].double() + k[:, 0].double().t() @ (left * v[:, 0].double())
    prompt(q, k, v, decay, state, 1e-6, segment, joined)
    return state[0, 0].double() - end, end


@pytest.mark.parametrize("segment,joined", [(0, False), (256, True), (4096, True), (1024, False)])
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (64, torch.float16), (128, torch.bfloat16),
                                     (256, torch.bfloat16), (256, torch.float16)])
@pytest.mark.parametrize("a", [0.0, -1e-6, -1e-5, -1e-4])
@pytest.mark.parametrize("first", [1.0, 1e6])
def test_states_of_many_tokens(first, a, d, dtype, segment, joined):
    """131,001 tokens of one sign, slow decays, behind a state like them or far above them: every sum is
    rounded to nearest, so errors of 2^-25 each grow by the square root of their number (6 sigma:
    2 sqrt(sums) 2^-24 where the state is as large throughout), and nothing is lost always the same
    way but what the weights are off by (eight roundings or last bits of an exponential)."""
    need_gpu()
    say(f"linear long states d={d} {dtype} a={a} first={first} segment={segment} joined={joined}")
    n = 131001
    err, end = long_state(n, d, dtype, a, first, segment, joined)
    sums = n / 32 if segment == 0 else segment / 32 + n / segment
    assert float((err / end).abs().max()) <= (2 * math.sqrt(sums) + 16) * 2.0 ** -24
    assert abs(float((err / end).mean())) <= 8 * 2.0 ** -24


@pytest.mark.parametrize("segment,joined", [(0, False), (96, False), (96, True), (32, True)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_fp16_small_values_before_large_ones(d, segment, joined):
    """Values of 2^-12, 32 large ones and small ones again, each kind with keys of its own: 22 bits of all."""
    need_gpu()
    say(f"linear fp16 small before large d={d} segment={segment} joined={joined}")
    n = 320
    q, k, v = (rows(n, 1, d, torch.float16, i) for i in range(3))
    large = torch.zeros(n, dtype=torch.bool, device=DEV)
    large[160:192] = True
    k[large, :, ::2] = 0
    k[~large, :, 1::2] = 0
    v[large] *= 2.0 ** 13
    v[~large] *= 2.0 ** -12
    state = torch.zeros((1, 1, d, d), device=DEV)
    decay = torch.full((1,), -0.02, device=DEV)
    _, _, end, end_size = lo.attend(q, k[:, 0], v[:, 0], float(decay[0]), 1e-4)
    prompt(q, k, v, decay, state, 1e-4, segment, joined)
    assert_state(state[0, 0], end, end_size, n, q.dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("a", [0.0, -1e-6, -1e-5, -1e-3])
def test_states_of_many_single_tokens(a, dtype):
    """4,000 steps of decode, k and v of one sign behind states of 1000: a step rounds a state once at its
    size (to nearest: 2^-24 of it at most, an error of 2^-24 / sqrt(3) each, 6 sigma over the steps), and
    nothing drifts."""
    need_gpu()
    say(f"linear many single tokens a={a} {dtype}")
    n, d = 4000, 64
    q, k, v = (rows(n, 1, d, dtype, i).abs() for i in range(3))
    state = torch.full((1, 1, d, d), 1000.0, device=DEV)
    ref, decay = state[0, 0].double(), torch.full((1,), a, device=DEV)
    step = torch.exp(decay.double())
    for t in range(n):
        flag_attn.linear_attention_decode(q[t:t + 1], k[t:t + 1], v[t:t + 1], decay, state)
        ref = ref * step + k[t, 0].double()[:, None] * v[t, 0].double()
    err = (state[0, 0].double() - ref) / ref
    assert float(err.abs().max()) <= 6 / math.sqrt(3) * math.sqrt(n) * 2.0 ** -24
    assert abs(float(err.mean())) <= 8 * 2.0 ** -24


@pytest.mark.parametrize("h,d", [(1, 64), (4, 64), (1, 128), (2, 128), (1, 256)])
@pytest.mark.parametrize("a", [-0.02, -0.1, -0.2, -0.6])
def test_fp16_small_rows_of_a_state_that_falls(a, h, d):
    """A state that only falls, q along rows that are 2^-10 of the others: a state's copy is off by 2^-11 of
    itself, or by 2^-20 of the largest of its column (2^-25 of a unit, which that is 2^-5 of, at least)."""
    need_gpu()
    say(f"linear fp16 falling state a={a} h={h} d={d}")
    n = min(400, int(40 / -a))
    q = rows(n, h, d, torch.float16, 1)
    q[..., ::2] = 0
    k = v = torch.zeros((n, 1, d), dtype=torch.float16, device=DEV)
    s0 = rows(1, d, d, torch.float32, 2)[0]
    s0[1::2] *= 2.0 ** -10
    decay = torch.full((1,), a, device=DEV)
    fall = torch.exp(float(decay[0]) * (1 + torch.arange(n, device=DEV).double()))[:, None, None]
    scale = 2.0 ** 10
    o = prompt(q, k, v, decay, s0[None, None].clone(), scale, 0)
    x = scale * q.double()
    ref, size = x @ s0.double() * fall, x.abs() @ s0.double().abs() * fall
    small = 2.0 ** -20 * x.abs().sum(-1, keepdim=True) * s0.double().abs().amax(0) * fall
    assert_out(o, ref, size, n, small)
