"""Tolerances of the rotary and linear-attention tests, from how the kernels round.

u is half a step of the output type (bf16 2^-8, fp16 2^-11).  Against the formula in 64 bits:

* rotary: the output is rounded once, u |y|; the angle is reduced to a part of a turn in 64 bits
  (positions below 2^31: off by 2^31 / 2 pi * 3 * 2^-53 turns, below 2^-22) and rounded to 32 (2^-25
  turns), so it is off by less than 2 pi (2^-22 + 2^-25) < 2^-19; the hardware's sine and cosine are
  taken to be within 2^-20 (``test_sine_of_a_turn`` holds them to it); fp32 products and a sum
  3 * 2^-24.  All in units of |x1| + |x2|: below 2^-18;
* linear attention, output: rounded once, u |o|, or by half of the smallest step.  Scores and the
  state's copy are rounded to the type to meet v and q: u of every term, u M with M the sum of
  magnitudes.  fp16 ones are taken relative to the largest of a token's 32 scores or of a
  column of the state: off by 2^-24 of that instead where they are small, 2^-24 (32 max|p| max|v| +
  sum|q| max|S| scale) in all, the maxima of v and S those of the output's column.  Scores are sums of D products, sums run over up to 64 terms a chunk
  and one per chunk, weights are off by (88 + 4) 2^-24 (an exponent above -88 and the function), two
  weights meet in a term;
* linear attention, state: the weighted values are split in two numbers of the type, whose rest is
  u^2; in fp16 no less than 2^-24 of the largest of their column of the chunk; the fall of a state is
  off by 2^-22 a chunk, its sums by 2^-24 times 32 terms.
"""
import torch

from tests._packed import HALF, TINY


def assert_turned(y, ref, size):
    tol = HALF[y.dtype] * ref.abs() + TINY[y.dtype] + 2.0 ** -18 * 1.01 * size
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), f"off by {float((err - tol).max()):.3e} past its tolerance"


def fp32_part(n, d):
    """What fp32 costs an output or a state in units of its magnitudes, n tokens, head dim d."""
    chunks = -(-n // 32)
    return (d + 64 + 2 * 92 + (4 + 32) * chunks) * 2.0 ** -24


def assert_out(o, ref, size, n, small=0.0):
    """o [n, G, D] against ref; size its magnitudes; small: what fp16's range costs."""
    u = HALF[o.dtype]
    tol = u * ref.abs() + TINY[o.dtype] + 1.02 * size * (u + u * u + fp32_part(n, o.shape[-1])) + small
    err = (o.double() - ref).abs()
    assert bool((err <= tol).all()), (
        f"{int((err > tol).sum())} of {err.numel()} outside: off by {float((err - tol).max()):.3e} past "
        f"its tolerance, error {float(err.max()):.3e}")


def assert_state(s, ref, size, n, dtype, small=0.0):
    u = HALF[dtype]
    tol = 1.02 * size * (u * u + fp32_part(n, s.shape[-1])) + small + 1e-37
    err = (s.double() - ref).abs()
    assert bool((err <= tol).all()), (
        f"state: {int((err > tol).sum())} of {err.numel()} outside: off by "
        f"{float((err - tol).max()):.3e} past its tolerance, error {float(err.max()):.3e}")


def small_out(q, k, v, state, scale):
    """What fp16's range costs an output of one KV head, at most: q [n, G, D], k, v [n, D]."""
    if q.dtype != torch.float16:
        return 0.0
    q, k, v = q.double().abs(), k.double().abs(), v.double().abs()
    row = q.sum(-1, keepdim=True)
    most_s = k.amax() * v.amax(0) * k.shape[0]  # of each column
    if state is not None:
        most_s = most_s + state.double().abs().amax(0)
    return 2.0 ** -24 * abs(scale) * row * (32 * k.max() * v.amax(0) + most_s)


def small_state(k, v, dtype):
    if dtype != torch.float16:
        return 0.0
    return 2.0 ** -24 * k.double().abs().sum(0)[:, None] * v.double().abs().amax(0)[None]
