"""Tolerances of the packed-attention and 4-bit-cache tests, from how the kernels round.

u is half a step of the output type (bf16 2^-8, fp16 2^-11).  Against the formula in 64 bits:

* the output is rounded once: u |o|; below the normal range by at most half of the smallest step;
* the weights are rounded to the type before they meet V: each off by u p, in all u a with
  a = sum p |v|; fp16 weights below 2^-14 of the row's largest are off by up to 2^-25 instead, so by
  at most 2^-25 n max|v| in all (the largest weight is 1, the row's sum at least that);
* a score is a sum of D products in fp32, in any order: off by at most (D + 2) 2^-24 ds, where ds
  is the sum of the products' magnitudes (times the scale); taking the exponent's argument
  rounds again by 2^-24 of its size, at most 4 ds 2^-24.  A weight and the row's sum
  are each off by that factor: 2 (D + 8) 2^-24 ds a;
* fp32 sums over n keys, exponentials, the split weights and the division: (n + 64) 2^-24 a, the
  n for partial sums that are each rounded.
"""
import ctypes

import torch

from flagattention_amd import _lib

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}  # half of the smallest step


def assert_rows(o, ref, a, ds, n, vmax):
    """o [..., D] of type fp16 / bf16 against float64 ref; a like ref, ds [...] per row, n keys."""
    u, d = HALF[o.dtype], o.shape[-1]
    tol = u * ref.abs() + TINY[o.dtype]
    tol = tol + a * (u + 2 * (d + 8) * 2.0 ** -24 * ds.unsqueeze(-1) + (n + 64) * 2.0 ** -24) * 1.01
    if o.dtype == torch.float16:
        tol = tol + 2.0 ** -25 * n * vmax
    err = (o.double() - ref).abs()
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(o), torch.isnan(ref)), "NaN in other places"
    assert torch.equal(torch.isinf(o), torch.isinf(ref)), "infinities in other places"
    bad = (err > tol) & fin
    assert not bool(bad.any()), (
        f"{int(bad.sum())} of {bad.numel()} outside: worst {float((err - tol)[bad].max()):.3e} past "
        f"its tolerance, error {float(err[bad].max()):.3e}")


def assert_largest_exact(o, ref, rest, ds, n, vmax, terms):
    """As assert_rows, where the rounding of the largest weight costs nothing: rest like ref, the sum of
    p |v| over the other keys, whose weights are each off by u p.  terms: the products of a score
    that are not 0 (the others add nothing, exactly).  The largest weight's own exponent is off by 2^-20
    at most (a reference below 2^5 is rounded by that), which P's rounding takes away, but not the
    row's sum."""
    u = HALF[o.dtype]
    fp32 = (2 * (terms + 8) * 2.0 ** -24 * ds.unsqueeze(-1) + (n + 64) * 2.0 ** -24 + 2.0 ** -20)
    tol = u * ref.abs() + TINY[o.dtype] + 1.01 * (u * rest + fp32 * (ref.abs() + 2 * rest))
    if o.dtype == torch.float16:
        tol = tol + 2.0 ** -25 * n * vmax
    err = (o.double() - ref).abs()
    assert bool((err <= tol).all()), (
        f"{int((err > tol).sum())} of {err.numel()} outside: worst {float((err - tol).max()):.3e} past "
        f"its tolerance, error {float(err[err > tol].max()):.3e}")


def assert_lse(lse, ref, ds, n, d):
    """lse: the scores' error, and that of a sum of n terms and of a logarithm in fp32."""
    assert torch.equal(torch.isneginf(lse), torch.isneginf(ref)), "-inf in other places"
    fin = torch.isfinite(ref)
    tol = (d + 8) * 2.0 ** -24 * ds + (n + 64) * 2.0 ** -24 + 2.0 ** -21 * ref.abs()
    err = (lse.double() - ref).abs()
    assert bool((err <= tol)[fin].all()), f"lse off by {float(err[fin].max()):.3e}"


def varlen_splits(total_q, total_k, seqs, h, hk, d, causal, max_q, max_k, cus):
    """(splits, tokens of each) that flash_attention_varlen takes."""
    args = _lib.VarlenArgs(num_seqs=seqs, total_q=total_q, total_k=total_k, h_q=h, h_kv=hk, d=d,
                           causal=int(causal))
    _lib.check(_lib.load().fa_varlen_plan(ctypes.byref(args), max_q, max_k, cus))
    return args.num_splits, args.split_tokens
