"""Oracle of packed prompt attention and of the 4-bit K/V cache, in float64.  TEST INFRASTRUCTURE
ONLY: written from the operators' definitions, on whatever device its inputs are on.

Beside each result stands what its tolerance is made of: the sums of magnitudes that roundings
scale with.
"""
from __future__ import annotations

import math

import torch

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def attend(q, k, v, scale, causal):
    """One head of one sequence: q [m, D], k, v [n, D] -> (o, lse, a, ds).

    a: sum of p |v| per output; ds: scale * max over the visible keys of sum |q| |k|, per row.
    A row without a visible key gets o = 0, lse = -inf.  A value of V at a key that a row does not
    see has no part in that row."""
    m, n = q.shape[0], k.shape[0]
    q, k, v = q.double(), k.double(), v.double()
    if n == 0:
        z = torch.zeros_like(q)
        return z, torch.full((m,), -math.inf, dtype=torch.float64, device=q.device), z, z[:, 0]
    s = (q @ k.t()) * scale
    mag = (q.abs() @ k.abs().t()) * abs(scale)
    if causal:
        seen = (torch.arange(n, device=q.device)[None, :] <=
                torch.arange(m, device=q.device)[:, None] + n - m)
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        mag = torch.where(seen, mag, torch.zeros_like(mag))
    else:
        seen = torch.ones_like(s, dtype=torch.bool)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen, torch.exp(s - lse[:, None]), torch.zeros_like(s))
    finite = torch.isfinite(v)
    o = p @ torch.where(finite, v, torch.zeros_like(v))
    a = p @ torch.where(finite, v, torch.zeros_like(v)).abs()
    if not bool(finite.all()):
        for j in (~finite).any(1).nonzero().flatten().tolist():
            bad = ~finite[j]
            o[:, bad] += torch.where(seen[:, j:j + 1], p[:, j:j + 1] * v[j, bad][None, :],
                                     torch.zeros((), dtype=v.dtype, device=v.device))
    return o, lse, a, mag.amax(-1)


def attend_rest(q, k, v, scale):
    """One head that sees every key: (o, rest, ds), rest the sum of p |v| but for each row's largest
    weight."""
    o, lse, a, ds = attend(q, k, v, scale, False)
    s = (q.double() @ k.double().t()) * scale
    top, at = s.max(-1)
    return o, a - torch.exp(top - lse)[:, None] * v.double()[at].abs(), ds


def varlen(q, k, v, cu_q, cu_k, scale, causal):
    """Packed attention: (o [total_q, H, D], lse [H, total_q], a like o, ds like lse)."""
    total, h, d = q.shape
    group = h // k.shape[1]
    o = torch.zeros((total, h, d), dtype=torch.float64, device=q.device)
    a = torch.zeros_like(o)
    lse = torch.full((h, total), -math.inf, dtype=torch.float64, device=q.device)
    ds = torch.zeros_like(lse)
    for i in range(len(cu_q) - 1):
        qs, ks = slice(cu_q[i], cu_q[i + 1]), slice(cu_k[i], cu_k[i + 1])
        if qs.start == qs.stop:
            continue
        for j in range(h):
            o[qs, j], lse[j, qs], a[qs, j], ds[j, qs] = attend(
                q[qs, j], k[ks, j // group], v[ks, j // group], scale, causal)
    return o, lse, a, ds


def pow2(byte):
    """2^(byte - 127) as float64, from the bits (a device's power function may be an ulp off)."""
    return ((byte.long() + (1023 - 127)) << 52).view(torch.float64)


def values(codes, scales):
    """float64 values of rows of codes [..., D / 2] with scale bytes [..., D / 32]."""
    table = torch.tensor(MAGNITUDES + tuple(-x for x in MAGNITUDES), dtype=torch.float64,
                         device=codes.device)
    nib = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    power = pow2(scales)
    power = torch.where(scales == 255, torch.full_like(power, math.nan), power)
    return (table[nib].unflatten(-1, (-1, 32)) * power.unsqueeze(-1)).flatten(-2)


def quantise(x):
    """(codes, scale bytes) of rows [..., D]: by trying every exponent and every magnitude."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1)
    ok = torch.isfinite(g).all(-1)
    byte = torch.zeros(top.shape, dtype=torch.int64, device=x.device)
    for e in range(254):
        byte += (top > 7 * 2.0 ** (e - 127)).long()
    byte = torch.where(ok, byte, torch.full_like(byte, 255))
    y = torch.where(ok.unsqueeze(-1), g, torch.zeros_like(g)) / pow2(byte).unsqueeze(-1)
    mags = torch.tensor(MAGNITUDES, dtype=torch.float64, device=x.device)
    dist = (y.abs().unsqueeze(-1) - mags).abs()
    best = dist.amin(-1, keepdim=True)
    near = dist == best  # one code, or two neighbours: then the even one
    even = torch.arange(8, device=x.device) % 2 == 0
    two = near.sum(-1, keepdim=True) > 1
    code = torch.where(two, near & even, near).long().argmax(-1)
    code = code | (torch.signbit(y).long() << 3)
    code = torch.where(ok.unsqueeze(-1), code, torch.zeros_like(code))
    code = code.flatten(-2).unflatten(-1, (-1, 2))
    return (code[..., 0] | (code[..., 1] << 4)).to(torch.uint8), byte.to(torch.uint8)


def write(codes, scales, x, slots):
    """The cache after writing rows x [T, H_kv, D] at slots (those outside are skipped)."""
    codes, scales = codes.clone(), scales.clone()
    block = codes.shape[2]
    c, s = quantise(x)
    for i, slot in enumerate(slots.tolist()):
        if 0 <= slot < codes.shape[0] * block:
            codes[slot // block, :, slot % block] = c[i]
            scales[slot // block, :, slot % block] = s[i]
    return codes, scales


def context(codes, scales, row, n):
    """(float64 [n, H_kv, D], bool [n]) tokens of the sequence whose blocks row lists; those of
    blocks outside the cache are zeros and False."""
    block = codes.shape[2]
    x = torch.zeros((n, codes.shape[1], 2 * codes.shape[3]), dtype=torch.float64,
                    device=codes.device)
    seen = torch.zeros(n, dtype=torch.bool, device=codes.device)
    for b in range(-(-n // block)):
        page = int(row[b]) if b < row.shape[0] else -1
        if 0 <= page < codes.shape[0]:
            at = slice(b * block, min((b + 1) * block, n))
            x[at] = values(codes[page], scales[page]).transpose(0, 1)[:at.stop - at.start]
            seen[at] = True
    return x, seen
