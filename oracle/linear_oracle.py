"""Oracle of rotary positions and of linear attention with a decay per head, in float64.  TEST
INFRASTRUCTURE ONLY: written from the operators' definitions, on whatever device its inputs are on.

Beside each result stands what its tolerance is made of: the sums of magnitudes that roundings
scale with.
"""
from __future__ import annotations

import torch


def powers(a, n):
    """e^(a n) of a float a and a tensor of whole numbers, 1 where they are 0."""
    n = n.double()
    return torch.where(n == 0, torch.ones_like(n), torch.exp(a * n))


def attend(q, k, v, a, scale, state=None):
    """One KV head of one sequence: q [n, G, D], k, v [n, D], a float, state [D, D] or None ->
    (o [n, G, D], size like o, state, state_size): o by its sum over the tokens seen, size the same
    sum of magnitudes."""
    n, _, d = q.shape
    q, k, v = q.double(), k.double(), v.double()
    s0 = torch.zeros((d, d), dtype=torch.float64, device=q.device) if state is None else state.double()
    i = torch.arange(n, device=q.device)
    gap = i[:, None] - i[None, :]
    w = torch.where(gap >= 0, powers(a, gap.clamp(min=0)), 0.0)
    o, size = torch.empty_like(q), torch.empty_like(q)
    since = powers(a, i + 1)[:, None]
    for g in range(q.shape[1]):
        x = q[:, g]
        o[:, g] = scale * ((x @ k.t() * w) @ v + since * (x @ s0))
        size[:, g] = abs(scale) * ((x.abs() @ k.abs().t() * w) @ v.abs() + since * (x.abs() @ s0.abs()))
    left = powers(a, n - 1 - i)[:, None]
    fall = powers(a, torch.full((1,), n, device=q.device))
    return (o, size, fall * s0 + k.t() @ (left * v), fall * s0.abs() + k.abs().t() @ (left * v.abs()))


def angles(positions, inv_freq, sections=None, mixed=False):
    """[tokens, pairs] in float64: the angle of each pair."""
    pairs = inv_freq.shape[0]
    p = positions.double().view(-1, positions.shape[-1])
    sections = (pairs,) if sections is None else sections
    axis = [0] * pairs
    if mixed:
        for a in range(1, len(sections)):
            for m in range(sections[a]):
                axis[m * len(sections) + a] = a
    else:
        axis = [a for a, m in enumerate(sections) for _ in range(m)]
    return torch.stack([p[axis[i]] * inv_freq[i].double() for i in range(pairs)], 1)


def turn(x, angle, adjacent=False):
    """x [tokens, heads, D] by angle [tokens, pairs] -> (y, size)."""
    x = x.double()
    y, size = x.clone(), x.abs()
    pairs = angle.shape[1]
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    one = slice(0, 2 * pairs, 2) if adjacent else slice(0, pairs)
    two = slice(1, 2 * pairs, 2) if adjacent else slice(pairs, 2 * pairs)
    u, w = x[..., one], x[..., two]
    y[..., one], y[..., two] = u * c - w * s, w * c + u * s
    size[..., one] = size[..., two] = u.abs() + w.abs()
    return y, size
