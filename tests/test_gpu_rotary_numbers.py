"""What the hardware's sine and cosine cost rotary positions, read finer than the output type."""
import math

import pytest
import torch

import flag_attn
from tests._helpers import DEV, need_gpu, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("start", [0, 1 << 30])
def test_sine_and_cosine_finer_than_the_type(start, adjacent):
    """x = (sin, cos) rounded to fp16: x1 cos - x2 sin is what those roundings left, 2^-11 at most, and rounded
    by 2^-11 of itself, so that an error of 2^-20 in either function shows.  The other output is 1.  The angle
    in turns is rounded to 2^-26 (2^-23 in radians), or by 2^-22 past 2^30 positions (three roundings of 2^30 / 2
    pi / 64 turns by 2^-53 are less), and fp32 products and a sum cost 3 * 2^-24."""
    need_gpu()
    say(f"rotary fine sine start={start} adjacent={adjacent}")
    n = 1 << 16
    pos = start + torch.arange(-n if start == 0 else 0, n, device=DEV)
    f = torch.tensor([2 * math.pi / n], device=DEV)
    angle = pos.double() * f.double()
    c, s = torch.cos(angle), torch.sin(angle)
    x = torch.stack((s, c), -1).half()[:, None].contiguous()
    y, z = flag_attn.rotary_embedding(x, x, pos, f, adjacent_pairs=adjacent)
    torch.cuda.synchronize()
    assert torch.equal(y, z)
    x = x.double()
    ref = x[..., 0] * c[:, None] - x[..., 1] * s[:, None]
    assert float(ref.abs().max()) <= 2.0 ** -11
    angle_off = 2.0 ** -23 if start == 0 else 2.0 ** -22
    tol = (2.0 ** -20 + angle_off + 3 * 2.0 ** -24) * x.abs().sum(-1) + 2.0 ** -11 * ref.abs() + 2.0 ** -25
    err = (y[..., 0].double() - ref).abs()
    print(f"worst {float(err.max()) * 2 ** 20:.3f} of 2^-20", flush=True)
    assert bool((err <= tol).all()), f"off by {float(err.max()):.3e}"
    one = x[..., 1] * c[:, None] + x[..., 0] * s[:, None]
    assert bool(((y[..., 1].double() - one).abs() <= 2.0 ** -11 * one.abs() + tol).all())
