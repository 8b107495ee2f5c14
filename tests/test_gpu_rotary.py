"""Rotary positions (flag_attn.rotary_embedding, rotary_cache_kv) against the formula in 64 bits, with
tolerances made of the roundings they make (tests/_linear.py)."""
import math

import pytest
import torch

import flag_attn
from oracle import linear_oracle as lo
from tests._helpers import DEV, need_gpu, say
from tests._linear import assert_turned

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def frequencies(pairs, base=1e4):
    return (base ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float().to(DEV)


def rows(n, h, d, dtype, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn((n, h, d), generator=gen, device=DEV).to(dtype)


def positions(n, axes, high, seed, dtype=torch.int64):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    shape = (n,) if axes == 0 else (axes, n)
    return torch.randint(-5, high, shape, generator=gen, device=DEV).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("n,h,hk,d,rot,sections,mixed", [
    (1, 1, 1, 64, 64, None, False), (37, 8, 2, 128, 128, None, False),
    (300, 5, 1, 128, 128, (16, 24, 24), False), (65, 3, 3, 128, 128, (22, 21, 21), True),
    (50, 4, 2, 256, 64, None, False), (33, 2, 2, 96, 48, (10, 0, 7, 7), False),
    (29, 3, 1, 80, 20, (4, 3, 3), True), (7, 2, 1, 70, 70, (35,), False), (19, 1, 1, 2, 2, None, False),
    (11, 2, 2, 136, 16, (5, 3), True), (12, 7, 7, 576, 64, None, False)])
def test_turns(n, h, hk, d, rot, sections, mixed, adjacent, dtype):
    """Whole and partial heads, sizes that are no multiples of 8, every kind of axes."""
    need_gpu()
    say(f"rotary n={n} h={h} hk={hk} d={d} rot={rot} {sections} mixed={mixed} adjacent={adjacent} {dtype}")
    f = frequencies(rot // 2)
    q, k = rows(n, h, d, dtype, 1), rows(n, hk, d, dtype, 2)
    for high, pt in ((50, torch.int32), (200000, torch.int64)):
        pos = positions(n, 0 if sections is None else len(sections), high, 3, pt)
        angle = lo.angles(pos, f, sections, mixed)
        y, z = flag_attn.rotary_embedding(q, k, pos, f, sections, mixed, adjacent)
        torch.cuda.synchronize()
        for out, x in ((y, q), (z, k)):
            assert out.shape == x.shape and out.dtype == dtype
            assert_turned(out, *lo.turn(x, angle, adjacent))
            assert torch.equal(out[..., rot:], x[..., rot:])
        a, b = q.clone(), k.clone()
        c, e = flag_attn.rotary_embedding(a, b, pos, f, sections, mixed, adjacent, inplace=True)
        assert c is a and e is b and torch.equal(a, y) and torch.equal(b, z)


def test_sine_of_a_turn():
    """Sine and cosine over a whole turn in steps of 2^-16 of it and next to its quarters, from
    positions of a frequency that makes them."""
    need_gpu()
    say("rotary sine")
    n = 1 << 16
    pos = torch.arange(-n, n, dtype=torch.int32, device=DEV)
    f = torch.tensor([2 * math.pi / n], device=DEV)
    # x = (1, 0) gives (cos, sin), read back from the sum of two fp16 numbers: 1, then 2^-11 more
    one = torch.zeros((2 * n, 1, 2), dtype=torch.float16, device=DEV)
    one[..., 0] = 1
    y, _ = flag_attn.rotary_embedding(one, one, pos, f)
    angle = pos.double() * f.double()
    ref = torch.stack((torch.cos(angle), torch.sin(angle)), -1)[:, None]
    # rounded to fp16 once: by 2^-11 of the value, or by 2^-25; the function itself within 2^-20
    err = (y.double() - ref).abs() - 2.0 ** -11 * ref.abs() - 2.0 ** -25
    assert float(err.max()) <= 2.0 ** -20 + 2.0 ** -19, f"off by {float(err.max()):.3e}"


@pytest.mark.parametrize("dtype", DTYPES)
def test_far_positions(dtype):
    """Positions up to 2^31 - 1 and past it keep their angles."""
    need_gpu()
    say(f"rotary far {dtype}")
    f = frequencies(32, 1e6)
    top = (1 << 31) - 1
    pos = torch.tensor([0, top, top - 1, -top, 1 << 24, (1 << 24) + 1], device=DEV)
    q, k = rows(6, 2, 64, dtype, 1), rows(6, 1, 64, dtype, 2)
    for p in (pos, pos.int()):
        y, z = flag_attn.rotary_embedding(q, k, p, f)
        assert_turned(y, *lo.turn(q, lo.angles(p, f)))
        assert_turned(z, *lo.turn(k, lo.angles(p, f)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    """Views of one packed projection, heads outermost, rows off the alignment, a slice of a longer
    head in place, last dim with a stride, one row seen by every token."""
    need_gpu()
    say(f"rotary strides {dtype}")
    n, d = 45, 64
    f = frequencies(d // 2)
    pos = positions(n, 0, 3000, 1)
    angle = lo.angles(pos, f)
    qkv = rows(n, 10, d, dtype, 1)
    heads = rows(6, n, d, dtype, 2).transpose(0, 1)
    off = rows(n, 6, d + 3, dtype, 3)[..., 3:]
    wide = rows(n, 6, 2 * d, dtype, 4)[..., ::2]
    once = rows(1, 6, d, dtype, 5).expand(n, 6, d)
    for x in (qkv, heads, off, wide, once):
        q, k = x[:, :4], x[:, 4:6]
        y, z = flag_attn.rotary_embedding(q, k, pos, f)
        assert_turned(y, *lo.turn(q, angle))
        assert_turned(z, *lo.turn(k, angle))
    for whole in (rows(n, 5, 576, dtype, 6), rows(n, 5, 575, dtype, 7)):
        before = whole.clone()
        part = whole[..., 512:512 + 60]
        g = frequencies(30)
        flag_attn.rotary_embedding(part[:, :3], part[:, 3:], pos, g, inplace=True)
        ref, size = lo.turn(before[..., 512:572], lo.angles(pos, g))
        assert_turned(part, ref, size)
        assert torch.equal(whole[..., :512], before[..., :512])
        assert torch.equal(whole[..., 572:], before[..., 572:])


def test_specials_stay_in_their_pair():
    need_gpu()
    say("rotary specials")
    f = frequencies(32)
    q = rows(9, 2, 64, torch.bfloat16, 1)
    k = rows(9, 2, 64, torch.bfloat16, 2)
    pos = positions(9, 0, 100, 1)
    y, _ = flag_attn.rotary_embedding(q, k, pos, f)
    q[4, 1, 7], q[2, 0, 40] = math.nan, math.inf
    y2, _ = flag_attn.rotary_embedding(q, k, pos, f)
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[4, 1, 7] = hit[4, 1, 39] = hit[2, 0, 40] = hit[2, 0, 8] = True
    assert torch.equal(y2[~hit], y[~hit])
    assert not bool(torch.isfinite(y2[hit]).any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("slot_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("n,h,hk,d,rot,block,sections", [
    (1, 8, 2, 64, 64, 16, None), (33, 4, 4, 128, 128, 64, (16, 24, 24)), (200, 6, 2, 256, 128, 16, None),
    (50, 3, 1, 80, 30, 7, None), (5, 2, 2, 128, 128, 1, None)])
def test_cache(n, h, hk, d, rot, block, sections, slot_type, dtype):
    """Rows go to their slots, slots of padding and past the cache are skipped, every other row stays."""
    need_gpu()
    say(f"rotary cache n={n} h={h} hk={hk} d={d} rot={rot} block={block} {dtype} {slot_type}")
    blocks = -(-n // block) + 3
    gen = torch.Generator(device=DEV).manual_seed(9)
    kc = rows(blocks * hk, block, d, dtype, 4).view(blocks, hk, block, d)
    vc = rows(blocks * block, hk, d, dtype, 5).view(blocks, block, hk, d).transpose(1, 2)
    slots = torch.randperm(blocks * block, generator=gen, device=DEV)[:n].to(slot_type)
    if n > 4:
        slots[1], slots[3] = -1, blocks * block
    q, k, v = rows(n, h, d, dtype, 1), rows(n, hk, d, dtype, 2), rows(n, hk, d, dtype, 3)
    f = frequencies(rot // 2)
    pos = positions(n, 0 if sections is None else len(sections), 9000, 3)
    kr, vr = kc.clone(), vc.clone()
    y = flag_attn.rotary_cache_kv(q, k, v, pos, f, kc, vc, slots, sections)
    torch.cuda.synchronize()
    y2, z2 = flag_attn.rotary_embedding(q, k, pos, f, sections)
    assert torch.equal(y, y2)
    assert_turned(y, *lo.turn(q, lo.angles(pos, f, sections)))
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < blocks * block:
            kr[slot // block, :, slot % block] = z2[t]
            vr[slot // block, :, slot % block] = v[t]
    assert torch.equal(kc, kr) and torch.equal(vc, vr)


def test_nothing():
    need_gpu()
    q = rows(0, 2, 64, torch.float16, 1)
    f = frequencies(32)
    y, z = flag_attn.rotary_embedding(q, q, positions(0, 0, 5, 1), f)
    assert y.shape == z.shape == (0, 2, 64)
    kc = torch.zeros((1, 2, 16, 64), dtype=torch.float16, device=DEV)
    assert flag_attn.rotary_cache_kv(q, q, q, positions(0, 0, 5, 1), f, kc, kc.clone(),
                                     torch.zeros(0, dtype=torch.int32, device=DEV)).shape == (0, 2, 64)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_step_of_a_model_with_both_kinds_of_layers(dtype):
    """A prompt, then tokens: rotary q and k, k and v into the paged cache, attention over the packed
    prompt and then over the cache; the same q and k through linear attention and its states."""
    need_gpu()
    say(f"rotary and both kinds of attention {dtype}")
    h, hk, d, block, lens = 4, 2, 128, 16, [37, 5]
    n, f = sum(lens), frequencies(d // 2)
    new = 3
    q, k, v = (rows(n + 2 * new, x, d, dtype, 10 + i) for i, x in enumerate((h, hk, hk)))
    kc = torch.zeros((10, hk, block, d), dtype=dtype, device=DEV)
    vc = torch.zeros_like(kc)
    table = torch.tensor([[7, 2, 5], [1, 9, 0]], dtype=torch.int32, device=DEV)
    a = torch.tensor([-0.2, -0.01], device=DEV)
    state = torch.full((2, hk, d, d), math.nan, device=DEV)
    cu = torch.tensor([0, 37, 42], dtype=torch.int32, device=DEV)

    def slots(seq, at):
        return table[seq, at // block].long() * block + at % block

    at = torch.cat([torch.arange(m, device=DEV) for m in lens])
    where = torch.cat([slots(s, torch.arange(m, device=DEV)) for s, m in enumerate(lens)])
    qr = flag_attn.rotary_cache_kv(q[:n], k[:n], v[:n], at, f, kc, vc, where)
    _, kr = flag_attn.rotary_embedding(q[:n], k[:n], at, f)
    o = flag_attn.flash_attention_varlen(qr, kr, v[:n], cu, cu, 37, 37, causal=True)
    lin = flag_attn.linear_attention_varlen(qr, kr, v[:n], a, cu, 37, state, None,
                                            torch.zeros(2, dtype=torch.bool, device=DEV))
    outs, lins = [o[:37], o[37:]], [lin[:37], lin[37:]]
    krs, vs = [kr[:37], kr[37:]], [v[:37], v[37:n]]
    qs = [qr[:37], qr[37:]]
    for step in range(new):
        row = slice(n + 2 * step, n + 2 * step + 2)
        ctx = torch.tensor([m + step for m in lens], device=DEV)
        where = torch.stack([slots(s, ctx[s]) for s in range(2)])
        q1 = flag_attn.rotary_cache_kv(q[row], k[row], v[row], ctx, f, kc, vc, where)
        _, k1 = flag_attn.rotary_embedding(q[row], k[row], ctx, f)
        o1 = flag_attn.paged_attention(q1, kc, vc, (ctx + 1).int(), table, d ** -0.5, 48)
        l1 = flag_attn.linear_attention_decode(q1, k1, v[row], a, state)
        for s in range(2):
            outs[s] = torch.cat((outs[s], o1[s:s + 1]))
            lins[s] = torch.cat((lins[s], l1[s:s + 1]))
            krs[s] = torch.cat((krs[s], k1[s:s + 1]))
            vs[s] = torch.cat((vs[s], v[row][s:s + 1]))
            qs[s] = torch.cat((qs[s], q1[s:s + 1]))
    torch.cuda.synchronize()
    from oracle import packed_oracle as po
    from tests._linear import assert_out, small_out
    from tests._packed import assert_rows
    for s in range(2):
        m = outs[s].shape[0]
        for j in range(hk):
            heads = slice(j * 2, j * 2 + 2)
            ref, size, _, _ = lo.attend(qs[s][:, heads], krs[s][:, j], vs[s][:, j], float(a[j]), d ** -0.5)
            assert_out(lins[s][:, heads], ref, size, 4 * m,
                       small_out(qs[s][:, heads], krs[s][:, j], vs[s][:, j], None, d ** -0.5))
            for g in range(2):
                ref, _, mag, ds = po.attend(qs[s][:, 2 * j + g], krs[s][:, j], vs[s][:, j], d ** -0.5, True)
                assert_rows(outs[s][:, 2 * j + g], ref, mag, ds, m, float(vs[s].abs().max()))
