"""The paged K/V cache in 4 bits (cache_kv_mxfp4, gather_kv_mxfp4, paged_attention_mxfp4): bytes
and read-back values exactly, attention against the formula in 64 bits over the cached values with
tolerances made of the roundings (tests/_packed.py)."""
import math

import pytest
import torch

import flag_attn
from oracle import packed_oracle as po
from tests._helpers import DEV, need_gpu, say
from tests._packed import assert_largest_exact, assert_rows

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]
DIMS = [64, 128, 256]


def new_cache(blocks, hk, block, d, seed=0):
    """A cache in use: random codes, scales between 2^-4 and 2^3."""
    gen = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        out.append(torch.randint(0, 256, (blocks, hk, block, d // 2), generator=gen).to(torch.uint8))
        out.append(torch.randint(123, 131, (blocks, hk, block, d // 32), generator=gen).to(torch.uint8))
    return [x.to(DEV) for x in out]


def all_patterns(dtype, d):
    """Rows that hold every finite value of the type among groups of 32 of like and unlike size."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype).float()
    bits = bits[torch.isfinite(bits)]
    gen = torch.Generator().manual_seed(7)
    order = torch.argsort(bits.abs(), stable=True)
    rows = [bits[order], bits[torch.randperm(bits.numel(), generator=gen)]]
    x = torch.cat([r[: r.numel() // (4 * d) * 4 * d].view(-1, 4, d) for r in rows])
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", DIMS)
def test_write_every_value(d, dtype):
    """Codes and scales of every finite value, in groups of neighbours and in mixed groups; ties,
    subnormals and signed zeros among them; every other slot is left as it was."""
    need_gpu()
    say(f"mxfp4 write d={d} {dtype}")
    x = all_patterns(dtype, d)
    t, hk = x.shape[:2]
    block = 64
    cache = new_cache(-(-2 * t // block), hk, block, d)
    slots = torch.randperm(2 * t, generator=torch.Generator().manual_seed(1))[:t]
    slots[3], slots[9] = -1, cache[0].shape[0] * block + 2
    want = [y.cpu() for y in cache]
    want = [*po.write(want[0], want[1], x, slots), *po.write(want[2], want[3], x.flip(0), slots)]
    flag_attn.cache_kv_mxfp4(x.to(DEV), x.flip(0).to(DEV), *cache, slots.to(DEV))
    for got, w in zip(cache, want):
        assert torch.equal(got.cpu(), w)


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_odd_values_and_layouts(dtype):
    """A NaN or an infinity makes its group NaN, and no other; int32 slots, sliced inputs (aligned
    and not), a cache whose tensors are slices of larger ones, no token at all."""
    need_gpu()
    say(f"mxfp4 write odd {dtype}")
    d, hk, block = 128, 2, 16
    gen = torch.Generator().manual_seed(3)
    x = torch.randn((40, hk, d), generator=gen).to(dtype)
    x[0, 0, 5], x[1, 1, 40], x[2, 0, 127] = math.nan, math.inf, -math.inf
    x[3, 0, :32] = 0.0
    x[3, 0, 32:64] = -0.0
    slots = torch.arange(40, dtype=torch.int32) + 7
    big = [y.repeat_interleave(2, 1) for y in new_cache(5, hk, block, d, seed=5)]
    cache = [y[:, 1::2] for y in big]
    before = [y.clone() for y in big]
    want = [y.cpu().contiguous() for y in cache]
    want = [*po.write(want[0], want[1], x, slots), *po.write(want[2], want[3], x, slots)]
    fused = torch.cat([x, x], 1).to(DEV)
    flag_attn.cache_kv_mxfp4(fused[:, :hk], fused[:, hk:], *cache, slots.to(DEV))
    for got, w, b, old in zip(cache, want, big, before):
        assert torch.equal(got.cpu(), w)
        assert torch.equal(b[:, 0::2], old[:, 0::2])
    k = po.values(cache[0], cache[1])[0, 0, 7]
    assert bool(torch.isnan(k[:32]).all()) and bool(torch.isfinite(k[32:]).all())
    odd = torch.zeros((40, hk, d + 1), dtype=dtype, device=DEV)
    odd[..., 1:] = x.to(DEV)
    again = [y[:, 1::2].contiguous() for y in before]
    flag_attn.cache_kv_mxfp4(odd[..., 1:], odd[..., 1:], *again, slots.long().to(DEV)[::1])
    assert all(torch.equal(y.cpu(), w) for y, w in zip(again, want))
    flag_attn.cache_kv_mxfp4(odd[:0, :, 1:], odd[:0, :, 1:], *again, slots[:0].to(DEV))
    assert all(torch.equal(y.cpu(), w) for y, w in zip(again, want))


@pytest.mark.parametrize("t,hk", [(20, 2), (1, 2), (1, 1)])
@pytest.mark.parametrize("d", DIMS)
def test_write_contiguous_rows_off_the_alignment(d, t, hk):
    """A misaligned base, and strides of dimensions of one that no row needs."""
    need_gpu()
    say(f"mxfp4 write off the alignment d={d} t={t} hk={hk}")
    x = queries(t, hk, d, torch.bfloat16, seed=d)
    slots = torch.arange(5, 5 + t, device=DEV)

    def written(k, v):
        cache = new_cache(2, hk, 16, d)
        flag_attn.cache_kv_mxfp4(k, v, *cache, slots)
        return cache

    want = new_cache(2, hk, 16, d)
    want = [*po.write(want[0], want[1], x, slots), *po.write(want[2], want[3], x, slots)]
    off = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape).copy_(x)
    assert off.is_contiguous() and off.data_ptr() % 16 == 2
    views = [off]
    if t == 1:
        views.append(x.as_strided(x.shape, (x.numel() + 3, d, 1)))
    if t == hk == 1:
        views.append(x.as_strided(x.shape, (d, d + 3, 1)))
    for y in views:
        for k, v in ((y, x), (x, y), (y, y)):
            assert all(torch.equal(a, b) for a, b in zip(written(k, v), want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("block", [16, 32, 128])
def test_gather(block, d, dtype):
    """Contexts of odd lengths (an empty one too) as packed rows, pages in any order, blocks
    outside the cache and a table that ends too early as zeros, rows behind the last as zeros."""
    need_gpu()
    say(f"mxfp4 gather block={block} d={d} {dtype}")
    lens, hk, blocks = [1, 130, 0, 17, 300], 3, 40
    cache = new_cache(blocks, hk, block, d, seed=block)
    gen = torch.Generator().manual_seed(2)
    bt = torch.randint(0, blocks, (5, -(-300 // block)), generator=gen, dtype=torch.int32)
    bt[1, 0], bt[4, 1] = -1, blocks
    cu = [0, 1, 131, 131, 148, 448]
    total = 470
    cud = torch.tensor(cu, dtype=torch.int32, device=DEV)
    for table in (bt, bt[:, :2]):
        k, v = flag_attn.gather_kv_mxfp4(*cache, table.to(DEV), cud, total, dtype)
        assert k.shape == (total, hk, d) and k.dtype == dtype and v.shape == k.shape
        for got, c, s in ((k, *cache[:2]), (v, *cache[2:])):
            want = torch.zeros((total, hk, d), dtype=torch.float64)
            for i, n in enumerate(lens):
                want[cu[i]:cu[i + 1]] = po.context(c.cpu(), s.cpu(), table[i], n)[0]
            assert torch.equal(got.cpu(), want.to(dtype))


@pytest.mark.parametrize("byte", [0, 100, 103, 126, 140, 141, 142, 254, 255])
def test_gather_rounds_to_the_type(byte):
    """Scales at the ends: below fp16's range the values round to it, past it they are infinities."""
    need_gpu()
    say(f"mxfp4 gather scale {byte}")
    cache = new_cache(1, 1, 16, 64, seed=byte)
    cache[1].fill_(byte), cache[3].fill_(byte)
    bt = torch.zeros((1, 1), dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 16], dtype=torch.int32, device=DEV)
    for dtype in DTYPES:
        k, v = flag_attn.gather_kv_mxfp4(*cache, bt, cu, 16, dtype)
        for got, codes, scales in ((k, cache[0], cache[1]), (v, cache[2], cache[3])):
            want = po.values(codes, scales)[0].transpose(0, 1).to(dtype)
            assert torch.equal(got.isnan(), want.isnan())
            assert torch.equal(got.nan_to_num(1.0, math.inf, -math.inf),
                               want.nan_to_num(1.0, math.inf, -math.inf))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", DIMS)
def test_gather_every_code_and_scale(d, dtype):
    """Every byte of two codes under every scale byte, a block for each of those."""
    need_gpu()
    say(f"mxfp4 gather every code d={d} {dtype}")
    codes = torch.arange(256, device=DEV).to(torch.uint8).repeat(256 * d // 32)
    cache = [codes.view(256, 1, 16, d // 2), None, codes.flip(0).view(256, 1, 16, d // 2), None]
    cache[1] = torch.arange(256, device=DEV).to(torch.uint8).view(256, 1, 1, 1).repeat(1, 1, 16, d // 32)
    cache[3] = cache[1].clone()
    bt = torch.arange(256, dtype=torch.int32, device=DEV)[None]
    cu = torch.tensor([0, 4096], dtype=torch.int32, device=DEV)
    for got, c, s in zip(flag_attn.gather_kv_mxfp4(*cache, bt, cu, 4096, dtype), cache[::2], cache[1::2]):
        want = po.values(c, s).transpose(1, 2).flatten(0, 1).to(dtype)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.isinf(), want.isinf())
        assert torch.equal(got.nan_to_num(1.0), want.nan_to_num(1.0))


def test_gather_of_no_rows_and_late_starts():
    need_gpu()
    say("mxfp4 gather edges")
    cache = new_cache(3, 1, 16, 64)
    bt = torch.zeros((1, 2), dtype=torch.int32, device=DEV)
    k, v = flag_attn.gather_kv_mxfp4(*cache, bt, torch.tensor([0, 0], dtype=torch.int32, device=DEV),
                                     0, torch.float16)
    assert k.shape == (0, 1, 64)
    k, v = flag_attn.gather_kv_mxfp4(*cache, bt, torch.tensor([4, 9], dtype=torch.int32, device=DEV),
                                     9, torch.bfloat16)
    assert bool((k[:4] == 0).all()) and torch.equal(
        k[4:].double(), po.values(cache[0], cache[1])[0].transpose(0, 1)[:5])
    k, v = flag_attn.gather_kv_mxfp4(*cache, bt[:0], torch.zeros(1, dtype=torch.int32, device=DEV),
                                     3, torch.float16)
    assert bool((k == 0).all()) and bool((v == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_gather_without_blocks_is_zeros(dtype):
    """A table without a column, as paged_attention_mxfp4 takes it: every token lies behind its end."""
    need_gpu()
    say(f"mxfp4 gather without blocks {dtype}")
    cache = new_cache(3, 2, 16, 128)
    bt = torch.zeros((2, 0), dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 4, 9], dtype=torch.int32, device=DEV)
    for x in flag_attn.gather_kv_mxfp4(*cache, bt, cu, 12, dtype):
        assert x.shape == (12, 2, 128) and x.dtype == dtype and bool((x == 0).all())


def run_decode(q, cache, lens, bt, scale=None, max_len=None, splits=0):
    d = q.shape[-1]
    ld = torch.tensor(lens, dtype=torch.int32, device=DEV)
    return flag_attn.paged_attention_mxfp4(q, *cache, ld, bt.to(DEV),
                                           d ** -0.5 if scale is None else scale,
                                           max(1, max(lens)) if max_len is None else max_len, splits)


def check_decode(q, cache, lens, bt, scale=None, max_len=None, splits=0):
    out = run_decode(q, cache, lens, bt, scale, max_len, splits)
    torch.cuda.synchronize()
    b, h, d = q.shape
    hk = cache[0].shape[1]
    scale = d ** -0.5 if scale is None else scale
    ref = torch.zeros((b, h, d), dtype=torch.float64, device=DEV)
    a, ds = torch.zeros_like(ref), torch.zeros((b, h), dtype=torch.float64, device=DEV)
    for i, n in enumerate(lens):
        k, seen = po.context(cache[0], cache[1], bt[i], n)
        v, _ = po.context(cache[2], cache[3], bt[i], n)
        for j in range(hk):
            r = slice(j * h // hk, (j + 1) * h // hk)
            ref[i, r], _, a[i, r], ds[i, r] = po.attend(q[i, r], k[seen, j], v[seen, j], scale, False)
    vmax = 6.0 * 2.0 ** (int(cache[3][cache[3] < 255].max()) - 127)
    assert out.shape == q.shape and out.dtype == q.dtype
    # fp16 values are halved on the way: those below 2^-13 lose a bit, at most 2^-25 each way
    assert_rows(out, ref, a, ds, max(lens), vmax)
    return out


def queries(b, h, d, dtype, seed=0, gain=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn((b, h, d), generator=gen, device=DEV) * gain).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("h,hk,block", [(4, 4, 16), (16, 2, 64), (7, 1, 128), (40, 2, 32)])
def test_decode(h, hk, block, d, dtype):
    """Contexts around tiles and pages, an empty one, groups of 1 .. 20 heads."""
    need_gpu()
    say(f"mxfp4 decode h={h} hk={hk} block={block} d={d} {dtype}")
    lens = [1, 15, 16, 33, 0, 129, 250]
    cache = new_cache(60, hk, block, d, seed=h)
    gen = torch.Generator().manual_seed(1)
    bt = torch.randint(0, 60, (len(lens), -(-250 // block)), generator=gen, dtype=torch.int32)
    out = check_decode(queries(len(lens), h, d, dtype, seed=d), cache, lens, bt)
    assert bool((out[4] == 0).all())


@pytest.mark.parametrize("splits", [0, 1, 3, 200])
@pytest.mark.parametrize("d", DIMS)
def test_decode_splits(d, splits):
    """Ragged contexts split along their keys; splits that lie behind a short context are empty."""
    need_gpu()
    say(f"mxfp4 decode splits={splits} d={d}")
    lens = [3000, 1, 0, 777]
    cache = new_cache(100, 2, 32, d, seed=4)
    gen = torch.Generator().manual_seed(2)
    bt = torch.randint(0, 100, (4, 94), generator=gen, dtype=torch.int32)
    check_decode(queries(4, 8, d, torch.bfloat16), cache, lens, bt, splits=splits)


@pytest.mark.parametrize("block", [16, 32, 64])
def test_decode_bad_blocks_are_masked(block):
    """Blocks outside the cache, and those behind the table's end, read as masked keys."""
    need_gpu()
    say(f"mxfp4 decode bad blocks {block}")
    lens = [200, 200, 100]
    cache = new_cache(20, 2, block, 128, seed=6)
    gen = torch.Generator().manual_seed(3)
    bt = torch.randint(0, 20, (3, -(-200 // block)), generator=gen, dtype=torch.int32)
    bt[0, 1], bt[0, 0], bt[1, :] = 20, -5, -1
    q = queries(3, 8, 128, torch.float16)
    out = check_decode(q, cache, lens, bt)
    assert bool((out[1] == 0).all())
    check_decode(q, cache, [200, 200, 200], bt[:, :2])
    assert bool((run_decode(q, cache, lens, bt[:, :0]) == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_nan_behind_the_context(dtype):
    """NaN scales in the rows behind a context, in its last page and in pages that only other
    sequences name, reach nobody; one inside it makes the row NaN, whatever the split."""
    need_gpu()
    say(f"mxfp4 decode NaN {dtype}")
    cache = new_cache(8, 1, 32, 64, seed=8)
    bt = torch.arange(8, dtype=torch.int32).view(2, 4)
    for x in (cache[1], cache[3]):
        x[3, :, 4:] = 255  # sequence 0: 100 tokens end at row 4 of block 3
    q = queries(2, 4, 64, dtype)
    for splits in (1, 4):
        check_decode(q, cache, [100, 128], bt, splits=splits)
    cache[1][5, 0, 3, 1] = 255
    for splits in (1, 2, 8):
        out = run_decode(q, cache, [100, 128], bt, splits=splits)
        assert bool(torch.isfinite(out[0]).all()) and bool(torch.isnan(out[1]).all())
    cache[1][4:] = 255  # every key of sequence 1
    for splits in (1, 4):
        assert bool(torch.isnan(run_decode(q, cache, [100, 128], bt, splits=splits)[1]).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_range_of_values(dtype):
    """The largest rows that the type can hold, and very small ones, written and attended to."""
    need_gpu()
    say(f"mxfp4 decode range {dtype}")
    top = 65504.0 if dtype == torch.float16 else 2.0 ** 100
    gen = torch.Generator().manual_seed(5)
    for size in (top, 2.0 ** -12):
        x = torch.rand((64, 2, 64), generator=gen).mul(0.4).add(0.6).to(dtype) * 1.0
        x = (x.float() * size).to(dtype)
        cache = new_cache(4, 2, 16, 64)
        slots = torch.arange(64, device=DEV)
        k = torch.randn((64, 2, 64), generator=gen).to(dtype)
        flag_attn.cache_kv_mxfp4(k.to(DEV), x.to(DEV), *cache, slots)
        check_decode(queries(1, 4, 64, dtype), cache, [64], torch.arange(4, dtype=torch.int32)[None])


def huge_case(d):
    """(cache, contexts, table, queries) for values of up to 1.5 * 2^127."""
    bt = torch.randperm(100, generator=torch.Generator().manual_seed(6)).int()
    return (new_cache(100, 2, 16, d, seed=3), [700, 33, 200],
            torch.stack([bt[:44], bt[44:88], bt[56:100]]), queries(3, 16, d, torch.bfloat16, seed=d))


@pytest.mark.parametrize("splits", [1, 5])
@pytest.mark.parametrize("d", DIMS)
def test_decode_huge_values(d, splits):
    """One key's values of up to 1.5 * 2^127, of any weight: the sums of a row stay within fp32 where
    its result does."""
    need_gpu()
    say(f"mxfp4 decode huge values d={d} splits={splits}")
    cache, lens, bt, q = huge_case(d)
    for i, at in enumerate((300, 31, 64)):
        cache[3][bt[i, at // 16], :, at % 16] = 252
    check_decode(q, cache, lens, bt, splits=splits)


def check_many_huge_values(d, splits):
    cache, lens, bt, q = huge_case(d)
    cache[3].fill_(252)
    check_decode(q, cache, lens, bt, splits=splits)
    cache[2].fill_(0x77)  # 6 * 2^125 everywhere, of equal weights
    check_decode(torch.zeros_like(q), cache, lens, bt, splits=splits)


@pytest.mark.parametrize("d", DIMS)
def test_decode_many_huge_values(d):
    """The same at every key."""
    need_gpu()
    say(f"mxfp4 decode many huge values d={d}")
    check_many_huge_values(d, 1)


@pytest.mark.parametrize("splits", [5, 40])
@pytest.mark.parametrize("d", DIMS)
def test_decode_many_huge_values_in_splits(d, splits):
    """The same where the keys are split: the merge's sums stay within fp32 too."""
    need_gpu()
    say(f"mxfp4 decode many huge values d={d} splits={splits}")
    check_many_huge_values(d, splits)


@pytest.mark.parametrize("gain", [5.0, 4000.0])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", DIMS)
def test_decode_rows_do_not_depend_on_their_neighbours(d, dtype, gain):
    """One head's query grows: every other head keeps its bits."""
    need_gpu()
    say(f"mxfp4 decode neighbours d={d} {dtype} gain={gain}")
    cache = new_cache(60, 2, 32, d, seed=3)
    bt = torch.randperm(60, generator=torch.Generator().manual_seed(6)).int().view(2, 30)
    q = queries(2, 16, d, dtype, seed=d)
    for splits in (1, 3):
        o = run_decode(q, cache, [900, 451], bt, splits=splits)
        for h in (0, 13):
            other = q.clone()
            other[0, h] *= gain
            o2 = run_decode(other, cache, [900, 451], bt, splits=splits)
            o2[0, h] = o[0, h]
            assert torch.equal(o, o2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", DIMS)
def test_decode_largest_weight_is_exact(d, dtype):
    """Two keys that a wave meets one after the other, the second e^0.6 .. e^4 times as heavy, among
    keys of next to no weight: the largest weight of a row is a power of two, whose rounding costs
    nothing, so that the first key's alone does."""
    need_gpu()
    say(f"mxfp4 decode largest weight d={d} {dtype}")
    k = torch.zeros((200, 2, d), dtype=dtype, device=DEV)
    k[..., 0] = -24.0
    k[3, :, 0], k[140, :, 0] = 2.0, 6.0  # tiles 0 and 4 of the first wave
    cache = new_cache(16, 2, 16, d, seed=d)
    v, _ = po.context(cache[2], cache[3], torch.arange(16), 200)
    flag_attn.cache_kv_mxfp4(k, v.to(dtype), *cache, torch.arange(200, device=DEV))
    bt = torch.arange(16, dtype=torch.int32)[None]
    q = torch.zeros((1, 32, d), dtype=dtype, device=DEV)
    q[..., 0] = torch.linspace(0.15, 1.0, 32, device=DEV).to(dtype)
    out = run_decode(q, cache, [200], bt, scale=1.0, splits=1)[0]
    ck, _ = po.context(cache[0], cache[1], bt[0], 200)
    cv, _ = po.context(cache[2], cache[3], bt[0], 200)
    assert torch.equal(ck, k.double())
    for j in range(2):
        r = slice(16 * j, 16 * j + 16)
        ref, rest, ds = po.attend_rest(q[0, r], ck[:, j], cv[:, j], 1.0)
        assert_largest_exact(out[r], ref, rest, ds, 200, 48.0, terms=1)


@pytest.mark.parametrize("scale", [0.0, -0.2, 30.0])
def test_decode_scales_and_layouts(scale):
    """Any finite scale; queries and caches as slices of larger tensors, repeated blocks."""
    need_gpu()
    say(f"mxfp4 decode scale {scale}")
    big = [y.repeat_interleave(2, 1) for y in new_cache(6, 2, 64, 128, seed=9)]
    cache = [y[:, 1::2] for y in big]
    q = queries(3, 24, 128, torch.bfloat16)[:, 8:16]
    bt = torch.tensor([[1, 1, 5], [0, 2, 0], [4, 3, 2]], dtype=torch.int32)
    check_decode(q, cache, [192, 100, 130], bt, scale=scale)


def test_offsets_past_32_bits():
    """Blocks that lie more than 2^32 bytes behind the cache's first row."""
    need_gpu()
    say("mxfp4 far offsets")
    blocks, hk, block, d = 70, 1, 16, 64
    stride = 1 << 26  # bytes from block to block
    wide = [torch.zeros(blocks * stride, dtype=torch.uint8, device=DEV) for _ in range(2)]
    views = []
    for i, w in enumerate(wide):
        views.append(w.as_strided((blocks, hk, block, d // 2), (stride, block * d // 2, d // 2, 1)))
        views.append(w.as_strided((blocks, hk, block, d // 32), (stride, block * d // 32, d // 32, 1),
                                  1 << 20))
    for v, n in zip(views, new_cache(blocks, hk, block, d, seed=10)):
        v.copy_(n)
    bt = torch.arange(blocks - 1, -1, -1, dtype=torch.int32)[None]
    lens = [blocks * block]
    check_decode(queries(1, 2, d, torch.float16), views, lens, bt)
    k, _ = flag_attn.gather_kv_mxfp4(*views, bt.to(DEV), torch.tensor([0, lens[0]], dtype=torch.int32,
                                                                     device=DEV), lens[0], torch.float16)
    assert torch.equal(k.double(), po.context(views[0], views[1], bt[0], lens[0])[0])
    x = torch.randn((2, hk, d), device=DEV).half()
    at = torch.tensor([blocks * block - 1, 0], device=DEV)
    flag_attn.cache_kv_mxfp4(x, x, *views, at)
    c, s = po.quantise(x)
    assert torch.equal(views[0][-1, :, -1], c[0]) and torch.equal(views[1][0, :, 0], s[1])


def test_serving_run():
    """A model's use of all of it: two prompts attended packed and cached, a second chunk over the
    contexts read back, then single tokens against the cache, under a captured graph."""
    need_gpu()
    say("mxfp4 serving run")
    h, hk, d, block = 8, 2, 128, 16
    dtype = torch.bfloat16
    cache = new_cache(64, hk, block, d)
    gen = torch.Generator(device=DEV).manual_seed(1)
    bt = torch.randperm(64, generator=torch.Generator().manual_seed(0)).int().view(2, 32)
    btd = bt.to(DEV)
    lens = [0, 0]

    def rows(n, heads):
        return torch.randn((n, heads, d), generator=gen, device=DEV).to(dtype)

    for chunk in ([70, 33], [50, 200]):
        new = [x + y for x, y in zip(lens, chunk)]
        k, v = rows(sum(chunk), hk), rows(sum(chunk), hk)
        slots = torch.cat([btd[i][torch.arange(a, b, device=DEV) // block].long() * block +
                           torch.arange(a, b, device=DEV) % block
                           for i, (a, b) in enumerate(zip(lens, new))])
        flag_attn.cache_kv_mxfp4(k, v, *cache, slots)
        cu_q = torch.tensor([0, chunk[0], sum(chunk)], dtype=torch.int32, device=DEV)
        cu_k = torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device=DEV)
        kk, vv = flag_attn.gather_kv_mxfp4(*cache, btd, cu_k, sum(new), dtype)
        q = rows(sum(chunk), h)
        o, lse = flag_attn.flash_attention_varlen(q, kk, vv, cu_q, cu_k, max(chunk), max(new), True,
                                                  return_log_normalizer=True)
        ck = [po.context(cache[0], cache[1], bt[i], n)[0] for i, n in enumerate(new)]
        cv = [po.context(cache[2], cache[3], bt[i], n)[0] for i, n in enumerate(new)]
        ref, _, a, ds = po.varlen(q, torch.cat(ck), torch.cat(cv), cu_q.tolist(), cu_k.tolist(),
                                  d ** -0.5, True)
        assert_rows(o, ref, a, ds.t(), max(new), 6.0)
        lens = new

    ld = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q, k, v = rows(2, h), rows(2, hk), rows(2, hk)
    slots = torch.zeros(2, dtype=torch.int64, device=DEV)

    def step():
        flag_attn.cache_kv_mxfp4(k, v, *cache, slots)
        return flag_attn.paged_attention_mxfp4(q, *cache, ld, btd, d ** -0.5, 512)

    slots.copy_(btd[[0, 1], [n // block for n in lens]].long() * block +
                torch.tensor([n % block for n in lens], device=DEV))
    ld += 1
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        lens = [n + 1 for n in lens]
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen, device=DEV))
        slots.copy_(btd[[0, 1], [n // block for n in lens]].long() * block +
                    torch.tensor([n % block for n in lens], device=DEV))
        ld += 1
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        torch.randn(4096, device=DEV).sum().item()
        assert torch.equal(got, check_decode(q, cache, [n + 1 for n in lens], bt, max_len=512))


def test_replays_and_other_streams():
    """Two captured graphs with their own splits' workspaces and a write and read back, replayed in
    turn on changed inputs, against the same calls on another stream."""
    need_gpu()
    say("mxfp4 graphs")
    d, hk, block = 128, 2, 32
    cache = new_cache(200, hk, block, d, seed=9)
    gen = torch.Generator(device=DEV).manual_seed(4)
    bt = torch.randperm(200, generator=torch.Generator().manual_seed(3)).int().view(2, 100).to(DEV)
    lens = torch.tensor([3000, 1701], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 40, 140], dtype=torch.int32, device=DEV)
    q = [queries(2, 8, d, torch.float16, seed=6), queries(2, 16, d, torch.float16, seed=7)]
    kv = queries(60, hk, d, torch.float16, seed=8)
    slots = torch.arange(64, 124, device=DEV)

    def calls(x):
        flag_attn.cache_kv_mxfp4(kv, kv, *cache, slots)
        return (flag_attn.paged_attention_mxfp4(x, *cache, lens, bt, 0.1, 3200),
                *flag_attn.gather_kv_mxfp4(*cache, bt, cu, 150, torch.float16))

    for x in q:
        calls(x)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in q:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(calls(x))
        graphs.append(g)
    stream = torch.cuda.Stream()
    for rep in range(3):
        for t in (*q, kv):
            t.copy_(torch.randn(t.shape, generator=gen, device=DEV))
        slots.copy_(torch.randperm(6400, device=DEV)[:60])
        lens.copy_(torch.tensor([3200 - 7 * rep, 1 + 33 * rep], dtype=torch.int32))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in outs]
        torch.randn(4096, device=DEV).sum().item()
        with torch.cuda.stream(stream):
            want = [calls(x) for x in q]
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(g, w)), rep
        check_decode(q[0], cache, lens.tolist(), bt.cpu(), scale=0.1, max_len=3200)
