"""Prompt attention over packed sequences (flag_attn.flash_attention_varlen) against the formula
in 64 bits, with tolerances made of the roundings it makes (tests/_packed.py)."""
import math
import random

import pytest
import torch

import flag_attn
from flagattention_amd import varlen
from oracle import packed_oracle as po
from tests._helpers import DEV, need_gpu, say
from tests._packed import assert_largest_exact, assert_lse, assert_rows, varlen_splits

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def inputs(lens_q, lens_k, h, hk, d, dtype, seed=0, extra_q=0, extra_k=0, spread=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def rows(n, heads, gain):
        return (torch.randn((n, heads, d), generator=gen, device=DEV) * gain).to(dtype)

    return (rows(sum(lens_q) + extra_q, h, spread), rows(sum(lens_k) + extra_k, hk, spread),
            rows(sum(lens_k) + extra_k, hk, 1.0), starts(lens_q), starts(lens_k))


def call(q, k, v, cu_q, cu_k, causal, scale=None, max_k=None):
    cq, ck = (torch.tensor(c, dtype=torch.int32, device=DEV) for c in (cu_q, cu_k))
    max_q = max((b - a for a, b in zip(cu_q, cu_q[1:])), default=0)
    if max_k is None:
        max_k = max((b - a for a, b in zip(cu_k, cu_k[1:])), default=0)
    return flag_attn.flash_attention_varlen(q, k, v, cq, ck, max_q, max_k, causal, scale,
                                            return_log_normalizer=True)


def check(q, k, v, cu_q, cu_k, causal, scale=None, max_k=None):
    o, lse = call(q, k, v, cu_q, cu_k, causal, scale, max_k)
    torch.cuda.synchronize()
    d = q.shape[-1]
    ref, ref_lse, a, ds = po.varlen(q, k, v, cu_q, cu_k, d ** -0.5 if scale is None else scale,
                                    causal)
    n = max((b - a for a, b in zip(cu_k, cu_k[1:])), default=0)
    vmax = float(v.float().abs().nan_to_num(0.0, 0.0, 0.0).max()) if v.numel() else 0.0
    assert o.dtype == q.dtype and o.shape == q.shape and lse.shape == (q.shape[1], q.shape[0])
    assert_rows(o, ref, a, ds.t(), n, vmax)
    assert_lse(lse, ref_lse, ds, n, d)
    return o, lse


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,hk,d", [(4, 4, 64), (8, 2, 128), (7, 1, 128), (4, 2, 256), (40, 8, 64)])
def test_whole_prompts(h, hk, d, dtype, causal):
    """Lengths around the tiles (one, odd, whole, one more), an empty sequence in the middle."""
    need_gpu()
    lens = [1, 31, 64, 65, 0, 127, 200, 2, 32]
    say(f"varlen prompts h={h} hk={hk} d={d} {dtype} causal={causal}")
    check(*inputs(lens, lens, h, hk, d, dtype, seed=d + h), causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16),
                                     (128, torch.bfloat16), (256, torch.bfloat16)])
def test_chunks_and_single_tokens(d, dtype, causal):
    """Chunks behind prefixes, single tokens, and more tokens than keys: the first of those see
    none (out 0, -inf)."""
    need_gpu()
    say(f"varlen chunks d={d} {dtype} causal={causal}")
    check(*inputs([40, 1, 1, 100, 17, 5], [300, 513, 1, 60, 17, 0], 8, 2, d, dtype, seed=3), causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", varlen.HEAD_DIMS)
@pytest.mark.parametrize("lens_q,lens_k", [([1], [5000]), ([3, 1], [2111, 40]), ([64], [3001])])
def test_split_keys(lens_q, lens_k, d, causal):
    """Few rows over many keys: the keys are split and the parts merged."""
    need_gpu()
    say(f"varlen splits {lens_q} {lens_k} d={d} causal={causal}")
    cu = torch.cuda.get_device_properties(0).multi_processor_count
    assert varlen_splits(sum(lens_q), sum(lens_k), len(lens_q), 4, 2, d, causal, max(lens_q),
                         max(lens_k), cu)[0] > 1
    check(*inputs(lens_q, lens_k, 4, 2, d, torch.bfloat16, seed=9), causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", varlen.HEAD_DIMS)
def test_split_keys_of_many_rows(d, causal):
    """More rows than the merge requests ahead, many without a key in the later splits."""
    need_gpu()
    say(f"varlen splits of many rows d={d} causal={causal}")
    cu = torch.cuda.get_device_properties(0).multi_processor_count
    assert varlen_splits(1110, 2500, 2, 8, 1, d, causal, 1100, 2490, cu)[0] > 1
    q, k, v, cq, ck = inputs([10, 1100], [10, 2490], 8, 1, d, torch.float16, seed=13)
    check(q, k, v, cq, ck, causal)


@pytest.mark.parametrize("max_k", [1, 700, 5000])
def test_length_bounds_do_not_choose_the_result(max_k):
    need_gpu()
    say(f"varlen max_k={max_k}")
    check(*inputs([2, 5], [2500, 900], 4, 1, 128, torch.float16, seed=1), True, max_k=max_k)


def test_rows_of_no_sequence_are_zero():
    """Rows behind the last sequence and before the first; NaN there and in the keys behind the
    last sequence reaches nobody."""
    need_gpu()
    say("varlen rows of no sequence")
    for d in varlen.HEAD_DIMS:
        q, k, v, cq, ck = inputs([70, 130], [70, 130], 4, 2, d, torch.bfloat16, seed=2, extra_q=300,
                                 extra_k=90)
        q[200:] = math.nan
        k[200:] = math.nan
        v[200:] = math.nan
        o, lse = call(q, k, v, cq, ck, True)
        assert bool((o[200:] == 0).all()) and bool(torch.isneginf(lse[:, 200:]).all())
        ref, ref_lse, a, ds = po.varlen(q[:200], k, v, cq, ck, d ** -0.5, True)
        assert_rows(o[:200], ref, a, ds.t(), 130, 6.0)
        assert_lse(lse[:, :200], ref_lse, ds, 130, d)
        late = [50, 120, 200]
        o, lse = call(q, k, v, late, ck, False)
        assert bool((o[:50] == 0).all()) and bool(torch.isneginf(lse[:, :50]).all())
        o, lse = call(q, k, v, [0], [0], False)
        assert bool((o == 0).all()) and bool(torch.isneginf(lse).all())


@pytest.mark.parametrize("d", varlen.HEAD_DIMS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_odd_values_reach_only_the_rows_that_see_them(d, dtype):
    """NaN and infinities in K and V at keys that a causal mask hides from earlier tokens."""
    need_gpu()
    say(f"varlen odd values d={d} {dtype}")
    q, k, v, cq, ck = inputs([150, 60, 100], [150, 90, 100], 4, 2, d, dtype, seed=5)
    v[149, 0, 3] = math.nan
    v[100, 1, 7] = math.inf
    v[150 + 70, 1, 0] = -math.inf
    v[150 + 89, 0, d - 1] = math.inf
    k[240 + 64, 0, 5] = math.nan
    o, lse = call(q, k, v, cq, ck, True)
    ref, ref_lse, a, ds = po.varlen(q, k, v, cq, ck, d ** -0.5, True)
    assert_rows(o, ref, a, ds.t(), 150, 6.0)
    assert torch.equal(torch.isnan(lse), torch.isnan(ref_lse))


@pytest.mark.parametrize("d", varlen.HEAD_DIMS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_odd_values_of_the_last_key_without_a_mask(d, dtype):
    """The rows past the end repeat the last key's: an infinity there stays one."""
    need_gpu()
    say(f"varlen odd last key d={d} {dtype}")
    q, k, v, cq, ck = inputs([150, 60, 3], [150, 90, 333], 4, 2, d, dtype, seed=5)
    v[149, 0, 3] = math.inf
    v[149, 1, 4] = math.nan
    v[239, 1, d - 1] = -math.inf
    v[572, 0, 0] = math.inf
    o, lse = call(q, k, v, cq, ck, False)
    ref, ref_lse, a, ds = po.varlen(q, k, v, cq, ck, d ** -0.5, False)
    assert bool(torch.isinf(ref).any())
    assert_rows(o, ref, a, ds.t(), 333, 6.0)
    assert torch.equal(torch.isnan(lse), torch.isnan(ref_lse))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,hk,d", [(4, 4, 64), (8, 2, 128), (7, 1, 128), (4, 2, 256), (32, 1, 64),
                                    (33, 1, 128)])
def test_few_rows_over_long_contexts(h, hk, d, dtype, causal):
    """Single tokens and short tails whose rows fill one wave at most, next to a prompt: contexts
    around the keys that four waves take at a time, and a tail of a longer prompt."""
    need_gpu()
    say(f"varlen few rows h={h} hk={hk} d={d} {dtype} causal={causal}")
    per = max(32 // (h // hk), 1)
    lens_q = [1, 1, per, 1, 2, 0, 1, 128 // (h // hk) + 1, 300]
    lens_k = [129, 1000, 257, 3001, 160, 500, 128, 700, 310]
    q, k, v, cq, ck = inputs(lens_q, lens_k, h, hk, d, dtype, seed=21)
    check(q, k, v, cq, ck, causal)
    check(q[:cq[5]], k[:ck[5]], v[:ck[5]], cq[:6], ck[:6], causal)  # in splits


@pytest.mark.parametrize("splits", [False, True])
@pytest.mark.parametrize("d", varlen.HEAD_DIMS)
def test_few_rows_with_odd_values(d, splits):
    need_gpu()
    say(f"varlen few rows, odd values d={d} splits={splits}")
    seqs = 10 if splits else 70
    q, k, v, cq, ck = inputs([5] * seqs, [390] * seqs, 4 * 4, 4, d, torch.float16, seed=22)
    for s, (where, x) in enumerate(((389, math.nan), (387, math.inf), (388, -math.inf), (10, math.inf),
                                    (386, math.nan))):
        v[ck[s] + where, s % 4, 3 + s] = x
    k[ck[5] + 388, 1, 5] = math.nan
    o, lse = call(q, k, v, cq, ck, True)
    ref, ref_lse, a, ds = po.varlen(q, k, v, cq, ck, d ** -0.5, True)
    assert_rows(o, ref, a, ds.t(), 390, 6.0)
    assert torch.equal(torch.isnan(lse), torch.isnan(ref_lse))


# one prompt and a chunk; short tails over dealt-out keys; few rows over keys in splits
SHAPES = [([200, 70], [200, 330]), ([5] * 40, [390] * 40), ([3, 1], [2111, 700])]


@pytest.mark.parametrize("lens_q,lens_k", SHAPES)
@pytest.mark.parametrize("d", varlen.HEAD_DIMS)
def test_huge_values(lens_q, lens_k, d):
    """The largest finite bf16 values at single keys of any weight: the sums of a row stay within fp32
    where its result does."""
    need_gpu()
    say(f"varlen huge values {lens_q[:2]} d={d}")
    top = torch.finfo(torch.bfloat16).max
    for causal in (True, False):
        q, k, v, cq, ck = inputs(lens_q, lens_k, 8, 2, d, torch.bfloat16, seed=d)
        for at in ck[:-1]:
            v[at + 50, 0], v[at + 7, 1] = -top, top
        check(q, k, v, cq, ck, causal)


def check_many_huge_values(lens_q, lens_k, d):
    for causal in (True, False):
        q, k, v, cq, ck = inputs(lens_q, lens_k, 8, 2, d, torch.bfloat16, seed=d)
        v.fill_(2.0 ** 127)  # off by no more than a weight's rounding: below 2^128
        check(q, k, v, cq, ck, causal)
        v.fill_(torch.finfo(torch.bfloat16).max)
        check(torch.zeros_like(q), k, v, cq, ck, causal)  # equal weights, all exact


@pytest.mark.parametrize("lens_q,lens_k", [([5] * 40, [390] * 40), ([300] * 60, [300] * 60)])
@pytest.mark.parametrize("d", varlen.HEAD_DIMS)
def test_many_huge_values(lens_q, lens_k, d):
    """The same at every key (nothing is split here)."""
    need_gpu()
    say(f"varlen many huge values {lens_q[:2]} d={d}")
    check_many_huge_values(lens_q, lens_k, d)


@pytest.mark.parametrize("lens_q,lens_k", [SHAPES[0], SHAPES[2], ([1], [70000])])
@pytest.mark.parametrize("d", varlen.HEAD_DIMS)
def test_many_huge_values_in_splits(lens_q, lens_k, d):
    """The same where the keys are split, but for some of the first: the merge's sums stay within fp32
    too."""
    need_gpu()
    say(f"varlen many huge values {lens_q[:2]} d={d} in splits")
    check_many_huge_values(lens_q, lens_k, d)


@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", varlen.HEAD_DIMS)
def test_largest_weight_of_few_rows_is_exact(d, dtype, tokens):
    """Single tokens: two keys that a wave meets one after the other, the second e^0.6 .. e^4 times as
    heavy, among keys of next to no weight: the largest weight of a row is a power of two, whose
    rounding costs nothing, so that the first key's alone does."""
    need_gpu()
    say(f"varlen largest weight d={d} {dtype} tokens={tokens}")
    n = 200
    q, k, v, cq, ck = inputs([1] * tokens, [n] * tokens, 32, 2, d, dtype, seed=d)
    q.zero_(), k.zero_()
    k[..., 0] = -24.0
    k[3::n, :, 0], k[140::n, :, 0] = 2.0, 6.0  # tiles 0 and 4 of the first wave
    q[..., 0] = torch.linspace(0.15, 1.0, 32, device=DEV).to(dtype)
    o, _ = call(q, k, v, cq, ck, True, scale=1.0)
    for i in range(tokens):
        for j in range(2):
            r, ks = slice(16 * j, 16 * j + 16), slice(ck[i], ck[i + 1])
            ref, rest, ds = po.attend_rest(q[i, r], k[ks, j], v[ks, j], 1.0)
            assert_largest_exact(o[i, r], ref, rest, ds, n, 6.0, terms=1)


@pytest.mark.parametrize("gain", [5.0, 4000.0])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens_q,lens_k", SHAPES)
@pytest.mark.parametrize("d", varlen.HEAD_DIMS)
def test_a_row_does_not_depend_on_its_neighbours(d, lens_q, lens_k, dtype, gain):
    """One token's query grows: every other row keeps its bits."""
    need_gpu()
    say(f"varlen neighbours {lens_q[:2]} d={d} {dtype} gain={gain}")
    q, k, v, cq, ck = inputs(lens_q, lens_k, 8, 2, d, dtype, seed=d)
    o, lse = call(q, k, v, cq, ck, True)
    for t, h in ((0, 0), (2, 5)):
        other = q.clone()
        other[t, h] *= gain
        o2, l2 = call(other, k, v, cq, ck, True)
        o2[t, h], l2[h, t] = o[t, h], lse[h, t]
        assert torch.equal(o, o2) and torch.equal(lse, l2)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-3, 40.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales(scale, dtype):
    need_gpu()
    say(f"varlen scale {scale} {dtype}")
    check(*inputs([90, 33], [150, 33], 4, 2, 64, dtype, seed=6), True, scale=scale)
    check(*inputs([1, 3, 16], [300, 1500, 129], 4, 2, 64, dtype, seed=6), True, scale=scale)


def test_strided_inputs():
    """q, k, v as slices of one fused projection, as a transposed tensor, and with rows that are
    not 16-byte aligned (copied)."""
    need_gpu()
    say("varlen strides")
    lens = [50, 77]
    cu = starts(lens)
    gen = torch.Generator(device=DEV).manual_seed(8)
    fused = torch.randn((127, 8, 128), generator=gen, device=DEV).bfloat16()
    check(fused[:, :4], fused[:, 4:6], fused[:, 6:], cu, cu, True)
    by_head = torch.randn((8, 127, 128), generator=gen, device=DEV).half().transpose(0, 1)
    check(by_head[:, :4], by_head[:, 4:6], by_head[:, 6:], cu, cu, False)
    odd = torch.randn((127, 4, 65), generator=gen, device=DEV).half()[..., 1:]
    check(odd, odd[:, :2], odd[:, 2:], cu, cu, True)
    wide = torch.randn((127, 2, 128), generator=gen, device=DEV).half()
    check(fused[:, :4].half(), wide.transpose(1, 2).contiguous().transpose(1, 2), wide, cu, cu, True)
    one = torch.randn((1, 2, 128), generator=gen, device=DEV).half().expand(127, 2, 128)
    check(fused[:, :4].half(), one, wide, cu, cu, True)


def off_base(t):
    """t's values in a contiguous tensor whose base is not 16-byte aligned."""
    out = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape)
    assert out.is_contiguous() and out.data_ptr() % 16 == 2
    return out.copy_(t)


@pytest.mark.parametrize("d", varlen.HEAD_DIMS)
def test_contiguous_rows_off_the_alignment(d):
    """A misaligned base, and strides of dimensions of one that no row needs: the same result."""
    need_gpu()
    say(f"varlen off the alignment d={d}")
    q, k, v, cq, ck = inputs([70, 1], [70, 300], 4, 2, d, torch.bfloat16, seed=3)
    want = check(q, k, v, cq, ck, True)
    for args in ((off_base(q), k, v), (q, off_base(k), v), (q, k, off_base(v)),
                 (off_base(q), off_base(k), off_base(v))):
        assert all(torch.equal(x, y) for x, y in zip(call(*args, cq, ck, True), want))
    one = inputs([1], [1], 1, 1, d, torch.float16, seed=4)
    want = check(*one, False)
    for strides in ((132, d, 1), (d, 132, 1), (1 << 24, 1 << 30, 1)):
        views = [t.as_strided((1, 1, d), strides) for t in one[:3]]
        assert all(torch.equal(x, y) for x, y in zip(call(*views, *one[3:], False), want))
    q, k, v, cq, ck = inputs([1], [1], 4, 2, d, torch.float16, seed=5)
    want = check(q, k, v, cq, ck, False)
    views = [t.as_strided(t.shape, (1 << 24, d, 1)) for t in (q, k, v)]
    assert all(torch.equal(x, y) for x, y in zip(call(*views, cq, ck, False), want))


def test_equals_the_rectangular_operator_where_both_apply():
    """Sequences of one length: the same rows as flash_attention, within both tolerances."""
    need_gpu()
    say("varlen against flash_attention")
    q, k, v, cq, ck = inputs([256] * 3, [256] * 3, 8, 2, 128, torch.float16, seed=11)
    o, lse = check(q, k, v, cq, ck, True)
    o2, l2 = flag_attn.flash_attention(*(x.view(3, 256, -1, 128).transpose(1, 2) for x in (q, k, v)),
                                       causal=True, return_log_normalizer=True)[:2]
    assert float((o.view(3, 256, 8, 128).transpose(1, 2).float() - o2.float()).abs().max()) < 4e-3
    assert float((lse.view(8, 3, 256).transpose(0, 1) - l2).abs().max()) < 1e-5


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("seqs", [62, 63, 200, 254, 255, 400])
def test_many_sequences(seqs, causal):
    """More sequences than a wave has lanes, and than are ordered by their cost; most of a few
    tokens, some empty."""
    need_gpu()
    say(f"varlen {seqs} sequences causal={causal}")
    gen = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 40, (seqs,), generator=gen).tolist()
    lens[seqs // 2] = 700
    keys = [n + int(x) for n, x in zip(lens, torch.randint(0, 30, (seqs,), generator=gen))]
    check(*inputs(lens, keys, 4, 1, 64, torch.bfloat16, seed=12, extra_q=130), causal)


def mixed_lengths(seqs, tokens, seed):
    """(new tokens, keys) of sequences with that many tokens in all, about: some empty, single tokens
    over short and long contexts, chunks behind a prefix, more tokens than keys, whole prompts."""
    gen = random.Random(seed)
    kinds = [gen.choice("eostcmpppp") for _ in range(seqs)]
    weights = [gen.uniform(0.2, 2.0) if x in "cmp" else 0.0 for x in kinds]
    out = []
    for kind, w in zip(kinds, weights):
        m = max(1, round(tokens * w / max(sum(weights), 1e-9)))
        out.append({"e": (0, 40), "o": (1, gen.randrange(1, 128)), "s": (1, gen.randrange(129, 900)),
                    "t": (2, 0), "c": (m, m + gen.randrange(1, 700)), "m": (m, m - m // 3),
                    "p": (m, m)}[kind])
    return [m for m, _ in out], [n for _, n in out]


# (h, hk, new tokens, keys): 8 KV heads, more than three rounds of work-groups; one KV head, the same;
# 8 KV heads, the last work-group in the second round; more KV heads than work-groups in a round; as
# many sequences as are ordered by their cost, and one more
ORDERS = [(32, 8, *mixed_lengths(21, 4000, 1)), (8, 1, *mixed_lengths(9, 13100, 2)),
          (32, 8, [58, 0, 0] * 20, [99, 40, 0] * 20), (300, 300, [137, 0], [150, 9]),
          (16, 4, *mixed_lengths(62, 5100, 3)), (16, 4, *mixed_lengths(63, 5100, 4))]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", varlen.HEAD_DIMS)
@pytest.mark.parametrize("case", range(len(ORDERS)))
def test_order_of_work_groups(case, d, causal):
    """Launches of more work-groups than run at once, which take the row blocks in another order (up to
    62 sequences): every row is written once, rows before, behind and between the sequences' too."""
    need_gpu()
    h, hk, lens, keys = ORDERS[case]
    seqs = len(lens)
    say(f"varlen order h={h} hk={hk} d={d} seqs={seqs} causal={causal}")
    q, k, v, cq, ck = inputs(lens, keys, h, hk, d, torch.bfloat16, seed=d, extra_q=150)
    cq = [c + 60 for c in cq]
    cu = torch.cuda.get_device_properties(0).multi_processor_count
    assert varlen_splits(q.shape[0], k.shape[0], seqs, h, hk, d, causal, max(lens), max(keys), cu)[0] == 1
    blocks = sum(-(-m * (h // hk) // 128) for m in (*lens, 60, 90))
    rounds = blocks / max(256 // hk, 1)
    assert 1 < rounds < 2 if case == 2 else rounds > 3
    assert (q.shape[0] * (h // hk) // 128 + seqs + 2) * hk > 768
    old = [torch.full_like(q, math.nan), torch.full((h, q.shape[0]), math.nan, device=DEV)]
    del old  # what the outputs' memory most likely holds
    check(q, k, v, cq, ck, causal)


def test_few_rows_strided_and_alone():
    """Short row blocks of fused and transposed tensors, and one row of one head over keys that end
    at, before and behind what the waves take in turn."""
    need_gpu()
    say("varlen few rows, strides")
    gen = torch.Generator(device=DEV).manual_seed(31)
    fused = torch.randn((1200, 8, 128), generator=gen, device=DEV).bfloat16()
    by_head = torch.randn((8, 1200, 128), generator=gen, device=DEV).bfloat16().transpose(0, 1)
    for x in (fused, by_head):
        check(x[:6, :4], x[:, 4:6], x[:, 6:], [0, 1, 6], [0, 700, 1200], True)
    for n in (129, 159, 160, 161, 255, 256, 257, 288, 512):
        for d in varlen.HEAD_DIMS:
            check(*inputs([1], [n], 1, 1, d, torch.float16, seed=n), n % 2 == 0)


def test_offsets_past_32_bits():
    """A key tensor whose last rows lie more than 2^32 bytes behind its first."""
    need_gpu()
    say("varlen far offsets")
    rows, stride = 1400, 1 << 21  # elements: 2.9e9 in all
    base = torch.empty(rows * stride, dtype=torch.float16, device=DEV)
    k = base.as_strided((rows, 2, 64), (stride, 64, 1))
    v = base.as_strided((rows, 2, 64), (stride, 64, 1), 128)
    gen = torch.Generator(device=DEV).manual_seed(3)
    k.copy_(torch.randn((rows, 2, 64), generator=gen, device=DEV))
    v.copy_(torch.randn((rows, 2, 64), generator=gen, device=DEV))
    q = torch.randn((40, 4, 64), generator=gen, device=DEV).half()
    check(q, k, v, [0, 10, 40], [0, 1000, 1400], True)


def test_replays_and_other_streams():
    """Two captured calls on changed inputs, replayed in turn, and a call on another stream."""
    need_gpu()
    say("varlen graph")
    lens = [100, 3, 257]
    a = inputs(lens, lens, 4, 2, 128, torch.float16, seed=1)
    b = inputs([2], [4000], 4, 2, 128, torch.float16, seed=2)
    call(*a, True), call(*b, False)
    torch.cuda.synchronize()
    cu = [[torch.tensor(c, dtype=torch.int32, device=DEV) for c in x[3:]] for x in (a, b)]
    graphs, outs = [], []
    for x, c, mq, mk in ((a, cu[0], 257, 257), (b, cu[1], 2, 4000)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(flag_attn.flash_attention_varlen(*x[:3], *c, mq, mk, True,
                                                         return_log_normalizer=True))
        graphs.append(g)
    for rep in range(3):
        for x in (a, b):
            for t in x[:3]:
                t.copy_(torch.randn_like(t))
        if rep == 2:  # the lengths are device data
            cu[0][0].copy_(torch.tensor([0, 200, 203, 360], dtype=torch.int32))
            cu[0][1].copy_(torch.tensor([0, 180, 203, 360], dtype=torch.int32))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in outs]
        torch.randn(4096, device=DEV).sum().item()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            want = [flag_attn.flash_attention_varlen(*x[:3], *c, mq, mk, True,
                                                     return_log_normalizer=True)
                    for x, c, mq, mk in ((a, cu[0], 257, 257), (b, cu[1], 2, 4000))]
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(g, w)), rep
