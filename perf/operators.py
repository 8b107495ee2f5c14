"""Performance cases of prompt attention over packed sequences and of the 4-bit K/V cache.

Three calls that a serving program makes one after the other: the new tokens of every sequence
attend to what their sequence has seen (packed, one call for all sequences); their K and V go
into a paged cache held in 4 bits, from which the next chunk of a prompt takes its context back;
and every further token attends to that cache.  ``op`` names the call of a case:

* ``prompt``  ``flash_attention_varlen``: packed new tokens against packed keys, grouped heads;
* ``append``  ``cache_kv_mxfp4`` of the new tokens, then ``gather_kv_mxfp4`` of the sequences'
              whole contexts, as a chunked prefill has it before its ``prompt`` call;
* ``decode``  ``paged_attention_mxfp4``: one token per sequence against the cache.

The cache holds e2m1 codes, two in a byte (the even dim in the low half), and one power-of-two
scale for 32 dims, kept as its exponent plus 127.  A scale is the smallest at which no code is
off by more than half of the widest step: amax <= 7 * scale.

Sequence lengths follow from the case alone (``lengths`` seeds them), so that its work does; the
seed decides every value and every page.
"""
import math
import random

import torch

own = False

DEV = "cuda"
GROUP = 32  # dims that share a scale
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # three chat turns of a few words on a small model: all launch latency
        dict(name="prompt_s3_n48_d64", op="prompt", seqs=3, longest=48, prefix=0, tokens=0,
             heads=8, kv_heads=2, dim=64, dtype="fp16", causal=True, lengths=1),
        # an ordinary batch of prompts of mixed lengths
        dict(name="prompt_s16_n2048_d128", op="prompt", seqs=16, longest=2048, prefix=0, tokens=0,
             heads=32, kv_heads=8, dim=128, dtype="bf16", causal=True, lengths=2),
        # whole documents, the longest prefill
        dict(name="prompt_s6_n8192_d128", op="prompt", seqs=6, longest=8192, prefix=0, tokens=0,
             heads=32, kv_heads=8, dim=128, dtype="bf16", causal=True, lengths=3),
        # a scheduler step that mixes one chunk of a prompt with the single tokens of 32 others
        dict(name="prompt_chunk2048_tokens32", op="prompt", seqs=33, longest=2048, prefix=4096,
             tokens=32, heads=32, kv_heads=8, dim=128, dtype="bf16", causal=True, lengths=4),
        # an encoder's texts: no mask, multi-head, head dim 256
        dict(name="prompt_s12_n1500_d256_full", op="prompt", seqs=12, longest=1500, prefix=0,
             tokens=0, heads=8, kv_heads=8, dim=256, dtype="fp16", causal=False, lengths=5),
        # one short chat
        dict(name="decode_b1_ctx500_d64", op="decode", seqs=1, longest=500, shortest=500, heads=8,
             kv_heads=2, dim=64, block=16, dtype="fp16", lengths=6),
        # an ordinary batch of ragged contexts
        dict(name="decode_b32_ctx4k_d128", op="decode", seqs=32, longest=4096, shortest=97,
             heads=32, kv_heads=8, dim=128, block=64, dtype="bf16", lengths=7),
        # a full batch of long contexts
        dict(name="decode_b64_g8_ctx8k_d128", op="decode", seqs=64, longest=8192, shortest=8192,
             heads=64, kv_heads=8, dim=128, block=16, dtype="fp16", lengths=8),
        # two very long contexts, multi-head, an odd length
        dict(name="decode_b2_h16_ctx131k_d128", op="decode", seqs=2, longest=131001,
             shortest=131001, heads=16, kv_heads=16, dim=128, block=64, dtype="bf16", lengths=9),
        # head dim 256, ragged
        dict(name="decode_b32_ctx3k_d256", op="decode", seqs=32, longest=3000, shortest=700,
             heads=16, kv_heads=4, dim=256, block=32, dtype="bf16", lengths=10),
        # drafted tokens of four short chats, written and read back with their contexts
        dict(name="append_s4_new8_ctx300", op="append", seqs=4, longest=8, prefix=300, kv_heads=4,
             dim=128, block=16, dtype="fp16", lengths=11),
        # the second chunk of eight long prompts
        dict(name="append_s8_new4096_ctx4k", op="append", seqs=8, longest=4096, prefix=4096,
             kv_heads=8, dim=128, block=64, dtype="bf16", lengths=12),
    ]


def _log_int(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(("prompt", "prompt", "decode", "decode", "append"))
        kv = rng.choice((1, 2, 4, 5, 8, 16))
        c = dict(op=op, kv_heads=kv, dim=rng.choice((64, 128, 128, 256)),
                 dtype=rng.choice(("fp16", "bf16")), lengths=rng.randrange(1, 1 << 30))
        if op == "prompt":
            c.update(heads=kv * rng.choice((1, 2, 4, 7, 8)), seqs=_log_int(rng, 1, 40),
                     longest=_log_int(rng, 1, 8192), causal=rng.random() < 0.7)
            c["prefix"] = _log_int(rng, 1, 8192) if rng.random() < 0.4 else 0
            c["tokens"] = rng.randrange(c["seqs"]) if c["prefix"] else 0
        elif op == "decode":
            c.update(heads=kv * rng.choice((1, 2, 4, 7, 8, 16)), seqs=_log_int(rng, 1, 96),
                     longest=_log_int(rng, 1, 131072), block=rng.choice((16, 32, 64, 128)))
            c["shortest"] = max(1, c["longest"] // rng.choice((1, 3, 30)))
        else:
            c.update(seqs=_log_int(rng, 1, 64), longest=_log_int(rng, 1, 4096),
                     prefix=_log_int(rng, 1, 8192) if rng.random() < 0.7 else 0,
                     block=rng.choice((16, 32, 64, 128)))
        top = [c2 for c2 in listed() if c2["op"] == op]
        w, tops = work(c), [work(c2) for c2 in top]
        if all(w[k] <= max(t[k] for t in tops) for k in w) and _plain_cost(c) <= max(
                map(_plain_cost, top)):
            return c


def _spread(case):
    """(new tokens, tokens before them) of every sequence: the first is the longest, the others
    lie evenly over the logarithm of the range."""
    rng = random.Random(case["lengths"])
    out = []
    for i in range(case["seqs"]):
        new = case["longest"] if i == 0 else _log_int(rng, max(1, case["longest"] // 16),
                                                      case["longest"])
        prefix = case.get("prefix", 0)
        before = 0 if not prefix else prefix if i == 0 else _log_int(rng, max(1, prefix // 16),
                                                                     prefix)
        if i >= case["seqs"] - case.get("tokens", 0):
            new = 1
        out.append((new, before))
    rng.shuffle(out)
    return out


def _contexts(case):
    rng = random.Random(case["lengths"])
    lens = [case["longest"]] + [rng.randint(case["shortest"], case["longest"])
                                for _ in range(case["seqs"] - 1)]
    rng.shuffle(lens)
    return lens


def _plain_cost(case):
    """Score matrix entries, or cached values: what the plain form's time and memory go by."""
    if case["op"] == "prompt":
        return sum(m * (m + p) for m, p in _spread(case)) * case["heads"]
    if case["op"] == "decode":
        return sum(_contexts(case)) * case["kv_heads"] * case["dim"]
    return sum(m + p for m, p in _spread(case)) * case["kv_heads"] * case["dim"]


def work(case):
    d, hk = case["dim"], case["kv_heads"]
    row4 = d // 2 + d // GROUP  # bytes of a cached row
    if case["op"] == "prompt":
        h = case["heads"]
        new = sum(m for m, _ in _spread(case))
        keys = sum(m + p for m, p in _spread(case))
        pairs = sum(m * p + (m * (m + 1) // 2 if case["causal"] else m * m)
                    for m, p in _spread(case))
        return {"bytes": 2 * d * (2 * h * new + 2 * hk * keys) + 4 * h * new,
                "flops": 4 * d * h * pairs}
    if case["op"] == "decode":
        h, keys = case["heads"], sum(_contexts(case))
        return {"bytes": 2 * hk * keys * row4 + 4 * case["seqs"] * h * d,
                "flops": 4 * d * h * keys}
    new = sum(m for m, _ in _spread(case))
    keys = sum(m + p for m, p in _spread(case))
    # each value is compared and scaled once on its way in and scaled once on its way out
    return {"bytes": 2 * hk * (new * (2 * d + row4) + keys * (row4 + 2 * d)),
            "flops": 2 * hk * d * (3 * new + keys)}


# ---- inputs ----

def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _rows(gen, n, heads, dim, dtype, spread):
    """Rows [n, heads, dim]; the dims of a head differ in size, as those of keys do."""
    gain = torch.exp(spread * torch.randn((1, heads, dim), generator=gen, device=DEV))
    x = torch.empty((n, heads, dim), dtype=dtype, device=DEV)
    step = max(1, (1 << 26) // (heads * dim))
    for i in range(0, n, step):
        part = x[i:i + step]
        part.copy_(torch.randn(part.shape, generator=gen, device=DEV) * gain)
    return x


def _pages(case, gen, lens):
    """A block table over shuffled pages, and the number of pages."""
    each = [-(-n // case["block"]) for n in lens]
    ids = torch.randperm(sum(each) + 3, generator=gen, device=DEV).to(torch.int32)
    table = torch.zeros((len(lens), max(each)), dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(each):
        table[i, :n] = ids[at:at + n]
        at += n
    return table, sum(each) + 3


def _cache(gen, pages, case, spread):
    """Codes and scales of a cache in use: quantised rows in every slot."""
    hk, d, block = case["kv_heads"], case["dim"], case["block"]
    codes = torch.empty((pages, hk, block, d // 2), dtype=torch.uint8, device=DEV)
    scales = torch.empty((pages, hk, block, d // GROUP), dtype=torch.uint8, device=DEV)
    gain = torch.exp(spread * torch.randn((1, hk, 1, d), generator=gen, device=DEV))
    step = max(1, (1 << 25) // (hk * block * d))
    for i in range(0, pages, step):
        n = min(step, pages - i)
        x = torch.randn((n, hk, block, d), generator=gen, device=DEV) * gain
        codes[i:i + n], scales[i:i + n] = _quantise(x)
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt, d, hk = DTYPES[case["dtype"]], case["dim"], case["kv_heads"]
    s = dict(op=case["op"])
    if case["op"] == "prompt":
        spread = _spread(case)
        new, keys = [m for m, _ in spread], [m + p for m, p in spread]
        s.update(q=_rows(gen, sum(new), case["heads"], d, dt, 0.0),
                 k=_rows(gen, sum(keys), hk, d, dt, 0.4), v=_rows(gen, sum(keys), hk, d, dt, 0.2),
                 cu_q=_i32(_starts(new)), cu_k=_i32(_starts(keys)), new=new, keys=keys,
                 causal=case["causal"], scale=d ** -0.5)
    elif case["op"] == "decode":
        lens = _contexts(case)
        table, pages = _pages(case, gen, lens)
        kc, ks = _cache(gen, pages, case, 0.4)
        vc, vs = _cache(gen, pages, case, 0.2)
        s.update(q=_rows(gen, case["seqs"], case["heads"], d, dt, 0.0), kc=kc, ks=ks, vc=vc, vs=vs,
                 lens=_i32(lens), table=table, host_lens=lens, scale=d ** -0.5)
    else:
        spread = _spread(case)
        new, keys = [m for m, _ in spread], [m + p for m, p in spread]
        table, pages = _pages(case, gen, keys)
        kc, ks = _cache(gen, pages, case, 0.4)
        vc, vs = _cache(gen, pages, case, 0.2)
        slots = []
        for i, (m, p) in enumerate(spread):
            at = torch.arange(p, p + m, device=DEV)
            slots.append(table[i, at // case["block"]].long() * case["block"] + at % case["block"])
        s.update(k=_rows(gen, sum(new), hk, d, dt, 0.4), v=_rows(gen, sum(new), hk, d, dt, 0.2),
                 kc=kc, ks=ks, vc=vc, vs=vs, table=table, slots=torch.cat(slots),
                 cu_k=_i32(_starts(keys)), keys=keys, dtype=dt)
    return s


# ---- one pass ----

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import flag_attn
    if s["op"] == "prompt":
        return flag_attn.flash_attention_varlen(
            s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], max(s["new"]), max(s["keys"]),
            causal=s["causal"], sm_scale=s["scale"], return_log_normalizer=True)
    if s["op"] == "decode":
        return flag_attn.paged_attention_mxfp4(
            s["q"], s["kc"], s["ks"], s["vc"], s["vs"], s["lens"], s["table"], s["scale"],
            max(s["host_lens"]))
    flag_attn.cache_kv_mxfp4(s["k"], s["v"], s["kc"], s["ks"], s["vc"], s["vs"], s["slots"])
    return flag_attn.gather_kv_mxfp4(s["kc"], s["ks"], s["vc"], s["vs"], s["table"], s["cu_k"],
                                     sum(s["keys"]), s["dtype"])


def _run_plain(s):
    return {"prompt": _plain_prompt, "decode": _plain_decode, "append": _plain_append}[s["op"]](s)


def _softmax_rows(scores):
    """Probabilities and natural-log normaliser of the last axis; a row of -inf gives zeros."""
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    lse = torch.where(total > 0, top + torch.log(total), top)
    return p / torch.where(total > 0, total, torch.ones_like(total)), lse.squeeze(-1)


def _plain_prompt(s):
    q, k, v = s["q"], s["k"], s["v"]
    h, hk, d = q.shape[1], k.shape[1], q.shape[2]
    group = h // hk
    out = torch.zeros_like(q)
    lse = torch.empty((h, q.shape[0]), dtype=torch.float32, device=q.device)
    q0 = k0 = 0
    for m, n in zip(s["new"], s["keys"]):
        if s["causal"]:
            hidden = (torch.arange(n, device=q.device)[None, :] >
                      torch.arange(n - m, n, device=q.device)[:, None])
        for j in range(hk):
            heads = slice(j * group, (j + 1) * group)
            qs = q[q0:q0 + m, heads].transpose(0, 1).float() * s["scale"]
            ks = k[k0:k0 + n, j].float()
            x = torch.matmul(qs.reshape(group * m, d), ks.t().contiguous()).view(group, m, n)
            if s["causal"]:
                x.masked_fill_(hidden, -math.inf)
            p, l = _softmax_rows(x)
            o = torch.matmul(p.view(group * m, n), v[k0:k0 + n, j].float())
            out[q0:q0 + m, heads] = o.view(group, m, d).transpose(0, 1).to(q.dtype)
            lse[heads, q0:q0 + m] = l
        q0 += m
        k0 += n
    return out, lse


def _values(codes, scales):
    """The fp32 values of cached rows [..., dim / 2] with scales [..., dim / 32]."""
    table = torch.tensor(MAGNITUDES + tuple(-x for x in MAGNITUDES), device=codes.device)
    pairs = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    x = table[pairs].unflatten(-1, (-1, GROUP))
    power = torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127)
    return (x * power.unsqueeze(-1)).flatten(-2)


def _context(codes, scales, row, n):
    """fp32 [heads, n, dim]: the first n tokens of the sequence whose pages row lists."""
    block = codes.shape[2]
    ids = row[:-(-n // block)].long()
    x = _values(codes[ids], scales[ids])
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


def _plain_decode(s):
    out = torch.empty_like(s["q"])
    hk = s["kc"].shape[1]
    h, d = s["q"].shape[1:]
    for i, n in enumerate(s["host_lens"]):
        k = _context(s["kc"], s["ks"], s["table"][i], n)
        v = _context(s["vc"], s["vs"], s["table"][i], n)
        q = s["q"][i].float().view(hk, h // hk, d) * s["scale"]
        p, _ = _softmax_rows(torch.matmul(q, k.transpose(1, 2).contiguous()))
        out[i] = torch.matmul(p, v.contiguous()).reshape(h, d).to(out.dtype)
    return out


def _quantise(x):
    """Codes [..., dim / 2] and scale bytes [..., dim / 32] of fp32 rows."""
    groups = x.unflatten(-1, (-1, GROUP))
    part, power = torch.frexp(groups.abs().amax(-1))  # amax = part * 2^power, part in [1/2, 1)
    power = torch.where(part > 0.875, power - 2, power - 3).clamp(min=-127)
    power = torch.where(part == 0, torch.full_like(power, -127), power)
    # divided in two steps: 2^127 is the largest power of two that fp32 holds
    half = torch.div(power, 2, rounding_mode="floor")
    a = torch.ldexp(torch.ldexp(groups, -half.unsqueeze(-1)), (half - power).unsqueeze(-1))
    sign = torch.signbit(a).to(torch.uint8) << 3
    a = a.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) +
            (a >= 3.5) + (a > 5.0)) | sign
    code = code.flatten(-2).unflatten(-1, (-1, 2))
    return code[..., 0] | (code[..., 1] << 4), (power + 127).to(torch.uint8)


def _plain_append(s):
    block = s["kc"].shape[2]
    page, at = s["slots"] // block, s["slots"] % block
    for x, codes, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        codes[page, :, at], scales[page, :, at] = _quantise(x.float())
    out = []
    for codes, scales in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
        rows = [_context(codes, scales, s["table"][i], n).transpose(0, 1).to(s["dtype"])
                for i, n in enumerate(s["keys"])]
        out.append(torch.cat(rows))
    return tuple(out)


# ---- the definitions in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    return {"prompt": _exact_prompt, "decode": _exact_decode, "append": _exact_append}[
        s["op"]](s)


def _attend(q, k, v, scale, first):
    """One head in float64: row i of q sees the keys below first + i + 1 (all without first)."""
    z = (q @ k.t()) * scale
    if first is not None:
        rows = torch.arange(q.shape[0], device=q.device) + first
        z = z.where(torch.arange(k.shape[0], device=q.device) <= rows[:, None],
                    z.new_tensor(-math.inf))
    l = torch.logsumexp(z, 1)
    return torch.exp(z - l[:, None]) @ v, l


def _exact_prompt(s):
    q, k, v = s["q"], s["k"], s["v"]
    h, hk = q.shape[1], k.shape[1]
    o = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.empty((h, q.shape[0]), dtype=torch.float64, device=q.device)
    cu_q, cu_k = _starts(s["new"]), _starts(s["keys"])
    for i in range(len(s["new"])):
        a, b, c, d = cu_q[i], cu_q[i + 1], cu_k[i], cu_k[i + 1]
        for head in range(h):
            kv = head * hk // h
            first = (d - c) - (b - a) if s["causal"] else None
            o[a:b, head], lse[head, a:b] = _attend(
                q[a:b, head].double(), k[c:d, kv].double(), v[c:d, kv].double(), s["scale"], first)
    return o, lse


def _decoded(byte):
    """float64 values of code bytes, from the bits: sign, two exponent bits, one of fraction."""
    nib = torch.stack((byte % 16, byte // 16), -1).flatten(-2).to(torch.int64)
    e, f = (nib % 8) // 2, (nib % 2).double()
    mag = torch.where(e == 0, f / 2, (1 + f / 2) * torch.pow(2.0, (e - 1).double()))
    return torch.where(nib >= 8, -mag, mag)


def _tokens64(codes, scales, row, n, head):
    at = torch.arange(n, device=codes.device)
    page, slot = row.long()[at // codes.shape[2]], at % codes.shape[2]
    x = _decoded(codes[page, head, slot])
    power = torch.pow(2.0, scales[page, head, slot].double() - 127)
    return x * power.repeat_interleave(GROUP, 1)


def _exact_decode(s):
    q = s["q"]
    h, hk = q.shape[1], s["kc"].shape[1]
    o = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    for i, n in enumerate(s["host_lens"]):
        for j in range(hk):
            heads = slice(j * h // hk, (j + 1) * h // hk)
            k = _tokens64(s["kc"], s["ks"], s["table"][i], n, j)
            v = _tokens64(s["vc"], s["vs"], s["table"][i], n, j)
            o[i, heads] = _attend(q[i, heads].double(), k, v, s["scale"], None)[0]
    return o


def _nearest(x):
    """The values that the cache holds for float64 rows: the nearest multiples, ties to even."""
    g = x.unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1, keepdim=True)
    # the smallest exponent with top <= 7 * 2^e
    e = torch.ceil(torch.log2(torch.where(top > 0, top, torch.ones_like(top)) / 7))
    e = torch.where(top > 7 * torch.pow(2.0, e), e + 1, e)
    e = torch.where(top <= 7 * torch.pow(2.0, e - 1), e - 1, e).clamp(min=-127)
    scale = torch.pow(2.0, e)
    y = g.abs() / scale
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0)).to(y.dtype)
    y = (torch.round(y / step) * step).clamp(max=6.0)  # torch.round goes to even
    return torch.where(torch.signbit(g), -y, y).mul(scale).flatten(-2)


def _exact_append(s):
    block, hk = s["kc"].shape[2], s["kc"].shape[1]
    out = []
    for x, codes, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        rows = torch.cat([torch.stack([_tokens64(codes, scales, s["table"][i], n, j)
                                       for j in range(hk)], 1) for i, n in enumerate(s["keys"])])
        # where the new tokens' slots lie among the packed rows
        where = torch.full((codes.shape[0] * block,), -1, dtype=torch.int64, device=x.device)
        at = 0
        for i, n in enumerate(s["keys"]):
            t = torch.arange(n, device=x.device)
            where[s["table"][i].long()[t // block] * block + t % block] = t + at
            at += n
        rows[where[s["slots"]]] = _nearest(x.double())
        out.append(rows)
    return tuple(out)
