"""Performance cases of rotary positions and of linear attention with a decay per head.

What a serving program of a model with softmax and linear attention layers calls around the
attention operators.  ``op`` names the call of a case:

* ``rotate``  ``rotary_embedding``: q and k of a step's tokens turned by their positions, of one axis
              (text) or three (time, height, width of images and video);
* ``store``   ``rotary_cache_kv``: the same where k and v go into the 16-bit paged cache;
* ``prompt``  ``linear_attention_varlen``: packed sequences from their states, which move on with them;
* ``token``   ``linear_attention_decode``: one token per sequence.

Linear attention of a KV head with log decay a: S_t = e^a S_{t-1} + k_t v_t^T, o_t = scale q_t S_t.

Sequence lengths follow from the case alone (``lengths`` seeds them), so that its work does; the
seed decides every value, slot and page.
"""
import math
import random

import torch

own = False

DEV = "cuda"
CHUNK = 128  # tokens that the plain form of ``prompt`` takes at once
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the tokens of three chats on a small model: all launch latency
        dict(name="rotate_t3_h8_d64", op="rotate", tokens=3, heads=8, kv_heads=2, dim=64, rot=64,
             axes=1, mixed=False, adjacent=False, reach=500, dtype="fp16", lengths=1),
        # an image and the text around it: three axes in runs
        dict(name="rotate_t8192_h32_d128_axes3", op="rotate", tokens=8192, heads=32, kv_heads=8,
             dim=128, rot=128, axes=3, mixed=False, adjacent=False, reach=8192, dtype="bf16",
             lengths=2),
        # far positions of long documents, a quarter of each head turned, adjacent pairs
        dict(name="rotate_t20001_h16_d256_part", op="rotate", tokens=20001, heads=16, kv_heads=16,
             dim=256, rot=64, axes=1, mixed=False, adjacent=True, reach=131072, dtype="fp16",
             lengths=3),
        # an ordinary decode step: one token of each of 32 sequences
        dict(name="store_t32_h32_d128", op="store", tokens=32, heads=32, kv_heads=8, dim=128,
             rot=128, axes=1, mixed=False, adjacent=False, reach=8192, block=64, dtype="bf16",
             lengths=4),
        # a chunk of a video, its three axes dealt out in turn
        dict(name="store_t16384_h64_d128_axes3", op="store", tokens=16384, heads=64, kv_heads=8,
             dim=128, rot=128, axes=3, mixed=True, adjacent=False, reach=131072, block=16,
             dtype="fp16", lengths=5),
        # three chat turns of a few words on a small model
        dict(name="prompt_s3_n48_d64", op="prompt", seqs=3, longest=48, heads=8, kv_heads=2, dim=64,
             kept=True, pad=0, dtype="fp16", lengths=6),
        # an ordinary batch of new prompts of mixed lengths
        dict(name="prompt_s16_n2048_d128", op="prompt", seqs=16, longest=2048, heads=32,
             kv_heads=32, dim=128, kept=False, pad=0, dtype="bf16", lengths=7),
        # one whole book: few heads, so the sequence itself has to fill the card
        dict(name="prompt_s1_n131001_d128", op="prompt", seqs=1, longest=131001, heads=16,
             kv_heads=16, dim=128, kept=False, pad=0, dtype="bf16", lengths=8),
        # the next chunk of eight prompts, grouped heads, head dim 256, padded behind
        dict(name="prompt_s8_n2048_g2_d256", op="prompt", seqs=8, longest=2048, heads=32,
             kv_heads=16, dim=256, kept=True, pad=77, dtype="fp16", lengths=9),
        # the next token of one chat on a small model
        dict(name="token_b1_h8_d64", op="token", seqs=1, heads=8, kv_heads=8, dim=64, pad=0,
             dtype="fp16", lengths=10),
        # an ordinary batch, padded to the size of a captured step
        dict(name="token_b64_h32_d128", op="token", seqs=61, heads=32, kv_heads=32, dim=128, pad=3,
             dtype="bf16", lengths=11),
        # a full batch, grouped heads, head dim 256
        dict(name="token_b256_h64_g4_d256", op="token", seqs=256, heads=64, kv_heads=16, dim=256,
             pad=0, dtype="bf16", lengths=12),
    ]


def _log_int(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(("rotate", "store", "prompt", "prompt", "token", "token"))
        kv = rng.choice((1, 2, 4, 5, 8, 16, 32))
        c = dict(op=op, kv_heads=kv, heads=kv * rng.choice((1, 1, 2, 4, 7, 8)),
                 dim=rng.choice((64, 128, 128, 256)), dtype=rng.choice(("fp16", "bf16")),
                 lengths=rng.randrange(1, 1 << 30))
        if op in ("rotate", "store"):
            c.update(tokens=_log_int(rng, 1, 32768), axes=rng.choice((1, 3)),
                     mixed=rng.random() < 0.5, adjacent=rng.random() < 0.3,
                     reach=_log_int(rng, 100, 1 << 20))
            c["rot"] = c["dim"] if rng.random() < 0.7 else rng.choice((16, 32, 48, 64))
            c["mixed"] = c["mixed"] and c["axes"] > 1
            if op == "store":
                c["block"] = rng.choice((16, 32, 64, 128))
        elif op == "prompt":
            c.update(seqs=_log_int(rng, 1, 40), longest=_log_int(rng, 1, 131072),
                     kept=rng.random() < 0.5, pad=rng.choice((0, 0, 5, 300)))
        else:
            c.update(seqs=_log_int(rng, 1, 512), pad=rng.choice((0, 0, 1, 7)))
        top = [c2 for c2 in listed() if c2["op"] == op]
        w, tops = work(c), [work(c2) for c2 in top]
        if all(w[k] <= max(t[k] for t in tops) for k in w) and _plain_cost(c) <= max(
                map(_plain_cost, top)):
            return c


def _new_tokens(case):
    """Tokens of every sequence: the first has the most, the others lie evenly over the logarithm of
    the range."""
    rng = random.Random(case["lengths"])
    n = [case["longest"]] + [_log_int(rng, max(1, case["longest"] // 16), case["longest"])
                             for _ in range(case["seqs"] - 1)]
    rng.shuffle(n)
    return n


def _plain_cost(case):
    """What the plain form's time goes by, apart from its bytes: steps one after the other."""
    if case["op"] == "prompt":
        return sum(-(-n // CHUNK) for n in _new_tokens(case))
    return 0


def work(case):
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] in ("rotate", "store"):
        n = case["tokens"]
        rows = h + hk if case["op"] == "rotate" else h + 2 * hk
        slots = 8 * n if case["op"] == "store" else 0
        return {"bytes": 4 * n * rows * d + 8 * n * case["axes"] + 2 * case["rot"] + slots,
                "flops": 3 * n * (h + hk) * case["rot"]}
    state = 4 * d * d * hk * case["seqs"]
    if case["op"] == "token":
        n = case["seqs"]
        return {"bytes": 2 * state + 4 * n * (h + hk) * d, "flops": n * d * d * (3 * hk + 2 * h)}
    n = sum(_new_tokens(case))
    return {"bytes": (2 if case["kept"] else 1) * state + 4 * n * (h + hk) * d,
            "flops": 2 * n * d * d * (h + hk)}


# ---- inputs ----

def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _rows(gen, n, heads, dim, dtype, gate=False):
    """Rows [n, heads, dim] of a projection; with ``gate`` behind x * sigmoid(x), as queries and keys
    of linear attention are."""
    x = torch.empty((n, heads, dim), dtype=dtype, device=DEV)
    step = max(1, (1 << 26) // (heads * dim))
    for i in range(0, n, step):
        y = torch.randn(x[i:i + step].shape, generator=gen, device=DEV)
        x[i:i + step] = y * torch.sigmoid(y) if gate else y
    return x


def _sections(case):
    """Frequencies of each axis: the first has a quarter or more, the others share the rest."""
    pairs = case["rot"] // 2
    if case["axes"] == 1:
        return None
    other = pairs * 3 // 8 if not case["mixed"] else pairs // 3
    return (pairs - 2 * other, other, other)


def _positions(case, gen):
    """int64 [axes, tokens] of one sequence that ends at ``reach``: text has the same position on
    every axis; a picture in the middle has its rows and columns on the second and third."""
    n = case["tokens"]
    at = torch.arange(n, device=DEV) + max(0, case["reach"] - n)
    jump = torch.randint(0, 50, (1,), generator=gen, device=DEV)
    if case["op"] == "store" and n <= 64:  # single tokens of many sequences
        at = torch.randint(0, case["reach"], (n,), generator=gen, device=DEV)
    at = at + jump
    if case["axes"] == 1:
        return at
    wide = max(1, math.isqrt(n // 2))
    i = torch.arange(n, device=DEV)
    inside = (i >= n // 4) & (i < n // 4 + wide * wide)
    k = i - n // 4
    first = at[n // 4]
    return torch.stack((torch.where(inside, first, at), torch.where(inside, first + k // wide, at),
                        torch.where(inside, first + k % wide, at)))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt, d, h, hk = DTYPES[case["dtype"]], case["dim"], case["heads"], case["kv_heads"]
    s = dict(op=case["op"])
    if case["op"] in ("rotate", "store"):
        n, pairs = case["tokens"], case["rot"] // 2
        i = torch.arange(pairs, dtype=torch.float64)
        s.update(q=_rows(gen, n, h, d, dt), k=_rows(gen, n, hk, d, dt),
                 positions=_positions(case, gen), sections=_sections(case), mixed=case["mixed"],
                 adjacent=case["adjacent"], inv_freq=(1e6 ** (-i / pairs)).float().to(DEV))
        if case["op"] == "store":
            blocks = -(-n // case["block"]) + 2
            shape = (blocks, hk, case["block"], d)
            s.update(v=_rows(gen, n, hk, d, dt), kc=torch.zeros(shape, dtype=dt, device=DEV),
                     vc=torch.zeros(shape, dtype=dt, device=DEV),
                     slots=torch.randperm(blocks * case["block"], generator=gen, device=DEV)[:n])
            if n > 64:  # whole pages one after the other, as a prompt's are
                page = torch.randperm(blocks, generator=gen, device=DEV)
                at = torch.arange(n, device=DEV)
                s["slots"] = page[at // case["block"]] * case["block"] + at % case["block"]
        return s
    # decays spread over the heads, from a memory of about two tokens to one of 256 and more
    a = -(2.0 ** (-8.0 * (torch.arange(hk, device=DEV) + 1) / hk))
    a = a * (0.5 + torch.rand(hk, generator=gen, device=DEV))
    lens = _new_tokens(case) if case["op"] == "prompt" else [1] * case["seqs"]
    n = sum(lens) + case["pad"]
    slots = case["seqs"] + 3
    size = (0.5 / torch.sqrt(-torch.expm1(2 * a))).view(hk, 1, 1)
    state = torch.empty((slots, hk, d, d), device=DEV)
    for i in range(slots):
        state[i] = torch.randn((hk, d, d), generator=gen, device=DEV) * size
    ids = torch.randperm(slots, generator=gen, device=DEV)[:case["seqs"]].to(torch.int32)
    s.update(q=_rows(gen, n, h, d, dt, True), k=_rows(gen, n, hk, d, dt, True),
             v=_rows(gen, n, hk, d, dt), log_decay=a, state=state, scale=d ** -0.5)
    if case["op"] == "prompt":
        s.update(ids=ids, host_ids=ids.tolist(), lens=lens, cu=_i32(_starts(lens)),
                 has=torch.full((case["seqs"],), case["kept"], dtype=torch.bool, device=DEV),
                 kept=case["kept"])
    else:
        s["ids"] = torch.cat((ids, _i32([-1] * case["pad"])))
        s["live"] = case["seqs"]
    return s


# ---- one pass ----

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import flag_attn
    if s["op"] == "rotate":
        return flag_attn.rotary_embedding(
            s["q"], s["k"], s["positions"], s["inv_freq"], sections=s["sections"],
            mixed_sections=s["mixed"], adjacent_pairs=s["adjacent"])
    if s["op"] == "store":
        q = flag_attn.rotary_cache_kv(
            s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["kc"], s["vc"], s["slots"],
            sections=s["sections"], mixed_sections=s["mixed"], adjacent_pairs=s["adjacent"])
        return q, s["kc"], s["vc"]
    if s["op"] == "prompt":
        o = flag_attn.linear_attention_varlen(
            s["q"], s["k"], s["v"], s["log_decay"], s["cu"], max(s["lens"]), state=s["state"],
            state_indices=s["ids"], has_state=s["has"], sm_scale=s["scale"])
    else:
        o = flag_attn.linear_attention_decode(s["q"], s["k"], s["v"], s["log_decay"], s["state"],
                                              state_indices=s["ids"], sm_scale=s["scale"])
    return o, s["state"]


def _run_plain(s):
    return {"rotate": _plain_rotate, "store": _plain_store, "prompt": _plain_prompt,
            "token": _plain_token}[s["op"]](s)


def _axis_positions(s):
    """[tokens, pairs]: the position that each frequency of each token takes."""
    pairs = s["inv_freq"].shape[0]
    if s["sections"] is None:
        return s["positions"][:, None].expand(-1, pairs)
    axis = []
    if s["mixed"]:
        axes = len(s["sections"])
        for i in range(pairs):
            a = i % axes
            axis.append(a if i // axes < s["sections"][a] else 0)
    else:
        for a, count in enumerate(s["sections"]):
            axis += [a] * count
    return s["positions"][torch.tensor(axis, device=s["positions"].device)].t()


def _plain_turn(s, x, cos, sin):
    pairs = cos.shape[-1]
    y = x[..., :2 * pairs].float()
    first, second = (y[..., 0::2], y[..., 1::2]) if s["adjacent"] else (y[..., :pairs],
                                                                        y[..., pairs:])
    a, b = first * cos - second * sin, second * cos + first * sin
    turned = torch.stack((a, b), -1).flatten(-2) if s["adjacent"] else torch.cat((a, b), -1)
    return torch.cat((turned.to(x.dtype), x[..., 2 * pairs:]), -1)


def _plain_rotate(s):
    angle = _axis_positions(s).double() * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    return _plain_turn(s, s["q"], cos, sin), _plain_turn(s, s["k"], cos, sin)


def _plain_store(s):
    q, k = _plain_rotate(s)
    block = s["kc"].shape[2]
    s["kc"][s["slots"] // block, :, s["slots"] % block] = k
    s["vc"][s["slots"] // block, :, s["slots"] % block] = s["v"]
    return q, s["kc"], s["vc"]


def _plain_prompt(s):
    q, k, v, scale = s["q"], s["k"], s["v"], s["scale"]
    h, hk, d = q.shape[1], k.shape[1], q.shape[2]
    group = h // hk
    out = torch.zeros_like(q)
    a = s["log_decay"].double().view(hk, 1, 1)
    i = torch.arange(CHUNK, device=q.device)
    gap = (i[:, None] - i[None, :]).double()
    within = torch.where(gap >= 0, torch.exp(a * gap.clamp(min=0)), 0.0).float()
    since = torch.exp(a * (i + 1).view(1, CHUNK, 1)).float()
    at = 0
    for n, slot in zip(s["lens"], s["host_ids"]):
        # the state is a sum over the whole sequence: kept in 64 bits
        state = s["state"][slot].double() if s["kept"] else torch.zeros((hk, d, d), device=q.device,
                                                                        dtype=torch.float64)
        for j in range(0, n, CHUNK):
            c = min(CHUNK, n - j)
            rows = slice(at + j, at + j + c)
            qs = q[rows].float().view(c, hk, group, d).permute(1, 2, 0, 3) * scale
            ks = k[rows].float().transpose(0, 1).contiguous()
            vs = v[rows].float().transpose(0, 1).contiguous()
            flat = qs.reshape(hk, group * c, d)
            x = torch.matmul(flat, ks.transpose(1, 2).contiguous()).view(hk, group, c, c)
            x = x * within[:, None, :c, :c]
            o = torch.matmul(x.view(hk, group * c, c), vs)
            past = torch.matmul(flat, state.float()).view(hk, group, c, d)
            o = o.view(hk, group, c, d) + past * since[:, None, :c]
            out[rows] = o.permute(2, 0, 1, 3).reshape(c, h, d).to(q.dtype)
            left = torch.exp(a * (c - 1 - i[:c]).view(1, c, 1)).float()
            new = torch.matmul(ks.transpose(1, 2).contiguous(), left * vs)
            state = torch.exp(a * c) * state + new
        s["state"][slot] = state.float()
        at += n
    return out, s["state"]


def _plain_token(s):
    n = s["live"]
    ids = s["ids"][:n].long()
    hk = s["k"].shape[1]
    group = s["q"].shape[1] // hk
    k, v = s["k"][:n].float(), s["v"][:n].float()
    decay = torch.exp(s["log_decay"]).view(1, hk, 1, 1)
    state = s["state"][ids] * decay + k[..., :, None] * v[..., None, :]
    q = s["q"][:n].float().unflatten(1, (hk, group)) * s["scale"]
    out = torch.zeros_like(s["q"])
    out[:n] = torch.matmul(q, state).flatten(1, 2).to(out.dtype)
    s["state"][ids] = state
    return out, s["state"]


# ---- the definitions in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("rotate", "store"):
        q, k = (_exact_turned(s, x) for x in (s["q"], s["k"]))
        if case["op"] == "rotate":
            return q, k
        caches = []
        for cache, rows in ((s["kc"], k), (s["vc"], s["v"].double())):
            flat = cache.double().transpose(1, 2).flatten(0, 1)
            flat[s["slots"]] = rows
            caches.append(flat.unflatten(0, (cache.shape[0], -1)).transpose(1, 2))
        return q, caches[0], caches[1]
    lens = s["lens"] if case["op"] == "prompt" else [1] * case["seqs"]
    if sum(lens) > 400000:
        return None
    return _exact_attention(case, s, lens)


def _exact_turned(s, x):
    """Each pair as a complex number times e^(i angle)."""
    pairs = s["inv_freq"].shape[0]
    positions = s["positions"].view(-1, x.shape[0]).cpu()
    angle = torch.empty((x.shape[0], pairs), dtype=torch.float64)
    sections = s["sections"] or (pairs,)
    freq = s["inv_freq"].double().cpu()
    if s["mixed"]:
        angle[:] = positions[0][:, None] * freq
        for a in range(1, len(sections)):
            take = torch.arange(sections[a]) * len(sections) + a
            angle[:, take] = positions[a][:, None] * freq[take]
    else:
        for a, (lo, hi) in enumerate(zip(_starts(sections), _starts(sections)[1:])):
            angle[:, lo:hi] = positions[a][:, None] * freq[lo:hi]
    turn = torch.polar(torch.ones_like(angle), angle).to(x.device)[:, None]
    y = x.double()
    if s["adjacent"]:
        z = torch.view_as_complex(y[..., :2 * pairs].unflatten(-1, (pairs, 2)).contiguous()) * turn
        y[..., :2 * pairs] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(y[..., :pairs].contiguous(), y[..., pairs:2 * pairs].contiguous()) * turn
        y[..., :pairs], y[..., pairs:2 * pairs] = z.real, z.imag
    return y


def _exact_attention(case, s, lens):
    """The recurrence, token after token."""
    q, k, v = (s[x] for x in "qkv")
    h, hk, d = q.shape[1], k.shape[1], q.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    states = s["state"].double()
    decay = torch.exp(s["log_decay"].double()).view(hk, 1, 1)
    at = 0
    for i, n in enumerate(lens):
        slot = s["host_ids"][i] if "host_ids" in s else int(s["ids"][i])
        state = states[slot] if case.get("kept", True) else torch.zeros_like(states[slot])
        block = 4096
        for j in range(at, at + n, block):
            rows = slice(j, min(j + block, at + n))
            qs = (q[rows].double() * s["scale"]).unflatten(1, (hk, h // hk))
            ks, vs = k[rows].double().unsqueeze(3), v[rows].double().unsqueeze(2)
            seen = []
            for t in range(qs.shape[0]):
                state = torch.addcmul(decay * state, ks[t], vs[t])
                seen.append(torch.matmul(qs[t], state))
            out[rows] = torch.stack(seen).flatten(1, 2)
        states[slot] = state
        at += n
    return out, states
