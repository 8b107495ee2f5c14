"""Views that share memory, as results of the rotary operators: refused where two of them may share an
element, and taken where packed projections and pools of caches keep them apart.  The Python path on the CPU
(what lies apart goes on to the next check, the device's); both host paths on the GPU."""
import itertools
import random

import pytest
import torch

import flag_attn
from flagattention_amd import ArgumentError, _lib, rotary
from tests._helpers import DEV, need_gpu, say


def views(x):
    """name -> (q, k, whether they lie apart) of x, 64-dim heads: [5, 8, 64] and other layouts of its memory."""
    flat = x.reshape(-1)
    rows = x.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    wide = x[:, :, None].expand(5, 8, 2, 64).contiguous()
    return {
        "packed": (x[:, :5], x[:, 5:7], True),
        "packed, k first": (x[:, 2:], x[:, :2], True),
        "heads between heads": (x[:, ::2], x[:, 1::2], True),
        "one head between heads": (x[:, ::2], x[:, 3:4], True),
        "heads outermost": (rows[:, :6], rows[:, 6:], True),
        "halves of wide heads": (wide[:, :, 0], wide[:, :, 1], True),
        "one token": (x[2:3, :5], x[2:3, 5:], True),
        "tokens apart": (x[:2].view(2, 8, 64), x[2:4, :1], True),
        "a head in both": (x[:, :4], x[:, 3:], False),
        "the same rows": (x, x, False),
        "inside": (x, x[:, 2:4], False),
        "a token on": (x[:4], x[1:], False),
        "half a head on": (flat[:4 * 512].view(4, 8, 64), flat[32:32 + 4 * 512].view(4, 8, 64), False),
        "half a wide head on": (wide[..., 0, :], wide.view(5, 8, 128)[..., 32:96], False),
        "other strides": (x[:, :1], flat[256:256 + 64 * 5].view(5, 1, 64), False),
    }


NAMES = sorted(views(torch.zeros((5, 8, 64), dtype=torch.float16)))


def call(q, k):
    t = min(q.shape[0], k.shape[0])
    return flag_attn.rotary_embedding(q[:t], k[:t], torch.zeros(t, dtype=torch.int32, device=q.device),
                                      torch.zeros(32, device=q.device), inplace=True)


@pytest.mark.parametrize("name", NAMES)
def test_in_place(name):
    q, k, apart = views(torch.zeros((5, 8, 64), dtype=torch.float16))[name]
    with pytest.raises(ArgumentError, match="CUDA" if apart else "q and k overlap"):
        call(q, k)


def caches(dev="cpu"):
    pool = torch.zeros((6, 2, 2, 16, 64), dtype=torch.float16, device=dev)  # [block, k / v, head, row, dim]
    one = torch.zeros((9, 2, 16, 64), dtype=torch.float16, device=dev)
    wide = torch.zeros((4, 2, 16, 128), dtype=torch.float16, device=dev)
    return {
        "block by block": (pool[:, 0], pool[:, 1], True),
        "a pool's parts": (one[:4], one[4:8], True),
        "every second block": (one[0:8:2], one[1:9:2], True),
        "halves of rows": (wide[..., :64], wide[..., 64:], True),
        "a block on": (one[:8], one[1:], False),
        "one block of both": (one[:5], one[4:], False),
        "the same half": (pool[:, 0], pool[:, 0], False),
        "a row on": (one.view(-1)[:8 * 2048].view(8, 2, 16, 64),
                     one.view(-1)[64:64 + 8 * 2048].view(8, 2, 16, 64), False),
    }


def store(kc, vc):
    n = min(kc.shape[0], vc.shape[0])
    rows = [torch.zeros((5, 2, 64), dtype=torch.float16, device=kc.device) for _ in range(3)]
    ids = torch.arange(5, dtype=torch.int32, device=kc.device)
    return flag_attn.rotary_cache_kv(*rows, ids, torch.zeros(32, device=kc.device), kc[:n], vc[:n], ids)


@pytest.mark.parametrize("name", sorted(caches()))
def test_caches(name):
    kc, vc, apart = caches()[name]
    with pytest.raises(ArgumentError, match="CUDA" if apart else "key_cache and value_cache overlap"):
        store(kc, vc)


def test_views_that_share_elements_are_never_taken():
    """2,000 pairs of views of one memory against the sets of their elements."""
    rng, memory = random.Random(1), torch.zeros(400, dtype=torch.float16)
    taken = refused = 0
    while taken + refused < 2000:
        pair = []
        for _ in range(2):
            size = [rng.randint(1, 4) for _ in range(2)] + [3]
            stride = [rng.choice((3, 4, 6, 9, 12, 18, 24, 36, 48)) for _ in range(2)] + [1]
            pair.append(memory.as_strided(size, stride, rng.randint(0, 60)))
        if not all(rotary._apart(x, (0, 1)) for x in pair):
            continue
        at = [{x.storage_offset() + i * x.stride(0) + j * x.stride(1) + e
               for i, j, e in itertools.product(*map(range, x.shape))} for x in pair]
        if rotary._meet(*pair):
            refused += 1
        else:
            taken += 1
            assert not at[0] & at[1]
    assert taken > 200 and refused > 200


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_both_host_paths_in_place(name):
    need_gpu()
    say(f"rotary overlap {name}")
    gen = torch.Generator(device=DEV).manual_seed(1)
    q, k, apart = views(torch.randn((5, 8, 64), generator=gen, device=DEV).half())[name]
    t = min(q.shape[0], k.shape[0])
    pos, f = torch.arange(t, device=DEV), torch.rand(32, generator=gen, device=DEV)
    if not apart:
        assert _lib.native().rotary(q[:t], k[:t], pos, f, None, False, False, True) is None
        with pytest.raises(ArgumentError, match="q and k overlap"):
            call(q, k)
        return
    want = flag_attn.rotary_embedding(q[:t], k[:t], pos, f)
    assert _lib.native().rotary(q[:t], k[:t], pos, f, None, False, False, True) is not None
    assert torch.equal(q[:t], want[0]) and torch.equal(k[:t], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(caches()))
def test_both_host_paths_caches(name):
    need_gpu()
    say(f"cache overlap {name}")
    kc, vc, apart = caches(DEV)[name]
    n = min(kc.shape[0], vc.shape[0])
    rows = torch.zeros((5, 2, 64), dtype=torch.float16, device=DEV)
    ids = torch.arange(5, device=DEV)
    done = _lib.native().rotary_cache(rows, rows, rows, ids, torch.zeros(32, device=DEV), kc[:n], vc[:n], ids, None,
                                      False, False)
    assert (done is not None) == apart
    if not apart:
        with pytest.raises(ArgumentError, match="overlap"):
            store(kc, vc)
