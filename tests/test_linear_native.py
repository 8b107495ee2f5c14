"""The native host path of the rotary and linear-attention operators: it takes exactly the calls that the
Python path would run, with the same results, and leaves every other call to it; and those operators in
graphs and on other streams."""
import math

import pytest
import torch

import flag_attn
from flagattention_amd import ArgumentError, _lib
from tests._helpers import DEV, need_gpu, say
from tests.test_gpu_graph import _capture_and_replay
from tests.test_native_host import _both, _same

pytestmark = pytest.mark.gpu


def half(*shape, dtype=torch.float16):
    return torch.randn(shape, device=DEV).to(dtype)


@pytest.mark.parametrize("sections,mixed,adjacent", [(None, False, False), ([10, 11, 11], False, True),
                                                     ((11, 11, 10), True, False)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rotary_matches_python_path(monkeypatch, sections, mixed, adjacent, dtype):
    need_gpu()
    say(f"rotary native {sections} {dtype}")
    fast = _lib.native()
    t, h, hk, d = 37, 6, 2, 64
    qkv = half(t, h + 2 * hk, d, dtype=dtype)
    q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    pos = torch.randint(0, 9000, (t,) if sections is None else (3, t), device=DEV)
    f = torch.rand(32, device=DEV)
    for p in (pos, pos.int()):
        args = (q, k, p, f, sections, mixed, adjacent, False)
        assert fast.rotary(*args) is not None
        _same(*_both(monkeypatch, lambda: flag_attn.rotary_embedding(*args)))

        def inplace():
            x = qkv.clone()
            out = flag_attn.rotary_embedding(x[:, :h], x[:, h:h + hk], *args[2:7], inplace=True)
            return (x,) + tuple(y.clone() for y in out)

        x = qkv.clone()
        assert fast.rotary(x[:, :h], x[:, h:h + hk], *args[2:7], True) is not None
        _same(*_both(monkeypatch, inplace))
    for change in ((0, q.float()), (1, k[:5]), (0, q[..., ::2]), (2, pos.float()), (3, f.double()),
                   (4, "ab"), (4, (40, -8)), (4, (16, 8)), (5, 1), (7, 0)):
        other = list(args)
        other[change[0]] = change[1]
        assert fast.rotary(*other) is None
    assert fast.rotary(q[:1].expand(t, h, d), k, pos.int(), f, sections, mixed, adjacent, True) is None
    for slots in (torch.randperm(80, device=DEV)[:t] - 3, torch.randperm(80, device=DEV)[:t].int()):
        def store():
            kc, vc = (torch.zeros((5, hk, 16, d), dtype=dtype, device=DEV) for _ in range(2))
            y = flag_attn.rotary_cache_kv(q, k, v, pos, f, kc, vc, slots, sections, mixed, adjacent)
            return y, kc, vc

        kc = torch.zeros((5, hk, 16, d), dtype=dtype, device=DEV)
        args = [q, k, v, pos, f, kc, kc.clone(), slots, sections, mixed, adjacent]
        assert fast.rotary_cache(*args) is not None
        _same(*_both(monkeypatch, store))
        for i, x in ((2, v[:3]), (5, kc[:, :1]), (5, kc[:1].expand(5, hk, 16, d)), (6, kc.float()),
                     (7, slots.float()), (7, slots[:4])):
            other = list(args)
            other[i] = x
            assert fast.rotary_cache(*other) is None


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("h,hk,d", [(4, 4, 64), (6, 2, 128), (2, 2, 256)])
def test_linear_matches_python_path(monkeypatch, h, hk, d, dtype):
    need_gpu()
    say(f"linear native h={h} hk={hk} d={d} {dtype}")
    fast = _lib.native()
    lens = [3, 0, 900, 40]
    n = sum(lens) + 5
    qkv = half(n, h + 2 * hk, d, dtype=dtype)
    q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    a = -torch.rand(hk, device=DEV)
    cu = torch.tensor([0, 3, 3, 903, 943], dtype=torch.int32, device=DEV)
    state0 = torch.randn((6, hk, d, d), device=DEV)
    ids = torch.tensor([5, 0, -1, 2], dtype=torch.int32, device=DEV)
    has = torch.tensor([1, 1, 0, 0], dtype=torch.uint8, device=DEV)

    def prompt(*extra):
        def call():
            state = state0.clone() if extra and extra[0] else None
            more = (state,) + extra[1:] if extra else ()
            return (flag_attn.linear_attention_varlen(q, k, v, a, cu, 900, *more), state)
        return call

    for extra in ((), (True,), (True, ids), (True, ids, has), (True, None, has.bool()), (True, ids, has, 0.25)):
        _same(*_both(monkeypatch, prompt(*extra)))
    args = [q, k, v, a, cu, 900, state0.clone(), ids, has, None]
    assert fast.linear_varlen(*args) is not None
    for i, x in ((0, q.float()), (0, qkv[:, 1:h + 1, 1:]), (1, k[:9]), (2, v[..., :8]), (3, a.double()), (4, cu.long()),
                 (5, -1), (5, 1.0), (6, state0[:, :, :8]), (6, state0[:1].expand(6, hk, d, d)),
                 (6, state0.transpose(2, 3)), (6, None), (7, ids.long()), (7, ids[:2]), (8, has.int()),
                 (8, has[:1]), (9, math.inf), (9, "x")):
        other = list(args)
        other[i] = x
        assert fast.linear_varlen(*other) is None
    rows = [x[:4] for x in (q, k, v)]

    def token(*extra):
        def call():
            state = state0.clone()
            return flag_attn.linear_attention_decode(*rows, a, state, *extra), state
        return call

    for extra in ((), (ids,), (ids, 0.5)):
        _same(*_both(monkeypatch, token(*extra)))
    args = [*rows, a, state0.clone(), ids, None]
    assert fast.linear_decode(*args) is not None
    for i, x in ((0, q[:5]), (4, None), (4, state0[:3]), (5, ids[:3]), (6, math.nan)):
        other = list(args)
        other[i] = x
        if i == 4 and x is not None:
            other[5] = None
        assert fast.linear_decode(*other) is None


def test_sizes_past_a_launch_are_left_to_python():
    """And raise argument errors there.  (Large tensors are one row seen many times.)"""
    need_gpu()
    fast = _lib.native()

    def many(*shape):
        return torch.zeros((1,) * (len(shape) - 1) + shape[-1:], device=DEV).half().expand(shape)

    f = torch.zeros(32, device=DEV)
    n = 1 << 24
    pos = torch.zeros(1, dtype=torch.int32, device=DEV).expand(n)
    assert fast.rotary(many(n, 16, 64), many(n, 2, 64), pos.contiguous(), f, None, False, False, False) is None
    with pytest.raises(ArgumentError, match="too many"):
        flag_attn.rotary_embedding(many(n, 16, 64), many(n, 2, 64), pos.contiguous(), f)
    b = 65536
    state = torch.zeros((1, 1, 64, 64), device=DEV)
    args = (many(b, 1, 64), many(b, 1, 64), many(b, 1, 64), torch.zeros(1, device=DEV), state,
            torch.zeros(b, dtype=torch.int32, device=DEV))
    assert fast.linear_decode(*args, None) is None
    with pytest.raises(ArgumentError, match="too many"):
        flag_attn.linear_attention_decode(*args)
    cu = torch.zeros(b + 1, dtype=torch.int32, device=DEV)
    assert fast.linear_varlen(*args[:4], cu, 1, None, None, None, None) is None
    with pytest.raises(ArgumentError, match="too many"):
        flag_attn.linear_attention_varlen(*args[:4], cu, 1)


@pytest.mark.parametrize("into", [0, 1, 2])
def test_rows_that_lie_in_the_caches_are_refused(into):
    """Before a launch: nothing is written."""
    need_gpu()
    fast = _lib.native()
    kc, vc = half(3, 2, 16, 64), half(3, 2, 16, 64)
    f, pos = torch.rand(32, device=DEV), torch.arange(5, device=DEV)
    for cache in (kc, vc):
        rows = [half(5, 2, 64) for _ in range(3)]
        rows[into] = cache[1, :, 3:8].transpose(0, 1)
        before = cache.clone()
        assert fast.rotary_cache(*rows, pos, f, kc, vc, pos, None, False, False) is None
        with pytest.raises(ArgumentError, match="must not lie in the caches"):
            flag_attn.rotary_cache_kv(*rows, pos, f, kc, vc, pos)
        assert torch.equal(cache, before)
        rows[into] = rows[into].clone()
        assert fast.rotary_cache(*rows, pos, f, kc, vc, pos, None, False, False) is not None


def test_graph_rotary_and_store():
    """Both in one graph; the replays see new rows, positions and slots."""
    need_gpu()
    say("rotary graph")
    t, h, hk, d = 70, 4, 2, 128
    q, k, v = half(t, h, d), half(t, hk, d), half(t, hk, d)
    pos = torch.randint(0, 1 << 20, (3, t), device=DEV)
    slots = torch.randperm(96, device=DEV)[:t]
    f = torch.rand(64, device=DEV)
    kc, vc = (torch.zeros((6, hk, 16, d), dtype=torch.float16, device=DEV) for _ in range(2))

    def eager():
        y, z = flag_attn.rotary_embedding(q, k, pos, f, (22, 21, 21), True)
        kc.zero_()
        vc.zero_()
        w = flag_attn.rotary_cache_kv(q, k, v, pos, f, kc, vc, slots, (16, 24, 24))
        return y, z, w, kc.clone(), vc.clone()

    def update(rep):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device=DEV))
        pos.copy_(torch.randint(0, 1 << 20, (3, t), device=DEV))
        slots.copy_(torch.randperm(99, device=DEV)[:t] - 1)

    _capture_and_replay(eager, update, ("q", "k", "stored q", "keys", "values"))


def test_rotary_on_a_stream_of_its_own():
    need_gpu()
    q, k = half(3000, 8, 128), half(3000, 2, 128)
    pos = torch.arange(3000, device=DEV)
    f = torch.rand(64, device=DEV)
    want = flag_attn.rotary_embedding(q, k, pos, f)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        x, y = q.clone(), k.clone()
        flag_attn.rotary_embedding(x, y, pos, f, inplace=True)
    stream.synchronize()
    assert torch.equal(x, want[0]) and torch.equal(y, want[1])
