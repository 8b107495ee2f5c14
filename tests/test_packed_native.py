"""The native host path of the packed-attention and 4-bit-cache operators: it takes exactly the calls
that the Python path would run, with the same results, and leaves every other call to it."""
import pytest
import torch

import flag_attn
from flagattention_amd import ArgumentError, _lib
from tests._helpers import DEV
from tests.test_native_host import _both, _same


def test_calls_without_gpu_tensors_are_left_to_python():
    fast = _lib.native()
    q = torch.zeros((4, 2, 64), dtype=torch.float16)
    cu = torch.zeros(2, dtype=torch.int32)
    c = [torch.zeros((2, 2, 16, n), dtype=torch.uint8) for n in (32, 2, 32, 2)]
    assert fast.varlen(q, q, q, cu, cu, 4, 4, True, None, True) is None
    assert fast.varlen(q) is None
    assert fast.mxfp4_write(q, q, *c, cu) is None
    assert fast.mxfp4_gather(*c, cu.view(1, 2), cu, 4, True) is None
    assert fast.mxfp4_decode(q, *c, cu, cu.view(1, 2), 1.0, 4, 0) is None
    assert fast.mxfp4_decode(*[None] * 10) is None


@pytest.mark.gpu
@pytest.mark.parametrize("lens_q,lens_k,h,hk,d,lse", [
    ([3, 0, 70], [3, 0, 70], 4, 2, 64, True), ([1], [3000], 8, 1, 128, True),
    ([200, 1], [200, 900], 8, 8, 256, False)])
def test_varlen_matches_python_path(monkeypatch, lens_q, lens_k, h, hk, d, lse):
    def cu(lens):
        return torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32)

    q = torch.randn((sum(lens_q), h, d), device=DEV).half()
    kv = torch.randn((sum(lens_k), 2 * hk, d), device=DEV).half()
    args = (q, kv[:, :hk], kv[:, hk:], cu(lens_q), cu(lens_k), max(lens_q), max(lens_k), True, None, lse)
    fast = _lib.native()
    assert fast.varlen(*args) is not None
    odd = torch.randn((sum(lens_q), h, d + 1), device=DEV).half()[..., 1:]
    for change in ((0, odd), (0, q.float()), (3, args[3].long()), (5, 1.5), (7, 1), (8, "x")):
        other = list(args)
        other[change[0]] = change[1]
        assert fast.varlen(*other) is None
    _same(*_both(monkeypatch, lambda: flag_attn.flash_attention_varlen(*args)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,block", [(64, 16), (128, 32), (256, 64)])
def test_mxfp4_matches_python_path(monkeypatch, d, block, dtype):
    hk, blocks, t = 3, 30, 90
    fast = _lib.native()

    def cache():
        return [torch.zeros((blocks, hk, block, n), dtype=torch.uint8, device=DEV)
                for n in (d // 2, d // 32, d // 2, d // 32)]

    k, v = (torch.randn((t, hk, d), device=DEV).to(dtype) for _ in range(2))
    for slots in (torch.randperm(blocks * block, device=DEV)[:t],
                  torch.randperm(blocks * block, device=DEV)[:t].int()):
        assert fast.mxfp4_write(k, v, *cache(), slots) is True
        assert fast.mxfp4_write(k, v, *cache(), slots.float()) is None
        assert fast.mxfp4_write(k.float(), v, *cache(), slots) is None

        def write():
            c = cache()
            flag_attn.cache_kv_mxfp4(k, v, *c, slots)
            return tuple(c)

        _same(*_both(monkeypatch, write))
    c = write()
    bt = torch.randint(0, blocks, (4, 12), dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 5, 5, 100, 300], dtype=torch.int32, device=DEV)
    assert fast.mxfp4_gather(*c, bt, cu, 310, True) is not None
    assert fast.mxfp4_gather(*c, bt, cu.long(), 310, True) is None
    assert fast.mxfp4_gather(*c, bt, cu, 0, True) is None
    _same(*_both(monkeypatch, lambda: flag_attn.gather_kv_mxfp4(*c, bt, cu, 310, dtype)))
    q = torch.randn((4, 4 * hk, d), device=DEV).to(dtype)
    lens = torch.tensor([0, 12 * block, 17, 16], dtype=torch.int32, device=DEV)
    for splits in (0, 1, 3, 40):
        args = (q, *c, lens, bt, d ** -0.5, 12 * block, splits)
        assert fast.mxfp4_decode(*args) is not None
        _same(*_both(monkeypatch, lambda: flag_attn.paged_attention_mxfp4(*args)))
    assert fast.mxfp4_decode(q, *c, lens, bt, d ** -0.5, 12 * block, -1) is None
    assert fast.mxfp4_decode(q.float(), *c, lens, bt, d ** -0.5, 12 * block, 0) is None
    assert fast.mxfp4_decode(q, *c[:3], c[3].half(), lens, bt, d ** -0.5, 12 * block, 0) is None


@pytest.mark.gpu
def test_sizes_past_a_launch_are_left_to_python():
    """And raise argument errors there.  (Large tensors are one row seen many times.)"""
    fast = _lib.native()

    def half(*shape):
        return torch.zeros((1,) * (len(shape) - 1) + shape[-1:], device=DEV).half().expand(shape)

    def i32(*shape):
        return torch.zeros(shape, dtype=torch.int32, device=DEV)

    def cache(hk):
        return [torch.zeros((4, 1, 16, n), dtype=torch.uint8, device=DEV).expand(4, hk, 16, n)
                for n in (32, 2, 32, 2)]

    q = half((1 << 29) - 1, 1, 64)
    args = (q, q[:8], q[:8], i32(1 << 24), i32(1 << 24), 4, 4, True, None, False)
    assert fast.varlen(*args) is None
    with pytest.raises(ArgumentError):
        flag_attn.flash_attention_varlen(*args[:9])
    n = (1 << 28) - 15
    slots = i32(n)
    assert fast.mxfp4_write(half(n, 1, 64), half(n, 1, 64), *cache(1), slots) is None
    with pytest.raises(ArgumentError):
        flag_attn.cache_kv_mxfp4(half(n, 1, 64), half(n, 1, 64), *cache(1), slots)
    assert fast.mxfp4_gather(*cache(1), i32(2, 4), i32(3), n, True) is None
    with pytest.raises(ArgumentError):
        flag_attn.gather_kv_mxfp4(*cache(1), i32(2, 4), i32(3), n, torch.float16)
    for seqs, h_q, hk, splits in ((65536, 1, 1, 0), (1, 65535 * 17, 65535, 0), (4097, 4096, 1, 2)):
        args = (half(seqs, h_q, 64), *cache(hk), i32(seqs), i32(seqs, 1), 1.0, 1000, splits)
        assert fast.mxfp4_decode(*args) is None
        with pytest.raises(ArgumentError):
            flag_attn.paged_attention_mxfp4(*args)
