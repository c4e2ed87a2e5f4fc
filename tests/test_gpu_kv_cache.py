"""The 8-bit key/value cache on the GPU: codes, scales and read-back values are
equal, bit for bit, to the rule of include/qwa.h computed in 64 bits."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import prefix_oracle as po  # noqa: E402

pytestmark = pytest.mark.gpu


def rows(seed, n, heads, dim, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, dim, generator=g) * torch.exp(
        3 * torch.randn(n, heads, 1, generator=g))
    return x.to(dtype)


def codes_of(t):
    return t.view(torch.uint8).cpu().numpy()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fmt", ["e4m3", "int8", "none"])
@pytest.mark.parametrize("n,heads,dim", [(1, 8, 128), (33, 8, 128), (5, 1, 16), (7, 3, 64),
                                         (4, 2, 256), (300, 4, 32)])
def test_write_and_read(pkg, cuda_dev, dtype, fmt, n, heads, dim):
    kc = pkg.kv_cache
    k, v = rows(n + dim, n, heads, dim, dtype), rows(n + dim + 1, n, heads, dim, dtype)
    cache = kc.KVCache(n + 9, fmt, heads, dim, dtype)
    slots = torch.randperm(n + 9, generator=torch.Generator().manual_seed(1))[:n].int()
    kc.kv_cache_write(cache, k.cuda(), v.cuda(), slots.cuda())
    others = np.setdiff1d(np.arange(n + 9), slots.numpy())
    got = kc.kv_cache_read(cache, slots.cuda())
    for x, held, scale, back in ((k, cache.k, cache.k_scale, got[0]),
                                 (v, cache.v, cache.v_scale, got[1])):
        if fmt == "none":
            assert torch.equal(held[slots.long().cuda()].cpu(), x)
            assert torch.equal(back.cpu(), x)
            assert not held[torch.from_numpy(others).cuda()].any()
            continue
        code, byte = po.quantise(x, fmt, dtype)
        assert np.array_equal(codes_of(held)[slots.numpy()], code.view(np.uint8))
        assert np.array_equal(scale.cpu().numpy()[slots.numpy()], byte)
        assert not codes_of(held)[others].any() and (scale.cpu().numpy()[others] == 127).all()
        values = po.dequantise(code, byte, fmt)
        assert np.array_equal(back.double().cpu().numpy(), values)
        # the rounding itself: half a step of the format against the largest value
        step = 2.0 ** -4 if fmt == "e4m3" else 2.0 ** -7
        big = x.double().abs().amax(-1, keepdim=True).numpy()
        lowest = np.exp2(byte.astype(float) - 127)[..., None] * (
            2.0 ** -10 if fmt == "e4m3" else 0.5)
        off = np.abs(values - x.double().numpy())
        limit = np.maximum(lowest, step * (np.abs(x.double().numpy()) if fmt == "e4m3" else big))
        assert (off <= limit).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_special_values(pkg, cuda_dev, dtype, fmt):
    """Zeros, the smallest and largest values, borders of the scale, ties, NaN
    and infinities."""
    kc = pkg.kv_cache
    top, tiny = float(torch.finfo(dtype).max), po.SMALLEST[dtype]
    heads = [[0.0] * 16, [-0.0, tiny, -tiny] + [0.0] * 13, [top, -top, top / 2, 1.0] + [3.0] * 12,
             [448.0] + [27.0] * 15, [449.0 if dtype == torch.float16 else 450.0] + [1.0] * 15,
             [127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 63.5] + [126.5] * 8, [128.0] + [1.5] * 15,
             [float("nan"), 1.0, -2.0] + [0.3] * 13, [float("nan")] * 16,
             [float("inf"), float("-inf"), 5.0] + [1.0] * 13,
             [240.0, 248.0, 232.0, 17.0, 18.0, 19.0] + [9.5] * 10,
             [tiny * 5, tiny * 3] + [tiny] * 14,
             [top * (1 - 2.0 ** -6)] + [top * 0.97] * 15]
    x = torch.tensor(heads, dtype=torch.float64).to(dtype)[None]
    cache = kc.KVCache(2, fmt, len(heads), 16, dtype)
    slot = torch.tensor([1], dtype=torch.int32, device="cuda")
    kc.kv_cache_write(cache, x.cuda(), -x.cuda(), slot)
    for held, scale, y in ((cache.k, cache.k_scale, x), (cache.v, cache.v_scale, -x)):
        code, byte = po.quantise(y, fmt, dtype)
        got = codes_of(held)[1]
        want = code.view(np.uint8)[0]
        nan = np.isnan(y[0].double().numpy())
        if fmt == "e4m3":  # any NaN code will do for NaN
            assert np.isnan(po.E4M3[got][nan]).all()
            got, want = np.where(nan, 0, got), np.where(nan, 0, want)
        assert np.array_equal(got, want)
        assert np.array_equal(scale.cpu().numpy()[1], byte[0])
    back, _ = kc.kv_cache_read(cache, slot)
    b = back[0].double().cpu().numpy()
    nan = np.isnan(x[0].double().numpy()) if fmt == "e4m3" else np.zeros((len(heads), 16), bool)
    assert np.array_equal(np.isnan(b), nan) and np.isfinite(b[~nan]).all()


def test_strides_and_slots_outside(pkg, cuda_dev):
    kc = pkg.kv_cache
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn(12, 4096, generator=g, device="cuda").half()
    k, v = qkv[:, 2048:3072].view(12, 8, 128), qkv[:, 3072:].view(12, 8, 128)
    slots = torch.tensor([0, -1, 3, 20, 19, 7, -5, 2 ** 31 - 1, 1, 2, 4, 5], dtype=torch.int32,
                         device="cuda")
    cache, plain = kc.KVCache(20), kc.KVCache(20)
    kc.kv_cache_write(cache, k, v, slots)
    inside = ((slots >= 0) & (slots < 20))
    kc.kv_cache_write(plain, k[inside].contiguous(), v[inside].contiguous(),
                      slots[inside].contiguous())
    for a, b in ((cache.k, plain.k), (cache.v, plain.v)):
        assert np.array_equal(codes_of(a), codes_of(b))
    assert torch.equal(cache.k_scale, plain.k_scale) and torch.equal(cache.v_scale, plain.v_scale)
    # reading: zeros for a slot that is not there, a slot twice gives it twice
    rk, rv = kc.kv_cache_read(cache, torch.tensor([3, 20, 3, -1], dtype=torch.int32,
                                                  device="cuda"))
    assert torch.equal(rk[0], rk[2]) and torch.equal(rv[0], rv[2]) and rk[0].any()
    assert not rk[1].any() and not rk[3].any() and not rv[1].any() and not rv[3].any()


def test_slots_past_32_bits(pkg, cuda_dev):
    """Codes at offsets above 2^31 bytes."""
    kc = pkg.kv_cache
    n = 2 ** 31 // 1024 + 5
    cache = kc.KVCache(n)
    x = rows(5, 3, 8, 128, torch.float16)
    slots = torch.tensor([n - 1, 2 ** 21 - 1, 0], dtype=torch.int32, device="cuda")
    kc.kv_cache_write(cache, x.cuda(), x.cuda(), slots)
    code, byte = po.quantise(x, "e4m3", torch.float16)
    for i, s in enumerate([n - 1, 2 ** 21 - 1, 0]):
        assert np.array_equal(codes_of(cache.v[s]), code[i])
    back, _ = kc.kv_cache_read(cache, slots)
    assert np.array_equal(back.double().cpu().numpy(), po.dequantise(code, byte, "e4m3"))


def test_captured(pkg, cuda_dev):
    kc = pkg.kv_cache
    k = rows(1, 6, 8, 128, torch.float16).cuda()
    cache = kc.KVCache(6, "int8")
    slots = torch.arange(6, dtype=torch.int32, device="cuda")
    kc.kv_cache_write(cache, k, k, slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kc.kv_cache_write(cache, k, k, slots)
        back, _ = kc.kv_cache_read(cache, slots)
    x = rows(2, 6, 8, 128, torch.float16)
    k.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(back.double().cpu().numpy(),
                          po.dequantise(*po.quantise(x, "int8", torch.float16), "int8"))


def test_refusals(pkg, cuda_dev):
    kc = pkg.kv_cache
    cache = kc.KVCache(4)
    k = torch.zeros(2, 8, 128, dtype=torch.float16, device="cuda")
    s = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (k.bfloat16(), k[:1], k[:, :4], k.cpu(), k.transpose(0, 1)):
        with pytest.raises(ValueError):
            kc.kv_cache_write(cache, bad, k, s)
    with pytest.raises(ValueError):
        kc.kv_cache_write(cache, k, k, s.long())
    with pytest.raises(ValueError):
        kc.KVCache(4, "fp4")
    with pytest.raises(ValueError):
        kc.KVCache.wrap(cache.k, cache.v)  # codes without scales
    with pytest.raises(ValueError):
        kc.KVCache.wrap(cache.k, cache.v, cache.k_scale, cache.v_scale[:2])
    with pytest.raises(pkg._lib.QwaError):
        odd = kc.KVCache(4, head_dim=96)
        kc.kv_cache_write(odd, torch.zeros(2, 8, 96, dtype=torch.float16, device="cuda"),
                          torch.zeros(2, 8, 96, dtype=torch.float16, device="cuda"), s)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    kc.kv_cache_write(cache, k[:0], k[:0], none)
    assert kc.kv_cache_read(cache, none)[0].shape == (0, 8, 128)
