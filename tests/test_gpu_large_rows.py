"""Rotary positions and cache writes of as many rows as take the kernels' forms for large
calls: several heads a thread (from 200000 heads x 16-byte units on), two vectors a
lane group (from 2^20 lanes on). The oracles and tolerances are those of the small calls."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import prefix_oracle as po  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype,n,hq,hk,dim,rotary", [
    (torch.float16, 1500, 16, 8, 128, 128),
    (torch.bfloat16, 1101, 64, 8, 128, 64),   # more heads than a block's threads take at once
    (torch.float16, 9001, 5, 1, 64, 64),
    (torch.bfloat16, 2100, 3, 2, 256, 128)])
def test_rope_of_several_heads_a_thread(pkg, cuda_dev, layout, dtype, n, hq, hk, dim, rotary):
    units = rotary // 16 + (dim - rotary) // 8 if layout == "half" else dim // 8
    assert n * (hq + hk) * units >= 200000
    g = torch.Generator(device="cuda").manual_seed(n)
    q, k = (torch.randn(n, h, dim, generator=g, device="cuda").to(dtype) for h in (hq, hk))
    table = pkg.rotary.rope_table(3000, rotary)
    pos = torch.randint(-5, 3000, (n,), generator=g, device="cuda", dtype=torch.int32)
    inside = (pos >= 0).cpu()
    for inverse in (False, True):
        outs = [torch.full_like(x, 7) for x in (q, k)]
        pkg.rotary.rope(q, k, table, pos, layout=layout, inverse=inverse, q_out=outs[0],
                        k_out=outs[1])
        for x, y in zip((q, k), outs):
            ref = po.rope(x, table, pos.clamp(0), rotary, layout, inverse)
            tol = po.rope_tolerance(x, ref, table, pos, dtype)
            off = (y.double().cpu() - ref).abs() - tol
            assert float(off[inside].max()) <= 0
            assert (y.cpu()[~inside] == 7).all()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype,n,heads,dim", [(torch.float16, 8201, 8, 128),
                                               (torch.bfloat16, 8192, 8, 128),
                                               (torch.float16, 43703, 3, 64),
                                               (torch.bfloat16, 32771, 1, 256)])
def test_cache_write_of_two_vectors_a_group(pkg, cuda_dev, fmt, dtype, n, heads, dim):
    assert 2 * n * heads * (dim // 16) >= 1 << 20
    kc, g = pkg.kv_cache, torch.Generator().manual_seed(n)
    k, v = ((torch.randn(n, heads, dim, generator=g)
             * torch.exp(3 * torch.randn(n, heads, 1, generator=g))).to(dtype) for _ in range(2))
    k[5::997, 0, 3] = float("nan")
    v[7::991, heads - 1, 9] = float("inf")
    k[11::983] = 0
    cache = kc.KVCache(n, fmt, heads, dim, dtype)
    slots = torch.randperm(n, generator=g).int()
    slots[3::1009] = -1  # rows that are skipped
    kc.kv_cache_write(cache, k.cuda(), v.cuda(), slots.cuda())
    there = (slots >= 0).numpy()
    at = slots.numpy()[there]
    empty = np.setdiff1d(np.arange(n), at)
    for x, held, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        code, byte = po.quantise(x, fmt, dtype)
        got = held.view(torch.uint8).cpu().numpy()
        want = code.view(np.uint8)[there]
        mine = got[at]
        if fmt == "e4m3":  # any NaN code will do for NaN
            nan = np.isnan(x.double().numpy())[there]
            assert np.isnan(po.E4M3[mine][nan]).all()
            mine, want = np.where(nan, 0, mine), np.where(nan, 0, want)
        assert np.array_equal(mine, want)
        assert np.array_equal(scale.cpu().numpy()[at], byte[there])
        assert not got[empty].any() and (scale.cpu().numpy()[empty] == 127).all()
