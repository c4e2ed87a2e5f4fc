"""Rotary positions on the GPU against 64 bits: layouts, parts of a head, odd
sizes, strides, in place, positions outside the table, the way back, and the
scaled tables. Tolerances: prefix_oracle.rope_tolerance."""
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import prefix_oracle as po  # noqa: E402

pytestmark = pytest.mark.gpu


def make(g, n, heads, dim, dtype):
    return torch.randn(n, heads, dim, generator=g, device="cuda").to(dtype)


def near(got, ref, tol):
    off = (got.double().cpu() - ref).abs() - tol
    assert float(off.max()) <= 0, float(off.max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("n,hq,hk,dim,rotary", [
    (1, 16, 8, 128, 128),     # one token
    (37, 16, 8, 128, 64),     # half of the head
    (5, 6, 2, 64, 18),        # pairs that no 16-byte unit holds
    (9, 3, 1, 256, 256),
    (4, 2, 2, 80, 34),        # a head that is no multiple of 32 values
    (3, 5, 1, 18, 2),         # nothing aligned
    (11, 40, 8, 128, 32),
    (2, 100, 28, 256, 66),    # more heads than a block holds at a time
    (1500, 2, 1, 64, 64),     # several heads a thread
])
def test_matches_64_bits(pkg, cuda_dev, dtype, layout, n, hq, hk, dim, rotary):
    g = torch.Generator(device="cuda").manual_seed(n * dim + rotary)
    q, k = make(g, n, hq, dim, dtype), make(g, n, hk, dim, dtype)
    table = pkg.rotary.rope_table(600, rotary)
    pos = torch.randint(0, 600, (n,), generator=g, device="cuda", dtype=torch.int32)
    for inverse in (False, True):
        yq, yk = pkg.rotary.rope(q, k, table, pos, layout=layout, inverse=inverse)
        for x, y in ((q, yq), (k, yk)):
            ref = po.rope(x, table, pos, rotary, layout, inverse)
            near(y, ref, po.rope_tolerance(x, ref, table, pos, dtype))
            assert torch.equal(y[..., rotary:], x[..., rotary:])


@pytest.mark.parametrize("rotary", [128, 34, 64])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides_in_place_and_skipped_rows(pkg, cuda_dev, layout, rotary):
    """q and k inside rows of a projection, rotated where they are; tokens with
    a position outside the table stay as they were, and so do the v columns."""
    g = torch.Generator(device="cuda").manual_seed(3)
    n = 21
    rows = torch.randn(n, 4096, generator=g, device="cuda").half()
    before = rows.clone()
    q, k = rows[:, :2048].view(n, 16, 128), rows[:, 2048:3072].view(n, 8, 128)
    table = pkg.rotary.rope_table(50, rotary)
    pos = torch.arange(n, dtype=torch.int32, device="cuda") * 3 - 3  # -3 .. 57
    pkg.rotary.rope(q, k, table, pos, layout=layout, q_out=q, k_out=k)
    inside = ((pos >= 0) & (pos < 50)).cpu()
    assert inside.sum() not in (0, n)
    ref = po.rope(before[:, :3072].view(n, 24, 128), table, pos.clamp(0, 49), rotary, layout, False)
    tol = po.rope_tolerance(before[:, :3072].view(n, 24, 128), ref, table, pos, torch.float16)
    near(rows[:, :3072].view(n, 24, 128)[inside], ref[inside], tol[inside])
    assert torch.equal(rows[~inside], before[~inside])
    assert torch.equal(rows[:, 3072:], before[:, 3072:])
    # the way back returns what was there, within two roundings
    pkg.rotary.rope(q, k, table, pos, layout=layout, inverse=True, q_out=q, k_out=k)
    off = (rows[:, :3072].double() - before[:, :3072].double()).abs().view(n, 24, 128)
    big = before[:, :3072].double().view(n, 24, 128).abs().amax(-1, keepdim=True)
    assert float((off - 3 * 2.0 ** -11 * 1.5 * big).max()) <= 0


def test_odd_strides_and_one_side(pkg, cuda_dev):
    """A token stride that is no multiple of eight, heads outermost, q alone."""
    g = torch.Generator(device="cuda").manual_seed(4)
    buf = torch.randn(7, 3 * 64 + 5, generator=g, device="cuda").half()
    q = buf[:, 3:3 + 192].unflatten(1, (3, 64))
    table = pkg.rotary.rope_table(16, 64)
    pos = torch.arange(7, dtype=torch.int32, device="cuda")
    y, none = pkg.rotary.rope(q, None, table, pos)
    assert none is None
    ref = po.rope(q, table, pos, 64, "half", False)
    near(y, ref, po.rope_tolerance(q, ref, table, pos, torch.float16))
    heads_first = torch.randn(3, 7, 64, generator=g, device="cuda").half()
    out = torch.empty_like(heads_first)
    _, k = pkg.rotary.rope(None, heads_first.transpose(0, 1), table, pos,
                           k_out=out.transpose(0, 1))
    ref = po.rope(heads_first.transpose(0, 1), table, pos, 64, "half", False)
    near(k, ref, po.rope_tolerance(heads_first.transpose(0, 1), ref, table, pos, torch.float16))


def test_gradient_by_differences(pkg, cuda_dev):
    """sum(w * rope(x)) has the gradient rope_inverse(w): against differences of
    the 64-bit form, exact for a linear map but for its rounding."""
    g = torch.Generator(device="cuda").manual_seed(8)
    for layout in ("half", "interleaved"):
        x, w = make(g, 2, 2, 32, torch.float16), make(g, 2, 2, 32, torch.float16)
        table = pkg.rotary.rope_table(9, 16)
        pos = torch.tensor([2, 8], dtype=torch.int32, device="cuda")
        dx, _ = pkg.rotary.rope(w, None, table, pos, layout=layout, inverse=True)
        base = x.double().cpu()
        for d in range(32):
            hi, lo = base.clone(), base.clone()
            hi[..., d] += 0.5
            lo[..., d] -= 0.5
            slope = ((po.rope(hi, table, pos, 16, layout, False)
                      - po.rope(lo, table, pos, 16, layout, False)) * w.double().cpu()).sum(-1)
            off = (dx[..., d].double().cpu() - slope).abs()
            assert float((off - (2.0 ** -11 * slope.abs() + 1e-5)).max()) <= 0


def _frequencies(rotary, theta, s):
    half, i = rotary // 2, np.arange(rotary // 2)
    f = theta ** (-i / half)
    if s["kind"] == "linear":
        return f / s["factor"], 1.0
    if s["kind"] == "ntk":
        return (theta * s["factor"] ** (rotary / (rotary - 2))) ** (-i / half), 1.0
    if s["kind"] == "yarn":
        L, fast, slow = s["original_positions"], s.get("beta_fast", 32), s.get("beta_slow", 1)
        dim = [half * math.log(L / (b * 2 * math.pi)) / math.log(theta) for b in (fast, slow)]
        low, high = max(math.floor(dim[0]), 0), min(math.ceil(dim[1]), rotary - 1)
        r = np.clip((i - low) / max(high - low, 0.001), 0, 1)
        m = s.get("attention_factor") or 0.1 * math.log(s["factor"]) + 1
        return f / s["factor"] * r + f * (1 - r), m
    if s["kind"] == "llama3":
        turns = s["original_positions"] * f / (2 * math.pi)
        t = np.clip((turns - 1) / 3, 0, 1)
        return (1 - t) * f / s["factor"] + t * f, 1.0
    return f, 1.0


@pytest.mark.parametrize("scaling", [
    dict(kind="none"), dict(kind="linear", factor=4.0), dict(kind="ntk", factor=2.5),
    dict(kind="yarn", factor=4.0, original_positions=32768),
    dict(kind="yarn", factor=8.0, original_positions=4096, beta_fast=16.0, attention_factor=0.75),
    dict(kind="llama3", factor=8.0, original_positions=8192)])
@pytest.mark.parametrize("rotary,theta,first,n", [(128, 1e6, 0, 1000), (64, 1e4, 131000, 77),
                                                  (2, 1e6, 5, 1), (256, 5e5, 1 << 30, 33),
                                                  (20, 1e6, 17, 31)])
def test_tables(pkg, cuda_dev, scaling, rotary, theta, first, n):
    if scaling["kind"] == "ntk" and rotary == 2:
        pytest.skip("ntk is not defined for one frequency")
    s = pkg.rotary.RopeScaling(**scaling)
    t = pkg.rotary.rope_table(n, rotary, theta, s, first=first).double().cpu().numpy()
    f, m = _frequencies(rotary, theta, scaling)
    a = (first + np.arange(n))[:, None] * f[None]
    ref = np.stack([np.cos(a) * m, np.sin(a) * m], -1)
    # f32 rounding, and the angle's in 64 bits (the frequency's too, a few roundings)
    tol = 2.0 ** -24 * np.abs(ref) + (8 * a[..., None] + 8) * 2.0 ** -52 * m
    assert np.all(np.abs(t - ref) <= tol), np.max(np.abs(t - ref) - tol)


def test_table_serves_the_fused_kernels(pkg, cuda_dev):
    """rope_table rows are what the Q/K norm kernel makes itself, and rows from P on
    shift its positions."""
    g = torch.Generator(device="cuda").manual_seed(6)
    qkv = torch.randn(40, 4096, generator=g, device="cuda").half()
    w = torch.ones(128, device="cuda")
    table = pkg.rotary.rope_table(200, 128)
    own = pkg.attention.qk_norm_rope(qkv, w, w, [0, 40])
    kern = pkg.attention.QKNormRopeKernel(0)
    outs = [torch.empty_like(t) for t in own]
    pkg.attention.encode_run(None, kern.create_run_varlen(
        qkv, w, w, outs[0], outs[1], [0, 40], input_stride=4096, rope_table=table))
    for a, b in zip(own, outs):
        assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -9 * 4  # a step at |x| < 8
    both = torch.cat([qkv[:7], qkv])
    whole = pkg.attention.qk_norm_rope(both, w, w, [0, 47])
    pkg.attention.encode_run(None, kern.create_run_varlen(
        qkv, w, w, outs[0], outs[1], [0, 40], input_stride=4096, rope_table=table[7:]))
    for a, b in zip(whole, outs):
        assert float((a[7:].float() - b.float()).abs().max()) <= 2.0 ** -9 * 4


def test_captured_and_on_another_stream(pkg, cuda_dev):
    g = torch.Generator(device="cuda").manual_seed(9)
    q, k = make(g, 64, 16, 128, torch.float16), make(g, 64, 8, 128, torch.float16)
    table = pkg.rotary.rope_table(64, 128)
    pos = torch.arange(64, dtype=torch.int32, device="cuda")
    ref = pkg.rotary.rope(q, k, table, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [torch.empty_like(q), torch.empty_like(k)]
    pkg.rotary.rope(q, k, table, pos, q_out=outs[0], k_out=outs[1], stream=side)
    side.synchronize()
    assert torch.equal(outs[0], ref[0]) and torch.equal(outs[1], ref[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = pkg.rotary.rope(q, k, table, pos)
    x = make(g, 64, 16, 128, torch.float16)
    q.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], pkg.rotary.rope(x, k, table, pos)[0])


def test_refusals(pkg, cuda_dev):
    rot = pkg.rotary
    q = torch.zeros(4, 2, 64, dtype=torch.float16, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    table = rot.rope_table(8, 64)
    with pytest.raises(ValueError):
        rot.rope(None, None, table, pos)
    with pytest.raises(ValueError):
        rot.rope(q.float(), None, table, pos)
    with pytest.raises(ValueError):
        rot.rope(q, None, table, pos.long())
    with pytest.raises(ValueError):
        rot.rope(q, None, table, pos[:3])
    with pytest.raises(ValueError):
        rot.rope(q, None, table, pos, layout="thirds")
    with pytest.raises(ValueError):
        rot.rope(q, q[:3], table, pos)
    with pytest.raises(pkg._lib.QwaError):  # a table for more values than the head has
        rot.rope(q, None, rot.rope_table(8, 128), pos)
    with pytest.raises(pkg._lib.QwaError):  # overlapping output rows
        rot.rope(q, None, table, pos, q_out=q[:1].expand(4, 2, 64))
    with pytest.raises(pkg._lib.QwaError):
        rot.rope_table(8, 63)
    with pytest.raises(pkg._lib.QwaError):
        rot.rope_table(8, 64, theta=1.0)
    with pytest.raises(pkg._lib.QwaError):
        rot.rope_table(8, 64, first=-1)
    with pytest.raises(pkg._lib.QwaError):
        rot.rope_table(8, 64, scaling=rot.RopeScaling("linear", 0.0))
    with pytest.raises(pkg._lib.QwaError):
        rot.rope_table(8, 64, scaling=rot.RopeScaling("yarn", 4.0))
    with pytest.raises(ValueError):
        rot.rope_table(8, 64, scaling=rot.RopeScaling("other"))
    empty = torch.zeros(0, 2, 64, dtype=torch.float16, device="cuda")
    assert rot.rope(empty, None, table, pos)[0].shape == (0, 2, 64)
    assert rot.rope_table(0, 64).shape == (0, 32, 2)
    with pytest.raises(pkg._lib.QwaError):  # more heads than 2^20
        rot.rope(q[:1, :1].expand(1, 2 ** 20 + 1, 64), None, table, pos)
    # in place, where a single token has no stride of its own
    one = q[:1]
    assert rot.rope(one, None, table, pos, q_out=one.as_strided((1, 2, 64), (999, 64, 1)))[0] \
        is not None
