"""Shared-prefix attention on the GPU against 64 bits, request by request.
Tolerances: prefix_oracle.prefix_attention."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import prefix_oracle as po  # noqa: E402

pytestmark = pytest.mark.gpu


def offsets(lengths):
    return [0] + [int(c) for c in np.cumsum(lengths)]


def problem(pkg, seed, queries, keys, prefix, hq, hk, dtype, fmt, spare=0):
    """(q, k, v, cache, the prefix's values in f64, offsets); the cache has
    `spare` slots before and after the prefix, with NaN codes or values."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    q = (1.5 * randn(sum(queries), hq, 128)).to(dtype)
    k = randn(sum(keys), hk, 128).to(dtype)
    v = (randn(sum(keys), hk, 128) * torch.exp(randn(sum(keys), hk, 1))).to(dtype)
    slots = prefix + 2 * spare
    cache = pkg.kv_cache.KVCache(max(slots, 1), fmt, hk, 128, dtype)
    if spare:
        bad = torch.full((slots, hk, 128), float("nan"), device="cuda").to(dtype)
        every = torch.arange(slots, dtype=torch.int32, device="cuda")
        pkg.kv_cache.kv_cache_write(cache, bad, bad, every)
    pk = randn(prefix, hk, 128).to(dtype)
    pv = (randn(prefix, hk, 128) * torch.exp(randn(prefix, hk, 1))).to(dtype)
    at = torch.arange(spare, spare + prefix, dtype=torch.int32, device="cuda")
    if prefix:
        pkg.kv_cache.kv_cache_write(cache, pk, pv, at)
        pk, pv = pkg.kv_cache.kv_cache_read(cache, at)  # what the cache stands for
    return q, k, v, cache, pk.double(), pv.double(), offsets(queries), offsets(keys)


def check(pkg, p, prefix, mode, first_slot=0, sparse_prefix=176, window=432, **kw):
    q, k, v, cache, pk, pv, cu_q, cu_k = p
    out = pkg.prefix.prefix_attention(q, k, v, cu_q, cache if prefix else None, prefix, first_slot,
                                      cu_k, mode, sparse_prefix, window, **kw)
    pkg.attention.Context.for_device(0).check()
    ref, tol = po.prefix_attention(q, k, v, cu_q, cu_k, pk, pv, mode == pkg.attention.MODE_SPARSE,
                                   sparse_prefix, window)
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(out), nan)
    inf = torch.isinf(ref)
    assert torch.equal(out[inf].double(), ref[inf])
    fine = ~nan & ~inf
    off = (out.double() - ref).abs()[fine] - tol[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())
    return out


FULL, SPARSE = 1, 2


@pytest.mark.parametrize("queries,prefix", [
    ([1], 1), ([1], 0), ([5], 16), ([130], 0), ([64, 64], 128), ([1] * 16, 100),
    ([15, 150, 1, 64], 176), ([300], 129), ([257], 40)])
@pytest.mark.parametrize("fmt", ["none", "e4m3", "int8"])
def test_few_tiles(pkg, cuda_dev, queries, prefix, fmt):
    p = problem(pkg, len(queries) + prefix, queries, queries, prefix, 16, 8, torch.float16, fmt)
    check(pkg, p, prefix, FULL)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fmt", ["none", "e4m3", "int8"])
@pytest.mark.parametrize("hq,hk", [(8, 8), (16, 8), (3, 1), (12, 4), (7, 1), (16, 1), (40, 8),
                                   (100, 1)])
def test_types_and_heads(pkg, cuda_dev, dtype, fmt, hq, hk):
    queries, before = [9, 1, 70, 33], [0, 45, 3, 0]
    keys = [a + b for a, b in zip(queries, before)]
    p = problem(pkg, hq, queries, keys, 211, hq, hk, dtype, fmt)
    check(pkg, p, 211, FULL)


@pytest.mark.parametrize("fmt", ["none", "e4m3"])
@pytest.mark.parametrize("queries,before,prefix,sparse_prefix,window", [
    ([700], [0], 900, 176, 432), ([600, 90, 1], [0, 500, 700], 300, 176, 432),
    ([50, 200], [0, 0], 100, 176, 432),      # the sparse prefix reaches into own keys
    ([40, 40], [0, 0], 1000, 0, 1),          # only itself
    ([33] * 8, [0] * 8, 555, 17, 64), ([300], [10], 0, 176, 100)])
def test_sparse(pkg, cuda_dev, fmt, queries, before, prefix, sparse_prefix, window):
    keys = [a + b for a, b in zip(queries, before)]
    p = problem(pkg, prefix + window, queries, keys, prefix, 16, 8, torch.float16, fmt)
    check(pkg, p, prefix, SPARSE, sparse_prefix=sparse_prefix, window=window)


@pytest.mark.parametrize("requests,prefix", [(1, 5000), (16, 2000), (2, 257)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_single_tokens(pkg, cuda_dev, requests, prefix, dtype):
    """One query a request behind its own keys: the tiles of a block are split over
    a cluster."""
    rng = np.random.default_rng(requests)
    keys = [int(x) for x in rng.integers(1, 200, requests)]
    p = problem(pkg, requests, [1] * requests, keys, prefix, 16, 8, dtype, "e4m3")
    check(pkg, p, prefix, FULL)


@pytest.mark.parametrize("dtype,fmt", [(torch.float16, "e4m3"), (torch.bfloat16, "none"),
                                       (torch.float16, "int8")])
def test_many_blocks(pkg, cuda_dev, dtype, fmt):
    """More blocks than SMs: CTAs run several, with and without a second tile."""
    queries = [900, 1, 513, 700, 64, 1000]
    p = problem(pkg, 77, queries, queries, 700, 16, 8, dtype, fmt)
    check(pkg, p, 700, FULL)
    p = problem(pkg, 78, [2000, 41], [2100, 900], 33, 32, 32, dtype, fmt)
    check(pkg, p, 33, FULL)


# lengths that the plan deals in each of its ways: (queries, prefix) -> tiles of a
# block, split or not (on the 148 SMs of a B200)
DEALS = {(1, True): ([20, 30, 10], 600), (1, False): ([60] * 18, 40),
         (2, True): ([128] * 3, 4000), (2, False): ([700] * 8, 300)}


@pytest.mark.parametrize("tiles,split", list(DEALS))
@pytest.mark.parametrize("dtype,fmt", [(torch.float16, "e4m3"), (torch.bfloat16, "none"),
                                       (torch.float16, "int8")])
def test_every_deal(pkg, cuda_dev, tiles, split, dtype, fmt):
    queries, prefix = DEALS[tiles, split]
    plan = pkg.prefix.PrefixPlan(offsets(queries), prefix, 16, 8, mode=FULL)
    assert (plan.block_tokens, plan.splits > 1) == (64 * tiles, split)
    p = problem(pkg, tiles + 2 * split, queries, queries, prefix, 16, 8, dtype, fmt)
    out = check(pkg, p, prefix, FULL)
    # an 8-bit prefix converted tile by tile, and once: the same numbers
    q, k, v, cache, _, _, cu, _ = p
    kern = pkg.prefix.PrefixAttentionKernel(0)
    plan.workspace = dict.fromkeys(plan.workspace, 0)
    other = torch.empty_like(out)
    kern.encode(None, kern.create_run(q, k, v, other, plan, cache))
    assert torch.equal(out, other)


def test_same_as_attention_without_a_prefix(pkg, cuda_dev):
    """With a prefix of no keys both operators compute the same (other tiles: a
    rounding apart); AUTO resolves to the same rule."""
    queries = [700, 33, 1200]
    p = problem(pkg, 3, queries, queries, 0, 16, 8, torch.float16, "none")
    q, k, v, _, _, _, cu, _ = p
    ref = pkg.attention.attention(q, k, v.reshape(-1, 1024), cu)
    out = pkg.prefix.prefix_attention(q, k, v, cu)
    check(pkg, p, 0, SPARSE)
    assert float((ref.float() - out.float()).abs().max()) <= 2e-3 * float(v.abs().max())


@pytest.mark.parametrize("fmt", ["none", "e4m3", "int8"])
def test_strides_slots_and_rows_behind(pkg, cuda_dev, fmt):
    """q, k, v inside rows of a projection, the prefix amid other slots, an
    output with rows behind the last request."""
    queries, prefix = [40, 3, 100], 75
    n = sum(queries)
    p = problem(pkg, 11, queries, queries, prefix, 16, 8, torch.float16, fmt, spare=9)
    q, k, v, cache, pk, pv, cu, _ = p
    rows = torch.full((n, 4104), float("nan"), dtype=torch.float16, device="cuda")
    rows[:, :2048], rows[:, 2048:3072], rows[:, 3072:4096] = (
        t.reshape(n, -1) for t in (q, k, v))
    p2 = (rows[:, :2048].unflatten(1, (16, 128)), rows[:, 2048:3072].unflatten(1, (8, 128)),
          rows[:, 3072:4096].unflatten(1, (8, 128)), cache, pk, pv, cu, cu)
    whole = torch.full((n + 5, 16, 128), 7.0, dtype=torch.float16, device="cuda")
    check(pkg, p2, prefix, FULL, first_slot=9, out=whole[:n])
    assert (whole[n:] == 7).all()


@pytest.mark.parametrize("mode", [FULL, SPARSE])
@pytest.mark.parametrize("fmt", ["none", "e4m3"])
@pytest.mark.parametrize("queries", [[20, 30, 25], [60] * 18, [400] * 20, [128, 25, 100]])
def test_values_that_are_not_finite_stay_with_their_rows(pkg, cuda_dev, mode, fmt, queries):
    """inf and NaN in V of one request, in its late keys and in the prefix: only
    rows that keep the key see it."""
    prefix = 300
    p = problem(pkg, 5, queries, queries, prefix, 16, 8, torch.float16, fmt)
    q, k, v, cache, pk, pv, cu, _ = p
    for row, dim, x in ((cu[1] + 12, 3, float("inf")), (cu[1] + 20, 3, float("-inf")),
                        (cu[1] + 18, 100, float("nan")), (cu[2] - 1, 5, float("-inf")),
                        (cu[0], 9, float("inf")), (cu[2] + 2, 64, float("-inf"))):
        v[row, 2, dim] = x
        v[row, 7, dim] = x
    if mode == SPARSE:  # keys of the prefix that later rows drop
        pvh = pv.half()
        pvh[200, 4, 17] = float("nan")
        pkg.kv_cache.kv_cache_write(cache, pk.half(), pvh,
                                    torch.arange(prefix, dtype=torch.int32, device="cuda"))
        pk, pv = (t.double() for t in pkg.kv_cache.kv_cache_read(
            cache, torch.arange(prefix, dtype=torch.int32, device="cuda")))
    p = (q, k, v, cache, pk, pv, cu, cu)
    check(pkg, p, prefix, mode, sparse_prefix=100, window=120)


def test_nan_key_reaches_only_rows_that_keep_it(pkg, cuda_dev):
    queries = [20, 30]
    p = problem(pkg, 6, queries, queries, 50, 16, 8, torch.float16, "none")
    q, k, v, cache, pk, pv, cu, _ = p
    clean = pkg.prefix.prefix_attention(q, k, v, cu, cache, 50)
    k[cu[1] + 4, 3, 60] = float("nan")
    out = pkg.prefix.prefix_attention(q, k, v, cu, cache, 50)
    hit = torch.zeros(50, 16, dtype=torch.bool, device="cuda")
    hit[cu[1] + 4:, 6:8] = True
    assert torch.isnan(out[hit]).all() and torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("fmt", ["none", "e4m3"])
def test_prefix_past_32_bits(pkg, cuda_dev, fmt):
    """The prefix at an offset above 2^31 bytes of its cache."""
    per_slot = 1024 * (2 if fmt == "none" else 1)
    prefix, first = 150, 2 ** 31 // per_slot + 7
    p = problem(pkg, 4, [40, 30], [40, 30], prefix, 16, 8, torch.float16, fmt)
    big = pkg.kv_cache.KVCache(first + prefix + 1, fmt)
    slots = torch.arange(first, first + prefix, dtype=torch.int32, device="cuda")
    pkg.kv_cache.kv_cache_write(big, p[4].half(), p[5].half(), slots)
    back = pkg.kv_cache.kv_cache_read(big, slots)
    check(pkg, (p[0], p[1], p[2], big, back[0].double(), back[1].double(), p[6], p[7]), prefix,
          FULL, first_slot=first)


def test_large_scores(pkg, cuda_dev):
    """Scores far apart: the running maximum moves by more than the lazy bound."""
    p = problem(pkg, 9, [50, 60], [50, 60], 500, 16, 8, torch.float16, "none")
    q, k, v, cache, pk, pv, cu, _ = p
    ramp = torch.linspace(0.05, 6, 500, device="cuda")[:, None, None]
    pk = (pk * ramp).half()
    pkg.kv_cache.kv_cache_write(cache, pk, pv.half(),
                                torch.arange(500, dtype=torch.int32, device="cuda"))
    check(pkg, (q * 4, k, v, cache, pk.double(), pv, cu, cu), 500, FULL)


def test_requests_without_queries_and_repeatable(pkg, cuda_dev):
    queries, keys = [0, 7, 0, 1, 0], [5, 7, 0, 9, 3]
    p = problem(pkg, 12, queries, keys, 64, 16, 8, torch.float16, "e4m3")
    a = check(pkg, p, 64, FULL)
    b = check(pkg, p, 64, FULL)
    assert torch.equal(a, b)
    empty = torch.empty(0, 16, 128, dtype=torch.float16, device="cuda")
    got = pkg.prefix.prefix_attention(empty, p[1][:5], p[2][:5], [0, 0], p[3], 64, 0, [0, 5])
    assert got.shape == (0, 16, 128)


def test_captured_graphs_and_streams(pkg, cuda_dev):
    """Two graphs of different lengths and the eager call share a context; each
    keeps its own plan, whatever plans come and go after it."""
    graphs = []
    for seed, queries in ((1, [30, 40]), (2, [1] * 9)):
        p = problem(pkg, seed, queries, queries, 200, 16, 8, torch.float16, "e4m3")
        ref = check(pkg, p, 200, FULL)
        q, k, v, cache, _, _, cu, _ = p
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = pkg.prefix.prefix_attention(q, k, v, cu, cache, 200, mode=FULL, cu_seqlens_k=cu)
        graphs.append((graph, out, ref, p))
    for n in range(1, pkg.prefix.MAX_PLANS + 3):  # other plans push the graphs' out of the list
        pkg.prefix.prefix_attention(q[:1], k[:1], v[:1], [0, 1], cache, n, mode=FULL)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for out in (g[1] for g in graphs):
        out.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (graph, _, _, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, ref, _ in graphs:
        assert torch.equal(out, ref)
    # on a stream given by the caller
    _, _, ref, p = graphs[0]
    out = torch.empty_like(ref)
    streams[0].wait_stream(torch.cuda.current_stream())
    pkg.prefix.prefix_attention(p[0], p[1], p[2], p[6], p[3], 200, cu_seqlens_k=p[7], mode=FULL,
                                out=out, stream=streams[0])
    streams[0].synchronize()
    assert torch.equal(out, ref)


def test_new_lengths_in_a_capture_are_refused(pkg, cuda_dev):
    p = problem(pkg, 1, [30], [30], 64, 16, 8, torch.float16, "none")
    q, k, v, cache = p[:4]
    pkg.prefix.prefix_attention(q, k, v, [0, 30], cache, 64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="before the capture"):
            pkg.prefix.prefix_attention(q, k, v, [0, 13, 30], cache, 64)
        out = pkg.prefix.prefix_attention(q, k, v, [0, 30], cache, 64)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, pkg.prefix.prefix_attention(q, k, v, [0, 30], cache, 64))


def test_refusals(pkg, cuda_dev):
    p = problem(pkg, 1, [30], [30], 64, 16, 8, torch.float16, "e4m3")
    q, k, v, cache = p[:4]
    fn = pkg.prefix.prefix_attention
    cu = [0, 30]
    with pytest.raises(ValueError):
        fn(q, k, v, cu, None, 64)                     # a prefix without its cache
    with pytest.raises(ValueError):
        fn(q, k, v, [0, 29], cache, 64)               # q has another number of rows
    with pytest.raises(ValueError):
        fn(q, k, v.bfloat16(), cu, cache, 64)
    with pytest.raises(ValueError):
        fn(q, k, v[:, :4], cu, cache, 64)
    with pytest.raises(ValueError):
        fn(q, k, v, cu, cache, 64, out=torch.empty(16, 30, 128, dtype=torch.float16,
                                                   device="cuda").transpose(0, 1))
    with pytest.raises(pkg._lib.QwaError):
        fn(q, k, v, cu, cache, 65)                    # more than the cache holds
    with pytest.raises(pkg._lib.QwaError):
        fn(q, k, v, cu, cache, 60, first_slot=5)
    with pytest.raises(pkg._lib.QwaError):
        fn(q, k, v, cu, cache, 60, first_slot=-1)
    with pytest.raises(pkg._lib.QwaError):
        fn(q, k, v, cu, pkg.kv_cache.KVCache(64, heads=8, dtype=torch.bfloat16), 64)
    with pytest.raises(pkg._lib.QwaError):
        fn(q, k, v, cu, pkg.kv_cache.KVCache(64, heads=4), 64)
    with pytest.raises(pkg._lib.QwaError):
        fn(q, k, v, cu, pkg.kv_cache.KVCache(64, head_dim=64), 64)
    with pytest.raises(pkg._lib.QwaError):
        fn(q[:, :12], k, v, cu, cache, 64)            # 12 heads over 8
    with pytest.raises(pkg._lib.QwaError):            # a token stride of no whole 16 bytes
        odd = torch.zeros(30, 16 * 128 + 4, dtype=torch.float16, device="cuda")
        fn(odd[:, :2048].unflatten(1, (16, 128)), k, v, cu, cache, 64)
    plan = pkg.prefix.PrefixPlan(cu, 64, 16, 8)
    run = pkg.prefix.PrefixAttentionKernel(0).create_run(q, k, v, torch.empty_like(q), plan, cache)
    plan.close()
    with pytest.raises(ValueError):
        pkg.attention.encode_run(None, run.commands[0])
    with pytest.raises(pkg._lib.QwaError):            # first_slot + 60 is past 64 bits
        fn(q, k, v, cu, cache, 60, first_slot=2 ** 63 - 20)


def test_two_threads_at_once(pkg, cuda_dev):
    """Each thread makes its own plans and calls on its own stream."""
    import threading
    work = []
    for seed in range(4):
        p = problem(pkg, seed, [seed + 1, 40 + seed], [seed + 1, 40 + seed], 600, 16, 8,
                    torch.float16, "e4m3")
        work.append((p, check(pkg, p, 600, FULL)))
    pkg.prefix._plans.clear()
    torch.cuda.synchronize()
    got, barrier = {}, threading.Barrier(4)

    def run(i):
        q, k, v, cache, _, _, cu, _ = work[i][0]
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            barrier.wait(10)
            for _ in range(20):
                out = pkg.prefix.prefix_attention(q, k, v, cu, cache, 600, mode=FULL)
            stream.synchronize()
            got[i] = out

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    for i, (_, ref) in enumerate(work):
        assert torch.equal(got[i], ref)


def test_captured_stream_must_be_the_current_one(pkg, cuda_dev):
    """A graph keeps its plan and its workspace only where the capture is that of
    the current stream."""
    q, k, v, cache, _, _, cu, _ = problem(pkg, 1, [30] * 20, [30] * 20, 600, 16, 8, torch.float16,
                                          "e4m3")
    ref = pkg.prefix.prefix_attention(q, k, v, cu, cache, 600)
    side, out = torch.cuda.Stream(), torch.empty_like(ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with torch.cuda.stream(torch.cuda.Stream()):
            with pytest.raises(ValueError, match="current one"):
                pkg.prefix.prefix_attention(q, k, v, cu, cache, 600, out=out, stream=side)
        pkg.prefix.prefix_attention(q, k, v, cu, cache, 600, out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ref)
