"""Calls on a stream that is not the current one. What a call makes for itself (outputs, a
workspace) must not be memory that work waiting on the current stream still
writes."""
import os
import sys

import numpy as np
import pytest
import torch

from oracle import q40 as oracle_q40

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_prefix import FULL, problem  # noqa: E402

pytestmark = pytest.mark.gpu

SLEEP = 100_000_000  # cycles: about 50 ms


def operators(pkg):
    """name -> a call of stream=, returning the tensors that it makes"""
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, cache, _, _, cu, _ = problem(pkg, 1, [70, 30], [70, 30], 400, 16, 8, torch.float16,
                                          "e4m3")
    table = pkg.rotary.rope_table(200)
    at = torch.randint(0, 200, (100,), generator=g, device="cuda", dtype=torch.int32)
    return {
        "rope": lambda stream: pkg.rotary.rope(q, k, table, at, stream=stream),
        "rope_table": lambda stream: (pkg.rotary.rope_table(3000, stream=stream),),
        "kv_cache_read": lambda stream: pkg.kv_cache.kv_cache_read(cache, at, stream=stream),
        "prefix_attention": lambda stream: (pkg.prefix.prefix_attention(
            q, k, v, cu, cache, 400, mode=FULL, stream=stream),),
    }


NAMES = ["rope", "rope_table", "kv_cache_read", "prefix_attention"]


def layer_operators(pkg):
    """The same of the framework's other calls with stream="""
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(300, 4096, generator=g, device="cuda").half()
    w = (torch.randn(4096, 1024, generator=g, device="cuda") / 32).half()
    hidden, ones, cu = x[:, :1024].contiguous(), torch.ones(128, device="cuda"), [0, 100, 300]
    q, k = pkg.attention.qk_norm_rope(x, ones, ones, cu)
    rng = np.random.default_rng(3)
    q40, _, _ = oracle_q40.pack_q40_tile32([(oracle_q40.random_q40_rows(rng, 1024, 1024), 1024)])
    packed = torch.from_numpy(q40).cuda()
    table = torch.from_numpy(np.frombuffer(pkg.prepacked.random_q6k_rows(rng, 64, 1024),
                                           np.uint8).copy()).cuda()
    ids = torch.randint(0, 64, (300,), generator=g, device="cuda", dtype=torch.int32)
    mm, att = pkg.matmul, pkg.attention

    def one(fn, *args):
        return lambda stream: (fn(*args, stream=stream),)
    return {
        "qk_norm_rope": lambda stream: att.qk_norm_rope(x, ones, ones, cu, stream=stream),
        "attention": one(att.attention, q, k, hidden, cu),
        "prefill_attention_layer": one(att.prefill_attention_layer, x, ones, ones, cu),
        "rms_norm": one(pkg.norm.rms_norm, hidden, torch.ones(1024, device="cuda")),
        "swiglu": one(pkg.ffn.swiglu, x, 2048),
        "embedding_lookup": one(pkg.ffn.embedding_lookup, ids, table),
        "last_token_pool": one(pkg.pooling.last_token_pool, hidden, cu),
        "q40_dequantize": one(mm.q40_dequantize, packed, 1024, 1024),
        "q40_matmul": one(mm.q40_matmul, hidden, packed, 1024, 1024),
        "matmul": one(mm.matmul, hidden, w),
        "matmul_swiglu": one(mm.matmul_swiglu, hidden, mm.interleave_gate_up(w)),
        "qkv_projection": lambda stream: mm.qkv_projection(hidden, w, ones, ones, cu,
                                                           stream=stream),
    }


LAYER_NAMES = ["qk_norm_rope", "attention", "prefill_attention_layer", "rms_norm", "swiglu",
               "embedding_lookup", "last_token_pool", "q40_dequantize", "q40_matmul", "matmul",
               "matmul_swiglu", "qkv_projection"]


@pytest.mark.parametrize("name", NAMES + LAYER_NAMES)
def test_outputs_are_not_memory_in_use_on_the_current_stream(pkg, cuda_dev, name):
    call = (operators if name in NAMES else layer_operators)(pkg)[name]
    ref = call(None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    call(side)
    torch.cuda.synchronize()
    torch.cuda._sleep(SLEEP)
    for r in ref:  # freed at once, written when the current stream gets there
        for _ in range(4):
            torch.empty_like(r).fill_(float("nan"))
    got = call(side)
    torch.cuda.synchronize()
    for a, b in zip(got, ref):
        assert torch.equal(a, b)


@pytest.mark.parametrize("name", NAMES + LAYER_NAMES)
def test_outputs_dropped_early_stay_of_their_stream(pkg, cuda_dev, name):
    """The memory of an output that is dropped before its stream has written it must not
    serve the current stream meanwhile."""
    call = (operators if name in NAMES else layer_operators)(pkg)[name]
    ref = call(None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    call(side)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(SLEEP)
    call(side)
    mine = [torch.empty_like(r).fill_(3.0) for r in ref for _ in range(4)]
    torch.cuda.synchronize()
    assert all((t == 3).all() for t in mine)


@pytest.mark.parametrize("name", NAMES)
def test_streams_by_handle(pkg, cuda_dev, name):
    """A stream's handle, that of the default stream (0) among them: the call runs behind
    what waits there."""
    call = operators(pkg)[name]
    ref = call(None)
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream, torch.cuda.default_stream().cuda_stream):
        call(stream)  # the stream's pool has memory then: allocating it may wait
        torch.cuda.synchronize()
        on = side if stream else torch.cuda.default_stream()
        with torch.cuda.stream(torch.cuda.Stream()):  # whatever the current one is
            with torch.cuda.stream(on):
                torch.cuda._sleep(4 * SLEEP)
            done = torch.cuda.Event()
            got = call(stream)
            done.record(on)
            assert not done.query()
            done.synchronize()
            for a, b in zip(got, ref):
                assert torch.equal(a, b)


def test_two_calls_have_workspaces_of_their_own(pkg, cuda_dev):
    """A long call on the current stream and one with another cache on a side stream, at
    once: each converts its prefix into a workspace that the other does not get."""
    work = []
    for seed, queries, prefix in ((1, [500] * 16, 2000), (2, [500] * 8, 2000)):
        q, k, v, cache, _, _, cu, _ = problem(pkg, seed, queries, queries, prefix, 16, 8,
                                              torch.float16, "e4m3")
        work.append((q, k, v, cu, cache, prefix))
    refs = [pkg.prefix.prefix_attention(*w, mode=FULL) for w in work]
    side = torch.cuda.Stream()
    outs = [torch.empty_like(r) for r in refs]
    for _ in range(20):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        pkg.prefix.prefix_attention(*work[0], mode=FULL, out=outs[0])
        pkg.prefix.prefix_attention(*work[1], mode=FULL, out=outs[1], stream=side)
        torch.cuda.synchronize()
        for out, ref in zip(outs, refs):
            assert torch.equal(out, ref)


def owned_run(pkg):
    """(out, reference, make): make() is a run that owns a workspace"""
    q, k, v, cache, _, _, cu, _ = problem(pkg, 5, [300] * 4, [300] * 4, 2000, 16, 8, torch.float16,
                                          "e4m3")
    ref = pkg.prefix.prefix_attention(q, k, v, cu, cache, 2000, mode=FULL)
    plan = pkg.prefix.PrefixPlan(cu, 2000, 16, 8, mode=FULL)
    kern, out = pkg.prefix.PrefixAttentionKernel(0), torch.empty_like(ref)

    def make():
        run = kern.create_run(q, k, v, out, plan, cache)
        assert [b.numel() for b in run.owned_buffers] == [plan.workspace["e4m3"]]
        return run
    return kern, out, ref, make


def test_workspace_of_a_run_is_not_in_use_elsewhere(pkg, cuda_dev):
    kern, out, ref, make = owned_run(pkg)
    side, nbytes = torch.cuda.Stream(), make().owned_buffers[0].numel()
    for _ in range(10):
        torch.cuda.synchronize()
        torch.cuda._sleep(SLEEP // 100)
        for _ in range(50):
            torch.empty(nbytes, dtype=torch.uint8, device="cuda").fill_(0x7e)
        run = make()
        for _ in range(20):
            kern.encode(side, run)
        torch.cuda.synchronize()
        assert torch.equal(out, ref)


def test_workspace_of_a_dropped_run_stays_of_its_stream(pkg, cuda_dev):
    kern, out, ref, make = owned_run(pkg)
    side, run = torch.cuda.Stream(), make()
    nbytes = run.owned_buffers[0].numel()
    kern.encode(side, run)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(SLEEP)
    out.zero_()
    side.wait_stream(torch.cuda.current_stream())
    kern.encode(side, run)
    del run
    mine = [torch.full((nbytes,), 3, dtype=torch.uint8, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    assert all((t == 3).all() for t in mine) and torch.equal(out, ref)


@pytest.mark.parametrize("name", ["rope", "kv_cache_read"])
def test_a_capture_keeps_what_its_calls_made(pkg, cuda_dev, name):
    """In a capture of a stream that is not the current one, outputs are of the graph's
    pool: it writes them at every replay."""
    call = operators(pkg)[name]
    ref = call(None)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = call(side)
    pools = {s["address"]: tuple(s["segment_pool_id"]) for s in torch.cuda.memory_snapshot()}
    for t in got:
        address = max(a for a in pools if a <= t.data_ptr())
        assert pools[address] == tuple(graph.pool())
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, ref):
        assert torch.equal(a, b)
