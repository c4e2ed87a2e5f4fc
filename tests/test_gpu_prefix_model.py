"""A whole model whose requests continue a cached text: rotary table, cache
write and shared-prefix attention together, as the engine runs them.

Against the same requests computed whole, each step's sums run in another order,
so stored f16 values may round the other way; the gate is the repository's own for
such differences (cosine >= 0.9999, tests/test_gpu_model.py). An 8-bit prefix is
compared with a 16-bit prefix that holds the values which the 8-bit one stands for:
the same numbers, the same gate."""
import asyncio
import importlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
VOCAB = 4096


@pytest.fixture(scope="module")
def model(pkg):
    data = pkg.model.synthetic_model_file(3, VOCAB, seed=2)
    return pkg.model.Qwen3EmbeddingModel(
        pkg.prepacked.PrepackedWeights(pkg.prepacked.parse_prepacked_model(data), 0))


def tokens(rng, lengths):
    return [rng.integers(0, VOCAB, n) for n in lengths]


def on_gpu(parts):
    ids = torch.from_numpy(np.concatenate(parts).astype(np.int32)).cuda()
    return ids, [0] + [int(c) for c in np.cumsum([len(p) for p in parts])]


@pytest.mark.parametrize("prefix,lengths", [(300, [15, 150, 1, 64]), (1, [40]), (777, [1] * 16),
                                            (640, [900, 20])])
def test_same_as_the_whole_requests(pkg, cuda_dev, model, prefix, lengths):
    rng = np.random.default_rng(prefix)
    (head,), parts = tokens(rng, [prefix]), tokens(rng, lengths)
    whole = model.embed(*on_gpu([np.concatenate([head, p]) for p in parts]))
    cached = model.cache_prefix(on_gpu([head])[0], "none")
    assert cached.length == prefix and len(cached.caches) == 3
    part = model.embed(*on_gpu(parts), prefix=cached)
    pkg.attention.Context.for_device(0).check()
    assert float((whole * part).sum(-1).min()) >= 0.9999


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_eight_bits_are_what_they_stand_for(pkg, cuda_dev, model, fmt):
    rng = np.random.default_rng(7)
    (head,), parts = tokens(rng, [500]), tokens(rng, [30, 100, 9])
    ids = on_gpu([head])[0]
    cached = model.cache_prefix(ids, fmt)
    values = model.cache_prefix(ids, "none")
    slots = torch.arange(500, dtype=torch.int32, device="cuda")
    for low, high in zip(cached.caches, values.caches):
        # what was stored is the layer's keys and values, rounded as the format does
        k, v = pkg.kv_cache.kv_cache_read(low, slots)
        # E4M3: half a step of 3 mantissa bits. INT8: half a step is 2^(e-1), and e is
        # the least with amax <= 127 * 2^e, so amax > 127 * 2^(e-1): at most amax / 127.
        step = 2.0 ** -4 if fmt == "e4m3" else 1 / 127
        for got, ref in ((k, high.k), (v, high.v)):
            big = ref.float().abs().amax(-1, keepdim=True)
            assert float(((got.float() - ref.float()).abs() - step * big).max()) <= 0
        pkg.kv_cache.kv_cache_write(high, k, v, slots)
    a = model.embed(*on_gpu(parts), prefix=cached)
    b = model.embed(*on_gpu(parts), prefix=values)
    assert float((a * b).sum(-1).min()) >= 0.9999
    assert cached.nbytes() < 0.52 * values.nbytes()


@pytest.mark.parametrize("packing", ["varlen", "padded"])
def test_engine_behind_a_prefix(pkg, cuda_dev, model, packing):
    eng_mod = importlib.import_module("qwen3-embedding-webgpu-prepacked_b200.engine")
    rng = np.random.default_rng(11)
    (head,), parts = tokens(rng, [200]), tokens(rng, [20, 70, 3, 130])
    runtime = model.with_prefix(model.cache_prefix(on_gpu([head])[0]))

    async def embed_all():
        eng = eng_mod.EmbeddingEngine(runtime, None, 16, 0, VOCAB - 1, packing=packing)
        return await asyncio.gather(*[eng.submit_tokens(list(p)) for p in parts])

    got = np.stack(asyncio.run(embed_all()))
    ref = runtime.embed(*on_gpu(parts)).cpu().numpy()
    assert (got * ref).sum(-1).min() >= 0.9999


def test_refusals(pkg, cuda_dev, model):
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        model.cache_prefix(empty)
    cached = model.cache_prefix(torch.zeros(5, dtype=torch.int32, device="cuda"))
    cached.caches.pop()
    with pytest.raises(ValueError):
        model.embed(torch.zeros(3, dtype=torch.int32, device="cuda"), [0, 3], prefix=cached)
    # caches that do not hold all tokens, or not all layers
    ids = torch.zeros(6, dtype=torch.int32, device="cuda")
    caches = [pkg.kv_cache.KVCache(5) for _ in range(3)]
    with pytest.raises(ValueError):
        model.forward(ids, [0, 6], store=caches)
    with pytest.raises(ValueError):
        model.forward(ids[:5], [0, 5], store=caches[:2])


def test_captured_before_longer_requests(pkg, cuda_dev, model):
    """A captured graph keeps its rotary table when longer requests need another;
    positions met for the first time are refused inside a capture."""
    rng = np.random.default_rng(11)
    (head,), parts = tokens(rng, [300]), tokens(rng, [20, 9])
    cached = model.cache_prefix(on_gpu([head])[0])
    ids, cu = on_gpu(parts)
    ref = model.forward(ids, cu, prefix=cached)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.forward(ids, cu, prefix=cached)
        far = pkg.model.CachedPrefix(10 ** 6, cached.mode, cached.caches)
        with pytest.raises(ValueError, match="before the capture"):
            model.forward(ids, cu, prefix=far)
    longer = on_gpu(tokens(rng, [2500]))
    side = torch.cuda.Stream()
    model.forward(*longer, prefix=cached)
    with torch.cuda.stream(side):  # the new table serves any stream
        again = model.forward(ids, cu, prefix=cached)
    side.synchronize()
    junk = [torch.full((1024, 64, 2), float("nan"), device="cuda") for _ in range(8)]
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    del junk
    assert torch.equal(out, ref) and torch.equal(again, ref)
