"""Requests that are longer than the sparse rule's range with their prefix, in a whole
model. Gate: that of tests/test_gpu_prefix_model.py."""
import warnings

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_modes_behind_a_long_prefix(pkg, cuda_dev):
    pp, attn = pkg.prepacked, pkg.attention
    model = pkg.model.Qwen3EmbeddingModel(pp.PrepackedWeights(pp.parse_prepacked_model(
        pkg.model.synthetic_model_file(2, 4096, seed=2)), 0))
    rng = np.random.default_rng(1)
    ids = torch.from_numpy(rng.integers(0, 4096, 8300).astype(np.int32)).cuda()
    head, own, cu = ids[:5000], ids[5000:], [0, 3300]
    pool = pkg.pooling.last_token_pool

    def behind(mode):
        cached = model.cache_prefix(head, "none", mode)
        return model.embed(own, cu, prefix=cached)
    for mode in (attn.MODE_FULL, attn.MODE_SPARSE):
        whole = pool(model.forward(ids, [0, 8300], mode), [0, 8300])
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            got = behind(mode)
        assert float((whole * got).sum(-1).min()) >= 0.9999
    with pytest.warns(UserWarning, match="MODE_FULL"):
        auto = behind(attn.MODE_AUTO)
    assert torch.equal(auto, got)  # the prefix's sparse rule
