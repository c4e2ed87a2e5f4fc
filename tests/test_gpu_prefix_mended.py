"""Shared-prefix attention on the GPU: calls that were once answered wrongly, against
64 bits (prefix_oracle.prefix_attention has the tolerances)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_prefix import FULL, check, problem  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,prefix", [("none", 0), ("e4m3", 16)])
def test_values_put_aside_by_warps_that_run_apart(pkg, cuda_dev, fmt, prefix):
    """Several blocks a CTA, one kv head of 0..3 and one of 4..7 in turn: the first have many
    NaN in the rows of the first preparing warp, the others one infinity in rows of
    another. The late note of the first must not hide the other's."""
    requests, n = 100, 96  # 75 blocks of 128 tokens for each of 8 kv heads, four to a CTA
    p = problem(pkg, 3, [n] * requests, [n] * requests, prefix, 16, 8, torch.float16, fmt)
    v = p[2].view(requests, n, 8, 128)
    for row in (32, 33, 34, 35, 48, 49, 50, 51, 64, 65, 66, 67):
        v[:, row, :4] = float("nan")
    v[:, 4, 4:, 77] = float("inf")
    first = check(pkg, p, prefix, FULL)
    assert torch.isinf(first.view(requests, n, 16, 128)[:, 4:, 8:, 77]).all()
    q, k, v, cache, _, _, cu, _ = p
    for _ in range(20):
        again = pkg.prefix.prefix_attention(q, k, v, cu, cache if prefix else None, prefix,
                                            mode=FULL)
        assert torch.equal(again.view(torch.int16), first.view(torch.int16))
