"""The cache's smallest numbers: f16 down to its smallest subnormal, bf16 down to its
smallest normal, as include/qwa.h states (not the kernel's exponents)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

LEAST = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_small_values_are_multiples_of_the_least(pkg, cuda_dev, fmt, dtype):
    least = LEAST[dtype]
    g = torch.Generator().manual_seed(1)
    # heads whose largest value is least * 2^-8 .. 2^11, and the borders themselves
    size = least * 2.0 ** torch.arange(-8, 12, dtype=torch.float64)[:, None]
    x = (torch.rand(20, 13, generator=g, dtype=torch.float64) * 2 - 1) * size
    x = torch.cat([x, size, least * torch.tensor([[0.5, 1.5]]).double().expand(20, 2)], 1)
    x = x.to(dtype)[None]
    cache = pkg.kv_cache.KVCache(1, fmt, 20, 16, dtype)
    slot = torch.zeros(1, dtype=torch.int32, device="cuda")
    pkg.kv_cache.kv_cache_write(cache, x.cuda(), -x.cuda(), slot)
    back, minus = (t.double().cpu() for t in pkg.kv_cache.kv_cache_read(cache, slot))
    assert torch.equal(back, -minus)
    steps = back / least
    assert torch.equal(steps, steps.round())
    # half a step of the format, or half of the least number
    top = x.double().abs().amax(-1, keepdim=True)
    step = 2.0 ** -4 * x.double().abs() if fmt == "e4m3" else top / 127
    assert ((back - x.double()).abs() <= step.clamp(min=least / 2)).all()
