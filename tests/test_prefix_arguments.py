"""Arguments of the rotary, cache and prefix bindings that are refused before any call of the
library, on the CPU."""
from types import SimpleNamespace

import pytest
import torch


@pytest.mark.parametrize("bad", [dict(first=2 ** 64), dict(first=2 ** 63), dict(first=-2 ** 64),
                                 dict(rotary_dim=2 ** 32 + 64)])
def test_numbers_of_a_table_past_their_bits(pkg, bad):
    """The C call would take their low bits."""
    with pytest.raises(ValueError, match="bit"):
        pkg.rotary.rope_table(**dict(dict(positions=0, rotary_dim=64), **bad))


@pytest.mark.parametrize("first_slot", [2 ** 64, 2 ** 64 + 5, -2 ** 64, 2 ** 63])
def test_slots_past_64_bits(pkg, first_slot):
    device = SimpleNamespace(device=-1)  # of CPU tensors
    q, k = (torch.zeros(3, heads, 128, dtype=torch.float16) for heads in (16, 8))
    plan = SimpleNamespace(ctx=device, handle=1, queries=3, keys=3, q_heads=16, kv_heads=8,
                           prefix_len=0)
    args = pkg.prefix._attention_args(device, plan, q, k, k, None, None, 7)[2]
    assert 7 in args
    with pytest.raises(ValueError, match="bit"):
        pkg.prefix._attention_args(device, plan, q, k, k, None, None, first_slot)


@pytest.mark.parametrize("factor", [float("inf"), float("nan"), 0.0, -1.0])
def test_attention_factors_of_no_use(pkg, factor):
    with pytest.raises(ValueError):
        pkg.rotary.RopeScaling("yarn", 4.0, 4096, attention_factor=factor).struct()
    assert pkg.rotary.RopeScaling("yarn", 4.0, 4096, attention_factor=0.5).struct()
