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


def test_rope_rows_are_on_the_device_and_enough(pkg):
    """Of the projection and of the Q/K norm, whose requests of `cu` begin behind a prefix."""
    def table(device=1, dtype=torch.float32, values=640, contiguous=True):
        return SimpleNamespace(get_device=lambda: device, dtype=dtype, is_cuda=device >= 0,
                               is_contiguous=lambda: contiguous, numel=lambda: values)
    cu = [0, 2, 7, 8]  # at most five positions
    pkg.attention._rope_rows(table(), cu, 1)
    for bad in (table(device=0), table(device=-1), table(dtype=torch.float64),
                table(values=639), table(contiguous=False)):
        with pytest.raises(ValueError, match="rope_table"):
            pkg.attention._rope_rows(bad, cu, 1)


def test_qk_norm_takes_no_short_rope_table(pkg, monkeypatch):
    """It read past the table's end."""
    attn = pkg.attention
    for name in ("_f16_cuda", "_f32_weight"):
        monkeypatch.setattr(attn, name, lambda *a: None)
    kern = attn.QKNormRopeKernel.__new__(attn.QKNormRopeKernel)
    kern.ctx = SimpleNamespace(device=-1, lib=None, handle=None)  # of CPU tensors
    x = torch.zeros(9, 4096)
    args = (x, x, x, x, x, [0, 4, 9])
    kern.create_run_varlen(*args, input_stride=4096, rope_table=torch.zeros(5, 64, 2))
    for bad in (torch.zeros(4, 64, 2), torch.zeros(5, 64, 2, dtype=torch.float64)):
        with pytest.raises(ValueError, match="rope_table"):
            kern.create_run_varlen(*args, input_stride=4096, rope_table=bad)
