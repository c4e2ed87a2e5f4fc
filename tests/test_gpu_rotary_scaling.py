"""Scalings whose table would hold values that are not finite are refused."""
import pytest

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("bad", [
    dict(kind="llama3", factor=8.0, original_positions=8192, low_freq_factor=-INF),
    dict(kind="llama3", factor=8.0, original_positions=8192, high_freq_factor=INF),
    dict(kind="llama3", factor=8.0, original_positions=8192, low_freq_factor=NAN),
    dict(kind="yarn", factor=8.0, original_positions=8192, beta_slow=NAN),
    dict(kind="linear", factor=1e-320), dict(kind="linear", factor=1e-305),
    dict(kind="ntk", factor=1e-320), dict(kind="linear", factor=NAN)])
def test_refusals(pkg, cuda_dev, bad):
    with pytest.raises(pkg._lib.QwaError):
        pkg.rotary.rope_table(8, 128, scaling=pkg.rotary.RopeScaling(**bad))


def test_refused_by_the_c_entry(pkg, cuda_dev):
    """attention_factor, which the binding refuses by itself."""
    import ctypes
    import torch
    ctx, out = pkg.attention.Context.for_device(0), torch.zeros(8, 64, 2, device="cuda")
    for factor in (INF, NAN, -INF):
        s = pkg.rotary.RopeScaling("yarn", 4.0, 4096).struct()
        s.attention_factor = factor
        assert ctx.lib.qwa_rope_table(ctx.handle, out.data_ptr(), 0, 8, 128, 1e6, ctypes.byref(s),
                                      None) != 0
    assert not out.any()


def test_large_finite_scalings_stay(pkg, cuda_dev):
    for s in (dict(kind="linear", factor=1e300), dict(kind="ntk", factor=1e6),
              dict(kind="yarn", factor=1e6, original_positions=1.0)):
        assert pkg.rotary.rope_table(8, 128, scaling=pkg.rotary.RopeScaling(**s)).isfinite().all()
