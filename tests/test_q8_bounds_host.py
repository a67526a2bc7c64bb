"""What an 8-bit row stands for, the f16 numbers n s, against the value that was written: the bound that
include/pelica_attn.h states, by the format's definition."""
import torch

from tests import q8_ref as q8


def test_a_value_is_off_by_half_a_scale_and_half_a_step_of_n_s():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2000, 3, 128, generator=g).double() * torch.logspace(-9, 4.1, 2000).double()[:, None, None]
    n, s = q8.quantise(x)
    d = s.double().repeat_interleave(32, -1)
    y = q8.values(n, s).double()
    off = (y - x).abs()
    assert (off <= d / 2 + n.double().abs() * d * 2.0 ** -11 + 2.0 ** -25).all()
    # 127 / 2048 and 1 / 2 of a scale; of normal data some values need more than half a scale
    assert (off <= 0.563 * d + 2.0 ** -25).all()
    assert (off[1000:] > d[1000:] * (0.5 + 2.0 ** -6)).any()


def test_infinities_are_of_large_groups_only():
    top = torch.cat((torch.linspace(60000, 65468, 400), torch.linspace(65469, 127 * 65504, 4000))).double()
    part = torch.linspace(-1, 1, 31).double()
    x = torch.cat((top[:, None], top[:, None] * part), 1)
    n, s = q8.quantise(x)
    y = q8.values(n, s).double()
    assert y[top <= 65468].isfinite().all()
    d = s.double()
    far = x.abs() >= 65520 - d / 2
    assert y[~far].isfinite().all()
    assert torch.equal(y.isinf(), n.double().abs() * d >= 65520)
    assert (y.isinf() & (x.abs() < 65468)).any()
