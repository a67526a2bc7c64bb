"""The 8-bit cache format by its definition, in 64 bits on the CPU."""
import torch

GROUP = 32
TOP = 65504.0
# every f16 number from 0 to the largest, in order
GRID = torch.arange(0x7C00, dtype=torch.int32).to(torch.int16).view(torch.float16).double()


def scales(x):
    """The smallest f16 numbers s with 127 s >= the largest magnitude of each group of x [..., hd]; NaN where it is none."""
    top = x.double().unflatten(-1, (-1, GROUP)).abs()
    bad = ~torch.isfinite(top).all(-1)
    top = torch.where(bad, 0.0, top.nan_to_num(0, 0, 0).amax(-1))
    bad |= top > 127 * TOP
    s = GRID[torch.searchsorted(GRID * 127, top.clamp(max=127 * TOP))]
    return torch.where(bad, torch.nan, s)


def quantise(x):
    """x [..., hd] (finite groups) as (int8 [..., hd], f16 [..., hd / 32])."""
    s = scales(x)
    d = torch.where(s > 0, s, 1.0)[..., None]
    n = (x.double().unflatten(-1, (-1, GROUP)) / d).round()
    return n.flatten(-2).to(torch.int8), s.to(torch.float16)


def values(n, s):
    """What int8 values and f16 scales stand for: f16 numbers."""
    y = n.unflatten(-1, (-1, GROUP)).double() * s.double()[..., None]
    return y.flatten(-2).to(torch.float16)
