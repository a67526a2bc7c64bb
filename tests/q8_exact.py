"""Rows written into 8-bit pages, integer by integer: the inputs of each form of
the qkv step, the definition in 64 bits, and a check that takes no other
integer or scale but where 64-bit sums decide."""
import torch

from oracle import oracle as orc
from tests import paged_ref as ref
from tests import q8_ref as q8

U64 = 2.0 ** -53
EPS = float(torch.tensor(1e-6, dtype=torch.float32))  # (as the call takes it)

# hd, kv heads, rows, rotated dims, NeoX pairs, position axes, norm.  About 2 million values each: of so
# many, f32's roundings of a norm or a turn put some beyond a border.
FORMS = {
    "64_neox": (64, 8, 4096, 64, True, 1, True),
    "128_neox_axes": (128, 4, 4096, 128, True, 3, True),
    "256_neox": (256, 2, 4096, 256, True, 1, True),
    "128_neighbours": (128, 4, 4096, 128, False, 1, True),
    "64_neighbours_no_norm": (64, 8, 4096, 64, False, 3, False),
    "128_part": (128, 4, 4096, 32, True, 1, True),
    "64_not_of_8": (64, 8, 4096, 36, True, 1, True),
    "128_not_of_8_neighbours": (128, 4, 4096, 100, False, 1, True),
    "256_not_of_8": (256, 2, 4096, 148, True, 2, True),
    "128_norm_only": (128, 4, 4096, 0, True, 1, True),
    "128_turn_only": (128, 4, 4096, 128, True, 1, False),
}


def inputs(form, seed=0, far=3000):
    """k, v [rows, n_kv, hd], the norm's weights, the rotary table, positions, each pair's axis."""
    hd, n_kv, T, rot, neox, axes, norm = FORMS[form]
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(T, n_kv, hd, generator=g) for _ in "kv")
    w = torch.rand(hd, generator=g) + 0.5 if norm else None
    table = torch.from_numpy(orc.rope_table(far, rot)) if rot else None
    pos = torch.randint(0, far, (axes, T), generator=g).to(torch.int32)
    return k, v, w, table, pos, [j % axes for j in range(rot // 2)]


def turned(form, k, w, table, pos, pair):
    """k normed and turned, in its own precision, and the magnitudes that the turn's terms have."""
    hd, n_kv, T, rot, neox, axes, norm = FORMS[form]
    y = k
    if norm:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.to(y.dtype)
    mag = y.abs()
    if rot:
        lo, hi = (slice(0, rot // 2), slice(rot // 2, rot)) if neox else (slice(0, rot, 2), slice(1, rot, 2))
        both = mag[..., lo] + mag[..., hi]
        mag[..., lo] = both
        mag[..., hi] = both
        cs = table[pos.long()[torch.tensor(pair)].T, torch.arange(rot // 2)].to(y.dtype)[:, None]  # [T, 1, rot/2, 2]
        a, b = y[..., lo], y[..., hi]
        z = y.clone()
        z[..., lo] = a * cs[..., 0] - b * cs[..., 1]
        z[..., hi] = b * cs[..., 0] + a * cs[..., 1]
        y = z
    return y, mag


def check(n, s, y, off):
    """Integers n and scales s (CPU) against those of y [..., hd] in f64, which is known to ``off``: the same, but for
    groups whose scale, and integers that, lie so near a border.  Returns how many of either were let pass."""
    want_n, want_s = q8.quantise(y)
    group = lambda t: t.unflatten(-1, (-1, 32))  # noqa: E731
    top, slack = group(y.abs()).amax(-1), group(off).amax(-1)
    ws = want_s.double()
    below = (want_s.view(torch.int16) - 1).clamp(min=0).view(torch.float16).double()
    near = ((127 * ws - top).abs() <= slack) | ((127 * below - top).abs() <= slack)
    near &= slack > 0
    assert ((s == want_s) | near).all(), f"{(~((s == want_s) | near)).sum()} scales are another one"
    # (of a group with the other scale the integers are the other one's)
    at = group(y) / torch.where(s > 0, s, 1.0).double()[..., None]
    border = (at - at.floor() - 0.5).abs()
    # (the quotient's own rounding: 2^-53 of at most 127)
    close = (border <= group(off) / torch.where(s > 0, s, 1.0).double()[..., None] + 128 * U64) & (group(off) > 0)
    right = group(n.double()) == at.round()
    assert (right | close).all(), f"{(~(right | close)).sum()} integers are another one"
    return int(near.sum() + close.sum())


def slack(form, mag):
    """How far two 64-bit computations of the same row may be apart: a sum of hd squares (half of it in the root), the
    root, three products and the turn's two, in each."""
    return mag * (FORMS[form][0] + 16) * U64 * (1.0 if FORMS[form][6] or FORMS[form][3] else 0.0)


def ties(seed=0):
    """Rows [n, 128] of f32 values on, and one f32 step beside, the borders between integers, whose groups' scales are
    known: every integer, f16 scales of every size."""
    g = torch.Generator().manual_seed(seed)
    s = torch.cat((torch.tensor([1, 2, 3, 1023, 1024, 1025, 0x7BFF, 0x3C00], dtype=torch.int16),
                   torch.randint(1, 0x7C00, (248,), generator=g).to(torch.int16))).view(torch.float16)
    half = torch.arange(-126, 126) + 0.5  # (252 borders, a group holds 31 beside its largest)
    x = []
    for v in s.tolist():
        at = half[torch.randint(0, 252, (4, 31), generator=g)] * v
        rows = torch.cat((torch.full((4, 1), 127.0 * v), at), 1).float()
        step = torch.randint(-1, 2, (4, 32), generator=g)
        step[:, 0] = 0
        rows = torch.where(rows == 0, rows, (rows.view(torch.int32) + step.int()).view(torch.float32))
        x.append(rows.flatten())
    return torch.stack(x), s
