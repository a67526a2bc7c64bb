"""The check of written 8-bit rows by planted mistakes: rows whose norm or turn was in f32, integers off by one."""
import pytest
import torch

from tests import q8_exact as ex
from tests import q8_ref as q8


@pytest.mark.parametrize("form", ex.FORMS)
def test_rows_in_f32_do_not_pass(form):
    k, v, w, table, pos, pair = ex.inputs(form)
    y, mag = ex.turned(form, k.double(), w, table, pos, pair)
    off = ex.slack(form, mag)
    n, s = q8.quantise(y)
    assert ex.check(n, s, y, off) <= 2
    f32, _ = ex.turned(form, k, w, table, pos, pair)
    with pytest.raises(AssertionError, match="another one"):
        ex.check(*q8.quantise(f32), y, off)


def test_one_integer_or_scale_off_does_not_pass():
    x, s = ex.ties()
    y = x.double()
    none = torch.zeros_like(y)
    n, got = q8.quantise(y)
    assert torch.equal(got, s[:, None].expand(-1, 4))
    assert ex.check(n, got, y, none) == 0
    for at in ((0, 5), (100, 127), (255, 33)):
        m = n.clone()
        m[at] += 1 if m[at] < 0 else -1
        with pytest.raises(AssertionError, match="1 integers"):
            ex.check(m, got, y, none)
    t = got.clone()
    t[3, 2] = (got[3, 2:3].view(torch.int16) + 1).view(torch.float16)[0]
    with pytest.raises(AssertionError, match="1 scales"):
        ex.check(n, t, y, none)
    # a border rounded away from zero instead of to the even integer
    away = torch.where(y < 0, -1, 1) * ((y.unflatten(-1, (-1, 32)) / got.double()[..., None]).abs() + 0.5).floor().flatten(-2)
    with pytest.raises(AssertionError, match="integers are another one"):
        ex.check(away.to(torch.int8), got, y, none)
