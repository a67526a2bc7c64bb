"""pages_read into rows beside its other arrays: every place that is not refused."""
import pytest
import torch

from pelica_amd import attn, paged
from tests import q8_ref as q8

pytestmark = pytest.mark.gpu
N_KV, HD, PAGE, T = 2, 64, 16, 40


def _pools(n_pages, g):
    k, v, ks, vs = paged.new_q8_pages(n_pages, PAGE, N_KV, HD)
    for t in (k, v):
        t.copy_(torch.randint(-127, 128, t.shape, generator=g).to(torch.int8))
    for t in (ks, vs):
        t.copy_(torch.rand(t.shape, generator=g).half())
    return k, v, ks, vs


def _want(n, s, slots):
    return q8.values(n.cpu().reshape(-1, N_KV, HD), s.cpu().reshape(-1, N_KV, HD // 32))[slots.cpu()]


def test_rows_that_take_turns_and_rows_side_by_side():
    g = torch.Generator().manual_seed(1)
    k, v, ks, vs = _pools(5, g)
    slots = torch.randperm(5 * PAGE, generator=g)[:T].cuda()
    for shape, pick in (((T, 2, N_KV, HD), lambda b: (b[:, 0], b[:, 1])), ((2, T, N_KV, HD), lambda b: (b[0], b[1])),
                        ((T, 3, N_KV, HD), lambda b: (b[:, 2], b[:, 0])), ((2, T, N_KV, HD), lambda b: (b[1], b[0]))):
        buf = torch.full(shape, 7.0, dtype=torch.float16, device="cuda")
        out = pick(buf)
        paged.pages_read(k, v, slots, k_scales=ks, v_scales=vs, out=out)
        torch.cuda.synchronize()
        assert torch.equal(out[0].cpu(), _want(k, ks, slots)) and torch.equal(out[1].cpu(), _want(v, vs, slots))
        if shape[1] == 3:
            assert (buf[:, 1] == 7.0).all()


def test_rows_between_two_pages_and_around_the_pool():
    """One buffer of f16 pages, each with room for T rows behind it: K's rows ahead of the pool, behind it, in a page's room."""
    g = torch.Generator().manual_seed(2)
    n, rows = 4, PAGE * N_KV * HD
    room = T * N_KV * HD
    buf = torch.full((room + n * (rows + room),), 7.0, dtype=torch.float16, device="cuda")
    k = buf[room:].view(n, rows + room)[:, :rows].view(n, PAGE, N_KV, HD)
    k.copy_(torch.randn(k.shape, generator=g))
    v = torch.zeros_like(buf)[room:].view(n, rows + room)[:, :rows].view(n, PAGE, N_KV, HD)
    v.copy_(torch.randn(v.shape, generator=g))
    slots = torch.randperm(n * PAGE, generator=g)[:T].cuda()
    want = k.reshape(-1, N_KV, HD)[slots].clone()
    vo = torch.zeros(T, N_KV, HD, dtype=torch.float16, device="cuda")
    for at in (0, room + rows, room + 2 * (rows + room) + rows, buf.numel() - room):
        out = buf[at:at + room].view(T, N_KV, HD)
        out.fill_(7.0)
        paged.pages_read(k, v, slots, out=(out, vo))
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(vo, v.reshape(-1, N_KV, HD)[slots])
        out.fill_(7.0)
    assert (buf[:room] == 7.0).all() and torch.equal(k.reshape(-1, N_KV, HD)[slots], want)
    with pytest.raises(attn.AttnError) as e:
        paged.pages_read(k, v, slots, out=(buf[room + rows - 8:2 * room + rows - 8].view(T, N_KV, HD), vo))
    assert e.value.code == attn.EINVAL
