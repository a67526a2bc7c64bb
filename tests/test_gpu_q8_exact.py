"""8-bit rows integer by integer: k in 64 bits through its norm and turn, v and
plain k exactly, by the definition."""
import pytest
import torch

from pelica_amd import paged
from tests import q8_exact as ex
from tests import q8_ref as q8
from tests import test_gpu_q8 as q8_tests

pytestmark = pytest.mark.gpu


def _rows(pool, slots):
    return pool.cpu().reshape(-1, *pool.shape[2:])[slots]


@pytest.mark.parametrize("form", ex.FORMS)
def test_keys_are_in_64_bits_and_values_exact(form):
    hd, n_kv, T, rot, neox, axes, norm = ex.FORMS[form]
    k, v, w, table, pos, pair = ex.inputs(form)
    page, n_head = 16, 2 * n_kv
    slots = torch.randperm(T + 3 * page, generator=torch.Generator().manual_seed(1))[:T]
    pools = paged.new_q8_pages(T // page + 3, page, n_kv, hd)
    paged.paged_qkv(torch.zeros(T, n_head, hd, device="cuda"), k.cuda(), v.cuda(), *pools[:2], slots.cuda(), k_scales=pools[2],
                    v_scales=pools[3], positions=pos.cuda() if rot else None, table=table.cuda() if rot else None, neox=neox,
                    pair_axis=pair if rot else None, q_norm=w.cuda() if norm else None, k_norm=w.cuda() if norm else None)
    torch.cuda.synchronize()
    y, mag = ex.turned(form, k.double(), w, table, pos, pair)
    assert ex.check(_rows(pools[0], slots), _rows(pools[2], slots), y, ex.slack(form, mag)) <= 2
    assert ex.check(_rows(pools[1], slots), _rows(pools[3], slots), v.double(), torch.zeros_like(v).double()) == 0


@pytest.mark.parametrize("n_kv,hd", [(2, 64), (1, 128), (1, 256)])
@pytest.mark.parametrize("T", [1, 7, 4000])
def test_borders_between_integers(T, n_kv, hd):
    """Of k without norm or turn and of v: ties to the even integer, one f32 step beside a border to its own side; every
    rotation of the rows so that a value meets every lane."""
    x, _ = ex.ties(seed=T + hd)
    x = torch.cat([x.roll(i, -1).flatten() for i in (0, 32, 64, 96)]).view(-1, n_kv, hd)
    x = x[torch.arange(T) % len(x)]
    kv = x, x.flip(0)
    pools = paged.new_q8_pages(-(-T // 8), 8, n_kv, hd)
    slots = torch.randperm(T, generator=torch.Generator().manual_seed(T))
    paged.paged_qkv(torch.zeros(T, n_kv, hd, device="cuda"), kv[0].cuda(), kv[1].cuda(), *pools[:2], slots.cuda(), k_scales=pools[2],
                    v_scales=pools[3])
    torch.cuda.synchronize()
    for i, y in enumerate(kv):
        assert ex.check(_rows(pools[i], slots), _rows(pools[2 + i], slots), y.double(), torch.zeros_like(y).double()) == 0


def test_two_level_table():
    """(cos, sin) of a two-level table are its two rows' f32 product, for k as for q: off by three roundings of 2^-24 of
    numbers up to 1 each, and k by that."""
    T, n_kv, hd, split = 2000, 4, 128, 12
    g = torch.Generator().manual_seed(5)
    ang = lambda at: at.double()[:, None] * 10000.0 ** (-torch.arange(hd // 2).double() / (hd // 2))  # noqa: E731
    rows = torch.cat((torch.arange(split) * 256, torch.arange(256)))
    table = torch.stack((ang(rows).cos(), ang(rows).sin()), -1).float()
    k, v = (torch.randn(T, n_kv, hd, generator=g) for _ in "kv")
    pos = torch.randint(0, 256 * split, (T,), generator=g)
    pools = paged.new_q8_pages(T // 16, 16, n_kv, hd)
    slots = torch.arange(T)
    paged.paged_qkv(torch.zeros(T, n_kv, hd, device="cuda"), k.cuda(), v.cuda(), *pools[:2], slots.cuda(), k_scales=pools[2],
                    v_scales=pools[3], positions=pos.int().cuda(), table=table.cuda(), table_split=split)
    torch.cuda.synchronize()
    far, near = table.double()[pos // 256], table.double()[split + pos % 256]
    c = (far[..., 0] * near[..., 0] - far[..., 1] * near[..., 1])[:, None]
    s = (far[..., 1] * near[..., 0] + far[..., 0] * near[..., 1])[:, None]
    a, b = k.double().chunk(2, -1)
    y = torch.cat((a * c - b * s, b * c + a * s), -1)
    mag = torch.cat((a.abs() + b.abs(),) * 2, -1)
    # (within half a scale and 3 roundings: the check of rows that are known to f32 roundings)
    q8_tests._check_rows(_rows(pools[0], slots), _rows(pools[2], slots), y, mag * 3 / 16, exact=False)


def test_replays_write_the_integers_of_new_rows():
    """A captured write and read of plain rows: every replay gives the definition's integers."""
    T, n_head, n_kv, hd, page = 40, 8, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(2)
    x = [torch.randn(T, h, hd, generator=g, device="cuda") for h in (n_head, n_kv, n_kv)]
    pools = paged.new_q8_pages(5, page, n_kv, hd)
    scales = dict(k_scales=pools[2], v_scales=pools[3])
    slots = torch.arange(T, device="cuda") + 7
    out = torch.zeros(T, n_head, hd, device="cuda")
    rows = [torch.zeros(T, n_kv, hd, dtype=torch.float16, device="cuda") for _ in "kv"]

    def both():
        paged.paged_qkv(*x, *pools[:2], slots, **scales, out=out)
        paged.pages_read(*pools[:2], slots, **scales, out=rows)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for i in range(4):
        for t in x:
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        # (a factor prime to the pool's 80 rows: no slot twice)
        slots.copy_((torch.arange(T, device="cuda") * (1, 3, 7, 9)[i]) % 80)
        graph.replay()
        torch.cuda.synchronize()
        for j in range(2):
            y, at = x[1 + j].cpu().double(), slots.cpu()
            assert ex.check(_rows(pools[j], at), _rows(pools[2 + j], at), y, torch.zeros_like(y)) == 0
            assert torch.equal(rows[j].cpu(), q8.values(*q8.quantise(y)))
        assert torch.equal(out, x[0])
