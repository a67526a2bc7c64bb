"""Rows quantised into 8-bit pages as they are written, and rows read back,
against the format's 64-bit definition."""
import math

import pytest
import torch

from oracle import oracle as orc
from pelica_amd import attn, paged
from tests import paged_ref as ref
from tests import q8_ref as q8

pytestmark = pytest.mark.gpu

U32 = ref.U32


def _pools(n_pages, page, n_kv, hd, layout):
    """Pages and scales of 8 bits, filled with what no test writes."""
    g = hd // 32
    make = lambda n, dt, fill: torch.full((n_pages, page, n_kv, n), fill, dtype=dt, device="cuda")  # noqa: E731
    if layout == "hnd":
        k, v, ks, vs = paged.new_q8_pages(n_pages, page, n_kv, hd)
        for t, fill in ((k, 99), (v, 99), (ks, 9.0), (vs, 9.0)):
            t.fill_(fill)
        return k, v, ks, vs
    if layout == "wide":  # rows of wider buffers
        wide = lambda n, dt, fill, more: torch.full((n_pages, page + 8, n_kv + 1, n + more), fill, dtype=dt,  # noqa: E731
                                                    device="cuda")[:, :page, :n_kv, :n]
        return wide(hd, torch.int8, 99, 16), wide(hd, torch.int8, 99, 16), wide(g, torch.float16, 9.0, 1), wide(g, torch.float16, 9.0, 1)
    if layout == "kv":  # K and V side by side, one buffer
        a = torch.full((n_pages, 2, page, n_kv, hd), 99, dtype=torch.int8, device="cuda")
        b = torch.full((n_pages, 2, page, n_kv, g), 9.0, dtype=torch.float16, device="cuda")
        return a[:, 0], a[:, 1], b[:, 0], b[:, 1]
    return make(hd, torch.int8, 99), make(hd, torch.int8, 99), make(g, torch.float16, 9.0), make(g, torch.float16, 9.0)


def _check_rows(n, s, x, mag, exact):
    """Rows n, s (on the CPU) of x [rows, n_kv, hd] f64, whose f32 result may be off by ``mag`` roundings of 2^-24."""
    off = mag * U32 * (0 if exact else 16)
    want = q8.scales(x)
    group = lambda t: t.unflatten(-1, (-1, 32))  # noqa: E731
    top, slack = group(x.abs()).amax(-1), group(off).amax(-1)
    sd = s.double()
    if exact:
        assert torch.equal(sd, want)
    # the smallest s with 127 s >= top, of a top that is as far off as the roundings allow
    assert (127 * sd >= top - slack).all()
    below = (s.view(torch.int16) - 1).clamp(min=0).view(torch.float16).double()
    assert ((127 * below <= top + slack) | (sd == 0)).all()
    y = group(n.double()) * sd[..., None]
    half = sd[..., None] * (0.5 + 2.0 ** -15)
    assert ((y - group(x)).abs() <= half + group(off)).all()
    assert n.abs().max() <= 127


def _write(T, n_head, n_kv, hd, *, axes=1, rot=None, neox=True, norm=False, half=False, page=16, seed=0, far=3000,
           skip=(), layout="hnd", in_place=False, x=None, graph=False, stream=None):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    rot = hd if rot is None else rot
    n_pages = -(-T // page) + 3
    tab = pos = None
    if rot:
        table = torch.from_numpy(orc.rope_table(far, rot))
        tab = table.cuda()
        pos = torch.randint(0, far, (axes, T), generator=g).to(torch.int32)
    pair = [j % axes for j in range(rot // 2)]
    q, k, v = rnd(T, n_head, hd), rnd(T, n_kv, hd), rnd(T, n_kv, hd)
    if x is not None:
        v = x
    qn, kn = (torch.rand(hd, generator=g) + 0.5, torch.rand(hd, generator=g) + 0.5) if norm else (None, None)
    slots = torch.randperm(n_pages * page, generator=g)[:T]
    for i, s in skip:
        slots[i] = s
    dq, dk, dv, ds = q.cuda(), k.cuda(), v.cuda(), slots.cuda()
    kp, vp, ks, vs = _pools(n_pages, page, n_kv, hd, layout)
    out = dq if in_place else torch.full((T, n_head, hd), 9.0, dtype=torch.float16 if half else torch.float32, device="cuda")
    args = dict(k_scales=ks, v_scales=vs, positions=None if pos is None else pos.cuda(), table=tab, rot=rot, neox=neox,
                pair_axis=pair if rot else None, q_norm=None if qn is None else qn.cuda(),
                k_norm=None if kn is None else kn.cuda())
    # q by the f16 path's call on the same rows: one formula
    k16, v16 = (torch.zeros(n_pages, page, n_kv, hd, dtype=torch.float16, device="cuda") for _ in "kv")
    plain = paged.paged_qkv(q.cuda(), dk, dv, k16, v16, ds, **{**args, "k_scales": None, "v_scales": None},
                            out=torch.full_like(out, 9.0))
    paged.paged_qkv(dq, dk, dv, kp, vp, ds, **args, out=out, stream=stream)
    torch.cuda.synchronize()
    live = (slots >= 0) & (slots < n_pages * page)
    assert torch.equal(out[live.cuda()], plain[live.cuda()])
    y = k.double()
    if norm:
        y = ref.norm(y, kn, 1e-6)
    mag = y.abs().clone()
    if rot:
        lo, hi = (slice(0, rot // 2), slice(rot // 2, rot)) if neox else (slice(0, rot, 2), slice(1, rot, 2))
        both = mag[..., lo] + mag[..., hi]
        mag[..., lo] = both
        mag[..., hi] = both
        y = ref.rope(y, table, pos, pair, rot, neox)
    at = slots[live]
    flat = lambda t: t.cpu().reshape(-1, *t.shape[2:])  # noqa: E731
    if x is None:
        _check_rows(flat(kp)[at], flat(ks)[at], y[live], mag[live], exact=not rot and not norm)
        _check_rows(flat(vp)[at], flat(vs)[at], v.double()[live], v.double().abs()[live], exact=True)
    others = torch.ones(n_pages * page, dtype=torch.bool)
    others[at] = False
    for t, fill in ((kp, 99), (vp, 99), (ks, 9.0), (vs, 9.0)):
        assert (flat(t)[others] == fill).all()
    # and back: bit for bit what the integers and scales stand for
    rows = [torch.full((T, n_kv, hd), 7.0, dtype=torch.float16, device="cuda") for _ in "kv"]
    paged.pages_read(kp, vp, ds, k_scales=ks, v_scales=vs, out=rows)
    torch.cuda.synchronize()
    for got, n, s in zip(rows, (kp, vp), (ks, vs)):
        want = q8.values(flat(n)[at], flat(s)[at])
        got = got.cpu()
        assert torch.equal(got[live].isnan(), want.isnan())
        assert torch.equal(got[live].nan_to_num(0), want.nan_to_num(0))
        assert (got[~live] == 7.0).all()
    return kp, vp, ks, vs, rows, slots


@pytest.mark.parametrize("T", [1, 2, 33, 700])
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 64, 8), (128, 32, 4), (256, 3, 1), (64, 5, 5), (128, 1, 1)])
def test_write(T, hd, n_head, n_kv):
    _write(T, n_head, n_kv, hd, norm=T % 2 == 1, half=T == 33, skip=[(T // 2, -1)] if T > 2 else (), seed=T)


@pytest.mark.parametrize("rot,neox", [(0, True), (128, False), (32, True), (32, False), (40, True), (6, True), (2, False)])
def test_write_partial_rope(rot, neox):
    _write(45, 6, 3, 128, rot=rot, neox=neox, norm=True, seed=rot)
    _write(45, 6, 2, 64, rot=min(rot, 64), neox=neox, seed=rot + 1)


@pytest.mark.parametrize("layout", ["hnd", "nhd", "wide", "kv"])
@pytest.mark.parametrize("page", [8, 16, 128])
def test_write_layouts(layout, page):
    _write(77, 8, 4, 64, page=page, layout=layout, axes=3, skip=[(3, -1), (10, 10 ** 9), (76, -5)])
    _write(77, 4, 2, 128, page=page, layout=layout, in_place=True)


def test_write_many_tokens():
    _write(4000, 32, 4, 128, axes=3, norm=True, half=True, page=64)


def test_write_on_another_stream():
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    _write(50, 8, 2, 64, stream=s)


def test_values_at_the_formats_ends():
    """Zeros, values that round to the smallest scale, the largest, infinities and NaN: a group is on its own."""
    T, n_kv, hd = 9, 2, 128
    x = torch.randn(T, n_kv, hd, generator=torch.Generator().manual_seed(1))
    x[0] = 0
    x[1] = -0.0
    x[2] *= 1e-9   # scales below 2^-24 / 2
    x[3] *= 1e-6   # subnormal scales
    x[4] = 0
    x[4, :, 5] = 1e-30
    x[5] = x[5].sign() * 65000
    x[6, 0, 40] = math.inf
    x[6, 1, 0] = -math.inf
    x[7, 0, 127] = math.nan
    x[8, 0, 3] = 3e38
    kp, vp, ks, vs, rows, slots = _write(T, 4, n_kv, hd, x=x, rot=0)
    got = rows[1].cpu()
    # what one group holds says nothing about the next
    bad = torch.zeros(T, n_kv, hd // 32, dtype=torch.bool)
    bad[6, 0, 1] = bad[6, 1, 0] = bad[7, 0, 3] = bad[8, 0, 0] = True
    bad = bad.repeat_interleave(32, -1)
    assert got[bad].isnan().all() and got[~bad].isfinite().all()
    s = q8.scales(x).repeat_interleave(32, -1)
    off = (got.double() - x.double()).abs()
    # half a scale, and f16's rounding of n s
    assert (off[~bad] <= (s * (0.5 + 2.0 ** -15) + 127 * s * 2.0 ** -11 + 2.0 ** -25)[~bad]).all()
    assert (got[0] == 0).all() and (got[1] == 0).all()
    assert (got[5].abs() >= 64900).all()


@pytest.mark.parametrize("hd,n_kv", [(64, 8), (128, 3), (256, 1)])
@pytest.mark.parametrize("layout", ["hnd", "nhd", "wide", "kv"])
def test_read_every_integer_and_scale(hd, n_kv, layout):
    """Rows of any bytes (-128 too) and scales, 8-bit and f16 pages, into rows of a wider buffer."""
    page, n_pages = 16, 7
    g = torch.Generator().manual_seed(hd)
    kp, vp, ks, vs = _pools(n_pages, page, n_kv, hd, layout)
    for t in (kp, vp):
        t.copy_(torch.randint(-128, 128, t.shape, generator=g).to(torch.int8))
    for t in (ks, vs):
        t.copy_(torch.randint(-2 ** 15, 2 ** 15, t.shape, generator=g).to(torch.int16).view(torch.float16))
    slots = torch.randint(-3, n_pages * page + 3, (301,), generator=g)
    slots[:2] = slots[2]  # the same row twice
    wide = torch.full((301, 2, n_kv * hd + 8), 7.0, dtype=torch.float16, device="cuda")
    out = [wide[:, i, :n_kv * hd].view(301, n_kv, hd) for i in range(2)]
    got = paged.pages_read(kp, vp, slots.cuda(), k_scales=ks, v_scales=vs, out=out)
    torch.cuda.synchronize()
    live = (slots >= 0) & (slots < n_pages * page)
    f16 = []
    for y, n, s in zip(got, (kp, vp), (ks, vs)):
        all_rows = q8.values(n.cpu().reshape(-1, n_kv, hd), s.cpu().reshape(-1, n_kv, hd // 32))
        want = all_rows[slots[live]]
        y = y.cpu()
        assert torch.equal(y[live].isnan(), want.isnan()) and torch.equal(y[live].nan_to_num(0), want.nan_to_num(0))
        assert (y[~live] == 7.0).all()
        f16.append(all_rows.view(n_pages, page, n_kv, hd).cuda())
    assert (wide[:, :, n_kv * hd:] == 7.0).all()
    k, v = paged.pages_read(f16[0], f16[1], slots.cuda())
    torch.cuda.synchronize()
    for a, b in zip((k, v), f16):
        assert torch.equal(a.cpu()[live].view(torch.int16), b.cpu().reshape(-1, n_kv, hd)[slots[live]].view(torch.int16))


def test_read_past_32_bits():
    """Pages whose last rows lie past 2^32 bytes and past 2^32 values."""
    page, n_kv, hd = 16, 2, 64
    stride = 1 << 28
    n = 18
    buf = torch.empty((n - 1) * stride + page * n_kv * hd, dtype=torch.int8, device="cuda")
    kp = buf.as_strided((n, page, n_kv, hd), (stride, n_kv * hd, hd, 1))
    sb = torch.empty((n - 1) * stride + page * n_kv * 2, dtype=torch.float16, device="cuda")
    ks = sb.as_strided((n, page, n_kv, 2), (stride, n_kv * 2, 2, 1))
    g = torch.Generator().manual_seed(3)
    last = torch.randint(-127, 128, (page, n_kv, hd), generator=g).to(torch.int8)
    sc = torch.rand(page, n_kv, 2, generator=g).half()
    kp[n - 1], ks[n - 1] = last.cuda(), sc.cuda()
    slots = torch.arange((n - 1) * page, n * page, device="cuda")
    k, v = paged.pages_read(kp, kp, slots, k_scales=ks, v_scales=ks)
    torch.cuda.synchronize()
    assert torch.equal(k.cpu(), q8.values(last, sc)) and torch.equal(v.cpu(), q8.values(last, sc))


def test_write_and_read_in_a_graph():
    T, n_head, n_kv, hd, page = 40, 8, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    x = [torch.randn(T, h, hd, generator=g, device="cuda") for h in (n_head, n_kv, n_kv)]
    pools = paged.new_q8_pages(5, page, n_kv, hd)
    slots = torch.arange(T, device="cuda") + 7
    out = torch.zeros(T, n_head, hd, device="cuda")
    rows = [torch.zeros(T, n_kv, hd, dtype=torch.float16, device="cuda") for _ in "kv"]

    def both():
        paged.paged_qkv(*x, *pools[:2], slots, k_scales=pools[2], v_scales=pools[3], out=out)
        paged.pages_read(*pools[:2], slots, k_scales=pools[2], v_scales=pools[3], out=rows)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for i in range(3):
        for t in x:
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        # (a factor prime to the pool's 80 rows: no slot twice)
        slots.copy_((torch.arange(T, device="cuda") * (1, 3, 7)[i]) % 80)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(rows, x[1:]):
            n, s = q8.quantise(want.cpu())
            y = q8.values(n, s).double()
            step = s.double().repeat_interleave(32, -1)
            # (an integer next to a border may be the other one)
            assert ((got.cpu().double() - y).abs() <= step * (1 + 2.0 ** -8)).all()
            assert (got.cpu().double() != y).float().mean() < 1e-2


@pytest.mark.parametrize("neox", [True, False])
def test_a_position_outside_the_table_gives_nan(neox):
    """k's groups that turn read as NaN, the others and the other rows as they are."""
    T, n_kv, hd, rot = 6, 2, 128, 64
    g = torch.Generator(device="cuda").manual_seed(5)
    x = [torch.randn(T, h, hd, generator=g, device="cuda") for h in (4, n_kv, n_kv)]
    pools = paged.new_q8_pages(2, 8, n_kv, hd)
    sc = dict(k_scales=pools[2], v_scales=pools[3])
    table = torch.from_numpy(orc.rope_table(100, rot)).cuda()
    pos = torch.tensor([0, 99, 100, -1, 5, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    slots = torch.arange(T, device="cuda")
    paged.paged_qkv(*x, *pools[:2], slots, **sc, positions=pos, table=table, neox=neox)
    k, v = paged.pages_read(*pools[:2], slots, **sc)
    torch.cuda.synchronize()
    bad = torch.tensor([False, False, True, True, False, True])
    assert k.cpu()[bad][..., :rot].isnan().all() and k.cpu()[bad][..., rot:].isfinite().all()
    assert k.cpu()[~bad].isfinite().all() and v.isfinite().all()


def test_refusals():
    k, v, ks, vs = paged.new_q8_pages(4, 16, 2, 64)
    slots = torch.arange(5, device="cuda")
    x = torch.zeros(5, 4, 64, device="cuda")
    kv = torch.zeros(5, 2, 64, device="cuda")
    bad = [dict(k_scales=None), dict(v_scales=None), dict(k_scales=None, v_scales=None), dict(k_scales=ks.float()),
           dict(k_scales=ks[:3]), dict(k_scales=ks[:3], v_scales=vs[:3]), dict(k_scales=ks[..., :1], v_scales=vs[..., :1]),
           dict(k_scales=ks.contiguous()), dict(k_scales=ks.cpu(), v_scales=vs.cpu()),
           dict(k_pages=k.half()), dict(k_pages=k.half(), v_pages=v.half())]
    for kw in bad:
        args = {**dict(k_pages=k, v_pages=v, k_scales=ks, v_scales=vs), **kw}
        with pytest.raises(attn.AttnError):
            paged.pages_read(slots=slots, **args)
        with pytest.raises(attn.AttnError):
            paged.paged_qkv(x, kv, kv, slots=slots, **args)
    good = dict(k_pages=k, v_pages=v, k_scales=ks, v_scales=vs)
    row = torch.zeros(5, 2, 64, dtype=torch.float16, device="cuda")
    for out in [(row, row[:4]), (row, row.float()), (row.cpu(), row), (row.expand(5, 2, 64)[:1].expand(5, 2, 64), row),
                (row, torch.zeros(5, 2, 128, dtype=torch.float16, device="cuda")[..., :64])]:
        with pytest.raises(attn.AttnError):
            paged.pages_read(**good, slots=slots, out=out)
    with pytest.raises(attn.AttnError):
        paged.pages_read(**good, slots=slots.int())
    with pytest.raises(attn.AttnError):
        paged.pages_read(**good, slots=slots[:0])
