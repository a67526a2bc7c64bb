"""The step before attention over pages against its 64-bit definition, and a run
of all the operators of a step together."""
import math

import pytest
import torch

from oracle import oracle as orc
from pelica_amd import attn, paged
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

U32, U16 = ref.U32, ref.U16


def _close(got, want, mag, u):
    """``mag``: the magnitude the roundings are relative to (a rotation adds two products)."""
    off = (got.cpu().double() - want).abs()
    tol = mag * (u + 16 * U32) + (2.0 ** -25 if u == U16 else 0)
    assert (off <= tol).all(), f"off by {(off / tol.clamp(min=1e-300)).max():.3g} of what roundings allow"


def _run(T, n_head, n_kv, hd, *, axes=1, rot=None, neox=True, split=False, norm=False, half=False, page=16, pair=None,
         fused=False, in_place=False, seed=0, far=3000, skip=(), layout="nhd"):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    rot = hd if rot is None else rot
    n_pages = -(-T // page) + 3
    tab = pos = table_ref = None
    n_split = 0
    if rot:
        table_ref = torch.from_numpy(orc.rope_table(far, rot))
        if split:
            two, n_split = orc.rope_table(far, rot, split=True)
            tab = torch.from_numpy(two).cuda()
        else:
            tab = table_ref.cuda()
        pos = torch.randint(0, far, (axes, T), generator=g).to(torch.int32)
        pos[:, 0] = far - 1
    pair = pair or [j % axes for j in range(rot // 2)]
    q, k, v = rnd(T, n_head, hd), rnd(T, n_kv, hd), rnd(T, n_kv, hd)
    qn, kn = (torch.rand(hd, generator=g) + 0.5, torch.rand(hd, generator=g) + 0.5) if norm else (None, None)
    slots = torch.randperm(n_pages * page, generator=g)[:T]
    for i, s in skip:
        slots[i] = s
    if fused:
        buf = torch.cat([q.reshape(T, -1), k.reshape(T, -1), v.reshape(T, -1), torch.zeros(T, 4)], 1).cuda()
        a, b, c = n_head * hd, (n_head + n_kv) * hd, (n_head + 2 * n_kv) * hd
        dq, dk, dv = buf[:, :a].view(T, n_head, hd), buf[:, a:b].view(T, n_kv, hd), buf[:, b:c].view(T, n_kv, hd)
    else:
        dq, dk, dv = q.cuda(), k.cuda(), v.cuda()
    shape = (n_pages, page, n_kv, hd)
    if layout == "hnd":
        kp, vp = (torch.full((n_pages, n_kv, page, hd), 9.0, dtype=torch.float16, device="cuda").transpose(1, 2) for _ in "kv")
    else:
        kp, vp = (torch.full(shape, 9.0, dtype=torch.float16, device="cuda") for _ in "kv")
    out = dq if in_place else torch.full((T, n_head, hd), 9.0, dtype=torch.float16 if half else torch.float32, device="cuda")
    paged.paged_qkv(dq, dk, dv, kp, vp, slots.cuda(), positions=None if pos is None else pos.cuda(), table=tab, rot=rot,
                    neox=neox, table_split=n_split, pair_axis=pair if rot else None,
                    q_norm=None if qn is None else qn.cuda(), k_norm=None if kn is None else kn.cuda(), out=out)
    torch.cuda.synchronize()
    live = (slots >= 0) & (slots < n_pages * page)
    x = [t.double() for t in (q, k)]
    if norm:
        x = [ref.norm(t, w, 1e-6) for t, w in zip(x, (qn, kn))]
    mags = [t.abs().clone() for t in x]
    if rot:
        half_ = rot // 2
        for m, t in zip(mags, x):  # a turned value is as large as its pair
            lo, hi = (slice(0, half_), slice(half_, rot)) if neox else (slice(0, rot, 2), slice(1, rot, 2))
            s = t[..., lo].abs() + t[..., hi].abs()
            m[..., lo] = s
            m[..., hi] = s
        x = [ref.rope(t, table_ref, pos, pair, rot, neox) for t in x]
    # (the two-level table composes two rows: their f32 roundings)
    more = 8 if split else 1
    _close(out[live.cuda()], x[0][live], mags[0][live] * more, U16 if half else U32)
    if not in_place:
        assert (out.cpu()[~live] == 9.0).all()
    for pool, want, mag in ((kp, x[1], mags[1]), (vp, v.double(), v.double().abs())):
        flat = pool.cpu().reshape(-1, n_kv, hd)
        _close(flat[slots[live]], want[live], mag[live] * more, U16)
        others = torch.ones(flat.shape[0], dtype=torch.bool)
        others[slots[live]] = False
        assert (flat[others] == 9.0).all()


@pytest.mark.parametrize("T", [1, 2, 33, 700])
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 64, 8), (128, 32, 4), (256, 3, 1), (64, 5, 5)])
def test_rows(T, hd, n_head, n_kv):
    _run(T, n_head, n_kv, hd, norm=True, seed=1)
    _run(T, n_head, n_kv, hd, axes=3, half=True, neox=False, seed=2)


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("rot", [0, 2, 6, 10, 20, 32, 64, 128])
def test_partial_rotation(rot, neox):
    _run(19, 4, 2, 128, rot=rot, neox=neox, axes=3 if rot else 1, norm=True, seed=3)


@pytest.mark.parametrize("axes", [1, 2, 3, 4])
@pytest.mark.parametrize("split", [False, True])
def test_axes_and_two_level_tables(axes, split):
    _run(50, 8, 2, 64, axes=axes, split=split, far=70000, seed=4)
    _run(50, 8, 2, 256, axes=axes, split=split, far=1000, seed=5, half=True)


def test_sections():
    assert paged.pair_axes((2, 1, 1)) == [0, 0, 1, 2]
    assert paged.pair_axes((4, 2, 2), interleaved=True) == [0, 1, 2, 0, 1, 2, 0, 0]
    _run(40, 4, 1, 128, axes=3, pair=paged.pair_axes((16, 24, 24)), seed=6)
    _run(40, 4, 1, 128, axes=3, pair=paged.pair_axes((24, 20, 20), interleaved=True), seed=7)


def test_skipped_rows_layouts_and_rows_in_place():
    skip = ((3, -1), (7, -2 ** 62), (11, (-(-30 // 16) + 3) * 16), (12, 2 ** 62))
    _run(30, 8, 2, 64, skip=skip, seed=8)
    _run(30, 8, 2, 64, skip=skip, half=True, fused=True, layout="hnd", seed=9)
    _run(30, 8, 2, 128, norm=True, in_place=True, fused=True, seed=10)
    _run(30, 8, 2, 128, page=8, in_place=True, rot=0, norm=True, seed=11)


def test_a_position_outside_the_table_gives_nan():
    T, hd = 4, 64
    x = torch.randn(T, 3, hd, device="cuda")
    tab = torch.from_numpy(orc.rope_table(100, hd)).cuda()
    pos = torch.tensor([[5, -1, 100, 2 ** 31 - 1]], dtype=torch.int32, device="cuda")
    kp = torch.zeros(2, 8, 1, hd, dtype=torch.float16, device="cuda")
    vp = kp.clone()
    slots = torch.arange(T, device="cuda")
    out = paged.paged_qkv(x[:, :1].contiguous(), x[:, 1:2].contiguous(), x[:, 2:].contiguous(), kp, vp, slots,
                          positions=pos, table=tab)
    assert out[0].isfinite().all() and out[1:].isnan().all()
    assert kp[0, 0].isfinite().all() and kp[0, 1:4].isnan().all() and vp.isfinite().all()


@pytest.mark.parametrize("half", [False, True])
def test_steps_of_an_engine(half):
    """Requests that come, are read in chunks, answer token by token and end,
    through pages, rope + rows and attention of two layers (window and full),
    against attention over each request's own tokens kept apart."""
    n_seq, page, n_pages, most, hd, n_head, n_kv, rows = 5, 16, 80, 20, 64, 8, 2, 160
    g = torch.Generator(device="cuda").manual_seed(20)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    tab = torch.full((n_seq, most), -1, dtype=torch.int32, device="cuda")
    lst = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    state = torch.tensor([0, n_pages], device="cuda")
    mid = torch.zeros_like(state)
    steps = [paged.PageStep(n_seq, rows), paged.PageStep(n_seq, rows)]
    rope = torch.from_numpy(orc.rope_table(most * page, hd)).cuda()
    kp = torch.full((2, n_pages, page, n_kv, hd), math.nan, dtype=torch.float16, device="cuda")
    vp = kp.clone()
    sinks = torch.randn(n_head, generator=g, device="cuda")
    plans = [[paged.PagedPlan(s.q_start, s.seq_kv_len, tab, n_head=n_head, n_kv=n_kv, hd=hd, page_size=page,
                              n_pages=n_pages, n_tokens=rows, max_q=rows, window=w) for w in (32, 0)] for s in steps]
    ws = [p.new_workspace() for p in plans[0]]
    cached = [0] * n_seq
    kept = [[[] for _ in range(n_seq)] for _ in range(2)]  # (k, v) rows of every request, by layer
    script = [[100, 7, 0, 0, 1], [60, 1, 30, 0, 1], [1, 1, 1, 90, 1], [1, 1, 1, 1, 1], [1, -1, 1, 20, 0], [2, 45, 3, 1, 1],
              [1, 1, 1, 1, 1]]
    for i, new in enumerate(script):
        ended = [int(n < 0) for n in new]
        new = [max(n, 0) for n in new]
        paged.pages_release(i32(ended), i32(cached), tab, lst, state, page_size=page, free_out=mid)
        for s in range(n_seq):
            if ended[s]:
                cached[s] = 0
                for layer in kept:
                    layer[s] = []
        step = paged.pages_append(i32(cached), i32(new), tab, lst, mid, page_size=page, step=steps[i % 2])
        state = step.free_state
        total = [c + n for c, n in zip(cached, new)]
        for layer in range(2):
            plan = plans[i % 2][layer].update()
            x = torch.randn(rows, (n_head + 2 * n_kv) * hd, generator=g, device="cuda")
            q, k, v = (t.view(rows, -1, hd) for t in x.split((n_head * hd, n_kv * hd, n_kv * hd), 1))
            qo = torch.zeros(rows, n_head, hd, dtype=torch.float16 if half else torch.float32, device="cuda")
            paged.paged_qkv(q, k, v, kp[layer], vp[layer], step.slots, positions=step.positions, table=rope, out=qo)
            out = paged.paged_attention(qo, kp[layer], vp[layer], plan, sinks=sinks, workspace=ws[layer])
            torch.cuda.synchronize()
            # the rows the step wrote, kept in order: one page a request
            at = 0
            kk = ref.rope(k.cpu().double(), rope.cpu(), step.positions.cpu()[None], [0] * (hd // 2), hd, True)
            slots = step.slots.cpu()[:sum(new)]
            got_k, got_v = (t[layer].reshape(-1, n_kv, hd)[slots.cuda()].cpu() for t in (kp, vp))
            mag = k.cpu().double()[:sum(new)].abs()
            mag = (mag + mag.roll(hd // 2, -1))
            _close(got_k, kk[:sum(new)], mag, U16)
            assert torch.equal(got_v, v.cpu()[:sum(new)].half())
            for s, n in enumerate(new):
                kept[layer][s] += [(got_k[at + t], got_v[at + t]) for t in range(n)]
                at += n
            big = max(total)
            pool = torch.zeros(2, n_seq, big, n_kv, hd, dtype=torch.float16)
            for s in range(n_seq):
                for j, (a, b) in enumerate(kept[layer][s]):
                    pool[0, s, j], pool[1, s, j] = a, b
            want, f32, f16 = ref.attention(qo.cpu(), pool[0], pool[1], [[s] for s in range(n_seq)], total, new, page=big,
                                           window=32 if layer == 0 else 0, sinks=sinks.cpu())
            ref.check(out, want, f32, f16 if half else None)
        cached = total


def test_refusals_of_the_binding():
    """What the checks of q, k, v, slots, norms, tables and positions refuse,
    before anything is launched."""
    T, H, hd = 3, 2, 64
    dev = dict(device="cuda")
    x = torch.zeros(T, 4 * H * hd, **dev)
    q, k, v = (x[:, i * H * hd:(i + 1) * H * hd].view(T, H, hd) for i in range(3))
    pages = torch.zeros(4, 16, H, hd, dtype=torch.float16, **dev)
    slots = torch.arange(T, **dev)
    table = torch.zeros(8, hd // 2, 2, **dev)
    pos = torch.zeros(T, dtype=torch.int32, **dev)
    good = dict(q=q, k=k, v=v, k_pages=pages, v_pages=pages, slots=slots, positions=pos, table=table)
    paged.paged_qkv(**good)
    bad = [
        dict(q=q.half()), dict(k=k.cpu()), dict(v=v[:2]), dict(v=v[:, :1]), dict(q=q[..., :32]),
        dict(q=q.contiguous()), dict(k=k.contiguous()), dict(v=v.contiguous()),
        dict(q=q.transpose(0, 1).contiguous().transpose(0, 1)), dict(q=torch.zeros(T, H, 2 * hd, **dev)[..., ::2]),
        dict(q=q[0]), dict(k_pages=pages.float()), dict(v_pages=pages[:2]), dict(k_pages=pages[:, :, :1]),
        dict(k_pages=pages.transpose(1, 2)), dict(slots=slots.int()), dict(slots=slots[:2]), dict(slots=slots.cpu()),
        dict(slots=torch.zeros(T, 1, dtype=torch.int64, **dev)), dict(q_norm=torch.ones(hd + 1, **dev)),
        dict(k_norm=torch.ones(hd, 1, **dev)), dict(q_norm=torch.ones(hd)), dict(table=table.half()),
        dict(table=table[:, :4, :1]), dict(table=table, rot=32), dict(table=table[0]), dict(positions=None),
        dict(positions=pos.long()), dict(positions=pos[:2]), dict(positions=torch.zeros(2, T, dtype=torch.int32, **dev)),
        dict(positions=torch.zeros(1, 1, T, dtype=torch.int32, **dev)), dict(pair_axis=[0] * 5), dict(pair_axis=[1] * (hd // 2)),
        dict(out=torch.zeros(T, H, 32, **dev)), dict(out=torch.zeros(T, H, hd, dtype=torch.bfloat16, **dev)),
        dict(out=torch.zeros(T, H, hd)),
    ]
    for kw in bad:
        with pytest.raises(attn.AttnError):
            paged.paged_qkv(**{**good, **kw})
