"""Attention of requests that share their first keys, walked once for a group,
against the 64-bit definition of every request by itself; f16 and 8-bit pages."""
import math

import pytest
import torch

from pelica_amd import attn, paged
from tests import paged_ref as ref
from tests import test_gpu_paged as f16_tests
from tests import test_gpu_paged_q8 as q8_tests

pytestmark = pytest.mark.gpu


def _case(base):
    class Case(base):
        """``groups``: (first request, behind the last, keys shared by the table, shared_len given)."""

        def __init__(self, lens, new, groups, **kw):
            super().__init__(lens, new, **kw)
            self.groups = groups
            for a, b, common, _ in groups:
                for s in range(a + 1, b):
                    n = min(common // self.page, len(self.table[s]))
                    self.table[s][:n] = self.table[a][:n]
            # pages that are no request's any more: nobody reads them
            used = {p for r in self.table for p in r}
            for p, i in self.live.items():
                if p not in used:
                    self.k[i] = self.v[i] = math.nan

        def device(self):
            super().device()
            i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
            starts, keys = [], []
            at = self.groups[0][0] if self.groups else 0
            for a, b, _, given in self.groups:
                if a > at:  # requests between two groups: one that shares nothing
                    starts.append(at)
                    keys.append(0)
                starts.append(a)
                keys.append(given)
                at = b
            self.group_start, self.shared_len = i32(starts + [at]), i32(keys)
            return self

        def plan(self, **kw):
            return super().plan(group_start=self.group_start, shared_len=self.shared_len, **kw)

    return Case


CASES = {"f16_pages": _case(f16_tests.Case), "8_bit_pages": _case(q8_tests.Case)}
f16_cases = pytest.mark.parametrize("pages", CASES)


# (lens, new, groups)
MIXES = {
    "two": ([100, 90], [1, 1], [(0, 2, 64, 64)]),
    "odd_shared": ([300, 170, 211], [1, 1, 1], [(0, 3, 160, 149)]),
    "longer_than_one_has": ([300, 97, 211], [1, 2, 1], [(0, 3, 160, 1000)]),
    "own_token_only": ([129, 129, 129], [1, 1, 1], [(0, 3, 128, 128)]),
    "drafts": ([200, 150, 333, 170], [4, 1, 3, 2], [(0, 4, 128, 128)]),
    "two_groups_and_more": ([400, 420, 70, 80, 33, 500, 90], [1, 2, 1, 1, 1, 1, 3], [(0, 2, 320, 320), (2, 4, 64, 64), (5, 6, 300, 300)]),
    "requests_ahead_and_behind": ([50, 200, 210, 60], [1, 1, 1, 1], [(1, 3, 192, 192)]),
    "a_gap": ([200, 210, 40, 300, 310], [1, 1, 1, 1, 1], [(0, 2, 96, 96), (3, 5, 256, 256)]),
    "empty_requests": ([200, 210, 0, 220, 30], [0, 1, 0, 1, 1], [(0, 4, 160, 160)]),
    "only_one_has_tokens": ([200, 210], [0, 1], [(0, 2, 160, 160)]),
    "nothing_shared": ([200, 210], [1, 1], [(0, 2, 0, 0)]),
    "below_a_chunk": ([200, 210], [1, 1], [(0, 2, 16, 31)]),
    "negative": ([200, 210], [1, 1], [(0, 2, 0, -5)]),
    "chunks": ([300, 250, 400], [70, 1, 130], [(0, 3, 160, 160)]),
    "a_prompt_that_has_all_but_its_tokens": ([96, 130, 97], [32, 60, 1], [(0, 3, 64, 64)]),
    "many": ([150 + 7 * i for i in range(40)], [1 + i % 3 for i in range(40)], [(0, 40, 144, 144)]),
}


@f16_cases
@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("mix", MIXES)
def test_groups(mix, hd, half, pages):
    lens, new, groups = MIXES[mix]
    CASES[pages](lens, new, groups, hd=hd, half=half, n_head=8, n_kv=2, seed=1).check()


@f16_cases
@pytest.mark.parametrize("n_head,n_kv", [(1, 1), (2, 1), (4, 4), (3, 1), (10, 2), (16, 1), (64, 8), (71, 1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_head_groups(n_head, n_kv, hd, pages):
    lens, new = [300, 170, 211, 290, 260], [1, 2, 1, 1, 3]
    CASES[pages](lens, new, [(0, 5, 160, 160)], n_head=n_head, n_kv=n_kv, hd=hd, half=hd == 64, sinks=True, seed=2).check()
    # all rows of a few requests in one narrow item
    CASES[pages](lens[:2], [1, 1], [(0, 2, 160, 160)], n_head=n_head, n_kv=n_kv, hd=hd, half=hd == 128, seed=3).check()


@f16_cases
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "wide", "kv"])
def test_pages_and_layouts(page, layout, pages):
    CASES[pages]([300, 270, 400], [1, 2, 1], [(0, 3, 256, 256)], page=page, layout=layout, hd=64, seed=4).check()
    CASES[pages]([300, 270, 400], [1, 60, 1], [(0, 3, 256, 200)], page=page, layout=layout, hd=128, half=True, seed=5).check()


@f16_cases
@pytest.mark.parametrize("cap", [0.0, 5.0, 50.0])
@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_scores(cap, sinks, hd, pages):
    for half in (False, True):
        CASES[pages]([300, 170, 211], [1, 3, 1], [(0, 3, 160, 160)], cap=cap, sinks=sinks, hd=hd, half=half, q_scale=6.0, seed=6).check()
        CASES[pages]([300, 190, 211], [100, 3, 1], [(0, 3, 160, 160)], cap=cap, sinks=sinks, hd=hd, half=half, seed=7).check()


@f16_cases
def test_scores_far_below_and_above(pages):
    # all weight on the shared keys, or on a request's own
    c = CASES[pages]([200, 190, 230], [1, 1, 1], [(0, 3, 160, 160)], q_scale=100.0, sinks=True, half=True, seed=8)
    c.check()
    CASES[pages]([200, 190, 230], [1, 1, 1], [(0, 3, 160, 160)], scale=1e-6, seed=9).check()


@f16_cases
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 64, 8), (128, 32, 4), (128, 16, 16), (64, 4, 1)])
def test_split_over_keys(hd, n_head, n_kv, pages):
    # long shared keys: cut into many ranges, and own keys cut as well
    kw = dict(hd=hd, n_head=n_head, n_kv=n_kv, sinks=True, page=64)
    CASES[pages]([5000, 4900, 4600], [1, 1, 2], [(0, 3, 4480, 4480)], seed=10, **kw).check()
    CASES[pages]([3000] * 20, [1] * 20, [(0, 20, 2944, 2944)], half=True, seed=11, **kw).check()
    CASES[pages]([400, 3000, 500, 410], [1, 1, 80, 1], [(0, 4, 320, 320)], half=True, seed=12, **kw).check()


def test_many_groups():
    # more items than one round of the planner's threads; groups' items among them
    lens, new, groups = [], [], []
    for g in range(500):
        n = 2 + g % 3
        groups.append((len(lens), len(lens) + n, 32, 32))
        lens += [40 + (g + i) % 9 for i in range(n)]
        new += [1] * n
    CASES["f16_pages"](lens, new, groups, n_head=2, n_kv=2, page=8, seed=13).check()
    lens = [100 + i % 50 for i in range(700)]
    CASES["f16_pages"](lens, [1 + i % 2 for i in range(700)], [(0, 700, 96, 96)], n_head=4, n_kv=1, hd=64, half=True, seed=14).check()


@f16_cases
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_random_mixes(hd, half, pages):
    g = torch.Generator().manual_seed(hd + half + len(pages))
    r = lambda a, b: int(torch.randint(a, b + 1, (1,), generator=g))  # noqa: E731
    for seed in range(8):
        page = (8, 16, 32, 64)[r(0, 3)]
        lens, new, groups = [], [], []
        for _ in range(r(1, 4)):
            n, common = r(1, 6), page * r(1, 20)
            first = len(lens)
            for _ in range(n):
                t = r(0, 3) if r(0, 5) else r(1, 60)
                lens.append(common + t + r(0, 150) if r(0, 9) else t + r(0, common))
                new.append(t)
            least = min(a - b for a, b in zip(lens[first:], new[first:]))
            groups.append((first, len(lens), min(common, least // page * page), r(0, common + 5) if r(0, 3) == 0 else min(common, least // page * page)))
            if groups[-1][3] > groups[-1][2]:  # (never more keys than the tables share)
                groups[-1] = (*groups[-1][:3], groups[-1][2])
        if sum(new) == 0:
            new[0], lens[0] = 1, max(lens[0], 1)
        hpk, n_kv = (1, 2, 3, 5, 8)[r(0, 4)], r(1, 3)
        CASES[pages](lens, new, groups, n_head=hpk * n_kv, n_kv=n_kv, hd=hd, half=half, page=page, sinks=r(0, 1) == 1, cap=(0.0, 30.0)[r(0, 1)],
                     layout=("hnd", "nhd", "wide", "kv")[r(0, 3)], pad=r(0, 3), seed=200 + seed).check()


def test_the_most_groups_and_empty_ones():
    n = 1100
    c = CASES["f16_pages"]([70] * n, [1] * n, [(0, n, 64, 64)], n_head=2, n_kv=1, page=16, seed=15).device()
    at = sorted([0, n] + [min(n, 5 * (i // 4)) for i in range(1023)])
    c.group_start = torch.tensor(at, dtype=torch.int32, device="cuda")
    c.shared_len = torch.full((1024,), 64, dtype=torch.int32, device="cuda")
    c.check(c.run())


def test_rows_behind_the_last_and_skipped_requests():
    # padding rows; a request of the group with fewer keys than tokens, one past its table's row
    c = CASES["f16_pages"]([200, 190, 180, 170], [1, 4, 2, 1], [(0, 4, 160, 160)], pad=6, seed=16).device()
    c.len[1] = 3
    c.len[2] = c.tab.shape[1] * c.page + 1
    out = c.run()
    want, f32, _ = ref.attention(c.q, c.k, c.v, [[c.live[p] for p in r] for r in c.table], [200, 3, 1, 170], [1, 4, 2, 1], page=16)
    ref.check(out, want, f32)
    assert (out[1:7] == 123.0).all() and (out[8:] == 123.0).all()


def test_rows_of_skipped_requests_may_hold_anything():
    c = CASES["f16_pages"]([200, 190, 180], [1, 1, 1], [(0, 3, 160, 160)], n_head=16, half=True, seed=17).device()
    c.len[1] = 0
    c.qd[1] = math.nan
    out = c.run()
    c.lens = [200, 0, 180]
    want, f32, f16 = ref.attention(c.q, c.k, c.v, [[c.live[p] for p in r] for r in c.table], c.lens, c.new, page=16)
    ref.check(out, want, f32, f16)
    assert (out[1] == 123.0).all()


def test_a_bad_page_of_the_shared_ones_is_the_groups():
    c = CASES["f16_pages"]([200, 190, 180], [1, 1, 1], [(0, 2, 160, 160)], seed=18).device()
    for bad in (-1, c.n_pages, 2 ** 31 - 1, -2 ** 31):
        c.tab[0, 2] = bad
        out = c.run()
        assert out[:2].isnan().all()
        want, f32, _ = c.reference()
        ref.check(out[2:], want[2:], f32[2:])


def test_first_requests_and_rows_that_decrease():
    c = CASES["f16_pages"]([200, 190, 180], [2, 40, 1], [(0, 3, 128, 128)], n_head=16, half=True, seed=19).device()
    good = c.group_start.clone()
    for start in ([1, 0], [0, 4], [-1, 3], [0, -3], [0, 2 ** 31 - 1]):
        c.group_start.copy_(torch.tensor(start, dtype=torch.int32))
        assert (c.run() == 123.0).all()
    c.group_start.copy_(good)
    rows = c.start.clone()
    c.start.copy_(torch.tensor([0, 42, 2, 43], dtype=torch.int32))
    assert (c.run() == 123.0).all()
    c.start.copy_(rows)
    c.check(c.run())


def test_plans_of_the_other_kind_write_nothing():
    c = CASES["f16_pages"]([2000, 1900], [1, 1], [(0, 2, 1600, 1600)], n_head=16, seed=20).device()
    shared = c.plan()
    plain = super(type(c), c).plan()
    for mine, desc in ((shared, plain), (plain, shared)):
        out = torch.full_like(c.qd, 123.0)
        call = paged.PagedPlan.__new__(paged.PagedPlan)
        call.__dict__.update(desc.__dict__)  # the other's descriptor and form, this one's list
        call._buffer, call._bytes, call.buffer = mine._buffer, max(mine._bytes, desc._bytes), mine.buffer
        if mine._bytes < desc._bytes:  # (room as the call needs it)
            call.buffer = torch.zeros(desc._bytes, dtype=torch.uint8, device="cuda")
            call.buffer[:mine._bytes] = mine.buffer
            call._buffer = call.buffer.data_ptr()
        paged.paged_attention(c.qd, c.kd, c.vd, call, out=out)
        assert (out == 123.0).all()


@f16_cases
def test_captured_steps_follow_new_lengths_and_groups(pages):
    a = CASES[pages]([2000, 1700, 1800, 90], [1, 1, 3, 1], [(0, 3, 1600, 1600)], n_head=16, n_kv=2, sinks=True, seed=21, pad=4).device()
    plan = a.plan()
    ws = plan.new_workspace()
    out = torch.full_like(a.qd, 123.0)
    kw = dict(sinks=a.dev(a.sinks), workspace=ws)
    if pages == "8_bit_pages":
        kw.update(k_scales=a.ks, v_scales=a.vs)
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        with torch.cuda.graph(graph, stream=st):
            plan.update()
            paged.paged_attention(a.qd, a.kd, a.vd, plan, out=out, **kw)
    torch.cuda.synchronize()
    for lens, new, keys in ((a.lens, a.new, 1600), ([1990, 1650, 0, 50], [2, 1, 0, 1], 1600), ([1700, 1603, 1700, 9], [3, 3, 1, 0], 777),
                            ([1700, 1603, 1700, 9], [1, 1, 1, 1], 0)):
        a.lens, a.new = lens, new
        start = [0]
        for t in new:
            start.append(start[-1] + t)
        a.start.copy_(torch.tensor(start, dtype=torch.int32))
        a.len.copy_(torch.tensor(lens, dtype=torch.int32))
        a.shared_len.fill_(keys)
        out.fill_(123.0)
        graph.replay()
        torch.cuda.synchronize()
        a.check(out)
        eager = torch.full_like(a.qd, 123.0)
        paged.paged_attention(a.qd, a.kd, a.vd, plan.update(), out=eager, **kw)
        assert torch.equal(eager, out)


def test_two_steps_at_once():
    runs = []
    for seed, pages in ((22, "f16_pages"), (23, "8_bit_pages")):
        c = CASES[pages]([3000, 2900, 2800, 500], [1, 1, 2, 1], [(0, 3, 2560, 2560)], n_head=16, n_kv=2, seed=seed).device()
        torch.cuda.synchronize()
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            plan = c.plan(stream=st)
            runs.append((c, st, plan, plan.new_workspace(), torch.full_like(c.qd, 123.0),
                         dict(k_scales=c.ks, v_scales=c.vs) if pages == "8_bit_pages" else {}))
    torch.cuda.synchronize()
    for _ in range(10):
        for c, st, plan, ws, out, kw in runs:
            plan.update(stream=st)
            paged.paged_attention(c.qd, c.kd, c.vd, plan, out=out, workspace=ws, stream=st, **kw)
    torch.cuda.synchronize()
    for c, _, _, _, out, _ in runs:
        c.check(out)


def test_token_rows_of_wider_buffers():
    c = CASES["f16_pages"]([300, 240, 230], [1, 3, 90], [(0, 3, 128, 128)], half=True, seed=24).device()
    n = c.n_head * c.hd
    wide = torch.full((c.rows, n + 48), 7.0, dtype=c.qd.dtype, device="cuda")
    wide[:, 16:16 + n] = c.qd.view(c.rows, n)
    c.qd = wide[:, 16:16 + n].view(c.rows, c.n_head, c.hd)
    to = torch.full((c.rows, n + 32), 123.0, dtype=c.qd.dtype, device="cuda")
    out = to[:, 8:8 + n].view(c.rows, c.n_head, c.hd)
    paged.paged_attention(c.qd, c.kd, c.vd, c.plan(), out=out)
    c.check(out)
    assert (to[:, :8] == 123.0).all() and (to[:, 8 + n:] == 123.0).all()


def test_refusals():
    c = CASES["f16_pages"]([200, 190], [1, 1], [(0, 2, 160, 160)], seed=25).device()
    args = dict(n_head=8, n_kv=2, hd=64, page_size=16, n_pages=c.n_pages, n_tokens=2, max_q=1)
    g, n = c.group_start, c.shared_len
    three = torch.zeros(3, dtype=torch.int32, device="cuda")
    for kw in (dict(group_start=g), dict(shared_len=n), dict(group_start=g.long(), shared_len=n), dict(group_start=g, shared_len=n.cpu()),
               dict(group_start=n, shared_len=n), dict(group_start=torch.zeros(4, dtype=torch.int32, device="cuda"), shared_len=three),
               dict(group_start=g, shared_len=n, window=64), dict(group_start=g, shared_len=n, prefix_len=c.len)):
        with pytest.raises(attn.AttnError):
            paged.PagedPlan(c.start, c.len, c.tab, **{**args, **kw})
    plan = c.plan()
    with pytest.raises(attn.AttnError) as e:
        paged.paged_attention(c.qd, c.kd, c.vd, plan, alibi=torch.ones(8, device="cuda"))
    assert e.value.code == attn.EUNSUPPORTED
