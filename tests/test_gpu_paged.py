"""Attention over a paged cache against its 64-bit definition: requests of one
token to long chunks in one call, pages that end inside a tile, windows,
prefixes, capped and biased scores, sinks, layouts.  Rows of the pool that no
token sees hold NaN and pages behind a window are gone from the table, so that
a read of them shows."""
import math

import pytest
import torch

from pelica_amd import paged
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, lens, new, *, n_head=8, n_kv=2, hd=64, page=16, window=0, prefix=None, sinks=False,
                 slopes=False, cap=0.0, half=False, seed=0, spare=3, layout="nhd", pad=0, scale=None, first_page=0,
                 n_pages=None, q_scale=1.0):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.lens, self.new, self.page, self.window, self.cap, self.scale = lens, new, page, window, cap, scale
        self.n_head, self.n_kv, self.hd, self.half = n_head, n_kv, hd, half
        self.prefix = prefix
        held = [-(-n // page) for n in lens]
        n_live = sum(held) + spare
        ids = (torch.randperm(n_live, generator=g) + first_page).tolist()
        self.n_pages = n_pages or n_live + first_page
        # a page of the pool is known by its place among the live ones
        self.live = {p: i for i, p in enumerate(sorted(ids))}
        k = torch.full((n_live, page, n_kv, hd), math.nan)
        v = k.clone()
        self.table = []
        for n, h, t in zip(lens, held, new):
            mine = [ids.pop() for _ in range(h)]
            lo = max(0, n - t - window + 1) if window else 0
            pre = 0 if prefix is None else prefix[len(self.table)]
            for j in range(n):
                if j >= lo or j < pre:
                    k[self.live[mine[j // page]], j % page] = rnd(n_kv, hd)
                    v[self.live[mine[j // page]], j % page] = rnd(n_kv, hd)
            for j in range(h):  # pages no token sees are gone
                if (j + 1) * page <= lo and j * page >= pre:
                    mine[j] = -1
            self.table.append(mine)
        self.k, self.v = k.half(), v.half()
        self.rows = sum(new) + pad
        q = rnd(self.rows, n_head, hd) * q_scale
        self.q = q.half() if half else q
        self.sinks = rnd(n_head) if sinks else None
        self.slopes = torch.exp2(-8 * (torch.arange(n_head) + 1.0) / n_head) if slopes else None
        self.layout = layout

    def pool(self, x):
        n, P, H, D = self.n_pages, self.page, self.n_kv, self.hd
        at = torch.tensor(sorted(self.live)).cuda()
        if self.layout == "hnd":
            t = torch.full((n, H, P, D), math.nan, dtype=torch.float16, device="cuda").transpose(1, 2)
        elif self.layout == "wide":  # rows of a wider buffer
            t = torch.full((n, P, H + 1, D + 8), math.nan, dtype=torch.float16, device="cuda")[:, :, :H, :D]
        else:
            t = torch.full((n, P, H, D), math.nan, dtype=torch.float16, device="cuda")
        t[at] = x.cuda()
        return t

    def device(self):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        start = [0]
        for t in self.new:
            start.append(start[-1] + t)
        most = max(1, max(map(len, self.table)))
        self.start, self.len = i32(start), i32(self.lens)
        self.tab = i32([r + [-7] * (most - len(r)) for r in self.table])
        self.pre = None if self.prefix is None else i32(self.prefix)
        if self.layout == "kv":  # K and V side by side, one buffer
            both = torch.full((self.n_pages, 2, self.page, self.n_kv, self.hd), math.nan, dtype=torch.float16, device="cuda")
            at = torch.tensor(sorted(self.live)).cuda()
            both[at, 0], both[at, 1] = self.k.cuda(), self.v.cuda()
            self.kd, self.vd = both[:, 0], both[:, 1]
        else:
            self.kd, self.vd = self.pool(self.k), self.pool(self.v)
        self.qd = self.q.cuda()
        self.dev = lambda x: None if x is None else x.cuda()
        return self

    def plan(self, **kw):
        return paged.PagedPlan(self.start, self.len, self.tab, n_head=self.n_head, n_kv=self.n_kv, hd=self.hd,
                               page_size=self.page, n_pages=self.n_pages, n_tokens=self.rows,
                               max_q=max(1, max(self.new)), window=self.window, prefix_len=self.pre, **kw)

    def run(self, plan=None, **kw):
        plan = plan or self.plan()
        out = torch.full_like(self.qd, 123.0)
        paged.paged_attention(self.qd, self.kd, self.vd, plan, sinks=self.dev(self.sinks), alibi=self.dev(self.slopes),
                              softcap=self.cap, scale=self.scale, out=out, **kw)
        return out

    def reference(self, **kw):
        names = [[self.live.get(p, -1) for p in r] for r in self.table]
        return ref.attention(self.q, self.k, self.v, names, self.lens, self.new, page=self.page, window=self.window,
                             prefix=self.prefix, sinks=self.sinks, slopes=self.slopes, cap=self.cap, scale=self.scale, **kw)

    def check(self, out=None, **kw):
        out = self.device().run() if out is None else out
        torch.cuda.synchronize()
        want, f32, f16 = self.reference(**kw)
        ref.check(out, want, f32, f16 if self.half else None)
        idle = want.isnan()
        assert (out.cpu()[idle] == 123.0).all(), "a row of no request was written"


MIXES = {
    "one": ([1], [1]),
    "one_of_two_keys": ([2], [1]),
    "page_ends": ([15, 16, 17, 31, 32, 33, 64, 65], [1] * 8),
    "ragged": ([300, 1, 77, 513, 128], [1, 1, 1, 1, 1]),
    "drafts": ([100, 41, 9, 260], [4, 1, 3, 2]),
    "empty_requests": ([0, 50, 0, 33, 20], [0, 1, 0, 2, 0]),
    "chunks": ([130, 40, 95], [65, 40, 1]),
    "fresh": ([257], [257]),
    "mixed": ([400, 7, 290, 64, 33], [1, 7, 129, 2, 33]),
}


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("mix", MIXES)
def test_requests(mix, hd, half):
    lens, new = MIXES[mix]
    Case(lens, new, hd=hd, half=half, n_head=8, n_kv=2, seed=1).check()


@pytest.mark.parametrize("n_head,n_kv", [(1, 1), (4, 4), (3, 1), (10, 2), (16, 1), (64, 8), (33, 1), (71, 1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_head_groups(n_head, n_kv, hd):
    Case([90, 33, 140], [1, 5, 70], n_head=n_head, n_kv=n_kv, hd=hd, half=hd == 64, seed=2).check()
    Case([90, 33, 140], [1, 1, 2], n_head=n_head, n_kv=n_kv, hd=hd, half=hd == 128, seed=3).check()


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("hd", [64, 128])
def test_page_sizes(page, hd):
    Case([257, 8, 100, 300], [1, 2, 1, 150], page=page, hd=hd, half=True, seed=4).check()
    Case([257, 8, 100, 600], [1, 2, 1, 1], page=page, hd=hd, seed=5).check()


@pytest.mark.parametrize("window", [1, 2, 16, 31, 33, 100, 1000])
@pytest.mark.parametrize("new", [[1, 1, 3], [90, 1, 40]], ids=["tokens", "chunks"])
@pytest.mark.parametrize("hd", [64, 128])
def test_windows(window, new, hd):
    Case([300, 40, 130], new, window=window, hd=hd, half=new[0] > 1, sinks=True, seed=6).check()


@pytest.mark.parametrize("window", [0, 24, 100])
@pytest.mark.parametrize("prefix", [[0, 1, 33], [64, 130, 200], [17, 5, 299], [1000, 1000, 1000]])
@pytest.mark.parametrize("new", [[1, 1, 2], [70, 130, 299]], ids=["tokens", "chunks"])
def test_prefixes(prefix, window, new):
    Case([300, 130, 300], new, prefix=prefix, window=window, hd=64, half=new[0] > 1, seed=7).check()
    Case([300, 130, 300], new, prefix=prefix, window=window, hd=128, page=8, half=new[0] == 1, seed=8).check()


@pytest.mark.parametrize("cap", [0.0, 5.0, 50.0, 1000.0])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_scores(cap, slopes, hd):
    kw = dict(cap=cap, slopes=slopes, hd=hd, sinks=True)
    Case([300, 40, 130], [1, 3, 1], seed=9, q_scale=8.0, **kw).check()
    Case([300, 40, 130], [90, 3, 130], seed=10, half=True, window=64, prefix=[50, 40, 0], **kw).check()
    Case([300, 40, 130], [90, 3, 130], seed=11, n_head=5, n_kv=1, **kw).check()


@pytest.mark.parametrize("cap", [50.0, 1000.0, 1e6])
@pytest.mark.parametrize("hd", [64, 128])
def test_scores_far_below_the_cap(cap, hd):
    # up to 0.55 of the cap a capped score is off by a part of itself, not of the cap
    Case([300, 40, 130], [1, 3, 1], seed=40, cap=cap, hd=hd).check(cap_off=0)
    Case([300, 40, 130], [90, 3, 130], seed=41, cap=cap, hd=hd, slopes=True).check(cap_off=0)
    Case([300, 40, 130], [90, 3, 130], seed=42, cap=cap, hd=hd, half=True).check(cap_off=0)


@pytest.mark.parametrize("cap", [1e-3, 1e-20])
def test_scores_far_above_the_cap(cap):
    # (all scores are the cap's: a mean of the values)
    Case([300, 40, 130], [1, 3, 1], seed=43, cap=cap, hd=64).check()
    Case([300, 40, 130], [90, 3, 130], seed=44, cap=cap, hd=128, half=True).check()


def test_scores_far_below_and_above():
    # scores of +-300 (natural log): sums stay finite, far keys vanish
    Case([200, 70], [1, 70], q_scale=100.0, half=True, seed=12).check()
    Case([200, 70], [1, 70], q_scale=100.0, sinks=True, seed=13).check()
    Case([200, 70], [1, 70], scale=1e-6, sinks=True, seed=14).check()


@pytest.mark.parametrize("layout", ["hnd", "wide", "kv"])
@pytest.mark.parametrize("hd", [64, 128])
def test_page_layouts(layout, hd):
    Case([300, 40, 130], [1, 3, 90], layout=layout, hd=hd, half=True, seed=15).check()
    Case([300, 40, 130], [1, 3, 1], layout=layout, hd=hd, n_head=4, n_kv=1, seed=16).check()


def test_single_page_pool():
    Case([5], [1], spare=0, n_kv=1, n_head=2, seed=17).check()


@pytest.mark.parametrize("half", [False, True])
def test_token_rows_of_wider_buffers(half):
    c = Case([300, 40, 130], [1, 3, 90], half=half, seed=18).device()
    n = c.n_head * c.hd
    wide = torch.full((c.rows, n + 48), 7.0, dtype=c.qd.dtype, device="cuda")
    wide[:, 16:16 + n] = c.qd.view(c.rows, n)
    c.qd = wide[:, 16:16 + n].view(c.rows, c.n_head, c.hd)
    to = torch.full((c.rows, n + 32), 123.0, dtype=c.qd.dtype, device="cuda")
    out = to[:, 8:8 + n].view(c.rows, c.n_head, c.hd)
    paged.paged_attention(c.qd, c.kd, c.vd, c.plan(), out=out)
    c.check(out)
    assert (to[:, :8] == 123.0).all() and (to[:, 8 + n:] == 123.0).all()


def test_rows_behind_the_last_and_skipped_requests():
    # 6 padding rows; a request with fewer keys than tokens and one past its table's row are skipped
    c = Case([100, 40, 30], [1, 4, 2], pad=6, seed=19).device()
    c.len[1] = 3
    c.len[2] = c.tab.shape[1] * c.page + 1
    out = c.run()
    c.lens = [100, 3, 30]
    want, f32, _ = ref.attention(c.q, c.k, c.v, [[c.live[p] for p in r] for r in c.table], [100, 3, 1], [1, 4, 2], page=16)
    ref.check(out, want, f32)
    assert (out[1:] == 123.0).all()


@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 64, 8), (128, 32, 4), (128, 16, 16), (64, 4, 1)])
def test_split_over_keys(hd, n_head, n_kv):
    # one request on an empty chip: cut into many key ranges, joined with the sinks
    Case([5000], [1], hd=hd, n_head=n_head, n_kv=n_kv, sinks=True, page=64, seed=20).check()
    Case([3001, 90], [3, 1], hd=hd, n_head=n_head, n_kv=n_kv, half=True, page=32, seed=21).check()
    Case([1500, 2000], [1, 40], hd=hd, n_head=n_head, n_kv=n_kv, sinks=True, half=True, seed=22).check()


def test_many_requests():
    # more items than fill the chip once, and more than one round of the planner's threads
    g = torch.Generator().manual_seed(23)
    lens = torch.randint(0, 60, (1500,), generator=g).tolist()
    Case(lens, [min(1, n) for n in lens], n_head=2, n_kv=2, page=8, seed=23).check()
    lens = torch.randint(1, 90, (700,), generator=g).tolist()
    Case(lens, [1 + n % 40 if n > 40 else 1 for n in lens], n_head=2, n_kv=1, hd=128, half=True, seed=24).check()


def test_bad_pages_give_nan_and_no_fault():
    c = Case([100, 100], [1, 1], seed=25).device()
    for bad in (-1, c.n_pages, 2 ** 31 - 1, -2 ** 31):
        c.tab[0, 2] = bad
        out = c.run()
        assert out[0].isnan().all()
        want, f32, _ = c.reference()
        ref.check(out[1:], want[1:], f32[1:])


def test_another_plan_writes_nothing():
    c = Case([100, 40], [1, 1], seed=26).device()
    plan = c.plan()
    other = Case([100, 40], [1, 1], window=20, seed=26).device()
    plan.desc.window = 20  # a descriptor that is not the plan's
    out = torch.full_like(c.qd, 123.0)
    paged.paged_attention(c.qd, c.kd, c.vd, plan, out=out)
    assert (out == 123.0).all()
    other.check()


def test_values_of_masked_keys_do_not_matter():
    # a later token's key row and value row (masked for the earlier ones) hold
    # infinities and NaN: the earlier tokens' outputs do not
    for half, hd in ((True, 64), (False, 64), (True, 128), (False, 128)):
        c = Case([80, 60], [40, 1], hd=hd, half=half, seed=27)
        want, f32, f16 = c.reference()
        c.k[c.live[c.table[0][75 // 16]], 75 % 16] = math.nan
        c.v[c.live[c.table[0][75 // 16]], 75 % 16, :, ::2] = math.inf
        c.v[c.live[c.table[0][76 // 16]], 76 % 16] = math.nan
        out = c.device().run()
        keep = torch.arange(41)[(torch.arange(41) < 35) | (torch.arange(41) == 40)]
        ref.check(out[keep.cuda()], want[keep], f32[keep], f16[keep] if half else None)
        assert out[35:40].isnan().any(-1).all()


def test_pool_past_4_gib():
    page, n_kv, hd = 256, 8, 64
    need = (5 << 30) // (page * n_kv * hd * 2)
    c = Case([700, 300], [1, 100], n_head=16, n_kv=n_kv, hd=hd, page=page, half=True, first_page=need, seed=28)
    c.check()


def test_another_stream_and_shared_workspace():
    c = Case([3000, 500], [1, 1], n_head=16, n_kv=2, sinks=True, seed=29).device()
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    plan = c.plan(stream=st)
    out = torch.full_like(c.qd, 123.0)
    torch.cuda.synchronize()
    got = paged.paged_attention(c.qd, c.kd, c.vd, plan, sinks=c.dev(c.sinks), out=out, stream=st)
    st.synchronize()
    c.check(got)
    # runs give the same bits
    for _ in range(3):
        assert torch.equal(c.run(plan), got)


def test_captured_step_follows_new_lengths():
    """A graph of plan + attention replayed with other lengths in the same
    arrays, with eager calls between the replays."""
    a = Case([2000, 120, 64], [1, 1, 3], n_head=16, n_kv=2, sinks=True, seed=30, pad=4).device()
    plan = a.plan()
    ws = plan.new_workspace()
    out = torch.full_like(a.qd, 123.0)
    sinks = a.dev(a.sinks)
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        with torch.cuda.graph(graph, stream=st):
            plan.update(stream=st)
            paged.paged_attention(a.qd, a.kd, a.vd, plan, sinks=sinks, out=out, workspace=ws, stream=st)
    torch.cuda.synchronize()
    lens0, new0 = list(a.lens), list(a.new)
    for lens, new in ((lens0, new0), ([1990, 100, 3], [2, 1, 3]), ([5, 120, 0], [3, 2, 0]), (lens0, new0)):
        a.lens, a.new = lens, new
        start = [0]
        for t in new:
            start.append(start[-1] + t)
        a.start.copy_(torch.tensor(start, dtype=torch.int32))
        a.len.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(123.0)
        graph.replay()
        torch.cuda.synchronize()
        a.check(out)
        eager = torch.full_like(a.qd, 123.0)
        paged.paged_attention(a.qd, a.kd, a.vd, plan.update(), sinks=sinks, out=eager, workspace=ws)
        assert torch.equal(eager, out)


def test_first_rows_that_decrease():
    # rows of two requests: nothing is planned, nothing written
    c = Case([200, 90, 140], [2, 40, 3], n_head=16, n_kv=2, seed=31, half=True).device()
    for start in ([0, 45, 5, 45], [0, 2, 1, 45], [45, 0, 45, 0]):
        c.start.copy_(torch.tensor(start, dtype=torch.int32))
        out = c.run(c.plan())
        torch.cuda.synchronize()
        assert (out == 123.0).all()
    c.start.copy_(torch.tensor([0, 2, 42, 45], dtype=torch.int32))
    c.check(c.run(c.plan()))


def test_two_steps_at_once():
    # two plans, workspaces and streams: split items of single tokens beside a chunk's
    a = Case([9000, 4000], [1, 1], n_head=16, n_kv=2, sinks=True, seed=32).device()
    b = Case([1500, 900], [200, 1], n_head=16, n_kv=2, hd=128, half=True, seed=33).device()
    runs = []
    torch.cuda.synchronize()
    for c in (a, b):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            plan = c.plan(stream=st)
            runs.append((c, st, plan, plan.new_workspace(), torch.full_like(c.qd, 123.0), c.dev(c.sinks)))
    torch.cuda.synchronize()
    for _ in range(10):
        for c, st, plan, ws, out, sinks in runs:
            plan.update(stream=st)
            paged.paged_attention(c.qd, c.kd, c.vd, plan, sinks=sinks, out=out, workspace=ws, stream=st)
    torch.cuda.synchronize()
    for c, _, _, _, out, _ in runs:
        c.check(out)


@pytest.mark.parametrize("new", [[1], [5], [200]], ids=["token", "draft", "chunk"])
@pytest.mark.parametrize("hd", [64, 128])
def test_many_equal_keys_far_below_one(new, hd):
    """Key 0 scores s, 20000 others 0, all values 1: the result is 1 to the
    roundings of sums, however the small weights are rounded on their way."""
    n, s = 20000, 13.3  # e^-13.3 = 1.75 x 2^-20
    c = Case([n], new, n_head=8, n_kv=1, hd=hd, page=64, seed=34)
    c.k[:], c.v[:] = 0, 1
    first = c.table[0][0]
    c.k[c.live[first], 0, 0, 0] = 4
    c.q[:] = 0
    c.q[..., 0] = s / 4 * math.sqrt(hd)
    out = c.device().run().double().cpu()
    # one rounding for each 32-key chunk a wave walks alone (a quarter of them)
    # and a few for the trees, in the sum and in the product
    tol = 2 * (n // 128 + 16) * ref.U32 if new[0] * 8 <= 32 else 2 * (n // 32 + 16) * ref.U32
    assert (out - 1).abs().max() <= tol


@pytest.mark.parametrize("new", [[1], [200]], ids=["token", "chunk"])
@pytest.mark.parametrize("hd", [64, 128])
def test_many_equal_f16_weights_far_below_one(new, hd):
    """f16 queries, the same keys, of which key 0 has the value 0: the others'
    share of the weights, 29.6 x 2^-24 each beside 1, is off by their one
    rounding (all alike) and the output's."""
    n, s = 20000, 13.25
    c = Case([n], new, n_head=8, n_kv=1, hd=hd, page=64, half=True, seed=35)
    c.k[:], c.v[:] = 0, 1
    at = c.live[c.table[0][0]]
    c.k[at, 0, 0, 0], c.v[at, 0] = 4, 0
    c.q[:] = 0
    c.q[..., 0] = s / 4 * math.sqrt(hd)
    want = c.reference()[0]
    out = c.device().run().double().cpu()
    tol = want * (2 * ref.U16 + ref.U16 ** 2 + 2 * (n // 32 + 16) * ref.U32)
    assert ((out - want).abs() <= tol).all()


# one token of each request, (lens, window, prefix): the prefix ends a few keys
# before the window, within one run of 8 rows; the keys between hold NaN
GAPS = {
    "first_chunk": ([130], 100, [26]),
    "only_chunk": ([31], 3, [26]),
    "last_chunk": ([300, 275, 64], 24, [275, 250, 33]),
    "one_key": ([300], 24, [275]),
}


@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_head,n_kv", [(8, 2), (20, 1), (40, 1)], ids=["rows8", "rows32", "wide"])
def test_keys_between_a_prefix_and_a_window(n_head, n_kv, hd, half, gap):
    lens, window, prefix = GAPS[gap]
    kw = dict(n_head=n_head, n_kv=n_kv, hd=hd, half=half, window=window, prefix=prefix, page=8)
    Case(lens, [1] * len(lens), seed=45, **kw).check()
    Case(lens, [1] * len(lens), seed=46, cap=5.0, sinks=True, **kw).check()
    Case(lens, [1] * len(lens), seed=47, slopes=True, **kw).check()
    Case(lens, [min(n, 3) for n in lens], seed=48, **kw).check()
