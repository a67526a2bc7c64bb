"""Attention over 8-bit pages: the cases of the f16 cache's tests over quantised
rows, against the 64-bit definition on the f16 numbers that the rows stand
for.  Rows that no token sees have NaN scales."""
import math

import pytest
import torch

from pelica_amd import attn, paged
from tests import q8_ref as q8
from tests import test_gpu_paged as f16_tests

pytestmark = pytest.mark.gpu


class Case(f16_tests.Case):
    """The f16 case, its rows quantised; ``k`` and ``v`` are what the rows stand for."""

    def __init__(self, *a, **kw):
        super().__init__(*a, **kw)
        self.stored = {}
        self.quantise()

    def quantise(self):
        """Groups of k and v that have changed since the last time."""
        for name in "kv":
            x = getattr(self, name)
            n, s = self.stored.get(name, (torch.zeros(x.shape, dtype=torch.int8),
                                          torch.full((*x.shape[:3], self.hd // 32), math.nan, dtype=torch.float16)))
            old, new = (t.unflatten(-1, (-1, 32)) for t in (q8.values(n, s), x))
            kept = ((old == new) | (old.isnan() & new.isnan())).all(-1)
            want = q8.scales(x).half()
            ints, _ = q8.quantise(x.nan_to_num(0, 0, 0))
            ints[want.isnan().repeat_interleave(32, -1)] = 55
            n = torch.where(kept.repeat_interleave(32, -1), n, ints)
            s = torch.where(kept, s, want)
            self.stored[name] = n, s
            setattr(self, name, q8.values(n, s))

    def pools(self, name, i, dtype, fill, more):
        """K's and V's pages (i = 0) or scales (1) in the layout's strides."""
        n, P, H = self.n_pages, self.page, self.n_kv
        D = self.stored["k"][i].shape[-1]
        at = torch.tensor(sorted(self.live)).cuda()
        if self.layout == "kv":
            both = torch.full((n, 2, P, H, D), fill, dtype=dtype, device="cuda")
            out = [both[:, 0], both[:, 1]]
        elif self.layout == "wide":
            out = [torch.full((n, P, H + 1, D + more), fill, dtype=dtype, device="cuda")[:, :, :H, :D] for _ in "kv"]
        elif self.layout == "hnd":
            out = [torch.full((n, H, P, D), fill, dtype=dtype, device="cuda").transpose(1, 2) for _ in "kv"]
        else:
            out = [torch.full((n, P, H, D), fill, dtype=dtype, device="cuda") for _ in "kv"]
        for t, name in zip(out, "kv"):
            t[at] = self.stored[name][i].cuda()
        return out

    def device(self):
        self.quantise()
        self.pool = lambda x: None
        layout, self.layout = self.layout, "hnd"
        super().device()
        self.layout = layout
        self.kd, self.vd = self.pools("pages", 0, torch.int8, 77, 16)
        self.ks, self.vs = self.pools("scales", 1, torch.float16, math.nan, 1)
        return self

    def run(self, plan=None, **kw):
        plan = plan or self.plan()
        out = torch.full_like(self.qd, 123.0)
        paged.paged_attention(self.qd, self.kd, self.vd, plan, k_scales=self.ks, v_scales=self.vs, sinks=self.dev(self.sinks),
                              alibi=self.dev(self.slopes), softcap=self.cap, scale=self.scale, out=out, **kw)
        return out


    def reference(self, **kw):
        # A weight's f16 parts keep 2^-22 of it, or half of f16's last step: 2^-25, of 2^14 for the largest.  (Quantised
        # values are 0 where the largest weight is often enough for that to be all there is.)
        want, f32, f16 = super().reference(**kw)
        return want, f32 + max(self.lens) * 2.0 ** -39 * self.v.nan_to_num(0, 0, 0).abs().max().double(), f16


@pytest.fixture(autouse=True)
def quantised(monkeypatch):
    monkeypatch.setattr(f16_tests, "Case", Case)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("mix", f16_tests.MIXES)
def test_requests(mix, hd, half):
    f16_tests.test_requests(mix, hd, half)


@pytest.mark.parametrize("n_head,n_kv", [(1, 1), (3, 1), (10, 2), (16, 1), (64, 8), (33, 1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_head_groups(n_head, n_kv, hd):
    f16_tests.test_head_groups(n_head, n_kv, hd)


@pytest.mark.parametrize("page", [8, 16, 32, 128])
@pytest.mark.parametrize("hd", [64, 128])
def test_page_sizes(page, hd):
    f16_tests.test_page_sizes(page, hd)


@pytest.mark.parametrize("window", [1, 16, 33, 100, 1000])
@pytest.mark.parametrize("new", [[1, 1, 3], [90, 1, 40]], ids=["tokens", "chunks"])
@pytest.mark.parametrize("hd", [64, 128])
def test_windows(window, new, hd):
    f16_tests.test_windows(window, new, hd)


@pytest.mark.parametrize("window", [0, 24])
@pytest.mark.parametrize("prefix", [[0, 1, 33], [17, 5, 299], [1000, 1000, 1000]])
@pytest.mark.parametrize("new", [[1, 1, 2], [70, 130, 299]], ids=["tokens", "chunks"])
def test_prefixes(prefix, window, new):
    f16_tests.test_prefixes(prefix, window, new)


@pytest.mark.parametrize("cap", [0.0, 5.0, 50.0])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_scores(cap, slopes, hd):
    f16_tests.test_scores(cap, slopes, hd)


@pytest.mark.parametrize("layout", ["nhd", "hnd", "wide", "kv"])
@pytest.mark.parametrize("hd", [64, 128])
def test_page_layouts(layout, hd):
    f16_tests.test_page_layouts(layout, hd)


@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 64, 8), (128, 32, 4), (128, 16, 16), (64, 4, 1)])
def test_split_over_keys(hd, n_head, n_kv):
    f16_tests.test_split_over_keys(hd, n_head, n_kv)


def test_scores_far_below_and_above():
    f16_tests.test_scores_far_below_and_above()


def test_single_page_pool():
    f16_tests.test_single_page_pool()


def test_many_requests():
    f16_tests.test_many_requests()


def test_bad_pages_give_nan_and_no_fault():
    f16_tests.test_bad_pages_give_nan_and_no_fault()


def test_values_of_masked_keys_do_not_matter():
    f16_tests.test_values_of_masked_keys_do_not_matter()


@pytest.mark.parametrize("gap", f16_tests.GAPS)
@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_head,n_kv", [(8, 2), (20, 1), (40, 1)], ids=["rows8", "rows32", "wide"])
def test_keys_between_a_prefix_and_a_window(n_head, n_kv, hd, half, gap):
    f16_tests.test_keys_between_a_prefix_and_a_window(n_head, n_kv, hd, half, gap)


def test_pages_past_4_gib():
    page, n_kv, hd = 256, 8, 64
    need = (5 << 30) // (page * n_kv * hd)
    Case([700, 300], [1, 100], n_head=16, n_kv=n_kv, hd=hd, page=page, half=True, first_page=need, seed=28).check()


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_captured_steps_follow_new_lengths(half):
    """A graph of plan and attention over 8-bit pages, other lengths, eager calls between the replays; the bits of eager calls."""
    a = Case([2000, 120, 64], [1, 1, 40], n_head=16, n_kv=2, sinks=True, half=half, seed=30, pad=4).device()
    plan = a.plan()
    ws = plan.new_workspace()
    out = torch.full_like(a.qd, 123.0)
    kw = dict(k_scales=a.ks, v_scales=a.vs, sinks=a.dev(a.sinks), workspace=ws)
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        with torch.cuda.graph(graph, stream=st):
            plan.update()
            paged.paged_attention(a.qd, a.kd, a.vd, plan, out=out, **kw)
    torch.cuda.synchronize()
    for lens, new in (([2000, 120, 64], [1, 1, 40]), ([1990, 100, 3], [2, 1, 3]), ([5, 120, 0], [3, 2, 0])):
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
        paged.paged_attention(a.qd, a.kd, a.vd, plan.update(), out=eager, **kw)
        assert torch.equal(eager, out)


@pytest.mark.parametrize("hd", [64, 128])
def test_a_step_writes_rows_and_reads_them(hd):
    """pages_append, paged_qkv into 8-bit pages, paged_attention over them: prompts, then tokens; the rows that pages_read
    gives are within the format's half scale of the f16 cache's, and attention over either agrees to that."""
    n_head, n_kv, page, n_pages = 8, 2, 16, 40
    g = torch.Generator(device="cuda").manual_seed(hd)
    dev = "cuda"
    pools = paged.new_q8_pages(n_pages, page, n_kv, hd)
    scales = dict(k_scales=pools[2], v_scales=pools[3])
    table = torch.full((3, 12), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(n_pages, generator=g, device=dev).int()
    state = torch.tensor([0, n_pages], device=dev)
    cached = torch.zeros(3, dtype=torch.int32, device=dev)
    rope = torch.zeros(200, hd // 2, 2, device=dev)
    ang = torch.arange(200, device=dev)[:, None] * 1e4 ** (-torch.arange(hd // 2, device=dev) / (hd // 2))
    rope[..., 0], rope[..., 1] = ang.cos(), ang.sin()
    for new in ([50, 7, 90], [1, 2, 1], [1, 0, 3]):
        T = sum(new)
        step = paged.pages_append(cached, torch.tensor(new, dtype=torch.int32, device=dev), table, free, state,
                                  page_size=page, n_tokens=T)
        assert (step.status == 0).all()
        x = [torch.randn(T, h, hd, generator=g, device=dev) for h in (n_head, n_kv, n_kv)]
        q = paged.paged_qkv(*x, *pools[:2], step.slots, positions=step.positions, table=rope, **scales)
        plan = paged.PagedPlan(step.q_start, step.seq_kv_len, table, n_head=n_head, n_kv=n_kv, hd=hd, page_size=page,
                               n_pages=n_pages, n_tokens=T, max_q=max(new))
        out = paged.paged_attention(q, *pools[:2], plan, **scales)
        # the whole pool as f16 pages
        k, v = (t.view(n_pages, page, n_kv, hd) for t in paged.pages_read(*pools[:2], torch.arange(n_pages * page, device=dev), **scales))
        same = paged.paged_attention(q, k, v, plan)
        torch.cuda.synchronize()
        # one operator, one set of numbers: the kernels differ in the order of f32 sums only
        assert torch.allclose(out, same, rtol=0, atol=2e-5)
        rows = v.reshape(-1, n_kv, hd)[step.slots]
        top = x[2].unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 32).flatten(-2)
        assert ((rows.float() - x[2]).abs() <= top * (0.5 / 127 + 2 * 2.0 ** -10)).all()
        cached, state = step.seq_kv_len, step.free_state


def test_refusals():
    c = Case([100, 40], [1, 1], seed=26).device()
    plan = c.plan()
    for kw in (dict(k_scales=None), dict(k_scales=None, v_scales=None), dict(v_scales=c.vs[:1]), dict(v_scales=c.vs.float()),
               dict(k_scales=c.ks[..., :1], v_scales=c.vs[..., :1]), dict(k_pages=c.kd.half(), v_pages=c.vd.half()),
               dict(v_pages=c.vd.half())):
        args = {**dict(k_pages=c.kd, v_pages=c.vd, k_scales=c.ks, v_scales=c.vs), **kw}
        with pytest.raises(attn.AttnError):
            paged.paged_attention(c.qd, plan=plan, **args)


# (lens, window, prefix): the prefix ends and the window begins within 16 or 32 rows that one load covers
@pytest.mark.parametrize("lens,window,prefix", [([130], 100, [20]), ([300, 275, 64], 24, [268, 242, 33]), ([300], 30, [257]),
                                                ([31], 3, [9]), ([420], 36, [353])])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_head,n_kv", [(8, 2), (20, 1), (40, 1)], ids=["rows8", "rows32", "wide"])
def test_keys_between_a_prefix_and_a_window_in_longer_pages(n_head, n_kv, hd, page, lens, window, prefix):
    for half in (False, True):
        kw = dict(n_head=n_head, n_kv=n_kv, hd=hd, half=half, window=window, prefix=prefix, page=page)
        Case(lens, [1] * len(lens), seed=45, **kw).check()
        Case(lens, [min(n, 3) for n in lens], seed=48, cap=5.0, sinks=True, **kw).check()


@pytest.mark.parametrize("page", [8, 16, 32, 128])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_random_mixes(page, hd, half):
    g = torch.Generator().manual_seed(page + hd + half)
    r = lambda a, b: int(torch.randint(a, b + 1, (1,), generator=g))  # noqa: E731
    for seed in range(6):
        n = r(1, 7)
        lens = [r(1, 700) for _ in range(n)]
        new = [min(a, r(1, (1, 3, 90)[r(0, 2)])) for a in lens]
        hpk, n_kv = (1, 2, 3, 5, 8)[r(0, 4)], r(1, 3)
        Case(lens, new, n_head=hpk * n_kv, n_kv=n_kv, hd=hd, half=half, page=page, window=(0, 0, r(1, 300))[r(0, 2)], sinks=r(0, 1) == 1,
             layout=("hnd", "nhd", "wide", "kv")[r(0, 3)], pad=r(0, 3), seed=100 + seed).check()
