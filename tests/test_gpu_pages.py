"""Page bookkeeping on the GPU against a plain Python walk of the requests: whole
numbers, equal or wrong."""
import ctypes

import pytest
import torch

from pelica_amd import attn, paged
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
i64 = lambda x: torch.tensor(x, dtype=torch.int64, device="cuda")  # noqa: E731


def _pool(cached, page, n_pages, max_pages, seed, taken=0):
    """A table of the cached tokens' pages and the queue of the others."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(n_pages, generator=g).tolist()
    table = []
    for c in cached:
        held = [ids.pop() for _ in range(-(-max(c, 0) // page))]
        table.append((held + [-1] * max_pages)[:max_pages])
    queue = [-1] * n_pages
    for i, p in enumerate(ids):
        queue[(taken + i) % n_pages] = p
    return table, queue, [taken, taken + len(ids)]


def _append(cached, new, table, queue, state, page, n_tokens, stream=None):
    tab = i32(table)
    step = paged.pages_append(i32(cached), i32(new), tab, i32(queue), i64(state), page_size=page, n_tokens=n_tokens,
                              stream=stream)
    torch.cuda.synchronize()
    got = {n: getattr(step, n).tolist() for n in ("q_start", "seq_kv_len", "status", "slots", "positions", "token_seq",
                                                  "free_state")}
    got["table"] = tab.tolist()
    return got


CASES = {
    "one_token": ([5], [1], 16),
    "first_token": ([0], [1], 16),
    "page_begins": ([16, 15, 17, 0, 31], [1, 1, 1, 0, 2], 16),
    "prompt": ([0, 7], [100, 33], 8),
    "nothing_new": ([40, 0, 9], [0, 0, 0], 16),
    "bad_lengths": ([-1, 30, 5, 2 ** 31 - 1], [3, -2, 4, 1], 16),
}


@pytest.mark.parametrize("taken", [0, 3, 10 ** 12 + 7])
@pytest.mark.parametrize("case", CASES)
def test_append(case, taken):
    cached, new, page = CASES[case]
    held = [c if 0 <= c < 10 ** 6 else 0 for c in cached]
    table, queue, state = _pool(held, page, 64, 24, 1, taken)
    for n_tokens in (max(1, sum(max(n, 0) for n in new)), 300):
        want = ref.pages_append(cached, new, table, queue, state, page, n_tokens, 24)
        assert _append(cached, new, table, queue, state, page, n_tokens) == want


@pytest.mark.parametrize("n_seq", [1, 255, 257, 1025, 4096])
def test_append_many(n_seq):
    g = torch.Generator().manual_seed(n_seq)
    cached = torch.randint(0, 100, (n_seq,), generator=g).tolist()
    new = torch.randint(0, 9, (n_seq,), generator=g).tolist()
    new[n_seq // 2] = 700
    n_pages = sum(-(-(c + n) // 8) for c, n in zip(cached, new)) + 3
    table, queue, state = _pool(cached, 8, n_pages, 120, 2, taken=77)
    n_tokens = sum(new) + 13
    assert _append(cached, new, table, queue, state, 8, n_tokens) == ref.pages_append(
        cached, new, table, queue, state, 8, n_tokens, 120)


@pytest.mark.parametrize("free", range(8))
def test_append_runs_out_of_pages(free):
    # needs, in order: 1, 0, 2, 0, 3 pages
    cached, new, page = [16, 3, 0, 20, 10], [1, 4, 32, 5, 50], 16
    table, queue, state = _pool(cached, page, 20, 10, 3)
    state = [state[0], state[0] + free]
    want = ref.pages_append(cached, new, table, queue, state, page, 120, 10)
    assert want["status"] == [int(free < 1), 0, int(free < 3), 0, int(free < 6)]
    assert _append(cached, new, table, queue, state, page, 120) == want


def test_append_past_the_table_or_the_rows():
    cached, new, page = [30, 60, 2, 1], [2, 8, 50, 1], 16
    table, queue, state = _pool(cached, page, 40, 4, 4)
    for n_tokens in (61, 60, 59, 10, 3, 1):
        want = ref.pages_append(cached, new, table, queue, state, page, n_tokens, 4)
        assert _append(cached, new, table, queue, state, page, n_tokens) == want
    assert 2 in want["status"] and 3 in want["status"]


def test_append_of_page_ids_outside_the_pool():
    cached, new, page = [20, 5], [20, 3], 16
    table, queue, state = _pool(cached, page, 30, 8, 5)
    table[0][1] = -3         # an entry that was there
    table[1][0] = 30
    queue[state[0] % 30] = 99  # the first free one
    want = ref.pages_append(cached, new, table, queue, state, page, 40, 8)
    got = _append(cached, new, table, queue, state, page, 40)
    # (what the queue held is no page: the table says so)
    assert got["table"][0][2] == -1
    got["table"][0][2] = want["table"][0][2]
    assert got == want and want["slots"][:12] == [-1] * 12


def _release(ended, cached, table, queue, state, page):
    lst = i32(queue)
    out = paged.pages_release(i32(ended), i32(cached), i32(table), lst, i64(state), page_size=page)
    torch.cuda.synchronize()
    return out.tolist(), lst.tolist()


@pytest.mark.parametrize("n_seq", [1, 5, 300, 3000])
def test_release(n_seq):
    g = torch.Generator().manual_seed(n_seq)
    cached = torch.randint(0, 60, (n_seq,), generator=g).tolist()
    ended = torch.randint(0, 2, (n_seq,), generator=g).tolist()
    n_pages = sum(-(-c // 8) for c in cached) + 5
    table, queue, state = _pool(cached, 8, n_pages, 9, 6, taken=10 ** 10 + 3)
    want, end = list(queue), state[1]
    for s in range(n_seq):
        if ended[s]:
            for j in range(-(-cached[s] // 8)):
                want[end % n_pages] = table[s][j]
                end += 1
    assert _release(ended, cached, table, queue, state, 8) == ([state[0], end], want)


def test_release_of_more_than_the_pool_holds_gives_nothing_back():
    table, queue, state = _pool([20], 8, 6, 4, 7)
    assert _release([1], [20], table, queue, [state[0], state[0] + 4], 8) == ([state[0], state[0] + 4], queue)


def test_steps_never_hand_out_a_page_twice():
    """Requests that come, grow and end over 40 steps, two PageSteps in turn."""
    n_seq, page, n_pages, most = 12, 8, 60, 12
    g = torch.Generator().manual_seed(8)
    cached = [0] * n_seq
    tab = torch.full((n_seq, most), -1, dtype=torch.int32, device="cuda")
    lst = i32(list(range(n_pages)))
    state = i64([0, n_pages])
    mid = torch.zeros(2, dtype=torch.int64, device="cuda")
    steps = [paged.PageStep(n_seq, 200), paged.PageStep(n_seq, 200)]
    refused = 0
    for i in range(40):
        ended = [int(c > 0 and torch.randint(0, 6, (1,), generator=g).item() == 0) for c in cached]
        paged.pages_release(i32(ended), i32(cached), tab, lst, state, page_size=page, free_out=mid)
        cached = [0 if e else c for e, c in zip(ended, cached)]
        new = [int(torch.randint(0, 16, (1,), generator=g)) if c + 16 < most * page else 0 for c in cached]
        step = paged.pages_append(i32(cached), i32(new), tab, lst, mid, page_size=page, step=steps[i % 2])
        state = step.free_state
        st = step.status.tolist()
        refused += sum(st)
        cached = [c if x else c + n for c, n, x in zip(cached, new, st)]
        held = [p for s, r in enumerate(tab.tolist()) for p in r[:-(-cached[s] // page)]]
        a, b = state.tolist()
        free = [lst.tolist()[j % n_pages] for j in range(a, b)]
        assert sorted(held + free) == list(range(n_pages)), i
    assert refused > 0  # (the pool ran dry at times)


def test_append_in_a_graph():
    cached, new, page = [5, 30, 0], [1, 2, 20], 16
    table, queue, state = _pool([5, 60, 40], page, 30, 8, 9)
    c, n, tab, lst, fs = i32(cached), i32(new), i32(table), i32(queue), i64(state)
    step = paged.PageStep(3, 40)
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(st), torch.cuda.graph(graph, stream=st):
        paged.pages_append(c, n, tab, lst, fs, page_size=page, step=step, stream=st)
    for cached, new in (([5, 30, 0], [1, 2, 20]), ([6, 32, 20], [3, 1, 0]), ([60, 1, 1], [1, 1, 30]), ([5, 30, 0], [1, 2, 20])):
        c.copy_(i32(cached))
        n.copy_(i32(new))
        tab.copy_(i32(table))
        want = ref.pages_append(cached, new, table, queue, state, page, 40, 8)
        graph.replay()
        torch.cuda.synchronize()
        assert tab.tolist() == want["table"] and step.slots.tolist() == want["slots"]
        assert step.free_state.tolist() == want["free_state"] and step.q_start.tolist() == want["q_start"]


def test_lengths_of_the_last_step_are_the_next_ones():
    """Two PageSteps in turn, the one's seq_kv_len the other's cached_len, in
    steps of many workgroups; the same PageStep is refused."""
    n_seq, page, n_pages, most = 300, 8, 2500, 20
    g = torch.Generator().manual_seed(10)
    lens = torch.randint(0, 40, (n_seq,), generator=g).tolist()
    table, queue, state = _pool(lens, page, n_pages, most, 11)
    tab, lst, fs, cached = i32(table), i32(queue), i64(state), i32(lens)
    steps = [paged.PageStep(n_seq, 2000), paged.PageStep(n_seq, 2000)]
    for i in range(6):
        new = torch.randint(0, 7, (n_seq,), generator=g).tolist()
        want = ref.pages_append(lens, new, table, queue, state, page, 2000, most)
        step = paged.pages_append(cached, i32(new), tab, lst, fs, page_size=page, step=steps[i % 2])
        torch.cuda.synchronize()
        for name in ("q_start", "seq_kv_len", "status", "slots", "positions", "token_seq", "free_state"):
            assert getattr(step, name).tolist() == want[name], (i, name)
        assert tab.tolist() == want["table"]
        cached, fs, table, state, lens = step.seq_kv_len, step.free_state, want["table"], want["free_state"], want["seq_kv_len"]
        with pytest.raises(attn.AttnError, match="overlaps cached_len"):
            paged.pages_append(cached, i32(new), tab, lst, steps[(i + 1) % 2].free_state, page_size=page, step=step)


def test_arrays_one_behind_the_other():
    # no gap between them, and none overlaps
    cached, new, page, n_tokens = [5, 30, 0, 7], [1, 2, 20, 700], 16, 1000
    table, queue, state = _pool(cached, page, 90, 50, 12)
    want = ref.pages_append(cached, new, table, queue, state, page, n_tokens, 50)
    parts = {"free_in": i64(state), "free_out": i64([0, 0]), "slots": i64([0] * n_tokens), "cached": i32(cached),
             "new": i32(new), "table": i32(table), "list": i32(queue), "q_start": i32([0] * 5), "len": i32([0] * 4),
             "positions": i32([0] * n_tokens), "token_seq": i32([0] * n_tokens), "status": i32([0] * 4)}
    buf = torch.cat([t.reshape(-1).view(torch.int32) for t in parts.values()])
    at, views = 0, {}
    for name, t in parts.items():
        n = t.numel() * t.element_size() // 4
        views[name] = buf[at:at + n].view(t.dtype)
        at += n
    order = ("cached", "new", "table", "list", "free_in", "free_out", "q_start", "len", "slots", "positions", "token_seq",
             "status")
    desc = attn.PageDesc(4, n_tokens, page, 90, 50)
    rc = attn.load_library().pelica_attn_pages_append(ctypes.byref(desc), *[views[n].data_ptr() for n in order],
                                                      attn._stream_ptr(None))
    torch.cuda.synchronize()
    assert rc == 0
    for name, key in (("q_start", "q_start"), ("len", "seq_kv_len"), ("slots", "slots"), ("positions", "positions"),
                      ("token_seq", "token_seq"), ("status", "status"), ("free_out", "free_state")):
        assert views[name].tolist() == want[key], name
    assert views["table"].view(4, 50).tolist() == want["table"]
    for name in ("cached", "new", "list", "free_in"):
        assert torch.equal(views[name], parts[name].view(-1)), name
