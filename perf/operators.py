"""The operators of a paged-cache serving step, as timed cases.

Kinds of case (``draw`` varies each over the range it stands for):

  pages    one step's block tables, slots and positions from the requests'
           lengths: the pages of requests that ended go back to the free
           list, then every running request gets the pages its new tokens
           need.
  qkv      the step between the projections and attention: per-head norms,
           rotary positions on one or three axes (text, or time / height /
           width of an image), queries out, key and value rows into the pages.
  attend   attention of each request's new tokens over its pages: single
           tokens, drafts, prompt chunks, and mixed batches of these, for
           ``layers`` layers of one step (one plan, then a call a layer).
  score    the same with capped scores, a bias by distance, or a prefix that
           every token sees.
"""
import math
import random

import torch

own = False

PAIRS = {64: 32, 128: 64}


def listed():
    oss = {"n_head": 64, "n_kv": 8, "hd": 64}
    qwen = {"n_head": 32, "n_kv": 4, "hd": 128}
    plain = {"cap": 0.0, "bias": False, "prefix": 0}
    return [
        # eight chats of one token each: the smallest step there is
        {"name": "pages_8_chats", "kind": "pages", "n_seq": 8, "page": 16, "lo": 100, "hi": 4000, "new_lo": 1,
         "new_hi": 1, "chunks": 0, "ended": 0, "lens_seed": 1},
        # a busy server: 500 requests, some of them prompts being read in
        # chunks, some slots just freed
        {"name": "pages_500_mixed", "kind": "pages", "n_seq": 500, "page": 16, "lo": 1, "hi": 16384, "new_lo": 1,
         "new_hi": 4, "chunks": 14, "ended": 31, "lens_seed": 2},
        # 32 single tokens of a text model with q / k norms
        {"name": "qkv_32_tokens", "kind": "qkv", **qwen, "tokens": 32, "page": 16, "axes": 1, "norm": True,
         "half": False, "lens_seed": 3},
        # an image and its text: 4000 tokens with three position axes, f16
        # queries for the prompt attention
        {"name": "qkv_image_4000", "kind": "qkv", **qwen, "tokens": 4000, "page": 64, "axes": 3, "norm": True,
         "half": True, "lens_seed": 4},
        # 32 requests of very different lengths, one token each
        {"name": "tokens_32_ragged", "kind": "attend", **qwen, **plain, "page": 16, "n_seq": 32, "lo": 512,
         "hi": 16384, "new_lo": 1, "new_hi": 1, "chunks": 0, "chunk": 0, "window": 0, "sinks": False, "half": False,
         "layers": 4, "lens_seed": 5},
        # 64 requests on the 128-key window layers of gpt-oss
        {"name": "tokens_64_window", "kind": "attend", **oss, **plain, "page": 32, "n_seq": 64, "lo": 300, "hi": 8000,
         "new_lo": 1, "new_hi": 1, "chunks": 0, "chunk": 0, "window": 128, "sinks": True, "half": False, "layers": 6,
         "lens_seed": 6},
        # one long chat: a single token over 32K keys (full gpt-oss layers)
        {"name": "token_32k", "kind": "attend", **oss, **plain, "page": 64, "n_seq": 1, "lo": 32768, "hi": 32768,
         "new_lo": 1, "new_hi": 1, "chunks": 0, "chunk": 0, "window": 0, "sinks": True, "half": False, "layers": 4,
         "lens_seed": 7},
        # a 512-token chunk of a long prompt
        {"name": "chunk_512_at_30k", "kind": "attend", **oss, **plain, "page": 64, "n_seq": 1, "lo": 30512,
         "hi": 30512, "new_lo": 1, "new_hi": 1, "chunks": 1, "chunk": 512, "window": 0, "sinks": True, "half": True,
         "layers": 1, "lens_seed": 8},
        # a fresh prompt of 4001 tokens, head dim 128
        {"name": "prompt_4001", "kind": "attend", **qwen, **plain, "page": 16, "n_seq": 1, "lo": 4001, "hi": 4001,
         "new_lo": 1, "new_hi": 1, "chunks": 1, "chunk": 4001, "window": 0, "sinks": False, "half": True, "layers": 1,
         "lens_seed": 9},
        # continuous batching: 28 chats answer while three prompts are read
        {"name": "mixed_31", "kind": "attend", **oss, **plain, "page": 32, "n_seq": 31, "lo": 200, "hi": 9000,
         "new_lo": 1, "new_hi": 3, "chunks": 3, "chunk": 700, "window": 0, "sinks": True, "half": True, "layers": 1,
         "lens_seed": 10},
        # capped scores, and an image of 600 tokens that everyone sees
        {"name": "capped_prefix_2000", "kind": "score", **qwen, "cap": 50.0, "bias": False, "prefix": 600, "page": 16,
         "n_seq": 1, "lo": 2000, "hi": 2000, "new_lo": 1, "new_hi": 1, "chunks": 1, "chunk": 2000, "window": 0,
         "sinks": False, "half": True, "layers": 1, "lens_seed": 11},
        # a model whose heads discount far keys, 16 chats, f32 queries
        {"name": "biased_16_tokens", "kind": "score", "n_head": 16, "n_kv": 16, "hd": 128, "cap": 0.0, "bias": True,
         "prefix": 0, "page": 32, "n_seq": 16, "lo": 300, "hi": 6000, "new_lo": 1, "new_hi": 1, "chunks": 0,
         "chunk": 0, "window": 0, "sinks": False, "half": False, "layers": 2, "lens_seed": 12},
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("pages", "qkv", "attend", "attend", "score", "score"))
    c = {"kind": kind, "page": rng.choice((8, 16, 32, 64, 128)), "lens_seed": rng.randrange(1 << 20)}
    if kind == "pages":
        n = _log(rng, 1, 600)
        lo = _log(rng, 1, 2000)
        return {**c, "n_seq": n, "lo": lo, "hi": _log(rng, lo, 16384), "new_lo": 1, "new_hi": rng.choice((1, 1, 4, 8)),
                "chunks": rng.randrange(0, min(n, 16) + 1), "ended": rng.randrange(0, n // 4 + 1)}
    n_kv, hpk = rng.choice((1, 2, 3, 4, 8, 16)), rng.choice((1, 2, 3, 5, 8, 16))
    n_kv = min(n_kv, 64 // hpk)
    c.update(n_head=n_kv * hpk, n_kv=n_kv, hd=rng.choice((64, 128)))
    if kind == "qkv":
        return {**c, "tokens": _log(rng, 1, 4000), "axes": rng.choice((1, 3)), "norm": rng.random() < 0.5,
                "half": rng.random() < 0.5}
    c.update(cap=0.0, bias=False, prefix=0, layers=1, sinks=rng.random() < 0.5,
             window=rng.choice((0, 0, 0, _log(rng, 16, 2000))))
    if rng.random() < 0.5:  # single tokens or drafts
        n = _log(rng, 1, 64)
        hi = _log(rng, 16, 24000 if n <= 8 else 6000)
        c.update(n_seq=n, lo=max(8, hi // 8), hi=hi, new_lo=1, new_hi=rng.choice((1, 1, 2, 4)), chunks=0, chunk=0,
                 half=rng.random() < 0.3)
    else:
        n, chunk = _log(rng, 1, 12), _log(rng, 9, 2000)
        c.update(n_seq=n, lo=chunk + 8, hi=chunk + _log(rng, 9, 4000 - chunk), new_lo=1, new_hi=2, chunk=chunk,
                 chunks=rng.randrange(1, min(n, 3 if chunk < 500 else 1) + 1), half=rng.random() < 0.75)
    if kind == "score":
        c["cap"] = rng.choice((0.0, 20.0, 30.0, 50.0))
        c["bias"] = c["cap"] == 0.0 or rng.random() < 0.3
        c["prefix"] = rng.choice((0, _log(rng, 1, c["lo"])))
    return c


def _lens(c):
    """(cached keys, new tokens) of each request, by the case alone."""
    r = random.Random(c["lens_seed"])
    if c["kind"] == "pages":
        total = [_log(r, c["lo"], c["hi"]) for _ in range(c["n_seq"])]
        new = [r.randint(c["new_lo"], c["new_hi"]) for _ in total]
        for s in r.sample(range(c["n_seq"]), c["chunks"]):
            new[s] = r.randint(100, 600)
        for s in r.sample(range(c["n_seq"]), c["ended"]):
            new[s] = 0  # (its slot stays empty until the next step)
        return total, new
    total = [r.randint(c["lo"], c["hi"]) for _ in range(c["n_seq"])]
    new = [r.randint(c["new_lo"], c["new_hi"]) for _ in total]
    for s in r.sample(range(c["n_seq"]), c["chunks"]):
        new[s] = min(c["chunk"], total[s])
    return [a - b for a, b in zip(total, new)], new


def _up(a, b):
    return -(-a // b)


def _starts(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    i64 = lambda v: torch.tensor(v, dtype=torch.int64, device="cuda")  # noqa: E731
    st = {"c": c}
    if c["kind"] == "pages":
        cached, new = _lens(c)
        page, n_seq = c["page"], c["n_seq"]
        ended = {s for s, b in enumerate(new) if b == 0}
        held = [_up(a, page) for a in cached]
        most = max(_up(a + b, page) for a, b in zip(cached, new)) + 1
        n_pages = sum(held) + sum(_up(a + b, page) for a, b in zip(cached, new)) + 64
        order = torch.randperm(n_pages, generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
        start = i64(_starts(held))
        col = torch.arange(most, device="cuda")
        at = (start[:-1, None] + col).clamp(max=n_pages - 1)
        table = torch.where(col < i64(held)[:, None], order[at], torch.full_like(order[at], -1))
        # the list's queue: some pages were taken and given back before
        taken, free = int(seed) % 1000, n_pages - sum(held)
        lst = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
        lst[(taken + torch.arange(free, device="cuda")) % n_pages] = order[sum(held):]
        st.update(cached=i32(cached), kept=i32([0 if s in ended else a for s, a in enumerate(cached)]),
                  ended=i32([1 if s in ended else 0 for s in range(n_seq)]), new=i32(new), table=table, list=lst,
                  state=i64([taken, taken + free]), mid=torch.zeros(2, dtype=torch.int64, device="cuda"),
                  rows=sum(new) + 5)
        if own:
            from pelica_amd import paged

            st["step"] = paged.PageStep(n_seq, st["rows"], device="cuda")
        return st
    n_head, n_kv, hd, page = c["n_head"], c["n_kv"], c["hd"], c["page"]
    if c["kind"] == "qkv":
        T = c["tokens"]
        width = (n_head + 2 * n_kv) * hd
        n_pages = _up(T, page) + 8
        far = 40000  # positions reach this far
        freq = 10000.0 ** (-torch.arange(hd // 2, device="cuda", dtype=torch.float64) / (hd // 2))
        ang = torch.arange(far, device="cuda", dtype=torch.float64)[:, None] * freq
        table = torch.stack((ang.cos(), ang.sin()), -1).float()
        pos = torch.randint(0, far, (1,), generator=g, device="cuda") % (far - T - 1)
        base = pos + torch.arange(T, device="cuda")
        if c["axes"] == 3:  # an image of 40 columns, then text: time, height, width
            n_img = T * 2 // 3
            k = torch.arange(T, device="cuda")
            img = k < n_img
            base = torch.stack((torch.where(img, pos, base), torch.where(img, pos + k // 40, base),
                                torch.where(img, pos + k % 40, base)))
        else:
            base = base[None]
        slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:T].contiguous()
        if T > 1:  # rows of a page one after the other, as tokens come
            pages = torch.randperm(n_pages, generator=g, device="cuda")
            t = torch.arange(T, device="cuda")
            slots = pages[t // page] * page + t % page
        slots[T // 2] = -1 if T > 20 else slots[T // 2]  # a padding row
        half = hd // 2
        axis = [min(j % 3, 2) if c["axes"] == 3 and j < 3 * (half // 4) else 0 for j in range(half)]
        st.update(x=rnd(T, width), table=table, pos=base.to(torch.int32).contiguous(), slots=slots, axis=axis,
                  axis_t=i64(axis),
                  qn=torch.rand(hd, generator=g, device="cuda") + 0.5 if c["norm"] else None,
                  kn=torch.rand(hd, generator=g, device="cuda") + 0.5 if c["norm"] else None,
                  k=torch.zeros(n_pages, page, n_kv, hd, dtype=torch.float16, device="cuda"),
                  v=torch.zeros(n_pages, page, n_kv, hd, dtype=torch.float16, device="cuda"),
                  q=torch.zeros(T, n_head, hd, dtype=torch.float16 if c["half"] else torch.float32, device="cuda"))
        return st
    cached, new = _lens(c)
    total = [a + b for a, b in zip(cached, new)]
    held = [_up(a, page) for a in total]
    n_pages, most = sum(held) + 3, max(held)
    order = torch.randperm(n_pages, generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    col = torch.arange(most, device="cuda")
    at = (i64(_starts(held))[:-1, None] + col).clamp(max=n_pages - 1)
    table = torch.where(col < i64(held)[:, None], order[at], torch.full_like(order[at], -1))
    kv = lambda: (0.5 * rnd(c["layers"], n_pages, page, n_kv, hd)).to(torch.float16)  # noqa: E731
    q = rnd(c["layers"], sum(new), n_head, hd)
    st.update(total=total, new=new, start=i32(_starts(new)), len=i32(total), table=table, k=kv(), v=kv(),
              q=q.to(torch.float16) if c["half"] else q, out=None,
              sinks=rnd(n_head) if c["sinks"] else None,
              slopes=torch.exp2(-8 * (torch.arange(n_head, device="cuda") + 1) / n_head).float() if c["bias"] else None,
              prefix=i32([min(c["prefix"], a) for a in total]) if c["prefix"] else None)
    st["out"] = torch.zeros_like(st["q"])
    if own:
        from pelica_amd import paged

        st["plan"] = paged.PagedPlan(st["start"], st["len"], table, n_head=n_head, n_kv=n_kv, hd=hd, page_size=page,
                                     n_pages=n_pages, n_tokens=sum(new), max_q=max(new), window=c["window"],
                                     prefix_len=st["prefix"])
        st["ws"] = st["plan"].new_workspace()
    return st


def run(st):
    return _own(st) if own else _plain(st)


def _own(st):
    from pelica_amd import paged

    c = st["c"]
    if c["kind"] == "pages":
        if c["ended"]:
            paged.pages_release(st["ended"], st["cached"], st["table"], st["list"], st["state"], page_size=c["page"],
                                free_out=st["mid"])
        step = paged.pages_append(st["kept"], st["new"], st["table"], st["list"],
                                  st["mid"] if c["ended"] else st["state"], page_size=c["page"], step=st["step"])
        return {"start": step.q_start, "len": step.seq_kv_len, "slots": step.slots, "pos": step.positions,
                "seq": step.token_seq, "status": step.status, "state": step.free_state, "table": st["table"],
                "list": st["list"]}
    if c["kind"] == "qkv":
        n_head, n_kv, hd, x = c["n_head"], c["n_kv"], c["hd"], st["x"]
        T, a, b = x.shape[0], n_head * hd, (n_head + n_kv) * hd
        paged.paged_qkv(x[:, :a].view(T, n_head, hd), x[:, a:b].view(T, n_kv, hd), x[:, b:].view(T, n_kv, hd), st["k"],
                        st["v"], st["slots"], positions=st["pos"], table=st["table"], pair_axis=st["axis"],
                        q_norm=st["qn"], k_norm=st["kn"], out=st["q"])
        return {"q": st["q"], "k": st["k"], "v": st["v"]}
    st["plan"].update()
    for i in range(c["layers"]):
        paged.paged_attention(st["q"][i], st["k"][i], st["v"][i], st["plan"], sinks=st["sinks"], alibi=st["slopes"],
                              softcap=c["cap"], out=st["out"][i], workspace=st["ws"])
    return st["out"]


def _plain(st):
    c = st["c"]
    if c["kind"] == "pages":
        return _plain_pages(st)
    if c["kind"] == "qkv":
        return _plain_qkv(st)
    for i in range(c["layers"]):
        _plain_attention(st, i)
    return st["out"]


def _plain_pages(st):
    page, table, lst, n = st["c"]["page"], st["table"], st["list"], st["list"].numel()
    cached, kept, new = st["cached"].long(), st["kept"].long(), st["new"].long()
    col = torch.arange(table.shape[1], device=table.device)
    state = st["state"]
    if st["c"]["ended"]:
        back = (st["ended"] != 0)[:, None] & (col < ((cached + page - 1) // page)[:, None])
        rank = torch.cumsum(back.reshape(-1).long(), 0) - 1
        ext = torch.cat((lst, lst[:1]))  # what is not given back goes to the row behind
        ext[torch.where(back.reshape(-1), (state[1] + rank) % n, torch.full_like(rank, n))] = table.reshape(-1)
        lst.copy_(ext[:n])
        state = torch.stack((state[0], state[1] + back.sum()))
        st["mid"].copy_(state)
    have, want = (kept + page - 1) // page, (kept + new + page - 1) // page
    need = want - have
    first = torch.cumsum(need, 0) - need
    lacks = (first + need > state[1] - state[0]) & (need > 0)
    ok = ~lacks
    fresh = (col >= have[:, None]) & (col < want[:, None]) & ok[:, None]
    pick = lst[(state[0] + first[:, None] + col - have[:, None]) % n]
    table.copy_(torch.where(fresh, pick, table))
    start = torch.cat((torch.zeros_like(new[:1]), torch.cumsum(new, 0)))
    row = torch.arange(st["rows"], device=table.device)
    seq = torch.searchsorted(start, row, right=True) - 1
    live = seq < new.numel()
    s = seq.clamp(max=new.numel() - 1)
    pos = kept[s] + row - start[s]
    there = live & ok[s]
    slots = table[s, (pos // page).clamp(max=table.shape[1] - 1)].long() * page + pos % page
    return {"start": start.int(), "len": torch.where(ok, kept + new, torch.zeros_like(new)).int(),
            "slots": torch.where(there, slots, torch.full_like(slots, -1)),
            "pos": torch.where(live, pos, torch.zeros_like(pos)).int(),
            "seq": torch.where(live, seq, torch.full_like(seq, -1)).int(), "status": lacks.int(),
            "state": torch.stack((state[0] + (need * ok).sum(), state[1])), "table": table, "list": lst}


def _plain_qkv(st):
    c = st["c"]
    n_head, n_kv, hd, x = c["n_head"], c["n_kv"], c["hd"], st["x"]
    T, half = x.shape[0], hd // 2
    x = x.view(T, n_head + 2 * n_kv, hd)
    q, k, v = x[:, :n_head], x[:, n_head:n_head + n_kv], x[:, n_head + n_kv:]
    if c["norm"]:
        q = q / (q.square().mean(-1, keepdim=True) + 1e-6).sqrt() * st["qn"]
        k = k / (k.square().mean(-1, keepdim=True) + 1e-6).sqrt() * st["kn"]
    cs = st["table"][st["pos"].long()[st["axis_t"]].T, torch.arange(half, device=x.device)]  # [T, half, 2]
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    turn = lambda y: torch.cat((y[..., :half] * cos - y[..., half:] * sin,  # noqa: E731
                                y[..., half:] * cos + y[..., :half] * sin), -1)
    there = st["slots"] >= 0
    st["q"].copy_(torch.where(there[:, None, None], turn(q).to(st["q"].dtype), st["q"]))
    for dst, y in ((st["k"], turn(k)), (st["v"], v)):
        flat = dst.view(-1, n_kv, hd)
        at = torch.where(there, st["slots"], st["slots"].max())  # (a padding row writes what lies there)
        old = y[torch.argmax(st["slots"])]
        flat[at] = torch.where(there[:, None, None], y, old).to(torch.float16)
    return {"q": st["q"], "k": st["k"], "v": st["v"]}


def _plain_weights(st, s, pos, key, seen):
    """Softmax weights of scores s (scaled products); pos, key and seen broadcast to them, heads at dims -4, -3."""
    c = st["c"]
    hpk = c["n_head"] // c["n_kv"]
    if c["cap"]:
        s = c["cap"] * torch.tanh(s / c["cap"])
    if c["bias"]:
        s = s - st["slopes"].view(c["n_kv"], hpk, 1, 1) * (pos - key).abs()
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True)
    if st["sinks"] is not None:
        sink = st["sinks"].view(c["n_kv"], hpk, 1, 1)
        top = torch.maximum(top, sink)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    if st["sinks"] is not None:
        total = total + torch.exp(sink - top)
    return p / total


def _plain_attention(st, i):
    c = st["c"]
    n_head, n_kv, hd, page = c["n_head"], c["n_kv"], c["hd"], c["page"]
    hpk, window = n_head // n_kv, c["window"]
    k, v, q, out = (st[n][i] for n in ("k", "v", "q", "out"))
    k, v = k.view(-1, n_kv, hd), v.view(-1, n_kv, hd)
    if max(st["new"]) == 1 and not c["prefix"]:
        # every request's last keys, side by side
        n = min(window, max(st["total"])) if window else max(st["total"])
        ln = st["len"].long()[:, None]
        key = ln - n + torch.arange(n, device=q.device)
        at = key.clamp(min=0)
        rows = st["table"].gather(1, at // page).long() * page + at % page
        kk, vv = (x[rows].permute(0, 2, 1, 3).float() for x in (k, v))       # [n_seq, n_kv, n, hd]
        s = torch.matmul(q.float().view(-1, n_kv, hpk, hd), kk.transpose(2, 3).contiguous()) / math.sqrt(hd)
        key = key[:, None, None, None]
        p = _plain_weights(st, s[:, :, :, None], ln[:, None, None, None] - 1, key, key >= 0)[:, :, :, 0]
        out.copy_(torch.matmul(p, vv).view(-1, n_head, hd))
        return
    first = 0
    for r, (total, new) in enumerate(zip(st["total"], st["new"])):
        key = torch.arange(total, device=q.device)
        pos = key[total - new:, None]
        rows = st["table"][r].long()[key // page] * page + key % page
        kk, vv = (x[rows].permute(1, 0, 2).float() for x in (k, v))          # [n_kv, total, hd]
        qq = q[first:first + new].float().view(new, n_kv, hpk, hd).permute(1, 2, 0, 3).reshape(n_kv, hpk * new, hd)
        s = torch.matmul(qq, kk.transpose(1, 2).contiguous()).view(n_kv, hpk, new, total) / math.sqrt(hd)
        seen = key <= pos
        if window:
            seen = seen & (key > pos - window)
        if c["prefix"]:
            seen = seen | (key < st["prefix"][r])
        p = _plain_weights(st, s, pos, key, seen).view(n_kv, hpk * new, total)
        o = torch.matmul(p, vv).view(n_kv, hpk, new, hd).permute(2, 0, 1, 3)
        out[first:first + new] = o.reshape(new, n_head, hd)
        first += new


def work(case):
    c = case
    if c["kind"] == "pages":
        cached, new = _lens(c)
        moved = sum(_up(a + b, c["page"]) - _up(a, c["page"]) if b else _up(a, c["page"]) for a, b in zip(cached, new))
        return {"bytes": 8 * moved + 16 * sum(new) + 24 * c["n_seq"] + 32, "flops": 0}
    n_head, n_kv, hd = c["n_head"], c["n_kv"], c["hd"]
    if c["kind"] == "qkv":
        T, e = c["tokens"], 2 if c["half"] else 4
        row = (n_head + 2 * n_kv) * hd * 4 + n_head * hd * e + 2 * n_kv * hd * 2 + 8 + 4 * c["axes"]
        rows = (T - T * 2 // 3) + 3 if c["axes"] == 3 else T  # (rows of the rotary table, at least)
        return {"bytes": T * row + rows * hd * 4, "flops": T * (n_head + 2 * n_kv) * hd * 6}
    cached, new = _lens(c)
    keys = pairs = 0
    for a, n in zip(cached, new):
        total, w, pre = a + n, c["window"], min(c["prefix"], a + n)
        lo = max(0, a + 1 - w) if w else 0
        keys += total - lo + min(pre, lo)
        # of token t: its window's keys, and the prefix's before and behind them
        for t in range(n):
            pos = a + t
            l0 = max(0, pos + 1 - w) if w else 0
            pairs += pos + 1 - l0 + min(pre, l0) + max(0, pre - pos - 1)
    e = 2 if c["half"] else 4
    byt = keys * n_kv * hd * 4 + 2 * sum(new) * n_head * hd * e + 4 * _up(keys, c["page"]) + 8 * c["n_seq"]
    return {"bytes": c["layers"] * byt, "flops": c["layers"] * 4 * hd * n_head * pairs}


def exact(case, seed):
    """The definition in 64 bits, request by request (kv head by kv head for attention)."""
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    c = st["c"]
    if c["kind"] == "pages":
        return None
    n_head, n_kv, hd, page = c["n_head"], c["n_kv"], c["hd"], c["page"]
    if c["kind"] == "qkv":
        x = st["x"].double()
        T, half = x.shape[0], hd // 2
        z = st["table"].double()
        f = torch.complex(z[..., 0], z[..., 1])
        ax = st["axis"]
        ang = torch.stack([f[st["pos"][ax[j]].long(), j] for j in range(half)], 1)  # [T, half]
        heads = x.view(T, -1, hd)
        q, k = torch.zeros_like(st["q"], dtype=torch.float64), st["k"].double()
        v = st["v"].double()
        for h in range(n_head + 2 * n_kv):
            y = heads[:, h]
            w = st["qn"] if h < n_head else st["kn"] if h < n_head + n_kv else None
            if w is not None:
                y = y * torch.rsqrt((y * y).sum(-1, keepdim=True) / hd + 1e-6) * w.double()
            if h < n_head + n_kv:
                y = torch.complex(y[:, :half].contiguous(), y[:, half:].contiguous()) * ang
                y = torch.cat((y.real, y.imag), 1)
            there = st["slots"] >= 0
            if h < n_head:
                q[there, h] = y[there]
            else:
                dst = (k if h < n_head + n_kv else v).view(-1, n_kv, hd)
                dst[st["slots"][there], (h - n_head) % n_kv] = y[there]
        return {"q": q, "k": k, "v": v}
    hpk = n_head // n_kv
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    for layer in range(c["layers"]):
        first = 0
        for r, (total, new) in enumerate(zip(st["total"], st["new"])):
            j = torch.arange(total, device=out.device)
            ids = st["table"][r].long()[: _up(total, page)]
            i = torch.arange(total - new, total, device=out.device)
            d = i[:, None] - j[None]
            hide = d < 0
            if c["window"]:
                hide |= d >= c["window"]
            if c["prefix"]:
                hide &= j[None] >= min(c["prefix"], total)
            for h in range(n_kv):
                kk = st["k"][layer][ids, :, h].reshape(-1, hd)[:total].double()
                vv = st["v"][layer][ids, :, h].reshape(-1, hd)[:total].double()
                for g in range(h * hpk, (h + 1) * hpk):
                    s = st["q"][layer][first:first + new, g].double() @ kk.t().contiguous() * hd ** -0.5
                    if c["cap"]:
                        s = torch.tanh(s / c["cap"]) * c["cap"]
                    if c["bias"]:
                        s = s - st["slopes"][g].double() * d.abs()
                    s = s.masked_fill(hide, -math.inf)
                    z = torch.logsumexp(s, 1, keepdim=True)
                    if st["sinks"] is not None:
                        z = torch.logaddexp(z, st["sinks"][g].double())
                    out[layer, first:first + new, g] = torch.exp(s - z) @ vv
            first += new
    return out
