"""The operators of a quantised paged cache and of a shared prefix, as timed cases.

Kinds of case (``draw`` varies each over the range it stands for):

  write    the step between the projections and attention over an 8-bit cache:
           per-head norms, rotary positions on one or three axes, queries out,
           key and value rows quantised into the pages; the rows that were
           written are read back, as a host that moves requests away reads them.
  read     rows of an 8-bit cache as f16 rows, request by request: a request
           that leaves the pool, or a prefix handed to the dense kernels.
  attend   attention of each request's new tokens over an 8-bit cache: single
           tokens, drafts, prompt chunks, for ``layers`` layers of one step (one
           plan, then a call a layer).
  shared   attention of requests whose first pages are the same (a system
           prompt, a document that many ask about), over f16 or 8-bit pages.

An 8-bit row holds, for each 32 values, integers n in [-127, 127] and an f16
scale s, the smallest with 127 s >= the largest magnitude; it stands for the
f16 numbers n s.
"""
import math
import random

import torch

own = False

GROUP = 32  # values that share a scale


def listed():
    oss = {"n_head": 64, "n_kv": 8, "hd": 64}
    qwen = {"n_head": 32, "n_kv": 4, "hd": 128}
    tok = {"new_lo": 1, "new_hi": 1, "chunks": 0, "chunk": 0, "cap": 0.0, "window": 0}
    return [
        # 32 single tokens of a text model with q / k norms
        {"name": "write_32_tokens", "kind": "write", **qwen, "tokens": 32, "page": 16, "axes": 1, "norm": True,
         "half": False, "lens_seed": 1},
        # an image and its text: 4000 tokens with three position axes, f16
        # queries for the prompt attention
        {"name": "write_image_4000", "kind": "write", **qwen, "tokens": 4000, "page": 64, "axes": 3, "norm": True,
         "half": True, "lens_seed": 2},
        # a short chat leaves the pool
        {"name": "read_333", "kind": "read", **oss, "tokens": 333, "page": 16, "lens_seed": 3},
        # a long document's rows
        {"name": "read_30000", "kind": "read", **qwen, "tokens": 30000, "page": 32, "lens_seed": 4},
        # 32 requests of very different lengths, one token each
        {"name": "tokens_32_ragged", "kind": "attend", **qwen, **tok, "page": 16, "n_seq": 32, "lo": 512, "hi": 16384,
         "sinks": False, "half": False, "layers": 4, "lens_seed": 5},
        # 64 requests on the 128-key window layers of gpt-oss
        {"name": "tokens_64_window", "kind": "attend", **oss, **tok, "page": 32, "n_seq": 64, "lo": 300, "hi": 8000,
         "window": 128, "sinks": True, "half": False, "layers": 6, "lens_seed": 6},
        # one long chat: a single token over 32K keys (full gpt-oss layers)
        {"name": "token_32k", "kind": "attend", **oss, **tok, "page": 64, "n_seq": 1, "lo": 32768, "hi": 32768,
         "sinks": True, "half": False, "layers": 4, "lens_seed": 7},
        # a 512-token chunk of a long prompt
        {"name": "chunk_512_at_30k", "kind": "attend", **oss, **tok, "page": 64, "n_seq": 1, "lo": 30512, "hi": 30512,
         "chunks": 1, "chunk": 512, "sinks": True, "half": True, "layers": 1, "lens_seed": 8},
        # eight chats behind one system prompt
        {"name": "shared_8_chats", "kind": "shared", **qwen, **tok, "page": 16, "n_seq": 8, "groups": 1, "lone": 0,
         "shared": 2000, "lo": 20, "hi": 900, "q8": False, "sinks": False, "half": False, "layers": 4, "lens_seed": 9},
        # 64 readers of one document
        {"name": "shared_64_document", "kind": "shared", **oss, **tok, "page": 64, "n_seq": 64, "groups": 1, "lone": 0,
         "shared": 16384, "lo": 50, "hi": 1500, "q8": False, "sinks": True, "half": False, "layers": 2,
         "lens_seed": 10},
        # drafts of four tokens over an 8-bit document, f16 queries
        {"name": "shared_32_drafts", "kind": "shared", **oss, **tok, "new_lo": 4, "new_hi": 4, "page": 32, "n_seq": 32,
         "groups": 1, "lone": 0, "shared": 12000, "lo": 100, "hi": 2000, "q8": True, "sinks": True, "half": True,
         "layers": 2, "lens_seed": 11},
        # a server with three system prompts and requests that share nothing
        {"name": "shared_3_prompts", "kind": "shared", **qwen, **tok, "page": 16, "n_seq": 60, "groups": 3, "lone": 9,
         "shared": 5000, "lo": 30, "hi": 3000, "q8": False, "sinks": False, "half": True, "layers": 2,
         "lens_seed": 12},
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("write", "read", "attend", "attend", "shared", "shared"))
    c = {"kind": kind, "page": rng.choice((8, 16, 32, 64, 128)), "lens_seed": rng.randrange(1 << 20)}
    n_kv, hpk = rng.choice((1, 2, 3, 4, 8, 16)), rng.choice((1, 2, 3, 5, 8, 16))
    n_kv = min(n_kv, 64 // hpk)
    c.update(n_head=n_kv * hpk, n_kv=n_kv, hd=rng.choice((64, 128)))
    if kind == "write":
        return {**c, "tokens": _log(rng, 1, 4000), "axes": rng.choice((1, 3)), "norm": rng.random() < 0.5,
                "half": rng.random() < 0.5}
    if kind == "read":
        return {**c, "tokens": _log(rng, 1, 30000)}
    c.update(cap=rng.choice((0.0, 0.0, 0.0, 30.0, 50.0)), window=0, layers=1, sinks=rng.random() < 0.5,
             chunks=0, chunk=0, new_lo=1, new_hi=rng.choice((1, 1, 2, 4)))
    if kind == "shared":
        n = _log(rng, 2, 96)
        c.update(n_seq=n, groups=rng.randrange(1, min(n // 2, 4) + 1), lone=rng.randrange(0, n // 4 + 1),
                 shared=_log(rng, 20, min(16384, 400000 // n)), lo=rng.choice((4, 20, 100)),
                 hi=_log(rng, 101, min(4000, 100000 // n)), q8=rng.random() < 0.5, half=rng.random() < 0.5)
        return c
    c.update(window=rng.choice((0, 0, 0, _log(rng, 16, 2000))))
    if rng.random() < 0.6:  # single tokens or drafts
        n = _log(rng, 1, 64)
        hi = _log(rng, 16, 24000 if n <= 8 else 6000)
        c.update(n_seq=n, lo=max(8, hi // 8), hi=hi, half=rng.random() < 0.3)
    else:
        n, chunk = _log(rng, 1, 6), _log(rng, 9, 1500)
        c.update(n_seq=n, lo=chunk + 8, hi=chunk + _log(rng, 9, 3000 - chunk), new_hi=2, chunk=chunk,
                 chunks=rng.randrange(1, min(n, 2 if chunk < 500 else 1) + 1), half=rng.random() < 0.75)
    return c


def _lens(c):
    """Of each request: keys ahead of its new tokens, new tokens, keys it shares; and where groups begin."""
    r = random.Random(c["lens_seed"])
    n = c["n_seq"]
    total = [r.randint(c["lo"], c["hi"]) for _ in range(n)]
    new = [r.randint(c["new_lo"], c["new_hi"]) for _ in total]
    for s in r.sample(range(n), c["chunks"]):
        new[s] = min(c["chunk"], total[s])
    shared, first = [0] * n, list(range(n + 1))
    if c["kind"] == "shared":
        # groups of about equal size, then the requests that share nothing
        joint = n - c["lone"]
        cut = [joint * g // c["groups"] for g in range(c["groups"] + 1)]
        first = cut + list(range(joint + 1, n + 1))
        for a, b in zip(cut, cut[1:]):
            common = max(1, round(c["shared"] * r.uniform(0.6, 1.0)) // c["page"]) * c["page"]
            for s in range(a, b):
                shared[s] = common
    return [a - b + e for a, b, e in zip(total, new, shared)], new, shared, first


def _up(a, b):
    return -(-a // b)


def _starts(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def _scales(x):
    """The f16 scales of x [..., groups, 32] (f32 or f64)."""
    top = x.abs().amax(-1)
    s = (top / 127).to(torch.float16)
    low = s.to(top.dtype) * 127 < top
    return torch.where(low, s.view(torch.int16) + 1, s.view(torch.int16)).view(torch.float16)


def _quantise(x):
    """x [..., hd] as int8 values and f16 scales [..., hd / 32]."""
    y = x.unflatten(-1, (-1, GROUP))
    s = _scales(y)
    d = s.to(y.dtype).unsqueeze(-1)
    n = torch.where(d > 0, y / torch.where(d > 0, d, torch.ones_like(d)), torch.zeros_like(y))
    return n.round().clamp(-127, 127).to(torch.int8).flatten(-2), s


def _values(n, s):
    """The f16 numbers that int8 values and their scales stand for."""
    return (n.unflatten(-1, (-1, GROUP)).float() * s.float().unsqueeze(-1)).flatten(-2).to(torch.float16)


def _pool(layers, n_pages, page, n_kv, width, dtype):
    """Pages whose rows of one head lie side by side, as [layers, n_pages, page, n_kv, width]."""
    return torch.zeros(layers, n_pages, n_kv, page, width, dtype=dtype, device="cuda").transpose(2, 3)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    i64 = lambda v: torch.tensor(v, dtype=torch.int64, device="cuda")  # noqa: E731
    st = {"c": c}
    n_head, n_kv, hd, page = c["n_head"], c["n_kv"], c["hd"], c["page"]

    def cache(layers, n_pages, q8):
        """Random pages: [k, v, k scales, v scales]."""
        rows = [0.5 * rnd(layers, n_pages, n_kv, page, hd) for _ in range(2)]
        if not q8:
            return [x.to(torch.float16).transpose(2, 3) for x in rows] + [None, None]
        (k, ks), (v, vs) = (_quantise(x) for x in rows)
        return [x.transpose(2, 3) for x in (k, v, ks, vs)]

    if c["kind"] in ("write", "read"):
        T = c["tokens"]
        n_pages = _up(T, page) + 8
        # rows of a page one after the other, as tokens come; pages as they were free
        pages = torch.randperm(n_pages, generator=g, device="cuda")
        t = torch.arange(T, device="cuda")
        slots = pages[t // page] * page + t % page
        if T > 20:
            slots[T // 2] = -1  # a padding row
        st.update(slots=slots)
        if c["kind"] == "read":
            k, v, ks, vs = (x[0] for x in cache(1, n_pages, True))
            st.update(k=k, v=v, ks=ks, vs=vs)
        else:
            width = (n_head + 2 * n_kv) * hd
            far = 40000  # positions reach this far
            freq = 10000.0 ** (-torch.arange(hd // 2, device="cuda", dtype=torch.float64) / (hd // 2))
            ang = torch.arange(far, device="cuda", dtype=torch.float64)[:, None] * freq
            pos = torch.randint(0, far, (1,), generator=g, device="cuda") % (far - T - 1)
            base = (pos + t)[None]
            if c["axes"] == 3:  # an image of 40 columns, then text: time, height, width
                img = t < T * 2 // 3
                base = torch.cat((torch.where(img, pos, base), torch.where(img, pos + t // 40, base),
                                  torch.where(img, pos + t % 40, base)))
            half = hd // 2
            axis = [min(j % 3, 2) if c["axes"] == 3 and j < 3 * (half // 4) else 0 for j in range(half)]
            st.update(x=rnd(T, width), table=torch.stack((ang.cos(), ang.sin()), -1).float(),
                      pos=base.to(torch.int32).contiguous(), axis=axis, axis_t=i64(axis),
                      qn=torch.rand(hd, generator=g, device="cuda") + 0.5 if c["norm"] else None,
                      kn=torch.rand(hd, generator=g, device="cuda") + 0.5 if c["norm"] else None,
                      k=_pool(1, n_pages, page, n_kv, hd, torch.int8)[0],
                      v=_pool(1, n_pages, page, n_kv, hd, torch.int8)[0],
                      ks=_pool(1, n_pages, page, n_kv, hd // GROUP, torch.float16)[0],
                      vs=_pool(1, n_pages, page, n_kv, hd // GROUP, torch.float16)[0],
                      q=torch.zeros(T, n_head, hd, dtype=torch.float16 if c["half"] else torch.float32, device="cuda"))
        st["rows"] = [torch.zeros(T, n_kv, hd, dtype=torch.float16, device="cuda") for _ in range(2)]
        return st
    cached, new, shared, first = _lens(c)
    total = [a + b for a, b in zip(cached, new)]
    # each request's own pages, behind those of its group
    leader = {s: a for a, b in zip(first, first[1:]) for s in range(a, b)}
    held = [_up(a, page) - (e // page if leader[s] != s else 0) for s, (a, e) in enumerate(zip(total, shared))]
    start, most = _starts(held), max(_up(a, page) for a in total)
    n_pages = sum(held) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    col = torch.arange(most, device="cuda")
    lead = i64([leader[s] for s in range(len(total))])
    begin, common = i64(start)[:-1, None], i64([e // page if leader[s] != s else 0 for s, e in enumerate(shared)])[:, None]
    at = torch.where(col < common, begin[lead] + col, begin + col - common).clamp(max=n_pages - 1)
    table = torch.where(col < i64([_up(a, page) for a in total])[:, None], order[at], torch.full_like(order[at], -1))
    q8 = c["kind"] == "attend" or c["q8"]
    k, v, ks, vs = cache(c["layers"], n_pages, q8)
    q = rnd(c["layers"], sum(new), n_head, hd)
    st.update(total=total, new=new, start=i32(_starts(new)), len=i32(total), table=table, k=k, v=v, ks=ks, vs=vs,
              q=q.to(torch.float16) if c["half"] else q, sinks=rnd(n_head) if c["sinks"] else None,
              groups=i32(first), shared=i32([shared[a] for a in first[:-1]]))
    st["out"] = torch.zeros_like(st["q"])
    if own:
        from pelica_amd import paged

        more = dict(group_start=st["groups"], shared_len=st["shared"]) if c["kind"] == "shared" else {}
        st["plan"] = paged.PagedPlan(st["start"], st["len"], table, n_head=n_head, n_kv=n_kv, hd=hd, page_size=page,
                                     n_pages=n_pages, n_tokens=sum(new), max_q=max(new), window=c["window"], **more)
        st["ws"] = st["plan"].new_workspace()
    return st


def run(st):
    return _own(st) if own else _plain(st)


def _own(st):
    from pelica_amd import paged

    c = st["c"]
    scales = dict(k_scales=st["ks"], v_scales=st["vs"])
    if c["kind"] == "write":
        n_head, n_kv, hd, x = c["n_head"], c["n_kv"], c["hd"], st["x"]
        T, a, b = x.shape[0], n_head * hd, (n_head + n_kv) * hd
        paged.paged_qkv(x[:, :a].view(T, n_head, hd), x[:, a:b].view(T, n_kv, hd), x[:, b:].view(T, n_kv, hd), st["k"],
                        st["v"], st["slots"], **scales, positions=st["pos"], table=st["table"], pair_axis=st["axis"],
                        q_norm=st["qn"], k_norm=st["kn"], out=st["q"])
        paged.pages_read(st["k"], st["v"], st["slots"], **scales, out=st["rows"])
        return {"q": st["q"], "k": st["rows"][0], "v": st["rows"][1]}
    if c["kind"] == "read":
        paged.pages_read(st["k"], st["v"], st["slots"], **scales, out=st["rows"])
        return {"k": st["rows"][0], "v": st["rows"][1]}
    st["plan"].update()
    for i in range(c["layers"]):
        if st["ks"] is not None:
            scales = dict(k_scales=st["ks"][i], v_scales=st["vs"][i])
        paged.paged_attention(st["q"][i], st["k"][i], st["v"][i], st["plan"], **scales, sinks=st["sinks"],
                              softcap=c["cap"], out=st["out"][i], workspace=st["ws"])
    return st["out"]


def _plain(st):
    c = st["c"]
    if c["kind"] == "write":
        return _plain_write(st)
    if c["kind"] == "read":
        return _plain_read(st)
    for i in range(c["layers"]):
        _plain_attention(st, i)
    return st["out"]


def _plain_read(st):
    there = st["slots"] >= 0
    at = st["slots"].clamp(min=0)
    for out, n, s in zip(st["rows"], (st["k"], st["v"]), (st["ks"], st["vs"])):
        page = n.shape[1]
        y = _values(n[at // page, at % page], s[at // page, at % page])
        out.copy_(torch.where(there[:, None, None], y, out))
    return {"k": st["rows"][0], "v": st["rows"][1]}


def _plain_write(st):
    """In 64 bits: an integer next to the border between two is decided by the last bits."""
    c = st["c"]
    n_head, n_kv, hd, x = c["n_head"], c["n_kv"], c["hd"], st["x"].double()
    T, half = x.shape[0], hd // 2
    x = x.view(T, n_head + 2 * n_kv, hd)
    q, k, v = x[:, :n_head], x[:, n_head:n_head + n_kv], x[:, n_head + n_kv:]
    if c["norm"]:
        q = q / (q.square().mean(-1, keepdim=True) + 1e-6).sqrt() * st["qn"]
        k = k / (k.square().mean(-1, keepdim=True) + 1e-6).sqrt() * st["kn"]
    cs = st["table"][st["pos"].long()[st["axis_t"]].T, torch.arange(half, device=x.device)].double()  # [T, half, 2]
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    turn = lambda y: torch.cat((y[..., :half] * cos - y[..., half:] * sin,  # noqa: E731
                                y[..., half:] * cos + y[..., :half] * sin), -1)
    there = st["slots"] >= 0
    st["q"].copy_(torch.where(there[:, None, None], turn(q).to(st["q"].dtype), st["q"]))
    slots = torch.where(there, st["slots"], st["slots"].max())  # (a padding row writes what lies there)
    last = torch.argmax(st["slots"])
    for pages, scales, y in ((st["k"], st["ks"], turn(k)), (st["v"], st["vs"], v)):
        page = pages.shape[1]
        n, s = _quantise(torch.where(there[:, None, None], y, y[last]))
        pages[slots // page, slots % page] = n
        scales[slots // page, slots % page] = s
    rows = _plain_read(st)
    return {"q": st["q"], **rows}


def _plain_weights(st, s, seen):
    """Softmax weights of scores s [n_seq, n_kv, hpk, T, keys] (scaled products)."""
    c = st["c"]
    if c["cap"]:
        s = c["cap"] * torch.tanh(s / c["cap"])
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True)
    if st["sinks"] is not None:
        sink = st["sinks"].view(c["n_kv"], c["n_head"] // c["n_kv"], 1, 1)
        top = torch.maximum(top, sink)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    if st["sinks"] is not None:
        total = total + torch.exp(sink - top)
    return p / total


def _plain_attention(st, i):
    """All requests side by side, each request's last keys and (up to) T last tokens."""
    c = st["c"]
    n_head, n_kv, hd, page, window = c["n_head"], c["n_kv"], c["hd"], c["page"], c["window"]
    hpk, q, table = n_head // n_kv, st["q"][i], st["table"].long()
    T = max(st["new"])
    n = min(max(st["total"]), window + T - 1) if window else max(st["total"])
    start, ln = st["start"].long(), st["len"].long()
    new = start[1:] - start[:-1]
    key = ln[:, None] - n + torch.arange(n, device=q.device)                  # [n_seq, n]
    at = key.clamp(min=0)
    ids, at = table.gather(1, at // page), at % page
    k, v = st["k"][i][ids, at], st["v"][i][ids, at]                           # [n_seq, n, n_kv, hd]
    if st["ks"] is not None:
        k, v = _values(k, st["ks"][i][ids, at]), _values(v, st["vs"][i][ids, at])
    kk, vv = (x.permute(0, 2, 1, 3).float() for x in (k, v))
    t = torch.arange(T, device=q.device)
    tok = (start[:-1, None] + t).clamp(max=q.shape[0] - 1)
    qq = q[tok].float().view(-1, T, n_kv, hpk, hd).permute(0, 2, 3, 1, 4).reshape(-1, n_kv, hpk * T, hd)
    s = (torch.matmul(qq, kk.transpose(2, 3).contiguous()) / math.sqrt(hd)).view(-1, n_kv, hpk, T, n)
    pos = ((ln - new)[:, None] + t)[:, None, None, :, None]
    key = key[:, None, None, None]
    seen = (key <= pos) & (key >= 0)
    if window:
        seen = seen & (key > pos - window)
    p = _plain_weights(st, s, seen).view(-1, n_kv, hpk * T, n)
    o = torch.matmul(p, vv).view(-1, n_kv, hpk, T, hd).permute(0, 3, 1, 2, 4)  # [n_seq, T, n_kv, hpk, hd]
    row = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(start, row, right=True) - 1
    st["out"][i].copy_(o[seq, row - start[seq]].reshape(-1, n_head, hd))


def work(case):
    c = case
    n_head, n_kv, hd = c["n_head"], c["n_kv"], c["hd"]
    row8 = 2 * n_kv * (hd + 2 * hd // GROUP)  # K and V of a token in 8 bits
    if c["kind"] in ("write", "read"):
        T = c["tokens"]
        back = T * (row8 + 2 * n_kv * hd * 2 + 8)
        if c["kind"] == "read":
            return {"bytes": back, "flops": T * 2 * n_kv * hd}
        e = 2 if c["half"] else 4
        row = (n_head + 2 * n_kv) * hd * 4 + n_head * hd * e + row8 + 8 + 4 * c["axes"]
        rows = (T - T * 2 // 3) + 3 if c["axes"] == 3 else T  # (rows of the rotary table, at least)
        return {"bytes": T * row + rows * hd * 4 + back, "flops": T * (n_head + 2 * n_kv) * hd * 6}
    cached, new, shared, first = _lens(c)
    keys = pairs = 0
    leaders = set(first)
    for s, (a, n, e) in enumerate(zip(cached, new, shared)):
        w = c["window"]
        lo = max(0, a + 1 - w) if w else 0
        keys += a + n - (lo if s in leaders else max(lo, e))
        pairs += sum(min(a + t + 1, w) if w else a + t + 1 for t in range(n))
    e = 2 if c["half"] else 4
    row = row8 if c["kind"] == "attend" or c["q8"] else 2 * n_kv * hd * 2
    byt = keys * row + 2 * sum(new) * n_head * hd * e + 4 * _up(keys, c["page"]) + 8 * c["n_seq"]
    return {"bytes": c["layers"] * byt, "flops": c["layers"] * 4 * hd * n_head * pairs}


def _exact_row(x):
    """x [..., hd] in 64 bits as what an 8-bit row of it stands for, by the definition: the grid of f16 numbers between
    0 and the largest is searched for the scale."""
    y = x.reshape(-1, GROUP)
    top = y.abs().max(1).values
    # (every f16 number from 0 to the largest finite one, in order)
    grid = torch.arange(0x7C00, dtype=torch.int32, device=x.device).to(torch.int16).view(torch.float16).double()
    s = grid[torch.searchsorted(grid * 127, top)]
    n = torch.div(y, s.clamp(min=2.0 ** -24)[:, None]).round()
    return (n * s[:, None]).half().double().view(x.shape)


def exact(case, seed):
    """The definition in 64 bits, request by request (kv head by kv head for attention)."""
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    c = st["c"]
    n_head, n_kv, hd, page = c["n_head"], c["n_kv"], c["hd"], c["page"]

    def stored(name, scales, layer, slots, h):
        """Rows `slots` of head h of a cache, in 64 bits."""
        x = st[name] if layer is None else st[name][layer]
        y = x[slots // page, slots % page, h].double()
        if st[scales] is None:
            return y
        z = (st[scales] if layer is None else st[scales][layer])[slots // page, slots % page, h].double()
        return (y * z.repeat_interleave(GROUP, -1)).half().double()

    if c["kind"] in ("write", "read"):
        there = (st["slots"] >= 0).nonzero()[:, 0]
        k, v = (torch.zeros(x.shape, dtype=torch.float64, device=x.device) for x in st["rows"])
        if c["kind"] == "read":
            for h in range(n_kv):
                k[there, h] = stored("k", "ks", None, st["slots"][there], h)
                v[there, h] = stored("v", "vs", None, st["slots"][there], h)
            return {"k": k, "v": v}
        x = st["x"].double()
        T, half = x.shape[0], hd // 2
        z = st["table"].double()
        f = torch.complex(z[..., 0], z[..., 1])
        ang = torch.stack([f[st["pos"][a].long(), j] for j, a in enumerate(st["axis"])], 1)  # [T, half]
        heads = x.view(T, -1, hd)
        q = torch.zeros(st["q"].shape, dtype=torch.float64, device=x.device)
        for h in range(n_head + 2 * n_kv):
            y = heads[:, h]
            w = st["qn"] if h < n_head else st["kn"] if h < n_head + n_kv else None
            if w is not None:
                y = y * torch.rsqrt((y * y).sum(-1, keepdim=True) / hd + 1e-6) * w.double()
            if h < n_head + n_kv:
                y = torch.complex(y[:, :half].contiguous(), y[:, half:].contiguous()) * ang
                y = torch.cat((y.real, y.imag), 1)
            if h < n_head:
                q[there, h] = y[there]
            else:
                (k if h < n_head + n_kv else v)[there, (h - n_head) % n_kv] = _exact_row(y[there])
        return {"q": q, "k": k, "v": v}
    hpk = n_head // n_kv
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    for layer in range(c["layers"]):
        first = 0
        for r, (total, new) in enumerate(zip(st["total"], st["new"])):
            lo = max(0, total - new + 1 - c["window"]) if c["window"] else 0
            j = torch.arange(lo, total, device=out.device)
            slots = st["table"][r].long()[j // page] * page + j % page
            d = torch.arange(total - new, total, device=out.device)[:, None] - j
            hide = (d < 0) | (d >= c["window"]) if c["window"] else d < 0
            for h in range(n_kv):
                kk, vv = stored("k", "ks", layer, slots, h), stored("v", "vs", layer, slots, h)
                own_q = st["q"][layer][first:first + new, h * hpk:(h + 1) * hpk].double()
                s = own_q.transpose(0, 1).contiguous() @ kk.t().contiguous() * hd ** -0.5  # [hpk, new, keys]
                if c["cap"]:
                    s = torch.tanh(s / c["cap"]) * c["cap"]
                s = s.masked_fill(hide, -math.inf)
                z = torch.logsumexp(s, -1, keepdim=True)
                if st["sinks"] is not None:
                    z = torch.logaddexp(z, st["sinks"][h * hpk:(h + 1) * hpk, None, None].double())
                out[layer, first:first + new, h * hpk:(h + 1) * hpk] = (torch.exp(s - z) @ vv).transpose(0, 1)
            first += new
    return out
