"""Plain 64-bit definitions of the paged operators, on the CPU, and the error
bounds that their kernels' roundings allow."""
from __future__ import annotations

import math

import torch

U16, U32 = 2.0 ** -11, 2.0 ** -24  # half a step of f16 / f32, relative


def attention(q, k_pages, v_pages, table, lens, new, *, page, window=0, prefix=None, sinks=None, slopes=None, cap=0.0,
              scale=None, cap_off=2 ** -21):
    """q [rows, n_head, hd], pages [n_pages, page, n_kv, hd], table a list of
    page lists, in f64.  Returns (out, bound): the rows of requests with
    tokens, NaN elsewhere, and how far a kernel may be off per value, split
    into (f32 part, f16 part)."""
    n_head, hd = q.shape[1:]
    n_kv = k_pages.shape[2]
    hpk = n_head // n_kv
    scale = 1 / math.sqrt(hd) if scale is None else scale
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    f32 = torch.zeros_like(out)
    f16 = torch.zeros_like(out)
    row = 0
    for s, (n, t) in enumerate(zip(lens, new)):
        if t == 0 or n < t:
            row += t
            continue
        rows = torch.tensor([table[s][j // page] * page + j % page for j in range(n)])
        pos = torch.arange(n - t, n)[:, None]
        key = torch.arange(n)[None]
        seen = key <= pos
        if window:
            seen &= key > pos - window
        if prefix is not None:
            seen |= key < prefix[s]
        # keys no token sees may sit in pages that are gone (-1), or be NaN
        live = seen.any(0)
        rows = torch.where(live, rows, torch.zeros_like(rows))
        kk = k_pages.reshape(-1, n_kv, hd)[rows].double()
        vv = v_pages.reshape(-1, n_kv, hd)[rows].double()
        kk[~live] = 0
        vv[~live] = 0
        for h in range(n_head):
            qq, kh, vh = q[row:row + t, h].double(), kk[:, h // hpk], vv[:, h // hpk]
            raw = qq @ kh.T * scale
            x = cap * torch.tanh(raw / cap) if cap else raw
            if slopes is not None:
                x = x - slopes[h].double() * (pos - key).abs()
            x = x.masked_fill(~seen, -math.inf)
            m = x.amax(1, keepdim=True)
            if sinks is not None:
                m = torch.maximum(m, sinks[h].double())
            p = torch.exp(x - m)
            den = p.sum(1, keepdim=True)
            if sinks is not None:
                den = den + torch.exp(sinks[h].double() - m)
            p = p / den
            out[row:row + t, h] = p @ vh
            a = p @ vh.abs()
            # a score's error (natural log): the product's hd roundings, those
            # of its scaling, bias and cap, and q's hi + lo parts (2^-22)
            dot = (qq.abs() @ kh.abs().T * scale).amax(1, keepdim=True)
            big = torch.where(seen, x, torch.zeros_like(x)).abs().amax(1, keepdim=True)
            dx = dot * ((hd + 4) * U32 + 2 ** -22) + big * 8 * U32 + cap * cap_off
            # weights are off by that twice (numerator, denominator), 2^-22 of
            # exp2 and of p's parts, and every f32 sum by a rounding a key
            f32[row:row + t, h] = a * (2 * dx + 2 ** -20 + 2 * n * U32)
            # f16: every p is rounded (in sum and product alike), and the output;
            # below 2^-14 a step of p is 2^-24 however small p, the rows' largest is >= 2^-14
            f16[row:row + t, h] = 2 * U16 * a + U16 * out[row:row + t, h].abs() + 2 ** -24 * vh.abs().sum(0) + 2 ** -25
        row += t
    return out, f32, f16


def check(got, ref, f32, f16=None):
    """``got`` where ``ref`` is a number; nothing is said of the rest."""
    got = got.detach().cpu().double()
    there = ~ref.isnan()
    assert got[there].isfinite().all(), "not finite"
    tol = f32 + (f16 if f16 is not None else 0)
    off = (got - ref).abs()[there] / tol[there].clamp(min=1e-300)
    assert off.numel() and off.max() <= 1, f"off by {off.max():.3g} of what roundings allow"


def rope(x, table, positions, pair_axis, rot, neox):
    """x [rows, heads, hd] f64, table [positions, rot/2, 2], positions [axes, rows]."""
    half = rot // 2
    y = x.clone()
    for j in range(half):
        cs = table[positions[pair_axis[j]].long(), j].double()
        c, s = cs[:, None, 0], cs[:, None, 1]
        a, b = (j, j + half) if neox else (2 * j, 2 * j + 1)
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def norm(x, w, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()


def pages_append(cached, new, table, free_list, state, page, n_tokens, max_pages):
    """Python lists in, a dict of lists out."""
    n_pages = len(free_list)
    taken, given = state
    table = [list(r) for r in table]
    q_start, lens, status = [0], [], []
    slots, positions, seqs = [-1] * n_tokens, [0] * n_tokens, [-1] * n_tokens
    at, dry, row = taken, False, 0
    for s, (c, n) in enumerate(zip(cached, new)):
        st = 0
        if c < 0 or n < 0 or c + n > 2 ** 31 - 1:
            st = 4
        rows = max(n, 0)
        pos0 = 0 if st == 4 else c
        have, want = -(-pos0 // page), -(-(pos0 + rows) // page)
        if st == 0 and want > max_pages:
            st = 2
        if st == 0 and rows and row + rows > n_tokens:
            st = 3
        need = want - have if st == 0 else 0
        if st == 0 and need and (dry or at + need > given):
            st, dry = 1, True
        if st == 0:
            for j in range(have, want):
                table[s][j] = free_list[at % n_pages]
                at += 1
        for i in range(rows):
            if row + i < n_tokens:
                seqs[row + i], positions[row + i] = s, pos0 + i
                if st == 0:
                    j = (pos0 + i) // page
                    p = table[s][j]
                    slots[row + i] = p * page + (pos0 + i) % page if 0 <= p < n_pages else -1
        row += rows
        q_start.append(min(row, n_tokens))
        lens.append(c + n if st == 0 else 0)
        status.append(st)
    return dict(q_start=q_start, seq_kv_len=lens, status=status, slots=slots, positions=positions, token_seq=seqs,
                free_state=[at, given], table=table)
