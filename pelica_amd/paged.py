"""Serving many requests from a paged cache: pages and slots from the requests'
lengths, the rope and cache-row step, attention over the pages
(include/pelica_attn.h, "serving many requests from a paged cache").

A step of an engine, all of it on the GPU:

    pages_release(ended, cached, table, free_list, state, page_size=16, free_out=mid)
    step = pages_append(cached, new, table, free_list, mid, page_size=16, step=step)
    plan.update()                      # a PagedPlan over step.q_start, step.seq_kv_len and table
    for each layer:
        paged_qkv(q, k, v, k_pages, v_pages, step.slots, positions=step.positions, table=rope_table, out=q)
        paged_attention(q, k_pages, v_pages, plan, out=attn, workspace=ws)

Pages are f16 tensors [n_pages, page_size, n_kv, hd], in any layout whose hd
values are contiguous (a transposed [n_pages, n_kv, page_size, hd], or K and V
side by side in one buffer).  Every call runs on the current device, on
``stream`` or the current stream; errors are ``AttnError``.
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import Optional, Sequence

from . import attn
from .attn import EINVAL, AttnError, PagedDesc, PagedRope, PageDesc

__all__ = ["PagedPlan", "PageStep", "paged_attention", "paged_qkv", "pages_append", "pages_release", "pair_axes"]

#: most requests of one step (PELICA_ATTN_PAGED_MAX_SEQ)
MAX_SEQ = 4096

#: values of PageStep.status
PAGES_OK, PAGES_NONE, PAGES_TABLE, PAGES_ROWS, PAGES_LENGTH = range(5)


def _need(ok, message: str) -> None:
    if not ok:
        raise AttnError(EINVAL, message)


_device = None


def _check(name: str, t, dtype, dim: Optional[int] = None, dense: bool = True):
    """A tensor argument: its type, dims, layout, and that it is on the current device."""
    global _device
    if _device is None:
        import torch

        _device = torch._C._cuda_getDevice if torch.cuda.is_available() else lambda: -1
    if t.dtype is not dtype or not t.is_cuda or (dim is not None and t.dim() != dim) or (
            dense and not t.is_contiguous()) or t.get_device() != _device():
        raise AttnError(EINVAL, f"{name}: a {'contiguous ' if dense else ''}{dtype} tensor"
                                f"{'' if dim is None else f' of {dim} dims'} on the current device is needed, got "
                                f"{t.dtype} {tuple(t.shape)} strides {tuple(t.stride())} on {t.device}")
    return t


def _on(stream):
    """Tensors made under it belong to the stream the call runs on."""
    if stream is None:
        return contextlib.nullcontext()
    import torch

    return torch.cuda.stream(stream)


class PageStep:
    """What ``pages_append`` writes: ``q_start`` [n_seq + 1], ``seq_kv_len``
    and ``status`` [n_seq] int32, ``slots`` [n_tokens] int64, ``positions`` and
    ``token_seq`` [n_tokens] int32, ``free_state`` [2] int64.  Keep it over the
    steps (its addresses stay, for a captured step)."""

    def __init__(self, n_seq: int, n_tokens: int, device="cuda"):
        import torch

        i32 = dict(dtype=torch.int32, device=device)
        self.n_seq, self.n_tokens = n_seq, n_tokens
        self.q_start = torch.zeros(n_seq + 1, **i32)
        self.seq_kv_len = torch.zeros(n_seq, **i32)
        self.status = torch.zeros(n_seq, **i32)
        self.slots = torch.full((n_tokens,), -1, dtype=torch.int64, device=device)
        self.positions = torch.zeros(n_tokens, **i32)
        self.token_seq = torch.full((n_tokens,), -1, **i32)
        self.free_state = torch.zeros(2, dtype=torch.int64, device=device)
        self._out = tuple(t.data_ptr() for t in (self.free_state, self.q_start, self.seq_kv_len, self.slots,
                                                 self.positions, self.token_seq, self.status))


def _page_args(lens, page_table, free_list, free_state, page_size, n_tokens):
    import torch

    n_seq = page_table.shape[0]
    _check("page_table", page_table, torch.int32, 2)
    _check("free_list", free_list, torch.int32, 1)
    _check("free_state", free_state, torch.int64, 1)
    _need(free_state.numel() == 2, "free_state: two values")
    for name, t in lens:
        _check(name, t, torch.int32, 1)
        _need(t.numel() == n_seq, f"{name}: one value for each of the {n_seq} rows of page_table")
    return PageDesc(n_seq, n_tokens, page_size, free_list.numel(), page_table.shape[1])


def pages_append(cached_len, new_len, page_table, free_list, free_state, *, page_size: int,
                 step: Optional[PageStep] = None, n_tokens: Optional[int] = None, stream=None) -> PageStep:
    """Pages, slots and positions for ``new_len[s]`` more tokens of every
    request (pelica_attn_pages_append): int32 [n_seq] lengths, int32
    ``page_table`` [n_seq, max_pages] (appended to), int32 ``free_list``
    [n_pages] and its queue ends ``free_state`` int64 [2].  Returns ``step``, or
    a new PageStep of ``n_tokens`` rows; its ``free_state`` is the next call's
    (of another PageStep: a call's may not be its own input)."""
    if step is None:
        _need(n_tokens is not None, "n_tokens or step is needed")
        with _on(stream):
            step = PageStep(page_table.shape[0], n_tokens, page_table.device)
    _need(n_tokens is None or n_tokens == step.n_tokens, "n_tokens is the step's")
    desc = _page_args((("cached_len", cached_len), ("new_len", new_len)), page_table, free_list, free_state, page_size,
                      step.n_tokens)
    _need(step.n_seq == desc.n_seq, "step: made for another number of requests")
    _need(step.q_start.device == page_table.device, "step: on another device")
    lib = attn.load_library()
    attn._check(lib.pelica_attn_pages_append(ctypes.byref(desc), cached_len.data_ptr(), new_len.data_ptr(),
                                             page_table.data_ptr(), free_list.data_ptr(), free_state.data_ptr(),
                                             *step._out, attn._stream_ptr(stream)))
    return step


def pages_release(ended, cached_len, page_table, free_list, free_state, *, page_size: int, free_out=None,
                  stream=None):
    """Gives the pages of the requests with ``ended[s] != 0`` back to the free
    list (pelica_attn_pages_release).  Returns ``free_out``, the queue ends
    after it (int64 [2], another tensor than ``free_state``)."""
    import torch

    if free_out is None:
        with _on(stream):
            free_out = torch.empty_like(free_state)
    _check("free_out", free_out, torch.int64, 1)
    _need(free_out.numel() == 2, "free_out: two values")
    desc = _page_args((("ended", ended), ("cached_len", cached_len)), page_table, free_list, free_state, page_size, 1)
    lib = attn.load_library()
    attn._check(lib.pelica_attn_pages_release(ctypes.byref(desc), ended.data_ptr(), cached_len.data_ptr(),
                                              page_table.data_ptr(), free_list.data_ptr(), free_state.data_ptr(),
                                              free_out.data_ptr(), attn._stream_ptr(stream)))
    return free_out


def _pool(name, t, shape=None):
    """The strides of a pool of pages: (page, row, head)."""
    import torch

    _check(name, t, torch.float16, 4, dense=False)
    st = t.stride()
    _need(st[3] == 1 and (shape is None or t.shape == shape), f"{name}: [n_pages, page_size, n_kv, hd] pages whose hd "
          f"values are contiguous, alike for k and v; got {tuple(t.shape)} strides {tuple(st)}")
    # (a dim of one has no stride of its own)
    return st[0] if t.shape[0] > 1 else 0, st[1], st[2] if t.shape[2] > 1 else 0


def _pools(k_pages, v_pages):
    a, b = _pool("k_pages", k_pages), _pool("v_pages", v_pages, k_pages.shape)
    _need(a == b, f"k_pages and v_pages: one layout for both, got strides {a} and {b}")
    return a


def _rows(name, t, dim=3):
    """The stride of token rows [n, heads, hd] (0: dense)."""
    if t.is_contiguous():
        return 0
    st = t.stride()
    _need(st[2] == 1 and (t.shape[1] == 1 or st[1] == t.shape[2]),
          f"{name}: token rows need contiguous heads, got strides {tuple(st)}")
    return st[0]


class PagedPlan:
    """The work list of a step's attention (pelica_attn_paged_plan), made on
    the GPU from ``q_start`` [n_seq + 1], ``seq_kv_len`` [n_seq], ``page_table``
    [n_seq, max_pages] and ``prefix_len`` [n_seq] or None (int32): ``update``
    makes it again when these have new contents.  Layers that differ in
    ``window`` need a plan each.  ``n_tokens``: rows of q; ``max_q``: most new
    tokens of one request."""

    def __init__(self, q_start, seq_kv_len, page_table, *, n_head: int, n_kv: int, hd: int, page_size: int,
                 n_pages: int, n_tokens: int, max_q: int, window: int = 0, prefix_len=None, stream=None):
        import torch

        n_seq = page_table.shape[0]
        _check("page_table", page_table, torch.int32, 2)
        for name, t, n in (("q_start", q_start, n_seq + 1), ("seq_kv_len", seq_kv_len, n_seq),
                           ("prefix_len", prefix_len, n_seq)):
            if t is not None:
                _check(name, t, torch.int32, 1)
                _need(t.numel() == n, f"{name}: {n} values for the {n_seq} rows of page_table")
        self._keep = (q_start, seq_kv_len, page_table, prefix_len)
        self.desc = PagedDesc(n_head, n_kv, hd, n_seq, n_tokens, max_q, page_size, n_pages, page_table.shape[1],
                              window, q_start.data_ptr(), seq_kv_len.data_ptr(), page_table.data_ptr(),
                              attn._ptr(prefix_len))
        lib = attn.load_library()
        n = lib.pelica_attn_paged_plan_bytes(ctypes.byref(self.desc))
        if n == 0:
            raise AttnError(EINVAL, lib.pelica_attn_last_error().decode(errors="replace"))
        self.device = page_table.device
        with _on(stream):
            self.buffer = torch.empty(n, dtype=torch.uint8, device=self.device)
        self.workspace_bytes = lib.pelica_attn_paged_workspace_bytes(ctypes.byref(self.desc))
        self.update(stream)

    def update(self, stream=None) -> "PagedPlan":
        """Make the work list from the arrays' present contents."""
        _check("page_table", self._keep[2], self._keep[2].dtype)
        attn._check(attn.load_library().pelica_attn_paged_plan(ctypes.byref(self.desc), self.buffer.data_ptr(),
                                                               self.buffer.numel(), attn._stream_ptr(stream)))
        return self

    def new_workspace(self):
        """A workspace for calls with this plan (uninitialised)."""
        import torch

        return torch.empty(max(self.workspace_bytes, 16), dtype=torch.uint8, device=self.device)


def paged_attention(q, k_pages, v_pages, plan: PagedPlan, *, sinks=None, alibi=None, softcap: float = 0.0,
                    scale: Optional[float] = None, out=None, workspace=None, stream=None):
    """Attention of every request's new tokens over its pages.  q: f16
    (pelica_attn_paged) or f32 (pelica_attn_paged_f32, products to f32's
    precision) [n_tokens, n_head, hd], contiguous or token rows of a wider
    buffer; ``sinks`` f32 [n_head]; ``alibi`` f32 [n_head] slopes of the
    distance bias; ``softcap`` c: scores c tanh(s / c).  Returns q's type;
    rows of requests without tokens or with lengths that do not fit, and rows
    behind the last, are left as they were (undefined in a new ``out``)."""
    import torch

    d = plan.desc
    f32 = q.dtype is torch.float32
    _need(f32 or q.dtype is torch.float16, f"q: f16 or f32, got {q.dtype}")
    shape = (d.n_tokens, d.n_head, d.hd)
    _check("q", q, q.dtype, 3, dense=False)
    _need(q.shape == shape, f"q: {shape} as planned, got {tuple(q.shape)}")
    page, row, head = _pools(k_pages, v_pages)
    _need(k_pages.shape == (d.n_pages, d.page_size, d.n_kv, d.hd),
          f"k_pages: {(d.n_pages, d.page_size, d.n_kv, d.hd)} as planned, got {tuple(k_pages.shape)}")
    if out is None:
        with _on(stream):
            out = torch.empty(shape, dtype=q.dtype, device=q.device)
    else:
        _check("out", out, q.dtype, 3, dense=False)
        _need(out.shape == shape, f"out: {shape}, got {tuple(out.shape)}")
    for name, t in (("sinks", sinks), ("alibi", alibi)):
        if t is not None:
            _check(name, t, torch.float32, 1)
            _need(t.numel() == d.n_head, f"{name}: one value for each of the {d.n_head} heads")
    if plan.workspace_bytes and (workspace is None or workspace.numel() * workspace.element_size() < plan.workspace_bytes):
        with _on(stream):
            workspace = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=q.device)
    elif workspace is not None:
        _check("workspace", workspace, workspace.dtype)
    x = PagedDesc.from_buffer_copy(d)
    x.alibi = attn._ptr(alibi)
    x.page_stride, x.row_stride, x.head_stride = page, row, head
    x.q_token_stride, x.out_token_stride = _rows("q", q), _rows("out", out)
    x.scale, x.softcap = 0.0 if scale is None else float(scale), float(softcap)
    lib = attn.load_library()
    fn = lib.pelica_attn_paged_f32 if f32 else lib.pelica_attn_paged
    attn._check(fn(ctypes.byref(x), plan.buffer.data_ptr(), q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                   attn._ptr(sinks), out.data_ptr(), attn._ptr(workspace),
                   0 if workspace is None else workspace.numel() * workspace.element_size(),
                   attn._stream_ptr(stream)))
    return out


def pair_axes(sections: Sequence[int], interleaved: bool = False) -> list:
    """The axis of each rotation pair for ``sections`` pairs per axis: one
    axis after the other, or interleaved (pair j turns by axis j mod n while
    that axis has pairs left, else by axis 0)."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    n, half = len(sections), sum(sections)
    return [j % n if j // n < sections[j % n] else 0 for j in range(half)]


def paged_qkv(q, k, v, k_pages, v_pages, slots, *, positions=None, table=None, rot: int = 0, neox: bool = True,
              table_split: int = 0, pair_axis: Optional[Sequence[int]] = None, q_norm=None, k_norm=None,
              eps: float = 1e-6, out=None, stream=None):
    """The step before attention over pages (pelica_attn_paged_qkv): per-head
    RMS norm of q and k (when q_norm / k_norm are given), rope by ``positions``
    (int32 [n_tokens], or [n_axes, n_tokens] with ``pair_axis``: the axis of
    each pair, see ``pair_axes``) with the f32 cos/sin ``table`` [rows, rot/2,
    2], k and v rows to f16 rows ``slots`` (int64 [n_tokens]; negative: the row
    is skipped) of the pages.  q: f32 [n_tokens, n_head, hd], k, v: f32
    [n_tokens, n_kv, hd], contiguous or views into one buffer of token rows.
    Returns ``out`` (f32, may be q; or f16), by default a new f32 tensor (its
    skipped rows undefined)."""
    import torch

    for name, t in (("q", q), ("k", k), ("v", v)):
        _check(name, t, torch.float32, 3, dense=False)
    T, n_head, hd = q.shape
    n_kv = k.shape[1]
    _need(k.shape == v.shape == (T, n_kv, hd), f"k and v: [{T}, n_kv, {hd}], got {tuple(k.shape)} and {tuple(v.shape)}")
    page, row, head = _pools(k_pages, v_pages)
    _need(k_pages.shape[2:] == (n_kv, hd), f"k_pages: [n_pages, page_size, {n_kv}, {hd}], got {tuple(k_pages.shape)}")
    st = {_rows(name, t) for name, t in (("q", q), ("k", k), ("v", v))}
    _need(len(st) == 1, "q, k and v: all contiguous, or views into rows of one stride")
    _check("slots", slots, torch.int64, 1)
    _need(slots.numel() == T, f"slots: one for each of the {T} rows")
    if out is None:
        with _on(stream):
            out = torch.empty((T, n_head, hd), dtype=torch.float32, device=q.device)
    _need(out.dtype in (torch.float16, torch.float32), f"out: f16 or f32, got {out.dtype}")
    _check("out", out, out.dtype, 3, dense=False)
    _need(out.shape == q.shape, f"out: {tuple(q.shape)}, got {tuple(out.shape)}")
    for name, t in (("q_norm", q_norm), ("k_norm", k_norm)):
        if t is not None:
            _check(name, t, torch.float32, 1)
            _need(t.numel() == hd, f"{name}: {hd} weights")
    rp = None
    if table is not None:
        _check("table", table, torch.float32, 3)
        rot = rot or 2 * table.shape[1]
        _need(table.shape[1:] == (rot // 2, 2), f"table: [rows, {rot // 2}, 2], got {tuple(table.shape)}")
        _need(positions is not None, "positions are needed with a table")
        _check("positions", positions, torch.int32)
        _need(positions.dim() in (1, 2) and positions.shape[-1] == T, f"positions: [{T}] or [n_axes, {T}]")
        n_axes = positions.shape[0] if positions.dim() == 2 else 1
        _need(n_axes == 1 or pair_axis is not None, "pair_axis is needed with more than one axis")
        axes = None
        if pair_axis is not None:
            _need(len(pair_axis) == rot // 2 and all(0 <= a < n_axes for a in pair_axis),
                  f"pair_axis: an axis below {n_axes} for each of the {rot // 2} pairs")
            axes = bytes(pair_axis)
        rp = PagedRope(rot, 1 if neox else 0, table_split, table.shape[0], table.data_ptr(), n_axes, axes,
                       positions.data_ptr(), T)
    d = PagedDesc(n_head=n_head, n_kv=n_kv, hd=hd, n_tokens=T, page_size=k_pages.shape[1], n_pages=k_pages.shape[0],
                  page_stride=page, row_stride=row, head_stride=head)
    attn._check(attn.load_library().pelica_attn_paged_qkv(
        ctypes.byref(d), None if rp is None else ctypes.byref(rp), q.data_ptr(), k.data_ptr(), v.data_ptr(), st.pop(),
        attn._ptr(q_norm), attn._ptr(k_norm), eps, slots.data_ptr(), out.data_ptr(),
        1 if out.dtype is torch.float16 else 0, _rows("out", out), k_pages.data_ptr(), v_pages.data_ptr(),
        attn._stream_ptr(stream)))
    return out
