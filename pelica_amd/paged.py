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

With 8-bit pages (``new_q8_pages``) the last two take ``k_scales`` and
``v_scales``, and ``pages_read`` gives rows back as f16 ones.  Requests that begin
with the same pages are groups of their PagedPlan (``group_start``, ``shared_len``).

Pages are f16 tensors [n_pages, page_size, n_kv, hd] (8-bit ones int8, with f16
scales [n_pages, page_size, n_kv, hd / 32]), in any layout whose hd
values are contiguous (a transposed [n_pages, n_kv, page_size, hd], or K and V
side by side in one buffer); an expanded dim (stride 0) is refused, of token
rows too.  Every call runs on the current device, on
``stream`` or the current stream; errors are ``AttnError``.
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import Optional, Sequence

from . import attn
from .attn import EINVAL, AttnError, PagedDesc, PagedQ8, PagedRope, PagedShared, PageDesc

__all__ = ["PagedPlan", "PageStep", "new_q8_pages", "paged_attention", "paged_qkv", "pages_append", "pages_read",
           "pages_release", "pair_axes"]

#: most requests of one step (PELICA_ATTN_PAGED_MAX_SEQ)
MAX_SEQ = 4096

#: values of an 8-bit row that share a scale
GROUP = 32

#: values of PageStep.status
PAGES_OK, PAGES_NONE, PAGES_TABLE, PAGES_ROWS, PAGES_LENGTH = range(5)


def _need(ok, message: str) -> None:
    if not ok:
        raise AttnError(EINVAL, message)


_torch = None
_device = None  # () -> the current device's index


def _start():
    """The names that a call looks up."""
    global _torch, _device
    import torch

    # (without a GPU: a device no tensor is on; those of the host are on -1)
    _device = torch._C._cuda_getDevice if torch.cuda.is_available() else lambda: -2
    _torch = torch
    return torch


def _check(name: str, t, dtype, dim: Optional[int] = None, dense: bool = True):
    """A tensor argument: its type, dims, layout, and that it is on the current device."""
    if _torch is None:
        _start()
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
    steps (its addresses stay, for a captured step).  None of them may be an
    input of the call that writes them: to pass ``seq_kv_len`` on as the next
    call's ``cached_len``, take two PageSteps in turn.  Made on the current
    stream."""

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
        self.device = self.slots.get_device()
        self._out = tuple(t.data_ptr() for t in (self.free_state, self.q_start, self.seq_kv_len, self.slots,
                                                 self.positions, self.token_seq, self.status))


def _pages_ok(dev, n_seq, a, b, page_table, free_list, free_state) -> bool:
    i32 = _torch.int32
    return (a.dtype is i32 and b.dtype is i32 and page_table.dtype is i32 and free_list.dtype is i32
            and free_state.dtype is _torch.int64 and a.get_device() == dev and b.get_device() == dev
            and page_table.get_device() == dev and free_list.get_device() == dev and free_state.get_device() == dev
            and a.dim() == 1 and b.dim() == 1 and free_list.dim() == 1 and a.numel() == n_seq and b.numel() == n_seq
            and free_state.numel() == 2 and a.is_contiguous() and b.is_contiguous() and page_table.is_contiguous()
            and free_list.is_contiguous() and free_state.is_contiguous())


def _refuse_pages(lens, page_table, free_list, free_state):
    """Names what is wrong with the arguments of a call over pages."""
    import torch

    _check("page_table", page_table, torch.int32, 2)
    _check("free_list", free_list, torch.int32, 1)
    _check("free_state", free_state, torch.int64, 1)
    _need(free_state.numel() == 2, "free_state: two values")
    for name, t in lens:
        _check(name, t, torch.int32, 1)
        _need(t.numel() == page_table.shape[0], f"{name}: one value for each of the {page_table.shape[0]} rows of page_table")
    raise AttnError(EINVAL, "arguments of a call over pages")


def pages_append(cached_len, new_len, page_table, free_list, free_state, *, page_size: int,
                 step: Optional[PageStep] = None, n_tokens: Optional[int] = None, stream=None) -> PageStep:
    """Pages, slots and positions for ``new_len[s]`` more tokens of every
    request (pelica_attn_pages_append): int32 [n_seq] lengths, int32
    ``page_table`` [n_seq, max_pages] (appended to), int32 ``free_list``
    [n_pages] and its queue ends ``free_state`` int64 [2].  Returns ``step``, or
    a new PageStep of ``n_tokens`` rows; its ``free_state`` is the next call's
    (of another PageStep: a call's outputs may not be its inputs)."""
    if _torch is None:
        _start()
    _need(page_table.dim() == 2, "page_table: [n_seq, max_pages]")
    n_seq, max_pages = page_table.shape
    dev = _device()
    if not _pages_ok(dev, n_seq, cached_len, new_len, page_table, free_list, free_state):
        _refuse_pages((("cached_len", cached_len), ("new_len", new_len)), page_table, free_list, free_state)
    if step is None:
        _need(n_tokens is not None, "n_tokens or step is needed")
        with _on(stream):
            step = PageStep(n_seq, n_tokens, page_table.device)
    if step.n_seq != n_seq or step.device != dev or not (n_tokens is None or n_tokens == step.n_tokens):
        raise AttnError(EINVAL, f"step: made for {step.n_seq} requests and {step.n_tokens} rows on device {step.device}, "
                                f"called with {n_seq}, {n_tokens} on {dev}")
    desc = PageDesc(n_seq, step.n_tokens, page_size, free_list.numel(), max_pages)
    lib = attn._lib or attn.load_library()
    rc = lib.pelica_attn_pages_append(ctypes.byref(desc), cached_len.data_ptr(), new_len.data_ptr(),
                                      page_table.data_ptr(), free_list.data_ptr(), free_state.data_ptr(), *step._out,
                                      attn._stream_ptr(stream))
    if rc:
        attn._check(rc)
    return step


def pages_release(ended, cached_len, page_table, free_list, free_state, *, page_size: int, free_out=None,
                  stream=None):
    """Gives the pages of the requests with ``ended[s] != 0`` back to the free
    list (pelica_attn_pages_release).  Returns ``free_out``, the queue ends
    after it (int64 [2], another tensor than ``free_state``)."""
    if _torch is None:
        _start()
    _need(page_table.dim() == 2, "page_table: [n_seq, max_pages]")
    n_seq, max_pages = page_table.shape
    if not _pages_ok(_device(), n_seq, ended, cached_len, page_table, free_list, free_state):
        _refuse_pages((("ended", ended), ("cached_len", cached_len)), page_table, free_list, free_state)
    if free_out is None:
        with _on(stream):
            free_out = _torch.empty_like(free_state)
    _check("free_out", free_out, _torch.int64, 1)
    _need(free_out.numel() == 2, "free_out: two values")
    desc = PageDesc(n_seq, 1, page_size, free_list.numel(), max_pages)
    lib = attn._lib or attn.load_library()
    rc = lib.pelica_attn_pages_release(ctypes.byref(desc), ended.data_ptr(), cached_len.data_ptr(),
                                       page_table.data_ptr(), free_list.data_ptr(), free_state.data_ptr(),
                                       free_out.data_ptr(), attn._stream_ptr(stream))
    if rc:
        attn._check(rc)
    return free_out


def _pools(k_pages, v_pages, dev, dtype=None, names=("k_pages", "v_pages"), last="hd"):
    """The strides of both pools of pages and their shape: page, row, head, shape."""
    st, shape = k_pages.stride(), k_pages.shape
    dtype = dtype or _torch.float16
    if not (k_pages.dtype is dtype and v_pages.dtype is dtype and len(st) == 4 and st[3] == 1
            and v_pages.stride() == st and shape == v_pages.shape and k_pages.get_device() == dev
            and v_pages.get_device() == dev and (0 not in st or all(s or n == 1 for s, n in zip(st, shape)))):
        for name, t in zip(names, (k_pages, v_pages)):
            _check(name, t, dtype, 4, dense=False)
        raise AttnError(EINVAL, f"{names[0]} and {names[1]}: [n_pages, page_size, n_kv, {last}] pages whose {last} values are "
                                f"contiguous, no stride of 0, one layout for both; got {tuple(k_pages.shape)} strides "
                                f"{tuple(st)} and {tuple(v_pages.shape)} strides {tuple(v_pages.stride())}")
    # (a dim of one has no stride of its own)
    return st[0] if shape[0] > 1 else 0, st[1], st[2] if shape[2] > 1 else 0, shape


def _q8_pools(k_pages, v_pages, k_scales, v_scales, dev):
    """Both pools' strides and shape as of ``_pools``, and their scales
    (PagedQ8; None for f16 pages, which come without)."""
    if k_scales is None and v_scales is None:
        return (*_pools(k_pages, v_pages, dev), None)
    _need(k_scales is not None and v_scales is not None, "k_scales and v_scales come together")
    st, shape, at, size = k_pages.stride(), k_pages.shape, k_scales.stride(), k_scales.shape
    i8, f16 = _torch.int8, _torch.float16
    if not (k_pages.dtype is i8 and v_pages.dtype is i8 and k_scales.dtype is f16 and v_scales.dtype is f16
            and len(st) == 4 and len(at) == 4 and st[3] == 1 and at[3] == 1 and v_pages.stride() == st
            and v_scales.stride() == at and v_pages.shape == shape and v_scales.shape == size
            and size[0] == shape[0] and size[1] == shape[1] and size[2] == shape[2] and size[3] * GROUP == shape[3]
            and k_pages.get_device() == dev and v_pages.get_device() == dev and k_scales.get_device() == dev
            and v_scales.get_device() == dev and 0 not in st and 0 not in at):
        # (names what is wrong; a dim of one may have a stride of 0)
        _pools(k_pages, v_pages, dev, i8)
        _pools(k_scales, v_scales, dev, None, ("k_scales", "v_scales"), "hd / 32")
        if size[:3] != shape[:3] or size[3] * GROUP != shape[3]:
            raise AttnError(EINVAL, f"k_scales: one for each {GROUP} values of the pages {tuple(shape)}, got {tuple(size)}")
    many, heads = shape[0] > 1, shape[2] > 1
    return (st[0] if many else 0, st[1], st[2] if heads else 0, shape,
            PagedQ8(k_scales.data_ptr(), v_scales.data_ptr(), at[0] if many else 0, at[1], at[2] if heads else 0))


def _weights(name, t, n, dev):
    """The address of a norm's ``n`` weights."""
    if not (t.dtype is _torch.float32 and t.get_device() == dev and t.shape == (n,) and t.is_contiguous()):
        _check(name, t, _torch.float32, 1)
        raise AttnError(EINVAL, f"{name}: {n} weights")
    return t.data_ptr()


def _per_head(name, t, n, dev):
    """The address of ``n`` heads' values."""
    if not (t.dtype is _torch.float32 and t.get_device() == dev and t.dim() == 1 and t.numel() == n and t.is_contiguous()):
        _check(name, t, _torch.float32, 1)
        raise AttnError(EINVAL, f"{name}: one value for each of the {n} heads")
    return t.data_ptr()


def _rows(name, t):
    """The stride of token rows [n, heads, hd] (0: dense)."""
    if t.is_contiguous():
        return 0
    st = t.stride()
    _need(st[2] == 1 and (t.shape[1] == 1 or st[1] == t.shape[2]) and st[0] > 0,
          f"{name}: token rows need contiguous heads and rows of their own, got strides {tuple(st)}")
    return st[0]


class PagedPlan:
    """The work list of a step's attention (pelica_attn_paged_plan), made on
    the GPU from ``q_start`` [n_seq + 1], ``seq_kv_len`` [n_seq], ``page_table``
    [n_seq, max_pages] and ``prefix_len`` [n_seq] or None (int32): ``update``
    makes it again when these have new contents.  Layers that differ in
    ``window`` need a plan each.  ``n_tokens``: rows of q; ``max_q``: most new
    tokens of one request.

    ``group_start`` [n_groups + 1] and ``shared_len`` [n_groups] (int32,
    together): requests ``group_start[g]`` .. ``group_start[g + 1]`` share their
    first ``shared_len[g]`` keys, which lie in the same pages (PelicaPagedShared):
    the plan walks those once for the whole group (no ``window``, ``prefix_len``
    or alibi).  Worth it for single tokens and drafts from about 4000 shared keys on,
    or 32 requests and 1000; not for few short ones, or prompts' chunks.  Its
    ``workspace_bytes`` grow with ``n_tokens``."""

    _shared = None

    def __init__(self, q_start, seq_kv_len, page_table, *, n_head: int, n_kv: int, hd: int, page_size: int,
                 n_pages: int, n_tokens: int, max_q: int, window: int = 0, prefix_len=None, group_start=None, shared_len=None,
                 stream=None):
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
        if group_start is not None or shared_len is not None:
            _need(group_start is not None and shared_len is not None, "group_start and shared_len come together")
            _check("group_start", group_start, torch.int32, 1)
            _check("shared_len", shared_len, torch.int32, 1)
            _need(group_start.numel() == shared_len.numel() + 1,
                  f"group_start: {shared_len.numel() + 1} values for {shared_len.numel()} groups, got {group_start.numel()}")
            self._keep += (group_start, shared_len)
            self._shared = PagedShared(shared_len.numel(), group_start.data_ptr(), shared_len.data_ptr())
        lib = attn.load_library()
        args = (ctypes.byref(self.desc),) if self._shared is None else (ctypes.byref(self.desc), ctypes.byref(self._shared))
        n = (lib.pelica_attn_paged_plan_bytes if self._shared is None else lib.pelica_attn_paged_shared_plan_bytes)(*args)
        if n == 0:
            raise AttnError(EINVAL, lib.pelica_attn_last_error().decode(errors="replace"))
        self.device = page_table.device
        self._dev = page_table.get_device()
        self._q_shape = (n_tokens, n_head, hd)
        self._page_shape = (n_pages, page_size, n_kv, hd)
        with _on(stream):
            self.buffer = torch.empty(n, dtype=torch.uint8, device=self.device)
        self._buffer, self._bytes = self.buffer.data_ptr(), n
        self.workspace_bytes = (lib.pelica_attn_paged_workspace_bytes if self._shared is None
                                else lib.pelica_attn_paged_shared_workspace_bytes)(*args)
        self.update(stream)

    def update(self, stream=None) -> "PagedPlan":
        """Make the work list from the arrays' present contents."""
        if _device() != self._dev:
            raise AttnError(EINVAL, f"the plan is on device {self._dev}, the current device is {_device()}")
        lib = attn._lib or attn.load_library()
        tail = (self._buffer, self._bytes, attn._stream_ptr(stream))
        if self._shared is None:
            rc = lib.pelica_attn_paged_plan(ctypes.byref(self.desc), *tail)
        else:
            rc = lib.pelica_attn_paged_shared_plan(ctypes.byref(self.desc), ctypes.byref(self._shared), *tail)
        if rc:
            attn._check(rc)
        return self

    def new_workspace(self, stream=None):
        """A workspace (uninitialised) for calls with this plan on ``stream`` or
        the current stream."""
        import torch

        with _on(stream):
            return torch.empty(max(self.workspace_bytes, 16), dtype=torch.uint8, device=self.device)


def paged_attention(q, k_pages, v_pages, plan: PagedPlan, *, k_scales=None, v_scales=None, sinks=None, alibi=None, softcap: float = 0.0,
                    scale: Optional[float] = None, out=None, workspace=None, stream=None):
    """Attention of every request's new tokens over its pages.  q: f16
    (pelica_attn_paged, probabilities rounded to f16 too) or f32
    (pelica_attn_paged_f32, products to f32's precision; values up to 65504)
    [n_tokens, n_head, hd], contiguous or token rows of a wider buffer; ``sinks`` f32 [n_head]; ``alibi`` f32 [n_head] slopes of the
    distance bias; 8-bit pages (int8) come with ``k_scales`` and ``v_scales``
    (pelica_attn_paged_q8); ``softcap`` c: scores c tanh(s / c); ``scale`` None or 0:
    1/sqrt(hd).  Returns q's type;
    rows of requests without tokens or with lengths that do not fit, and rows
    behind the last, are left as they were (undefined in a new ``out``)."""
    torch, dev, shape = _torch, plan._dev, plan._q_shape
    dtype = q.dtype
    f32 = dtype is torch.float32
    if not ((f32 or dtype is torch.float16) and q.shape == shape and q.get_device() == dev and dev == _device()):
        _need(f32 or dtype is torch.float16, f"q: f16 or f32, got {dtype}")
        _check("q", q, dtype, 3, dense=False)
        _need(q.shape == shape, f"q: {shape} as planned, got {tuple(q.shape)}")
        raise AttnError(EINVAL, f"the plan is on device {dev}, q on {q.device}")
    page, row, head, pool, q8 = _q8_pools(k_pages, v_pages, k_scales, v_scales, dev)
    if pool != plan._page_shape:
        raise AttnError(EINVAL, f"k_pages: {plan._page_shape} as planned, got {tuple(k_pages.shape)}")
    if out is None:
        with _on(stream):
            out = torch.empty(shape, dtype=dtype, device=q.device)
    elif not (out.dtype is dtype and out.shape == shape and out.get_device() == dev):
        _check("out", out, dtype, 3, dense=False)
        raise AttnError(EINVAL, f"out: {shape}, got {tuple(out.shape)}")
    if sinks is not None:
        sinks = _per_head("sinks", sinks, shape[1], dev)
    if alibi is not None:
        alibi = _per_head("alibi", alibi, shape[1], dev)
    need, ws, ws_bytes = plan.workspace_bytes, None, 0
    if need:
        ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
        if ws_bytes < need:
            with _on(stream):
                workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
            ws_bytes = need
        elif workspace.get_device() != dev or not workspace.is_contiguous():
            _check("workspace", workspace, workspace.dtype)
        ws = workspace.data_ptr()
    x = PagedDesc.from_buffer_copy(plan.desc)
    if alibi is not None:
        x.alibi = alibi
    x.page_stride, x.row_stride, x.head_stride = page, row, head
    if not q.is_contiguous():
        x.q_token_stride = _rows("q", q)
    if not out.is_contiguous():
        x.out_token_stride = _rows("out", out)
    if scale is not None:
        x.scale = scale
    if softcap:
        x.softcap = softcap
    lib = attn._lib
    tail = (k_pages.data_ptr(), v_pages.data_ptr(), sinks, out.data_ptr(), ws,
            ws_bytes, attn._stream_ptr(stream))
    if plan._shared is not None:
        rc = lib.pelica_attn_paged_shared(ctypes.byref(x), ctypes.byref(plan._shared), None if q8 is None else ctypes.byref(q8),
                                          plan._buffer, plan._bytes, q.data_ptr(), not f32, *tail)
    elif q8 is not None:
        rc = lib.pelica_attn_paged_q8(ctypes.byref(x), ctypes.byref(q8), plan._buffer, plan._bytes, q.data_ptr(), not f32, *tail)
    else:
        rc = (lib.pelica_attn_paged_f32 if f32 else lib.pelica_attn_paged)(ctypes.byref(x), plan._buffer, plan._bytes,
                                                                           q.data_ptr(), *tail)
    if rc:
        attn._check(rc)
    return out


def pair_axes(sections: Sequence[int], interleaved: bool = False) -> list:
    """The axis of each rotation pair for ``sections`` pairs per axis: one
    axis after the other, or interleaved (pair j turns by axis j mod n while
    that axis has pairs left, else by axis 0)."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    n, half = len(sections), sum(sections)
    return [j % n if j // n < sections[j % n] else 0 for j in range(half)]


def new_q8_pages(n_pages: int, page_size: int, n_kv: int, hd: int, device="cuda"):
    """Empty 8-bit pages, ``(k_pages, v_pages, k_scales, v_scales)``: int8
    [n_pages, page_size, n_kv, hd] and f16 [n_pages, page_size, n_kv, hd / 32]
    (PelicaPagedQ8), zeros, a head's rows side by side, as attention reads them."""
    import torch

    _need(n_pages > 0 and page_size > 0 and n_kv > 0 and hd > 0 and hd % GROUP == 0,
          f"pages of [{n_pages}, {page_size}, {n_kv}, {hd}]: positive, hd a multiple of {GROUP}")
    pool = lambda n, t: torch.zeros(n_pages, n_kv, page_size, n, dtype=t, device=device).transpose(1, 2)  # noqa: E731
    return (pool(hd, torch.int8), pool(hd, torch.int8), pool(hd // GROUP, torch.float16), pool(hd // GROUP, torch.float16))


def pages_read(k_pages, v_pages, slots, *, k_scales=None, v_scales=None, out=None, stream=None):
    """Rows of the pages as f16 rows (pelica_attn_pages_read): ``slots`` int64
    [n] (negative or past the pool: the row is left as it was).  8-bit pages
    (int8, with ``k_scales`` and ``v_scales``) or f16 ones.  Returns ``out``, (k_rows,
    v_rows) of f16 [n, n_kv, hd], contiguous or rows of wider buffers of one
    stride, by default new ones (skipped rows undefined)."""
    if _torch is None:
        _start()
    dev, f16 = _device(), _torch.float16
    page, row, head, (n_pages, page_size, n_kv, hd), q8 = _q8_pools(k_pages, v_pages, k_scales, v_scales, dev)
    if not (slots.dtype is _torch.int64 and slots.get_device() == dev and slots.dim() == 1 and slots.is_contiguous()):
        _check("slots", slots, _torch.int64, 1)
    shape = (slots.numel(), n_kv, hd)
    if out is None:
        with _on(stream):
            out = (_torch.empty(shape, dtype=f16, device=k_pages.device), _torch.empty(shape, dtype=f16, device=k_pages.device))
    k_out, v_out = out
    if not (k_out.dtype is f16 and v_out.dtype is f16 and k_out.shape == shape and v_out.shape == shape
            and k_out.get_device() == dev and v_out.get_device() == dev):
        for t in out:
            _check("out", t, f16, 3, dense=False)
        raise AttnError(EINVAL, f"out: two of {shape}, got {tuple(k_out.shape)} and {tuple(v_out.shape)}")
    stride = 0 if k_out.is_contiguous() else _rows("out", k_out)
    if (0 if v_out.is_contiguous() else _rows("out", v_out)) != stride:
        raise AttnError(EINVAL, "out: both contiguous, or rows of one stride")
    d = PagedDesc(n_kv, n_kv, hd, 0, shape[0], 0, page_size, n_pages, 0, 0, None, None, None, None, None, page, row, head)
    lib = attn._lib or attn.load_library()
    rc = lib.pelica_attn_pages_read(ctypes.byref(d), None if q8 is None else ctypes.byref(q8), slots.data_ptr(),
                                    k_pages.data_ptr(), v_pages.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), stride,
                                    attn._stream_ptr(stream))
    if rc:
        attn._check(rc)
    return out


def paged_qkv(q, k, v, k_pages, v_pages, slots, *, k_scales=None, v_scales=None, positions=None, table=None, rot: int = 0, neox: bool = True,
              table_split: int = 0, pair_axis: Optional[Sequence[int]] = None, q_norm=None, k_norm=None,
              eps: float = 1e-6, out=None, stream=None):
    """The step before attention over pages (pelica_attn_paged_qkv): per-head
    RMS norm of q and k (when q_norm / k_norm are given), rope by ``positions``
    (int32 [n_tokens], or [n_axes, n_tokens] with ``pair_axis``: the axis of
    each pair, see ``pair_axes``) with the f32 cos/sin ``table`` [rows, rot/2,
    2], k and v rows to f16 rows ``slots`` (int64 [n_tokens]; negative: the row
    is skipped) of the pages; 8-bit pages (int8, with ``k_scales`` and
    ``v_scales``) take the rows quantised (pelica_attn_paged_qkv_q8; no slot twice).  q: f32 [n_tokens, n_head, hd], k, v: f32
    [n_tokens, n_kv, hd], contiguous or views into one buffer of token rows.
    Returns ``out`` (f32, may be q; or f16), by default a new f32 tensor (its
    skipped rows undefined)."""
    if _torch is None:
        _start()
    f32, dev = _torch.float32, _device()
    shape, kv_shape = q.shape, k.shape
    at_q, at_k, at_v = q.stride(), k.stride(), v.stride()
    if not (q.dtype is f32 and k.dtype is f32 and v.dtype is f32 and len(shape) == 3 and len(kv_shape) == 3
            and v.shape == kv_shape and kv_shape[0] == shape[0] and kv_shape[2] == shape[2]
            and q.get_device() == dev and k.get_device() == dev and v.get_device() == dev):
        for name, t in (("q", q), ("k", k), ("v", v)):
            _check(name, t, f32, 3, dense=False)
        raise AttnError(EINVAL, f"q, k, v: [n_tokens, heads, hd], k and v alike; got {tuple(shape)}, {tuple(kv_shape)} and "
                                f"{tuple(v.shape)}")
    T, n_head, hd = shape
    n_kv = kv_shape[1]
    page, row, head, (n_pages, page_size, heads, dims), q8 = _q8_pools(k_pages, v_pages, k_scales, v_scales, dev)
    if heads != n_kv or dims != hd:
        raise AttnError(EINVAL, f"k_pages: [n_pages, page_size, {n_kv}, {hd}], got {tuple(k_pages.shape)}")
    stride = at_q[0] if T > 1 else 0
    if not (at_q[2] == 1 and (at_q[1] == hd or n_head == 1) and at_k[2] == 1 and (at_k[1] == hd or n_kv == 1)
            and at_v[2] == 1 and (at_v[1] == hd or n_kv == 1) and (T == 1 or at_k[0] == at_v[0] == stride > 0)):
        stride = _rows("q", q)
        if _rows("k", k) != stride or _rows("v", v) != stride:
            raise AttnError(EINVAL, "q, k and v: all contiguous, or views into rows of one stride")
    if not (slots.dtype is _torch.int64 and slots.get_device() == dev and slots.shape == (T,) and slots.is_contiguous()):
        _check("slots", slots, _torch.int64, 1)
        raise AttnError(EINVAL, f"slots: one for each of the {T} rows")
    if out is None:
        with _on(stream):
            out = _torch.empty(shape, dtype=f32, device=q.device)
    half = out.dtype is _torch.float16
    if not ((half or out.dtype is f32) and out.shape == shape and out.get_device() == dev):
        _need(out.dtype in (_torch.float16, f32), f"out: f16 or f32, got {out.dtype}")
        _check("out", out, out.dtype, 3, dense=False)
        raise AttnError(EINVAL, f"out: {tuple(shape)}, got {tuple(out.shape)}")
    wq, wk = q_norm, k_norm
    if wq is not None:
        wq = _weights("q_norm", wq, hd, dev)
    if wk is not None:
        wk = _weights("k_norm", wk, hd, dev)
    rp = None
    if table is not None:
        size = table.shape
        if not (table.dtype is f32 and table.get_device() == dev and len(size) == 3 and size[2] == 2
                and (rot == 0 or rot == 2 * size[1]) and table.is_contiguous()):
            _check("table", table, f32, 3)
            raise AttnError(EINVAL, f"table: [rows, {rot // 2 or 'rot / 2'}, 2], got {tuple(table.shape)}")
        rot = 2 * size[1]
        _need(positions is not None, "positions are needed with a table")
        at = positions.shape
        n_axes = at[0] if len(at) == 2 else 1
        if not (positions.dtype is _torch.int32 and positions.get_device() == dev and 1 <= len(at) <= 2 and at[-1] == T
                and positions.is_contiguous()):
            _check("positions", positions, _torch.int32)
            raise AttnError(EINVAL, f"positions: [{T}] or [n_axes, {T}], got {tuple(positions.shape)}")
        axes = None
        if pair_axis is not None:
            try:
                axes = bytes(pair_axis)  # (the call checks them against n_axes)
            except (TypeError, ValueError) as e:
                raise AttnError(EINVAL, f"pair_axis: an axis below {n_axes} for each pair: {e}") from None
            _need(len(axes) == rot // 2, f"pair_axis: an axis for each of the {rot // 2} pairs")
        _need(n_axes == 1 or axes is not None, "pair_axis is needed with more than one axis")
        rp = ctypes.byref(PagedRope(rot, 1 if neox else 0, table_split, size[0], table.data_ptr(), n_axes, axes,
                                    positions.data_ptr(), T))
    # (in the order of PagedDesc._fields_)
    d = PagedDesc(n_head, n_kv, hd, 0, T, 0, page_size, n_pages, 0, 0, None, None, None, None, None, page, row, head)
    lib = attn._lib or attn.load_library()
    tail = (q.data_ptr(), k.data_ptr(), v.data_ptr(), stride, wq, wk, eps, slots.data_ptr(), out.data_ptr(), half,
            _rows("out", out), k_pages.data_ptr(), v_pages.data_ptr(), attn._stream_ptr(stream))
    if q8 is None:
        rc = lib.pelica_attn_paged_qkv(ctypes.byref(d), rp, *tail)
    else:
        rc = lib.pelica_attn_paged_qkv_q8(ctypes.byref(d), rp, ctypes.byref(q8), *tail)
    if rc:
        attn._check(rc)
    return out
