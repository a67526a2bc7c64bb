"""The calls over 8-bit pages without a GPU: struct layout, refusals, the format's definition."""
import ctypes
import os
import subprocess

import pytest
import torch

from pelica_amd import attn, paged
from tests import q8_ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 64  # an address that is aligned for everything and never read: the calls below end before a launch


def _desc(**kw):
    d = dict(n_head=8, n_kv=2, hd=64, n_seq=4, n_tokens=16, max_q=4, page_size=16, n_pages=100, max_pages=10,
             q_start=A, seq_kv_len=A, page_table=A)
    return attn.PagedDesc(**{**d, **kw})


def _q8(**kw):
    return attn.PagedQ8(**{**dict(k_scales=A, v_scales=A), **kw})


def _error(rc, code, word):
    text = attn.load_library().pelica_attn_last_error().decode()
    assert rc == code and word in text, (rc, text)


def test_struct_layout(tmp_path):
    src = tmp_path / "layout.c"
    cls, name = attn.PagedQ8, "PelicaPagedQ8"
    body = "".join(f'printf("{f} %zu\\n", offsetof({name}, {f}));\n' for f, _ in cls._fields_)
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "pelica_attn.h"\nint main(void) {\n' + body
                   + f'printf("size %zu\\n", sizeof({name}));\nreturn 0;\n}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    out = dict(x.split() for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(out["size"]) == ctypes.sizeof(cls)
    for f, _ in cls._fields_:
        assert int(out[f]) == getattr(cls, f).offset, f


BAD = [
    (_desc(n_kv=3), _q8(), attn.EINVAL, "n_head"), (_desc(n_tokens=0), _q8(), attn.EINVAL, "n_tokens"),
    (_desc(page_size=12), _q8(), attn.EUNSUPPORTED, "page_size"), (_desc(n_pages=0), _q8(), attn.EINVAL, "n_pages"),
    # pages' strides: whole 16-byte pieces of 8-bit values
    (_desc(row_stride=136), _q8(), attn.EINVAL, "multiples of 16"), (_desc(head_stride=72), _q8(), attn.EINVAL, "multiples of 16"),
    (_desc(page_stride=2056), _q8(), attn.EINVAL, "multiples of 16"), (_desc(row_stride=48), _q8(), attn.EINVAL, "at least hd"),
    (_desc(row_stride=1 << 24), _q8(), attn.EUNSUPPORTED, "too large"),
    (_desc(), _q8(k_scales=None), attn.EINVAL, "k_scales"), (_desc(), _q8(v_scales=0), attn.EINVAL, "v_scales"),
    (_desc(), _q8(k_scales=A + 1), attn.EINVAL, "aligned"), (_desc(), _q8(v_scales=A + 1), attn.EINVAL, "aligned"),
    (_desc(), _q8(row_stride=1), attn.EINVAL, "at least hd / 32"), (_desc(), _q8(head_stride=-2), attn.EINVAL, "at least"),
    (_desc(), _q8(page_stride=1), attn.EINVAL, "at least"), (_desc(), _q8(row_stride=1 << 24), attn.EUNSUPPORTED, "scales"),
    (_desc(page_size=65536), _q8(row_stride=1 << 14), attn.EUNSUPPORTED, "scales"),
    (_desc(), _q8(head_stride=1 << 40), attn.EUNSUPPORTED, "scales"),
]


@pytest.mark.parametrize("d,x,code,word", BAD)
def test_bad_descriptors(d, x, code, word):
    lib = attn.load_library()
    _error(lib.pelica_attn_paged_qkv_q8(d, None, x, A, A, A, 0, None, None, 0.0, A, A, 0, 0, A, A, None), code, word)
    _error(lib.pelica_attn_pages_read(d, x, A, A, A, A, A, 0, None), code, word)


def test_null_and_misaligned_arguments():
    lib = attn.load_library()
    d, x = _desc(), _q8()
    _error(lib.pelica_attn_paged_qkv_q8(d, None, None, A, A, A, 0, None, None, 0.0, A, A, 0, 0, A, A, None), attn.EINVAL, "q8")
    _error(lib.pelica_attn_paged_qkv_q8(None, None, x, A, A, A, 0, None, None, 0.0, A, A, 0, 0, A, A, None), attn.EINVAL, "desc")
    qkv = dict(d=d, rope=None, x=x, q=A, k=A, v=A, stride=0, wq=None, wk=None, eps=0.0, slots=A, out=A, half=0, so=0, kp=A,
               vp=A, st=None)
    for kw, word in ((dict(q=None), "NULL"), (dict(kp=None), "NULL"), (dict(vp=None), "NULL"), (dict(slots=None), "NULL"),
                     (dict(kp=A + 8), "aligned"), (dict(vp=A + 8), "aligned"), (dict(stride=500), "token_stride"),
                     (dict(out=A, half=1, q=A), "q_out"), (dict(eps=-1.0), "eps")):
        _error(lib.pelica_attn_paged_qkv_q8(*{**qkv, **kw}.values()), attn.EINVAL, word)
    _error(lib.pelica_attn_paged_qkv_q8(*{**qkv, "d": _desc(hd=96)}.values()), attn.EUNSUPPORTED, "hd")
    read = dict(d=d, x=x, slots=A, kp=A, vp=A, ko=2 * A, vo=3 * A, so=0, st=None)
    for kw, word in ((dict(d=None), "desc"), (dict(slots=None), "NULL"), (dict(kp=None), "NULL"), (dict(vp=None), "NULL"),
                     (dict(ko=None), "NULL"), (dict(vo=None), "NULL"), (dict(kp=A + 8), "aligned"), (dict(ko=A + 8), "aligned"),
                     (dict(ko=3 * A), "different"), (dict(vo=A), "different"), (dict(ko=A), "different"),
                     (dict(slots=A + 4), "aligned"), (dict(so=127), "out_stride"), (dict(so=132), "out_stride"),
                     (dict(so=-128), "out_stride"), (dict(so=1 << 31), "out_stride")):
        for form in (x, None):  # 8-bit and f16 pages
            _error(lib.pelica_attn_pages_read(*{**read, "x": form, **kw}.values()), attn.EINVAL, word)
    _error(lib.pelica_attn_pages_read(*{**read, "x": None, "d": _desc(hd=96, row_stride=192, head_stride=96)}.values()),
           attn.EUNSUPPORTED, "hd")
    _error(lib.pelica_attn_pages_read(*{**read, "d": _desc(n_tokens=1 << 20, n_head=1 << 10, n_kv=1 << 10)}.values()),
           attn.EUNSUPPORTED, "2^33")


def test_the_binding_refuses_rows_of_the_host_and_odd_pools():
    k, v, ks, vs = paged.new_q8_pages(3, 8, 2, 64, device="cpu")
    assert k.shape == (3, 8, 2, 64) and ks.shape == (3, 8, 2, 2) and k.dtype is torch.int8 and ks.dtype is torch.float16
    assert k.stride(1) == 64 and ks.stride(1) == 2 and not (k.any() or vs.any())
    with pytest.raises(attn.AttnError):
        paged.pages_read(k, v, torch.zeros(2, dtype=torch.int64), k_scales=ks, v_scales=vs)
    for bad in ((0, 8, 2, 64), (3, 8, 2, 48), (3, 8, -1, 64)):
        with pytest.raises(attn.AttnError):
            paged.new_q8_pages(*bad, device="cpu")


def test_strides_of_zero_are_refused(monkeypatch):
    """Rows or scales of an expanded dim: where the call would write or read, it goes by strides alone."""
    calls = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: calls.append(name) or 0

    paged._start()
    monkeypatch.setattr(paged, "_device", lambda: -1)
    monkeypatch.setattr(attn, "_lib", Lib())
    monkeypatch.setattr(attn, "_stream_ptr", lambda s: None)
    k, v, ks, vs = paged.new_q8_pages(3, 8, 2, 64, device="cpu")
    slots, rows = torch.arange(5), torch.zeros(5, 2, 64)
    good = dict(k_pages=k, v_pages=v, slots=slots, k_scales=ks, v_scales=vs)
    paged.pages_read(**good)
    paged.paged_qkv(rows, rows, rows, **good, out=torch.zeros(5, 2, 64))
    assert calls == ["pelica_attn_pages_read", "pelica_attn_paged_qkv_q8"]
    few, few_s = k[:1].expand(3, -1, -1, -1), ks[:, :1].expand(-1, 8, -1, -1)
    for kw in (dict(k_pages=few, v_pages=few), dict(k_scales=few_s, v_scales=few_s), dict(k_scales=few_s),
               dict(k_scales=ks.transpose(2, 3), v_scales=vs.transpose(2, 3))):
        with pytest.raises(attn.AttnError):
            paged.pages_read(**{**good, **kw})
        with pytest.raises(attn.AttnError):
            paged.paged_qkv(rows, rows, rows, **{**good, **kw})
    assert len(calls) == 2


def test_the_format_keeps_half_a_scale():
    x = torch.randn(500, 3, 128, generator=torch.Generator().manual_seed(0)).double() * torch.logspace(-8, 4, 500).double()[:, None, None]
    n, s = q8_ref.quantise(x)
    d = s.double().repeat_interleave(32, -1)
    assert ((n.double() * d - x).abs() <= d / 2).all()
    below = (s.view(torch.int16) - 1).clamp(min=0).view(torch.float16).double()
    top = x.abs().unflatten(-1, (-1, 32)).amax(-1)
    assert (127 * s.double() >= top).all() and ((127 * below < top) | (s == 0)).all()
