"""The calls over shared keys without a GPU: struct layout, refusals, sizes."""
import ctypes
import os
import subprocess

import pytest

from pelica_amd import attn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 64  # an address that is aligned for everything and never read: the calls below end before a launch


def _desc(**kw):
    d = dict(n_head=8, n_kv=2, hd=64, n_seq=4, n_tokens=16, max_q=4, page_size=16, n_pages=100, max_pages=10,
             q_start=A, seq_kv_len=A, page_table=A)
    return attn.PagedDesc(**{**d, **kw})


def _shared(**kw):
    return attn.PagedShared(**{**dict(n_groups=2, group_start=A, shared_len=A), **kw})


def _error(rc, code, word):
    text = attn.load_library().pelica_attn_last_error().decode()
    assert rc == code and word in text, (rc, text)


def test_struct_layout_and_limit(tmp_path):
    src = tmp_path / "layout.c"
    cls, name = attn.PagedShared, "PelicaPagedShared"
    body = "".join(f'printf("{f} %zu\\n", offsetof({name}, {f}));\n' for f, _ in cls._fields_)
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "pelica_attn.h"\nint main(void) {\n' + body
                   + f'printf("size %zu\\n", sizeof({name}));\nprintf("most %d\\n", PELICA_ATTN_PAGED_MAX_GROUPS);\nreturn 0;\n}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    out = dict(x.split() for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(out["size"]) == ctypes.sizeof(cls) and int(out["most"]) == 1024
    for f, _ in cls._fields_:
        assert int(out[f]) == getattr(cls, f).offset, f


BAD = [
    (_desc(n_kv=3), _shared(), attn.EINVAL, "n_head"), (_desc(hd=96), _shared(), attn.EUNSUPPORTED, "hd"),
    (_desc(max_q=0), _shared(), attn.EINVAL, "max_q"), (_desc(q_start=None), _shared(), attn.EINVAL, "q_start"),
    (_desc(), _shared(n_groups=0), attn.EINVAL, "n_groups"), (_desc(), _shared(n_groups=-1), attn.EINVAL, "n_groups"),
    (_desc(), _shared(n_groups=5), attn.EINVAL, "n_groups"), (_desc(n_seq=2000), _shared(n_groups=1025), attn.EINVAL, "n_groups"),
    (_desc(), _shared(group_start=None), attn.EINVAL, "group_start"), (_desc(), _shared(shared_len=None), attn.EINVAL, "shared_len"),
    (_desc(), _shared(group_start=A + 2), attn.EINVAL, "aligned"), (_desc(), _shared(shared_len=A + 1), attn.EINVAL, "aligned"),
    (_desc(window=1), _shared(), attn.EUNSUPPORTED, "window"), (_desc(prefix_len=A), _shared(), attn.EUNSUPPORTED, "prefix_len"),
    (_desc(alibi=A), _shared(), attn.EUNSUPPORTED, "alibi"),
    (_desc(n_tokens=1 << 20, n_head=512, n_kv=2), _shared(), attn.EUNSUPPORTED, "2^28"),
]


@pytest.mark.parametrize("d,x,code,word", BAD)
def test_bad_descriptors(d, x, code, word):
    lib = attn.load_library()
    _error(lib.pelica_attn_paged_shared_plan(d, x, A, 1 << 30, None), code, word)
    _error(lib.pelica_attn_paged_shared(d, x, None, A, 1 << 30, A, 0, A, A, None, A, A, 1 << 40, None), code, word)
    for size in (lib.pelica_attn_paged_shared_plan_bytes, lib.pelica_attn_paged_shared_workspace_bytes):
        assert size(d, x) == 0 and word in lib.pelica_attn_last_error().decode()


def test_null_and_misaligned_arguments():
    lib = attn.load_library()
    d, x = _desc(), _shared()
    need, ws = lib.pelica_attn_paged_shared_plan_bytes(d, x), lib.pelica_attn_paged_shared_workspace_bytes(d, x)
    assert need > 0 and ws > 0
    _error(lib.pelica_attn_paged_shared_plan(d, None, A, need, None), attn.EINVAL, "shared")
    _error(lib.pelica_attn_paged_shared_plan(None, x, A, need, None), attn.EINVAL, "desc")
    _error(lib.pelica_attn_paged_shared_plan(d, x, None, need, None), attn.EINVAL, "plan")
    _error(lib.pelica_attn_paged_shared_plan(d, x, A + 8, need, None), attn.EINVAL, "plan")
    _error(lib.pelica_attn_paged_shared_plan(d, x, A, need - 1, None), attn.EWORKSPACE, "plan")
    call = dict(d=d, x=x, q8=None, plan=A, n=need, q=A, half=0, k=A, v=A, sinks=None, out=A, ws=A, wsn=ws, st=None)
    for kw, code, word in ((dict(plan=None), attn.EINVAL, "NULL"), (dict(q=None), attn.EINVAL, "NULL"), (dict(k=None), attn.EINVAL, "NULL"),
                           (dict(out=A + 8), attn.EINVAL, "aligned"), (dict(sinks=A + 2), attn.EINVAL, "sinks"),
                           (dict(n=need - 1), attn.EWORKSPACE, "plan"), (dict(wsn=ws - 1), attn.EWORKSPACE, "workspace"),
                           (dict(ws=None), attn.EWORKSPACE, "workspace"),
                           (dict(q8=attn.PagedQ8(None, A)), attn.EINVAL, "k_scales"), (dict(x=None), attn.EINVAL, "shared")):
        _error(lib.pelica_attn_paged_shared(*{**call, **kw}.values()), code, word)


def test_a_workspace_holds_every_rows_partials():
    """A row of each token and head from its request and one from its group, and the pieces of split items."""
    lib = attn.load_library()
    for n_head, n_kv, hd, tokens in ((64, 8, 64, 64), (32, 4, 128, 300), (1, 1, 64, 2), (16, 16, 128, 4096)):
        d = _desc(n_head=n_head, n_kv=n_kv, hd=hd, n_tokens=tokens, max_q=1, n_seq=min(tokens, 4096))
        assert lib.pelica_attn_paged_shared_workspace_bytes(d, _shared()) >= 2 * tokens * n_head * (hd + 2) * 4
