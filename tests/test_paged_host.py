"""The paged calls without a GPU: the ctypes mirrors, the refusals of the C entry
points and of the binding, and the address rules of the kernels walked key by key."""
import ctypes
import os
import random
import subprocess

import pytest
import torch

from pelica_amd import attn, paged

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("name,cls", [("PelicaPageDesc", attn.PageDesc), ("PelicaPagedDesc", attn.PagedDesc),
                                      ("PelicaPagedRope", attn.PagedRope)])
def test_struct_layouts(name, cls, tmp_path):
    src = tmp_path / "layout.c"
    body = "".join(f'printf("{f} %zu\\n", offsetof({name}, {f}));\n' for f, _ in cls._fields_)
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "pelica_attn.h"\nint main(void) {\n' + body
                   + f'printf("size %zu\\n", sizeof({name}));\nreturn 0;\n}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    out = dict(x.split() for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(out["size"]) == ctypes.sizeof(cls)
    for f, _ in cls._fields_:
        assert int(out[f]) == getattr(cls, f).offset, f


def test_constants_match_the_header():
    text = open(os.path.join(ROOT, "include", "pelica_attn.h")).read()
    assert f"#define PELICA_ATTN_PAGED_MAX_SEQ {paged.MAX_SEQ}\n" in text
    for i, n in enumerate(("OK", "NONE", "TABLE", "ROWS", "LENGTH")):
        assert f"#define PELICA_ATTN_PAGES_{n} {i}" in text


A = 64  # an address that is aligned for everything and never read: the calls below end before a launch


def _desc(**kw):
    d = dict(n_head=8, n_kv=2, hd=64, n_seq=4, n_tokens=16, max_q=4, page_size=16, n_pages=100, max_pages=10, window=0,
             q_start=A, seq_kv_len=A, page_table=A)
    d.update(kw)
    return attn.PagedDesc(**d)


def _error(rc, code, word):
    text = attn.load_library().pelica_attn_last_error().decode()
    assert rc == code and word in text, (rc, text)


BAD = [
    (dict(n_kv=3), attn.EINVAL, "n_head"), (dict(n_head=0), attn.EINVAL, "n_head"), (dict(n_kv=-1), attn.EINVAL, "n_head"),
    (dict(hd=96), attn.EUNSUPPORTED, "hd"), (dict(n_seq=0), attn.EINVAL, "n_seq"), (dict(n_seq=4097), attn.EINVAL, "n_seq"),
    (dict(n_tokens=0), attn.EINVAL, "n_tokens"), (dict(n_tokens=(1 << 20) + 1), attn.EINVAL, "n_tokens"),
    (dict(max_q=0), attn.EINVAL, "max_q"), (dict(max_q=17), attn.EINVAL, "max_q"),
    (dict(page_size=4), attn.EUNSUPPORTED, "page_size"), (dict(page_size=24), attn.EUNSUPPORTED, "page_size"),
    (dict(page_size=1 << 17), attn.EUNSUPPORTED, "page_size"), (dict(page_size=0), attn.EUNSUPPORTED, "page_size"),
    (dict(page_size=-16), attn.EUNSUPPORTED, "page_size"),
    (dict(n_pages=0), attn.EINVAL, "n_pages"), (dict(max_pages=0), attn.EINVAL, "max_pages"),
    (dict(max_pages=(1 << 26) + 1), attn.EINVAL, "max_pages"), (dict(window=-1), attn.EINVAL, "window"),
    (dict(scale=-1.0), attn.EINVAL, "scale"), (dict(scale=float("nan")), attn.EINVAL, "scale"),
    (dict(scale=float("inf")), attn.EINVAL, "scale"), (dict(softcap=-1.0), attn.EINVAL, "softcap"),
    (dict(softcap=float("nan")), attn.EINVAL, "softcap"), (dict(softcap=1e-35), attn.EUNSUPPORTED, "softcap"),
    (dict(softcap=1e35), attn.EUNSUPPORTED, "softcap"), (dict(row_stride=60), attn.EINVAL, "strides"),
    (dict(row_stride=132), attn.EINVAL, "strides"), (dict(head_stride=4), attn.EINVAL, "strides"),
    (dict(page_stride=-8), attn.EINVAL, "strides"), (dict(row_stride=1 << 24), attn.EUNSUPPORTED, "strides"),
    (dict(q_start=None), attn.EINVAL, "NULL"), (dict(seq_kv_len=None), attn.EINVAL, "NULL"),
    (dict(page_table=None), attn.EINVAL, "NULL"),
    (dict(q_start=A + 2), attn.EINVAL, "aligned"), (dict(seq_kv_len=A + 1), attn.EINVAL, "aligned"),
    (dict(page_table=A + 2), attn.EINVAL, "aligned"), (dict(prefix_len=A + 2), attn.EINVAL, "aligned"),
    (dict(alibi=A + 2), attn.EINVAL, "aligned"),
]


@pytest.mark.parametrize("kw,code,word", BAD, ids=[str(b[0]) for b in BAD])
def test_bad_descriptors(kw, code, word):
    lib, d = attn.load_library(), _desc(**kw)
    assert lib.pelica_attn_paged_plan_bytes(ctypes.byref(d)) == 0
    assert word in lib.pelica_attn_last_error().decode()
    assert lib.pelica_attn_paged_workspace_bytes(ctypes.byref(d)) == 0
    _error(lib.pelica_attn_paged_plan(ctypes.byref(d), A, 1 << 30, None), code, word)
    for f in (lib.pelica_attn_paged, lib.pelica_attn_paged_f32):
        _error(f(ctypes.byref(d), A, 1 << 40, A, A, A, None, A, A, 1 << 40, None), code, word)


def test_null_and_misaligned_arguments():
    lib, d = attn.load_library(), _desc(max_q=16)
    ref = ctypes.byref(d)
    need = lib.pelica_attn_paged_plan_bytes(ref)
    _error(lib.pelica_attn_paged_plan(ref, None, need, None), attn.EINVAL, "plan")
    _error(lib.pelica_attn_paged_plan(ref, A + 4, need, None), attn.EINVAL, "plan")
    _error(lib.pelica_attn_paged_plan(ref, A, need - 1, None), attn.EWORKSPACE, "plan")
    _error(lib.pelica_attn_paged_plan(None, A, need, None), attn.EINVAL, "desc")
    ws = lib.pelica_attn_paged_workspace_bytes(ref)
    assert ws > 0
    good = [A, need, A, A, A, None, A, A, ws, None]
    for f in (lib.pelica_attn_paged, lib.pelica_attn_paged_f32):
        for i in (0, 2, 3, 4, 6):
            _error(f(ref, *[None if j == i else x for j, x in enumerate(good)]), attn.EINVAL, "NULL")
            _error(f(ref, *[A + 8 if j == i else x for j, x in enumerate(good)]), attn.EINVAL, "aligned")
        _error(f(ref, *[None if j == 7 else x for j, x in enumerate(good)]), attn.EWORKSPACE, "workspace")
        _error(f(ref, *[ws - 1 if j == 8 else x for j, x in enumerate(good)]), attn.EWORKSPACE, "workspace")
        _error(f(ref, *[need - 1 if j == 1 else x for j, x in enumerate(good)]), attn.EWORKSPACE, "plan")
        _error(f(ref, *[A + 2 if j == 5 else x for j, x in enumerate(good)]), attn.EINVAL, "sinks")
    for kw in (dict(q_token_stride=8), dict(out_token_stride=511), dict(q_token_stride=516), dict(out_token_stride=1 << 31)):
        d = _desc(max_q=16, **kw)
        _error(lib.pelica_attn_paged(ctypes.byref(d), *good), attn.EINVAL, "stride")


def test_pages_arguments():
    lib = attn.load_library()
    good = attn.PageDesc(4, 16, 16, 100, 10)
    args = [A, A, A, A, 128, 256, A, A, A, A, A, A, None]
    for i in range(12):
        _error(lib.pelica_attn_pages_append(ctypes.byref(good), *[None if j == i else x for j, x in enumerate(args)]),
               attn.EINVAL, "NULL")
        _error(lib.pelica_attn_pages_append(ctypes.byref(good), *[x + 2 if j == i else x for j, x in enumerate(args)]),
               attn.EINVAL, "aligned")
    for out in (120, 128, 136):
        _error(lib.pelica_attn_pages_append(ctypes.byref(good), *[out if j == 5 else x for j, x in enumerate(args)]),
               attn.EINVAL, "overlaps")
    rel = [A, A, A, A, 128, 256, None]
    for i in range(6):
        _error(lib.pelica_attn_pages_release(ctypes.byref(good), *[None if j == i else x for j, x in enumerate(rel)]),
               attn.EINVAL, "NULL")
    _error(lib.pelica_attn_pages_release(ctypes.byref(good), A, A, A, A, 128, 128, None), attn.EINVAL, "overlaps")
    for bad, code, word in (((0, 16, 16, 100, 10), attn.EINVAL, "n_seq"), ((4097, 16, 16, 100, 10), attn.EINVAL, "n_seq"),
                            ((4, 16, 12, 100, 10), attn.EUNSUPPORTED, "page_size"),
                            ((4, 16, 16, 0, 10), attn.EINVAL, "n_pages"), ((4, 16, 16, 100, 0), attn.EINVAL, "max_pages")):
        d = attn.PageDesc(*bad)
        _error(lib.pelica_attn_pages_append(ctypes.byref(d), *args), code, word)
        _error(lib.pelica_attn_pages_release(ctypes.byref(d), *rel), code, word)
    for n in (0, (1 << 20) + 1):
        d = attn.PageDesc(4, n, 16, 100, 10)
        _error(lib.pelica_attn_pages_append(ctypes.byref(d), *args), attn.EINVAL, "n_tokens")


def _apart(counts):
    """An address for each array of so many values, one behind the other."""
    at, out = 1 << 20, []
    for n, size in counts:
        out.append(at)
        at += -(-n * size // 64) * 64 + 64
    return out


def test_pages_outputs_may_not_overlap_another_array():
    # workgroups read the inputs while another writes the outputs (lengths
    # updated in place went wrong in steps of more than one workgroup)
    lib = attn.load_library()
    n_seq, n_tokens, n_pages, most = 4, 1000, 100, 10
    d = ctypes.byref(attn.PageDesc(n_seq, n_tokens, 16, n_pages, most))
    sizes = [(n_seq, 4), (n_seq, 4), (n_seq * most, 4), (n_pages, 4), (2, 8), (2, 8), (n_seq + 1, 4), (n_seq, 4),
             (n_tokens, 8), (n_tokens, 4), (n_tokens, 4), (n_seq, 4)]
    at = _apart(sizes)
    for o in (2, *range(5, 12)):  # outputs: page_table, free_out, q_start ... status
        for i in range(12):
            if i == o:
                continue
            (n, size), (m, width) = sizes[i], sizes[o]
            # on it, its last value, and the output's last value on its first
            for x in (at[i], (at[i] + n * size - 1) // 8 * 8, (at[i] - m * width) // 8 * 8 + 8):
                args = [x if j == o else a for j, a in enumerate(at)]
                _error(lib.pelica_attn_pages_append(d, *args, None), attn.EINVAL, "overlaps")
    sizes = [(n_seq, 4), (n_seq, 4), (n_seq * most, 4), (n_pages, 4), (2, 8), (2, 8)]
    at = _apart(sizes)
    for o in (3, 5):  # free_list, free_out
        for i in range(6):
            if i != o:
                args = [at[i] if j == o else a for j, a in enumerate(at)]
                _error(lib.pelica_attn_pages_release(d, *args, None), attn.EINVAL, "overlaps")


def test_qkv_arguments():
    lib = attn.load_library()
    args = [A, A, A, 0, None, None, 1e-6, A, 128, 0, 0, A, A, None]

    def call(d=None, rope=None, **at):
        d = d or _desc(hd=128)
        a = [at.get(f"a{i}", x) for i, x in enumerate(args)]
        return lib.pelica_attn_paged_qkv(ctypes.byref(d), None if rope is None else ctypes.byref(rope), *a)

    for i in (0, 1, 2, 7, 8, 11, 12):
        _error(call(**{f"a{i}": None}), attn.EINVAL, "NULL")
        _error(call(**{f"a{i}": A + 4}), attn.EINVAL, "aligned")
    _error(call(a4=A + 8), attn.EINVAL, "aligned")
    _error(call(a3=100), attn.EINVAL, "token_stride")
    _error(call(a3=1026), attn.EINVAL, "token_stride")
    _error(call(a10=1000), attn.EINVAL, "q_out_stride")
    _error(call(a8=A, a9=1), attn.EINVAL, "q_out")
    _error(call(a8=A, a3=1536), attn.EINVAL, "q_out")
    _error(call(a6=float("nan")), attn.EINVAL, "eps")
    _error(call(_desc(hd=96)), attn.EUNSUPPORTED, "hd")
    _error(call(_desc(hd=128, page_size=7)), attn.EUNSUPPORTED, "page_size")
    _error(call(_desc(hd=128, n_tokens=0)), attn.EINVAL, "n_tokens")
    pair = bytes([0] * 63 + [3])
    base = dict(rot=128, neox=1, table_split=0, table_rows=100, table=A, n_axes=3, pair_axis=None, positions=A,
                axis_stride=16)
    for kw, word in ((dict(rot=7), "rot"), (dict(rot=130), "rot"), (dict(rot=-2), "rot"), (dict(table=None), "table"),
                     (dict(table=A + 4), "table"), (dict(table_rows=0), "table"), (dict(table_split=10), "two-level"),
                     (dict(n_axes=0), "n_axes"), (dict(n_axes=5), "n_axes"), (dict(positions=None), "positions"),
                     (dict(axis_stride=15), "axis_stride"), (dict(pair_axis=pair), "axis 3")):
        _error(call(rope=attn.PagedRope(**{**base, **kw})), attn.EINVAL, word)


def test_the_binding_refuses_cpu_tensors_and_wrong_types():
    i = torch.zeros(4, dtype=torch.int32)
    for f in (lambda: paged.pages_append(i, i, i.view(2, 2), i, torch.zeros(2, dtype=torch.int64), page_size=16, step=None),
              lambda: paged.PagedPlan(i, i, i.view(2, 2), n_head=1, n_kv=1, hd=64, page_size=16, n_pages=4, n_tokens=4, max_q=1),
              lambda: paged.paged_qkv(*[torch.zeros(1, 1, 64)] * 3, i, i, i)):
        with pytest.raises(attn.AttnError) as e:
            f()
        assert e.value.code == attn.EINVAL


def test_rows_of_the_host_are_refused():
    x, pages = torch.zeros(2, 1, 64), torch.zeros(4, 16, 1, 64, dtype=torch.float16)
    with pytest.raises(attn.AttnError) as e:
        paged.paged_qkv(x, x, x, pages, pages, torch.zeros(2, dtype=torch.int64), out=x)
    assert e.value.code == attn.EINVAL and "device" in str(e.value)


def test_strides_of_zero_are_refused(monkeypatch):
    """To the C calls 0 means dense; of a tensor it is one row for all, and the
    rows that a dense tensor would have lie behind its storage.  (Host tensors,
    and no call: whatever passes the checks ends in the recorder.)"""
    calls = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: calls.append(name) or 0

    paged._start()
    monkeypatch.setattr(paged, "_device", lambda: -1)
    monkeypatch.setattr(attn, "_lib", Lib())
    monkeypatch.setattr(attn, "_stream_ptr", lambda s: None)
    n, page, heads, hd = 3, 16, 4, 64
    pool = torch.zeros(n, page, heads, hd, dtype=torch.float16)
    one = [pool[:1].expand(n, -1, -1, -1), pool[:, :1].expand(-1, page, -1, -1), pool[:, :, :1].expand(-1, -1, heads, -1)]
    T = 5
    rows = torch.zeros(T, heads, hd)
    slots = torch.arange(T)
    few = rows[:1].expand(T, -1, -1)
    good = dict(q=rows, k=rows, v=rows, k_pages=pool, v_pages=pool, slots=slots, out=rows)
    # dims of one have any stride: a single page, head, token
    fine = [{}, dict(k_pages=pool[:1].expand(1, -1, -1, -1), v_pages=pool[:1])]
    single = torch.zeros(1, page, 1, hd, dtype=torch.float16)
    x = torch.zeros(1, 1, hd)
    fine.append(dict(q=x, k=x, v=x, k_pages=single, v_pages=single, slots=slots[:1], out=x))
    x = torch.as_strided(torch.zeros(hd), (1, 1, hd), (0, 0, 1))
    fine.append(dict(q=x, k=x, v=x, k_pages=torch.as_strided(single, single.shape, (0, hd, 0, 1)),
                     v_pages=torch.as_strided(single, single.shape, (0, hd, 0, 1)), slots=slots[:1], out=x))
    for kw in fine:
        paged.paged_qkv(**{**good, **kw})
    assert len(calls) == len(fine)
    bad = [dict(k_pages=p, v_pages=p) for p in one]
    bad += [dict(q=few, k=few, v=few), dict(q=few), dict(k=few), dict(v=few), dict(k=few, v=few), dict(out=few)]
    bad += [dict(q=rows[:, :1].expand(-1, heads, -1)), dict(k=rows[:, :1].expand(-1, heads, -1))]
    for kw in bad:
        with pytest.raises(attn.AttnError) as e:
            paged.paged_qkv(**{**good, **kw})
        assert e.value.code == attn.EINVAL and "stride" in str(e.value)
    assert len(calls) == len(fine)

    plan = paged.PagedPlan.__new__(paged.PagedPlan)
    plan._dev, plan._q_shape, plan._page_shape = -1, (T, heads, hd), (n, page, heads, hd)
    plan.workspace_bytes, plan.desc, plan._buffer, plan._bytes = 0, attn.PagedDesc(), None, 0
    good = dict(q=rows, k_pages=pool, v_pages=pool, plan=plan, out=rows)
    paged.paged_attention(**good)
    assert len(calls) == len(fine) + 1
    for kw in [dict(k_pages=p, v_pages=p) for p in one] + [dict(q=few), dict(out=few)]:
        with pytest.raises(attn.AttnError) as e:
            paged.paged_attention(**{**good, **kw})
        assert e.value.code == attn.EINVAL and "stride" in str(e.value)
    assert len(calls) == len(fine) + 1


def test_a_workspace_belongs_to_its_stream(monkeypatch):
    """Memory of the stream that the calls run on: another's may be in use."""
    import contextlib

    on = []

    @contextlib.contextmanager
    def _on(stream):
        on.append(stream)
        yield
        on.append("made")

    plan = paged.PagedPlan.__new__(paged.PagedPlan)
    plan.device, plan.workspace_bytes = torch.device("cpu"), 100
    monkeypatch.setattr(paged, "_on", _on)
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: on.append("empty") or empty(*a, **kw))
    st = object()
    assert plan.new_workspace(st).numel() == plan.new_workspace(stream=st).numel() == 100
    assert on == [st, "empty", "made"] * 2
    plan.new_workspace()
    assert on[6:] == [None, "empty", "made"]


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    so = tmp_path_factory.mktemp("plan") / "plan.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-o", str(so),
                    os.path.join(ROOT, "tests", "paged_plan_shim.cpp")], check=True)
    lib = ctypes.CDLL(str(so))
    lib.plan_items_of.restype = ctypes.c_int64
    lib.plan_items_of.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int32, ctypes.c_int32]
    return lib


def _seen(pos, window, pe):
    lo = pos - window + 1 if window and pos >= window else 0
    return set(range(lo, pos + 1)) | set(range(pe))


def test_an_items_chunks_hold_every_key_its_rows_see_once(rules):
    r = random.Random(1)
    out6, out2 = (ctypes.c_int * 6)(), (ctypes.c_int * 2)()
    for _ in range(3000):
        length = r.randint(1, 700)
        first = r.randint(0, length - 1)
        last = r.randint(first, min(length - 1, first + r.choice((0, 3, 40))))
        window = r.choice((0, 0, 1, 5, 32, 64, 300))
        prefix = r.choice((0, 0, 1, 31, 32, 33, 200, 1000))
        rules.item_keys_of(first, last, length, window, prefix, out6)
        n_pre, lo_base, n_chunks, lo, kend, pe = out6
        assert pe == min(prefix, length) and kend == last + 1
        want = set().union(*(_seen(p, window, pe) for p in range(first, last + 1)))
        got = []
        for c in range(n_chunks):
            key = rules.chunk_key_of(c, n_pre, lo_base)
            assert key % 32 == 0
            for n in (4, 8):  # rows of a load at head dim 128, 64
                touched = []
                for kg in range(key, key + 32, n):
                    rules.group_rows_of(kg, n, lo, kend, pe, out2)
                    f, cnt = out2
                    assert 0 <= f and f + cnt <= n
                    rows = list(range(kg + f, kg + f + cnt))
                    # every wanted row, none past the request's keys, and what lies between the prefix
                    # and the window within one group (of one page) only
                    assert set(range(kg, kg + n)) & want <= set(rows)
                    assert all(x in want or (kg <= pe - 1 < kg + n and x < kend) for x in rows)
                    assert not rows or rows[-1] < max(kend, pe)
                    touched += rows
            got += [x for x in touched if x in want]
        assert len(got) == len(set(got)) and set(got) == want


def test_rows_that_one_token_loads_and_does_not_see_are_told(rules):
    """An item whose rows share one position: its loads touch a key that it does
    not see where, and only where, gap_in_run says so."""
    r = random.Random(4)
    out6, out2 = (ctypes.c_int * 6)(), (ctypes.c_int * 2)()
    told = 0
    for _ in range(6000):
        length = r.randint(1, 200)
        window = r.choice((0, 1, 3, 24, 100))
        begin = max(0, length - window)
        prefix = max(0, r.choice((0, 5, begin - 1, begin - 2, begin - 7, begin - 8, begin, begin + 3)))
        rules.item_keys_of(length - 1, length - 1, length, window, prefix, out6)
        n_pre, lo_base, n_chunks, lo, kend, pe = out6
        unseen = set()
        for c in range(n_chunks):
            key = rules.chunk_key_of(c, n_pre, lo_base)
            for kg in range(key, key + 32, 8):  # runs of 8, as the kernels address them
                rules.group_rows_of(kg, 8, lo, kend, pe, out2)
                unseen |= set(range(kg + out2[0], kg + sum(out2))) - _seen(length - 1, window, pe)
        assert bool(unseen) == bool(rules.gap_in_run_of(lo, pe)), (length, window, prefix, unseen)
        told += bool(unseen)
    assert 300 < told < 3000


def test_pieces_of_an_item(rules):
    rules.item_pieces_of.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_float]
    r = random.Random(3)
    for _ in range(2000):
        chunks = r.choice((1, 2, 5, 100, 5000, 1 << 25))
        cost = chunks * r.choice((1, 3))
        limit = r.choice((4.0, 4.7, 37.2, 1000.5, 1e9))
        k = rules.item_pieces_of(cost, chunks, limit)
        # (in f32: a piece may pass the limit by its roundings)
        assert 1 <= k <= chunks and (k == chunks or k * limit * (1 + 2 ** -21) >= cost)
        cuts = [chunks * i // k for i in range(min(k, 300) + 1)]
        assert cuts[0] == 0 and all(a < b for a, b in zip(cuts, cuts[1:])) and chunks * k // k == chunks


def test_the_bound_on_items_holds(rules):
    r = random.Random(2)
    for _ in range(500):
        hpk, hd = r.choice((1, 2, 3, 8, 16, 71)), r.choice((64, 128))
        new = [r.choice((0, 1, 2, 5, 40, 300)) for _ in range(r.randint(1, 40))]
        W = 256 if hd == 64 else 128
        items = sum(1 if n * hpk <= 32 else -(-n * hpk // W) for n in new if n)
        if sum(new):
            assert items <= rules.plan_items_of(len(new), sum(new), hpk, hd)
