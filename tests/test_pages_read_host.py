"""pages_read without a GPU: outputs that share bytes with another array of the call are refused."""
import pytest

from pelica_amd import attn

# one array after another with room between; the calls below end before a launch
MB = 1 << 20
T, N_KV, HD, PAGE, PAGES = 16, 2, 64, 16, 100
ROW = 2 * N_KV * HD  # bytes of an output row
SLOTS, KP, VP, KS, VS, KO, VO = (MB * (10 + i) for i in range(7))
POOL = {True: PAGES * PAGE * N_KV * HD, False: 2 * PAGES * PAGE * N_KV * HD}  # bytes of 8-bit, of f16 pages


def _read(q8, ko=KO, vo=VO, stride=0, slots=SLOTS, page_stride=0, scale_page=0):
    d = attn.PagedDesc(n_head=N_KV, n_kv=N_KV, hd=HD, n_tokens=T, page_size=PAGE, n_pages=PAGES, page_stride=page_stride)
    x = attn.PagedQ8(KS, VS, scale_page, 0, 0) if q8 else None
    lib = attn.load_library()
    return lib.pelica_attn_pages_read(d, x, slots, KP, VP, ko, vo, stride, None), lib.pelica_attn_last_error().decode()


def _refused(word, q8=True, **kw):
    rc, text = _read(q8, **kw)
    assert rc == attn.EINVAL and word in text, (rc, text)


def test_outputs_over_each_other():
    for by in (16, ROW, ROW * (T - 1), ROW * T - 16):
        _refused("k_out overlaps v_out", vo=KO + by)
        _refused("k_out overlaps v_out", ko=VO + by, q8=False)
    # rows that take turns too closely
    for by in (16, ROW - 16, ROW + 16, 3 * ROW - 16):
        _refused("k_out overlaps v_out", vo=KO + by, stride=ROW)  # (values: rows and as much between them)


@pytest.mark.parametrize("q8", [True, False], ids=["8_bit", "f16"])
def test_outputs_over_the_pages(q8):
    for name, pool in (("k_pages", KP), ("v_pages", VP)):
        for at in (pool - ROW * T + 16, pool + 16, pool + POOL[q8] // 2, pool + POOL[q8] - 16):
            _refused(f"k_out overlaps {name}", q8, ko=at)
            _refused(f"v_out overlaps {name}", q8, vo=at)


def test_outputs_over_scales_and_slots():
    for name, at, n in (("k_scales", KS, PAGES * PAGE * N_KV * 4), ("v_scales", VS, PAGES * PAGE * N_KV * 4), ("slots", SLOTS, 8 * T)):
        for to in (at - ROW * T + 16, at + n - 16):
            _refused(f"k_out overlaps {name}", ko=to)
            _refused(f"v_out overlaps {name}", vo=to)


def test_outputs_between_two_pages_that_reach_into_one():
    page = PAGE * N_KV * HD
    gap = ROW * T + 64
    kw = dict(page_stride=page + gap)
    for at in (page - 16, page + gap - ROW * T + 16, page + gap // 2):
        _refused("k_out overlaps k_pages", ko=KP + 3 * (page + gap) + at, **kw)
    # a row in each gap: the rows' step is not the pages'
    _refused("k_out overlaps k_pages", ko=KP + page, stride=(page + gap) // 2 + 8, **kw)


def test_rows_of_f16_pages_themselves():
    """The pool's own rows as the output: the same step, the same places."""
    _refused("k_out overlaps k_pages", False, ko=KP + ROW)
    _refused("different", False, ko=KP)
