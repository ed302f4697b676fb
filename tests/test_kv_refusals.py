"""What the paged cache, its attention and the grouped router decline: before any side effect, with or without a GPU."""
import ctypes as C

import pytest

FAKE = 1 << 20  # a 16-byte aligned address that no declined call touches


@pytest.fixture(scope="module")
def lib():
    from fucina_b200._lib import load

    return load()


def pages(**kw):
    from fucina_b200._lib import KvPagesStruct

    a = dict(fmt=1, k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, n_pages=8, page_tokens=16, kv_heads=2, d=128, page_stride=0, scale_stride=0)
    a.update(kw)
    return C.byref(KvPagesStruct(**a))


BAD_PAGES = [dict(fmt=2), dict(fmt=-1), dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=FAKE + 8), dict(v_scale=FAKE + 2),
             dict(n_pages=0), dict(n_pages=1 << 31), dict(page_tokens=0), dict(page_tokens=24), dict(page_tokens=8192), dict(kv_heads=0),
             dict(kv_heads=513), dict(d=0), dict(d=48), dict(d=288), dict(fmt=0, d=24), dict(fmt=0, d=264), dict(page_stride=16 * 2 * 128 - 16),
             dict(page_stride=16 * 2 * 128 + 8), dict(page_stride=1 << 60), dict(scale_stride=1), dict(scale_stride=129)]


def append(lib, p, k=FAKE, v=FAKE, stride=0, seq=FAKE, pos=FAKE, n=4, table=FAKE, n_seqs=2, max_pages=4):
    return lib.fq_kv_append_dev(p, k, v, stride, seq, pos, n, table, n_seqs, max_pages, None)


def read(lib, p, k=FAKE, v=FAKE, half=0, seq=FAKE, pos=FAKE, n=4, table=FAKE, n_seqs=2, max_pages=4):
    return lib.fq_kv_read_dev(p, k, v, half, seq, pos, n, table, n_seqs, max_pages, None)


def attend(lib, p, q=FAKE, stride=0, table=FAKE, lens=FAKE, n_seqs=2, max_pages=4, max_len=0, heads=8, scale=1.0, window=0, out=FAKE, stats=None,
           ws=None, ws_bytes=0):
    return lib.fq_attn_paged_dev(p, q, stride, table, lens, n_seqs, max_pages, max_len, heads, scale, window, out, stats, ws, ws_bytes, None)


def route(lib, x=FAKE, seq=4, e=64, score=0, bias=None, groups=1, kept=1, rank=0, k=4, norm=1, scale=1.0, sel=FAKE, w=FAKE):
    return lib.fq_router_groups_dev(x, seq, e, score, bias, groups, kept, rank, k, norm, scale, sel, w, None)


@pytest.mark.parametrize("kw", BAD_PAGES)
def test_pages_that_make_no_cache(lib, kw):
    assert append(lib, pages(**kw)) == 1
    assert read(lib, pages(**kw)) == 1
    assert attend(lib, pages(**kw)) == 1
    assert lib.fq_attn_paged_workspace_bytes(pages(**kw), 1, 8, 1 << 20) == 0


def test_rows_tables_and_pointers(lib):
    p = pages()
    for kw in (dict(k=None), dict(v=None), dict(seq=None), dict(pos=None), dict(table=None), dict(k=FAKE + 4), dict(stride=252), dict(stride=258),
               dict(stride=1 << 40), dict(n=1 << 40), dict(n_seqs=0), dict(n_seqs=1 << 40), dict(max_pages=0), dict(max_pages=1 << 40)):
        assert append(lib, p, **kw) == 1, kw
    for kw in (dict(k=None, v=None), dict(seq=None), dict(pos=None), dict(table=None), dict(v=FAKE + 8), dict(n=1 << 40), dict(n_seqs=0), dict(max_pages=0),
               dict(max_pages=1 << 30)):
        assert read(lib, p, **kw) == 1, kw
    assert append(lib, None) == 1 and read(lib, None) == 1 and attend(lib, None) == 1
    for kw in (dict(q=None), dict(out=None), dict(table=None), dict(lens=None), dict(heads=0), dict(heads=7), dict(heads=8192), dict(n_seqs=0),
               dict(n_seqs=65536), dict(max_pages=0), dict(max_pages=1 << 32), dict(stride=1020), dict(stride=1025), dict(q=FAKE + 4), dict(out=FAKE + 8)):
        assert attend(lib, p, **kw) == 1, kw


def test_router_arguments(lib):
    for kw in (dict(x=None), dict(sel=None), dict(w=None), dict(seq=0), dict(seq=1 << 40), dict(e=0), dict(e=4097), dict(score=2), dict(score=-1),
               dict(rank=2), dict(groups=0), dict(groups=3), dict(groups=65, e=65), dict(kept=0), dict(kept=2), dict(k=0), dict(k=33),
               dict(groups=32, kept=1, k=3)):
        assert route(lib, **kw) == 1, kw


def test_good_arguments_get_past_the_checks_without_a_gpu(lib):
    """The same calls without a mistake: only the missing GPU stops them."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("the pointers are made up")
    p = pages()
    assert append(lib, p) == 2 and read(lib, p) == 2 and attend(lib, p) == 2 and route(lib) == 2
    assert read(lib, p, k=None) == 2 and append(lib, p, stride=260) == 2 and route(lib, groups=8, kept=4, rank=1, score=1) == 2
    assert attend(lib, pages(fmt=0, d=80, k_scale=None, v_scale=None)) == 2
