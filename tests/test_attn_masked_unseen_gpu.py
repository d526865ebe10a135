"""mi_attn_masked: what no row sees has no part in the outputs, and rows that see nothing give zeros, whatever their q, the
cache and the page table hold there. The tolerances are test_attn_masked_gpu.py's."""
import numpy as np
import pytest

from mipkg import host, mi, stream
from test_attn_masked_gpu import Case

pytestmark = pytest.mark.gpu

# The few-rows kernel and the chunk's, at rows of 128 and 256, in one part of the keys, in up to eight and in more (the
# parts have a join each).
WAYS = [(2, 60, 10, 2, 128), (3, 60, 10, 2, 128), (2, 60, 16, 2, 256), (3, 700, 10, 2, 128), (2, 600, 16, 2, 256),
        (3, 5000, 10, 2, 128), (2, 5000, 16, 2, 256),
        (70, 90, 10, 2, 128), (70, 90, 16, 2, 256), (333, 333, 40, 8, 128), (500, 4500, 32, 8, 128),
        (130, 1500, 16, 2, 256), (20, 4020, 40, 8, 128), (40, 6000, 16, 2, 256)]


def padded_rows(T):
    """rows that see nothing, between the others and at the end"""
    return np.arange(T) % 3 == 1


@pytest.mark.parametrize("q", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("T,keys,qh,kvh,hd", WAYS)
def test_padded_rows_whose_queries_are_not_finite(T, keys, qh, kvh, hd, q):
    pad = padded_rows(T)
    c = Case(T + keys, T, keys, qh, kvh, hd, hi=np.where(pad, 0, np.arange(T) + keys - T + 1))
    c.q[pad] = np.float32(q)
    got = c.run().astype(np.float64)
    c.q[pad] = 0  # (no part in the oracle's)
    want, tol = c.exact()
    assert not got[pad].any()
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("poison", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("T,keys,qh,kvh,hd", WAYS)
def test_keys_that_no_row_sees_beside_seen_ones(T, keys, qh, kvh, hd, poison, padded):
    """infinities and NaN in K rows of the tiles of 32 keys that a row sees in part: before lo, behind hi, behind the prefix"""
    pad = padded_rows(T) if padded else np.zeros(T, bool)
    prefix, lo, hi = 5, 42, keys - 3
    c = Case(T + keys, T, keys, qh, kvh, hd, lo=np.full(T, lo), hi=np.where(pad, 0, hi), prefix=prefix)
    unseen = np.r_[prefix:lo, hi:keys]
    assert not c.seen()[0][:, unseen].any()
    k = c.k.copy()
    k[:, unseen] = poison
    want, tol = c.exact()
    got = c.run(k=k).astype(np.float64)
    assert not got[pad].any()
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("T,lo,page", [(1, 90, 16), (1, 100, 24), (3, 90, 16), (70, 90, 16), (70, 100, 24), (300, 90, 8),
                                       (40, 600, 32)])
@pytest.mark.parametrize("prefix", [0, 5])
def test_pages_that_no_row_sees_may_be_outside_the_cache(T, lo, page, prefix):
    """a window over a cache whose older pages are given back, and pages behind the rows' last key that are not there yet"""
    qh, kvh, hd = (10, 2, 128) if T != 300 else (16, 2, 256)
    keys, hi = 1200, 1100
    c = Case(T + lo + page, T, keys, qh, kvh, hd, lo=np.full(T, lo), hi=np.full(T, hi), prefix=prefix, page=page)
    want, tol = c.exact()
    at = np.arange(-(-keys // page)) * page
    given_back = ((at + page <= lo) & (at >= prefix)) | (at >= hi)
    pages = np.where(given_back, np.uint32(0xFFFFFFFF), c.order).astype(np.uint32)
    got = c.run(pages=pages).astype(np.float64)  # (run holds the flag to 0)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("T,page", [(1, 16), (3, 24), (70, 24), (70, 64)])
def test_pages_between_the_rows_spans_may_be_outside_the_cache(T, page):
    """rows that see far apart keys, in one block of rows"""
    keys = 1500
    second = np.arange(T) % 2 == 1
    lo, hi = np.where(second, 1300, 90), np.where(second, 1400, 200)
    c = Case(T + page, T, keys, 10, 2, 128, lo=lo, hi=hi, page=page)
    want, tol = c.exact()
    seen = c.seen()[0].any(0)
    used = [seen[i:i + page].any() for i in range(0, keys, page)]
    pages = np.where(used, c.order, np.uint32(c.n_pages)).astype(np.uint32)
    got = c.run(pages=pages).astype(np.float64)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("T,page,prefix", [(1, 16, 0), (3, 24, 0), (70, 24, 0), (70, 64, 0), (70, 24, 5), (2, 1, 5), (70, 1, 0)])
def test_one_seen_key_on_a_page_outside_the_cache_is_reported(T, page, prefix):
    lo, hi = 90, 1100
    c = Case(T + page, T, 1200, 10, 2, 128, lo=np.full(T, lo), hi=np.full(T, hi), prefix=prefix, page=page)
    c.fill = np.float16(0)
    for key in [lo, hi - 1] + ([prefix - 1] if prefix else []):
        pages = c.order.copy()
        pages[key // page] = c.n_pages
        b = c.bind(pages=pages)
        mi.call("mi_attn_masked", *b["args"], stream())
        c.result(b)
        assert int(host(b["flag"], np.uint32)[0]) == mi.STATUS_BAD_PAGE, key


@pytest.mark.parametrize("T", [3, 70])
def test_rows_that_see_the_prefix_alone_need_no_other_page(T):
    """lo == hi: such a row beside others, and alone; its pages behind the prefix are not there"""
    page, prefix, keys = 16, 20, 900
    for alone in (False, True):
        lo = np.where((np.arange(T) % 2 == 0) | alone, 600, 300)
        hi = np.where(lo == 600, 600, 340)
        c = Case(T, T, keys, 10, 2, 128, lo=lo, hi=hi, prefix=prefix, page=page)
        want, tol = c.exact()
        seen = c.seen()[0].any(0)
        pages = np.where([seen[i:i + page].any() for i in range(0, keys, page)], c.order, np.uint32(0xFFFFFFFF)).astype(np.uint32)
        got = c.run(pages=pages).astype(np.float64)
        assert np.all(np.abs(got - want) <= tol)
