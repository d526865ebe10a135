"""mi_attn_masked: what no row sees has no part in the outputs, and rows that see nothing give zeros, whatever their q and
the cache hold there. The tolerances are test_attn_masked_gpu.py's."""
import numpy as np
import pytest

from test_attn_masked_gpu import Case

pytestmark = pytest.mark.gpu

# The few-rows kernel and the chunk's, at rows of 128 and 256, in one part of the keys, in up to eight and in more (the
# parts have a join each).
WAYS = [(2, 60, 10, 2, 128), (3, 60, 10, 2, 128), (2, 60, 16, 2, 256), (3, 700, 10, 2, 128), (2, 600, 16, 2, 256),
        (3, 5000, 10, 2, 128), (2, 5000, 16, 2, 256), (70, 90, 10, 2, 128), (70, 90, 16, 2, 256), (333, 333, 40, 8, 128), (500, 4500, 32, 8, 128),
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
