"""mi_logprobs against the definition in 64 bits. Ranks and ids are equal; probabilities and entropy are held to the
roundings of their formulas (u = 2^-24): d = x - m is off by u |d|, an exponential by (3 |d| + 3) u of its value, a sum of n
terms by its longest chain of additions, n / 256 + 40 of them, a logarithm by 2 u of its value."""
import numpy as np
import pytest

from mipkg import dev, empty, host, mi, ptr, stream, sync, torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
NONE = 0xFFFFFFFF


def call(x, tokens, used, top, st=None, entropy=True):
    T = torch()
    M, stride = x.shape
    dx = dev(x)
    dt = dev(tokens.astype(np.uint32)) if tokens is not None else None
    lp, rk = (empty((M,), np.float32), empty((M,), np.uint32)) if tokens is not None else (None, None)
    en = empty((M,), np.float32) if entropy else None
    ids, tl = (empty((M * top + 4,), np.uint32), empty((M * top + 4,), np.float32)) if top else (None, None)
    if top:
        ids.fill_(-7)
        tl.fill_(9.0)
    need = mi.lib().mi_logprobs_ws(M, used, top)
    ws = T.full((need + 64,), 77, dtype=T.uint8, device="cuda")
    mi.call("mi_logprobs", ptr(dx), stride, ptr(dt), M, used, top, ptr(lp), ptr(rk), ptr(en), ptr(ids), ptr(tl), ptr(ws), need,
            st if st is not None else stream())
    sync()
    assert (ws[need:] == 77).all()
    got = {"lp": host(lp, np.float32) if lp is not None else None, "rank": host(rk, np.uint32) if rk is not None else None,
           "entropy": host(en, np.float32) if en is not None else None}
    if top:
        assert (host(ids, np.int32)[M * top:] == -7).all() and (host(tl, np.float32)[M * top:] == 9.0).all()
        got["ids"] = host(ids, np.uint32)[:M * top].reshape(M, top)
        got["top"] = host(tl, np.float32)[:M * top].reshape(M, top)
    return got


def check_row(x, token, top, got, r):
    """one row x fp32 [used], finite or -inf, not all -inf"""
    n = len(x)
    xd = x.astype(np.float64)
    m = xd.max()
    d = xd - m
    e = np.exp(d)
    z = e.sum()
    p = e / z
    ad = np.where(e > 0, np.abs(d), 0.0)
    D, D2, logz = (p * ad).sum(), (p * ad * ad).sum(), np.log(z)
    chain = n / 256 + 40
    sum_z = U * (chain + 3 * D + 3)  # of log z
    if got["entropy"] is not None:
        tol = sum_z + 2 * U * logz + U * (D * (2 * chain + 8) + 4 * D2 + D + logz + 1)
        assert abs(got["entropy"][r] - (logz + D)) <= tol, (got["entropy"][r], logz + D, tol)

    def near(v, i):
        want = d[i] - logz
        if want == -np.inf:
            return v == -np.inf
        return abs(float(v) - want) <= sum_z + U * (2 * abs(d[i]) + 3 * logz + abs(want))

    if token is not None:
        assert near(got["lp"][r], token), (got["lp"][r], d[token] - logz)
        want = int((x > x[token]).sum() + (x[:token] == x[token]).sum())
        assert got["rank"][r] == want
    if top:
        order = np.lexsort((np.arange(n), -xd))[:top]
        k = len(order)
        assert np.array_equal(got["ids"][r][:k], order.astype(np.uint32)), (got["ids"][r], order)
        assert all(near(got["top"][r][i], order[i]) for i in range(k))
        assert (got["ids"][r][k:] == NONE).all() and (got["top"][r][k:] == -np.inf).all()


SIZES = [(1, 1, 1), (1, 2, 5), (3, 5, 64), (2, 63, 20), (1, 64, 64), (4, 100, 3), (2, 1023, 1), (2, 1025, 20), (1, 4096, 64),
         (5, 4099, 20), (1, 50257, 20), (3, 151669, 5), (1, 151936, 64), (40, 32001, 20), (300, 8192, 7), (1500, 2049, 20)]


@pytest.mark.parametrize("kind", ["normal", "ties", "peaked", "masked", "rising", "flat"])
@pytest.mark.parametrize("M,n,top", SIZES)
def test_against_the_definition(M, n, top, kind):
    rng = np.random.default_rng(n + top)
    pad = int(rng.integers(0, 9))
    x = rng.normal(0, 2, (M, n + pad)).astype(np.float32)
    if kind == "ties":
        x = np.round(x)
    elif kind == "peaked":
        x[np.arange(M), rng.integers(0, n, M)] += 40
    elif kind == "masked":
        keep = rng.random(n + pad) < max(0.02, 2 / n)
        keep[rng.integers(0, n)] = True
        x[:, ~keep] = -np.inf
    elif kind == "rising":
        x = np.sort(x, 1)
    elif kind == "flat":
        x[:] = np.float32(3.25)
        x[:, 0] = -0.0 if n > 1 else 3.25
    x[:, n:] = 1e30  # behind the vocabulary
    tokens = rng.integers(0, n, M)
    if kind == "masked":
        tokens[:] = np.flatnonzero(x[0, :n] > -np.inf)[0]
    got = call(x, tokens, n, top)
    for r in sorted(set(range(M)) if M <= 8 else {0, 1, M // 2, M - 1}):
        check_row(x[r, :n], int(tokens[r]), top, got, r)


@pytest.mark.parametrize("kind", ["normal", "ties", "flat", "falling", "rising", "few", "last", "nan"])
@pytest.mark.parametrize("M,n,top", [(1, 700001, 20), (2, 530000, 64), (1, 151936, 33), (3, 2500, 64), (1, 1 << 23, 5)])
def test_best_tokens_of_a_cut_row(M, n, top, kind):
    """rows in slices: the best tokens come from few runs, from runs of equal logits, from all of them"""
    rng = np.random.default_rng(n + top)
    x = rng.normal(0, 2, (M, n)).astype(np.float32)
    if kind == "ties":
        x = np.round(x)
    elif kind == "flat":
        x[:] = -1.5
    elif kind == "falling":
        x = -np.sort(-x, 1)
    elif kind == "rising":
        x = np.sort(x, 1)
    elif kind == "few":  # fewer finite than asked, at the end
        x[:, :n - 3] = -np.inf
    elif kind == "last":  # equal ones but for the last, and one large
        x[:] = 0
        x[:, n - 1] = 1
    elif kind == "nan":  # a NaN is behind every token, the others keep their places
        x[:, ::3] = np.nan
        x[:, :1024] = np.nan
    tokens = rng.integers(0, n, M)
    got = call(x, tokens, n, top)
    for r in range(M):
        if kind != "nan":
            check_row(x[r, :n], int(tokens[r]) if x[r, tokens[r]] > -np.inf else None, top, got, r)
        else:
            order = np.lexsort((np.arange(n), np.where(np.isnan(x[r]), np.inf, -x[r])))[:min(top, int((~np.isnan(x[r])).sum()))]
            assert np.array_equal(got["ids"][r][:len(order)], order.astype(np.uint32))


@pytest.mark.parametrize("n", [7, 5000, 70001])
def test_rows_without_finite_answers(n):
    rng = np.random.default_rng(n)
    low = np.float32(np.finfo(np.float32).min)
    x = rng.normal(0, 1, (7, n)).astype(np.float32)
    x[0] = -np.inf
    x[1, n // 2] = np.nan
    x[2, n - 1] = np.inf
    x[3] = low            # the type's lowest value everywhere: a flat row
    x[4, 1:] = low        # one token left
    x[4, 0] = 2.0
    x[5, n // 3] = -np.inf
    tokens = np.array([0, 1, n - 1, 2, 0, n // 3, n])
    got = call(x, tokens, n, 3)
    assert np.isnan(got["lp"][[0, 1, 2]]).all() and np.isnan(got["entropy"][[0, 1, 2]]).all()
    assert got["ids"][0].tolist() == [0, 1, 2] and np.isnan(got["top"][0]).all()
    clean = np.where(np.isnan(x[1]), -np.inf, x[1])
    assert got["ids"][1].tolist() == np.lexsort((np.arange(n), -clean))[:3].tolist()  # a NaN is behind every token
    assert got["ids"][2][0] == n - 1
    assert abs(got["lp"][3] + np.log(n)) < 1e-4 and abs(got["entropy"][3] - np.log(n)) < 1e-4 and got["rank"][3] == 2
    assert got["lp"][4] == 0 and got["entropy"][4] == 0 and got["ids"][4].tolist() == [0, 1, 2]
    assert got["lp"][5] == -np.inf and got["rank"][5] == n - 1
    check_row(x[5], None, 3, got, 5)
    assert np.isnan(got["lp"][6]) and got["rank"][6] == NONE  # a token outside the vocabulary
    check_row(x[6], None, 3, got, 6)
    nan_token = call(x[1:2], np.array([n // 2]), n, 0)
    assert np.isnan(nan_token["lp"][0]) and nan_token["rank"][0] == NONE


@pytest.mark.parametrize("M,n", [(1, 9001), (200, 3001)])
def test_parts_may_be_left_out(M, n):
    rng = np.random.default_rng(M)
    x, tokens = rng.normal(0, 2, (M, n)).astype(np.float32), rng.integers(0, n, M)
    whole = call(x, tokens, n, 9)
    for kw in ({"tokens": None, "top": 9}, {"tokens": tokens, "top": 0}, {"tokens": tokens, "top": 9, "entropy": False}):
        part = call(x, kw["tokens"], n, kw["top"], entropy=kw.get("entropy", True))
        for k, v in part.items():
            assert v is None or np.array_equal(v, whole[k]), k


def test_other_stream_and_replayed_graph():
    T = torch()
    rng = np.random.default_rng(5)
    side = T.cuda.Stream()
    with T.cuda.stream(side):
        x, tokens = rng.normal(0, 2, (2, 40000)).astype(np.float32), np.array([5, 39999])
        got = call(x, tokens, 40000, 20, st=side.cuda_stream)
        for r in range(2):
            check_row(x[r], int(tokens[r]), 20, got, r)
    for M, n in ((1, 20011), (700, 2000)):
        dx, dt = empty((M, n), np.float32), dev(np.zeros(M, np.uint32))
        lp, rk, en = empty((M,), np.float32), empty((M,), np.uint32), empty((M,), np.float32)
        ids, tl = empty((M, 4), np.uint32), empty((M, 4), np.float32)
        need = mi.lib().mi_logprobs_ws(M, n, 4)
        ws = T.empty(max(need, 1), dtype=T.uint8, device="cuda")
        dx.zero_()
        g = T.cuda.CUDAGraph()
        with T.cuda.graph(g):
            mi.call("mi_logprobs", ptr(dx), n, ptr(dt), M, n, 4, ptr(lp), ptr(rk), ptr(en), ptr(ids), ptr(tl), ptr(ws), need, stream())
        for _ in range(3):
            x, tokens = rng.normal(0, 2, (M, n)).astype(np.float32), rng.integers(0, n, M)
            dx.copy_(dev(x))
            dt.copy_(dev(tokens.astype(np.uint32)))
            g.replay()
            sync()
            got = {"lp": host(lp, np.float32), "rank": host(rk, np.uint32), "entropy": host(en, np.float32),
                   "ids": host(ids, np.uint32).reshape(M, 4), "top": host(tl, np.float32).reshape(M, 4)}
            for r in {0, M - 1}:
                check_row(x[r], int(tokens[r]), 4, got, r)
