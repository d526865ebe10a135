"""The scoring entries at the edges of what their documentation allows: two calls at once, graphs that share a workspace, the
least alignment, the most rows, a page that stands twice in the table."""
import numpy as np
import pytest

from mipkg import dev, empty, host, mi, ptr, stream, sync, torch
from test_attn_masked_gpu import Case
from test_linear_w8a8_gpu import check as check_linear, rows, tile, weights
from test_logprobs_gpu import check_row

pytestmark = pytest.mark.gpu


class Calls:
    """One call of each entry, bound to inputs and outputs of its own; `shared`: a workspace for all of them."""

    def __init__(self, seed, M, shared=None):
        rng = np.random.default_rng(seed)
        T, L = torch(), mi.lib()
        K, N, V, top = 1536, 528, 30001, 7
        self.x, (self.w, self.ws) = rows(rng, M, K), weights(rng, N, K)
        self.logits, self.tokens = rng.normal(0, 2, (M, V)).astype(np.float32), rng.integers(0, V, M)
        self.case = Case(seed, M, 900 + M, 16, 2, 256 if seed % 2 else 128, cap=30.0)
        self.b = self.case.bind()
        need = max(L.mi_linear_w8a8_ws(M, K), L.mi_logprobs_ws(M, V, top), self.b["need"], 16)
        ws = shared if shared is not None else T.empty(need, dtype=T.uint8, device="cuda")
        assert ws.numel() >= need
        self.keep = [dev(self.x.view(np.uint16)), dev(tile(self.w)), dev(self.ws), dev(self.logits), dev(self.tokens.astype(np.uint32)), ws]
        dx, dw, dws, dl, dt, _ = self.keep
        self.out = empty((M, N), np.float32)
        self.lp, self.rank, self.en = empty((M,), np.float32), empty((M,), np.uint32), empty((M,), np.float32)
        self.ids, self.tl = empty((M, top), np.uint32), empty((M, top), np.float32)
        a = self.b["args"]
        self.run = lambda st: (
            mi.call("mi_linear_w8a8", ptr(dx), K, ptr(dw), ptr(dws), ptr(ws), ws.numel(), ptr(self.out), mi.OUT_F32, N, M, K, N, st),
            mi.call("mi_attn_masked", *a[:12], ptr(ws), ws.numel(), a[14], a[15], st),
            mi.call("mi_logprobs", ptr(dl), V, ptr(dt), M, V, top, ptr(self.lp), ptr(self.rank), ptr(self.en), ptr(self.ids), ptr(self.tl),
                    ptr(ws), ws.numel(), st))

    def clear(self):
        for t in (self.out, self.lp, self.rank, self.en, self.ids, self.tl):
            t.zero_()
        self.b["out"][:-32] = 0

    def results(self):
        sync()
        return [self.out.cpu().numpy(), self.case.result(self.b).view(np.uint16)] + [
            t.cpu().numpy() for t in (self.lp, self.rank, self.en, self.ids, self.tl)]

    def check(self):
        out, _, lp, rank, en, ids, tl = self.results()
        check_linear(out, self.x, self.w, self.ws, mi.OUT_F32)
        want, tol = self.case.exact()
        assert np.all(np.abs(self.case.result(self.b).astype(np.float64) - want) <= tol)
        got = {"lp": lp, "rank": rank.view(np.uint32), "entropy": en, "ids": ids.view(np.uint32), "top": tl}
        for m in {0, len(self.x) - 1}:
            check_row(self.logits[m], int(self.tokens[m]), 7, got, m)


@pytest.mark.parametrize("M", [1, 40])
def test_two_calls_at_once(M):
    T = torch()
    sides = [T.cuda.Stream(), T.cuda.Stream()]
    calls = [Calls(10 + i, M) for i in range(2)]
    for c in calls:
        c.run(stream())
        c.check()
    alone = [c.results() for c in calls]
    for _ in range(3):
        for c in calls:
            c.clear()
        sync()
        for _ in range(10):
            for c, s in zip(calls, sides):
                c.run(s.cuda_stream)
        for c, want in zip(calls, alone):
            assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(c.results(), want))


@pytest.mark.parametrize("M", [1, 40])
def test_two_graphs_share_a_workspace(M):
    T = torch()
    ws = T.full((1 << 24,), 0xFF, dtype=T.uint8, device="cuda")
    calls = [Calls(20, M, ws), Calls(21, M + 3, ws)]
    graphs = []
    for c in calls:
        c.run(stream())
        c.check()
    alone = [c.results() for c in calls]
    for c in calls:
        g = T.cuda.CUDAGraph()
        with T.cuda.graph(g):
            c.run(stream())
        graphs.append(g)
    for order in ((0, 1), (1, 0), (0, 0, 1, 1)):
        for c in calls:
            c.clear()
        ws.fill_(0xA5)
        for i in order:
            graphs[i].replay()
        calls[0].run(stream())  # an eager call between the replays
        for c, want in zip(calls, alone):
            assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(c.results(), want))


def shifted(a, elements):
    """the array on the device, `elements` of its own behind an allocation's start"""
    T = torch()
    t = dev(a)
    buf = T.empty(t.numel() + elements, dtype=t.dtype, device="cuda")
    buf[elements:] = t.reshape(-1)
    return buf[elements:]


@pytest.mark.parametrize("M", [1, 6, 70])
def test_least_alignment(M):
    T, L = torch(), mi.lib()
    rng = np.random.default_rng(M)
    K, N = 320, 80
    x, (w, ws) = rows(rng, M, K), weights(rng, N, K)
    dx, dw, dws = dev(x.view(np.uint16)), dev(tile(w)), shifted(ws, 1)
    scratch = T.empty(L.mi_linear_w8a8_ws(M, K), dtype=T.uint8, device="cuda")
    for kind, np_t in ((mi.OUT_F32, np.float32), (mi.OUT_F16, np.uint16)):
        out = empty((M * N + 1,), np_t)[1:]
        mi.call("mi_linear_w8a8", ptr(dx), K, ptr(dw), ptr(dws), ptr(scratch), scratch.numel(), ptr(out), kind, N, M, K, N, stream())
        sync()
        got = host(out, np_t).reshape(M, N)
        check_linear(got if kind == mi.OUT_F32 else got.view(np.float16), x, w, ws, kind)

    n, top = 20011, 6
    logits, tokens = rng.normal(0, 2, (M, n)).astype(np.float32), rng.integers(0, n, M)
    dl, dt = shifted(logits, 1), shifted(tokens.astype(np.uint32), 1)
    lp, rk, en = (empty((M + 1,), t)[1:] for t in (np.float32, np.uint32, np.float32))
    ids, tl = empty((M * top + 1,), np.uint32)[1:], empty((M * top + 1,), np.float32)[1:]
    lws = T.empty(max(L.mi_logprobs_ws(M, n, top), 1), dtype=T.uint8, device="cuda")
    mi.call("mi_logprobs", ptr(dl), n, ptr(dt), M, n, top, ptr(lp), ptr(rk), ptr(en), ptr(ids), ptr(tl), ptr(lws), lws.numel(), stream())
    sync()
    got = {"lp": host(lp, np.float32), "rank": host(rk, np.uint32), "entropy": host(en, np.float32),
           "ids": host(ids, np.uint32).reshape(M, top), "top": host(tl, np.float32).reshape(M, top)}
    for m in {0, M - 1}:
        check_row(logits[m], int(tokens[m]), top, got, m)

    for hd, splits in ((128, False), (256, True)):
        c = Case(M + hd, M, M + (1500 if splits else 20), 8, 2, hd, slopes=True)
        b = c.bind()
        q, out = shifted(c.q, 1), empty((c.q.size + 1,), np.uint16)[1:]
        sl = shifted(c.slopes, 1)
        b["mask"].slopes = ptr(sl)
        mi.call("mi_attn_masked", ptr(q), *b["args"][1:14], ptr(out), None, stream())
        sync()
        want, tol = c.exact()
        assert np.all(np.abs(host(out, np.uint16).view(np.float16).reshape(want.shape).astype(np.float64) - want) <= tol)


def test_the_most_rows_of_a_linear():
    T, L = torch(), mi.lib()
    M, K, N = 1 << 20, 64, 16
    rng = np.random.default_rng(1)
    w, ws = weights(rng, N, K)
    dx = T.randn(M, K, device="cuda").half()
    scratch = T.empty(L.mi_linear_w8a8_ws(M, K), dtype=T.uint8, device="cuda")
    out, dw, dws = empty((M, N), np.float32), dev(tile(w)), dev(ws)
    mi.call("mi_linear_w8a8", ptr(dx), K, ptr(dw), ptr(dws), ptr(scratch), scratch.numel(), ptr(out), mi.OUT_F32, N, M, K, N, stream())
    sync()
    at = np.r_[0:40, M // 2:M // 2 + 40, M - 40:M]
    check_linear(out[at].cpu().numpy(), dx[at].cpu().numpy(), w, ws, mi.OUT_F32)


def test_the_most_rows_of_log_probabilities():
    T = torch()
    M, n, top = 65535, 1030, 3
    x = T.randn(M, n, device="cuda")
    tokens = np.arange(M) % n
    dt, lp, rk, en = dev(tokens.astype(np.uint32)), empty((M,), np.float32), empty((M,), np.uint32), empty((M,), np.float32)
    ids, tl = empty((M, top), np.uint32), empty((M, top), np.float32)
    assert mi.lib().mi_logprobs_ws(M, n, top) == 0
    mi.call("mi_logprobs", ptr(x), n, ptr(dt), M, n, top, ptr(lp), ptr(rk), ptr(en), ptr(ids), ptr(tl), None, 0, stream())
    sync()
    got = {"lp": host(lp, np.float32), "rank": host(rk, np.uint32), "entropy": host(en, np.float32), "ids": host(ids, np.uint32),
           "top": host(tl, np.float32)}
    for m in (0, 1, 30000, M - 1):
        check_row(x[m].cpu().numpy(), int(tokens[m]), top, got, m)


@pytest.mark.parametrize("qh,kvh,hd", [(1, 1, 128), (2, 1, 256)])
def test_the_most_rows_of_attention(qh, kvh, hd):
    M, keys = 65535, 2000
    pos = (np.arange(M) * 7) % keys
    lo, hi = np.maximum(pos - 30, 0), pos + 1
    hi[-3:] = 0  # padding
    c = Case(hd, M, keys, qh, kvh, hd, lo=lo, hi=hi, pos=pos)
    got = c.run()
    at = np.r_[0:5, 40000:40005, M - 6:M]
    some = Case(hd, 1, keys, qh, kvh, hd)
    some.T, some.q, some.k, some.v = len(at), c.q[at], c.k, c.v
    some.lo, some.hi, some.pos = c.lo[at], c.hi[at], c.pos[at]
    want, tol = some.exact()
    assert np.all(np.abs(got[at].astype(np.float64) - want) <= tol)
    assert not got[-3:].any() and np.isfinite(got).all()


@pytest.mark.parametrize("T,page", [(1, 32), (60, 64), (60, 24)])
def test_a_page_that_stands_twice(T, page):
    c = Case(T + page, T, 8 * page + 5, page=page)
    c.order[3] = c.order[1]  # the keys of the page 3 are those of the page 1
    for x in (c.k, c.v):
        x[:, 3 * page:4 * page] = x[:, page:2 * page]
    c.check()
