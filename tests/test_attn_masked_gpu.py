"""mi_attn_masked against the definition in 64 bits.

Tolerance, per output: a score is off by at most ds = scale * (2^-21 + head_dim 2^-23) sum|q k| (q in f16 high and low
parts, sums in fp32), with a cap by 2^-20 cap more, with slopes by 2^-22 of the bias; a weight by that and by its f16
rounding, 2^-11 of it (weights under 2^-24 of 1/128 of the largest: 2^-32 each at most). The weights' sum is taken before
that rounding. So |out - exact| <= (2^-11 + 2.1 max ds + 2^-19) sum p|v| + keys 2^-32 max|v| + half a step of f16."""
import numpy as np
import pytest

from mipkg import dev, empty, host, mi, ptr, stream, sync, torch

pytestmark = pytest.mark.gpu
GUARD = 32


class Case:
    """Inputs of one call; K and V as [kv_head][key][dim] f16, placed into a cache when called."""

    def __init__(self, seed, T, keys, qh=10, kvh=2, hd=128, lo=None, hi=None, pos=None, pos0=None, prefix=0, cap=0.0,
                 slopes=False, scale=None, page=0, q_std=1.0):
        rng = np.random.default_rng(seed)
        self.T, self.keys, self.qh, self.kvh, self.hd, self.page = T, keys, qh, kvh, hd, page
        self.q = (rng.standard_normal((T, qh, hd)) * q_std).astype(np.float32)
        self.k, self.v = (rng.standard_normal((kvh, keys, hd)).astype(np.float16) for _ in range(2))
        self.lo, self.hi, self.pos = (None if a is None else np.asarray(a, np.uint32) for a in (lo, hi, pos))
        self.pos0 = max(keys - T, 0) if pos0 is None else pos0
        self.prefix, self.cap = prefix, cap
        self.slopes = (2.0 ** (-8.0 / qh * np.arange(1, qh + 1))).astype(np.float32) if slopes else None
        self.scale = hd ** -0.5 if scale is None else scale
        self.order = rng.permutation(-(-keys // page) + 3)[:-(-keys // page)].astype(np.uint32) if page else None
        self.n_pages = -(-keys // page) + 3 if page else 0
        self.fill = np.float16(np.nan)  # what the cache holds where no key is

    def seen(self):
        p = self.pos.astype(np.int64) if self.pos is not None else self.pos0 + np.arange(self.T)
        hi = np.minimum(self.hi.astype(np.int64) if self.hi is not None else p + 1, self.keys)
        lo = self.lo.astype(np.int64) if self.lo is not None else np.zeros(self.T, np.int64)
        j = np.arange(self.keys)
        return (j < hi[:, None]) & ((j >= lo[:, None]) | (j < self.prefix)), p

    def exact(self, k=None, v=None):
        k, v = self.k if k is None else k, self.v if v is None else v
        seen, p = self.seen()
        out, tol = np.zeros((self.T, self.qh, self.hd)), np.zeros((self.T, self.qh, self.hd))
        far = np.abs(p[:, None] - np.arange(self.keys)).astype(np.float64)
        for h in range(self.qh):
            kd, vd = k[h // (self.qh // self.kvh)].astype(np.float64), v[h // (self.qh // self.kvh)].astype(np.float64)
            qd = self.q[:, h].astype(np.float64)
            s = qd @ kd.T * self.scale
            ds = abs(self.scale) * (2.0 ** -21 + self.hd * 2.0 ** -23) * (np.abs(qd) @ np.abs(kd).T)
            if self.cap:
                s = self.cap * np.tanh(s / self.cap)
                ds = ds + 2.0 ** -20 * self.cap
            if self.slopes is not None:
                s = s - float(self.slopes[h]) * far
                ds = ds + 2.0 ** -22 * float(self.slopes[h]) * far
            s = np.where(seen, s, -np.inf)
            m = s.max(1, keepdims=True)
            e = np.where(seen, np.exp(s - np.where(np.isfinite(m), m, 0)), 0)
            z = e.sum(1, keepdims=True)
            w = e / np.where(z > 0, z, 1)
            out[:, h] = w @ vd
            near = np.where(w > 1e-12, ds, 0).max(1, keepdims=True)
            tol[:, h] = (2.0 ** -11 + 2.1 * near + 2.0 ** -19) * (w @ np.abs(vd)) + self.keys * 2.0 ** -32 * np.abs(vd).max()
        return out, tol + 2.0 ** -11 * np.abs(out) + 2.0 ** -25

    def place(self, x, by_row):
        """the cache: paged or not, head-major or row-major, with `fill` wherever no key is"""
        rows = self.n_pages * self.page if self.page else self.keys + 5
        j = np.arange(self.keys)
        at = self.order[j // self.page].astype(np.int64) * self.page + j % self.page if self.page else j
        c = np.full((rows, self.kvh, self.hd + 8) if by_row else (self.kvh, rows, self.hd), self.fill, np.float16)
        if by_row:
            c[at, :, :self.hd] = x.transpose(1, 0, 2)
        else:
            c[:, at] = x
        return dev(c.view(np.uint16)), ((self.kvh * (self.hd + 8), self.hd + 8) if by_row else (self.hd, rows * self.hd))

    def shape(self, act=0):
        return mi.AttnShape(self.qh, self.kvh, self.hd, self.hd, 0, (self.qh + 2 * self.kvh) * self.hd, self.qh * self.hd,
                            (self.qh + self.kvh) * self.hd, self.scale, 1e-6, act)

    def bind(self, by_row=False, k=None, v=None, kv_len=None, pages=None, act=0):
        T = torch()
        dk, (rs, hs) = self.place(self.k if k is None else k, by_row)
        dv, _ = self.place(self.v if v is None else v, by_row)
        keep = {n: dev(getattr(self, n)) for n in ("lo", "hi", "pos", "slopes", "q")}
        keep["pages"] = dev(self.order if pages is None else pages) if self.page else None
        sh = self.shape(act)
        mask = mi.AttnMask(lo=ptr(keep["lo"]), hi=ptr(keep["hi"]), pos=ptr(keep["pos"]), pos0=self.pos0, prefix=self.prefix,
                           cap=self.cap, slopes=ptr(keep["slopes"]))
        n = kv_len or self.keys
        need = mi.lib().mi_attn_masked_ws(self.T, n, mi.C.byref(sh))
        ws = T.full((need + GUARD,), 77, dtype=T.uint8, device="cuda")
        out = empty((self.T * self.qh * self.hd + GUARD,), np.uint16)
        out.fill_(1234)
        flag = dev(np.zeros(1, np.uint32))
        args = (ptr(keep["q"]), ptr(dk), ptr(dv), rs, hs, ptr(keep["pages"]), self.page, self.n_pages, n, self.T,
                mi.C.byref(sh), mi.C.byref(mask), ptr(ws), need, ptr(out), ptr(flag))
        keep.update(k=dk, v=dv, sh=sh, mask=mask, ws=ws, out=out, flag=flag, need=need, args=args)
        return keep

    def result(self, b):
        sync()
        assert (b["ws"][b["need"]:] == 77).all()
        o = host(b["out"], np.uint16)
        assert (o[-GUARD:] == 1234).all()
        return o[:-GUARD].view(np.float16).reshape(self.T, self.qh, self.hd)

    def run(self, st=None, **kw):
        b = self.bind(**kw)
        mi.call("mi_attn_masked", *b["args"], st if st is not None else stream())
        got = self.result(b)
        assert int(host(b["flag"], np.uint32)[0]) == 0
        return got

    def check(self, **kw):
        want, tol = self.exact()
        got = self.run(**kw).astype(np.float64)
        assert np.isfinite(got).all()
        assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)
        return got


HEADS = [(10, 2, 128), (8, 8, 128), (16, 2, 256), (12, 2, 256), (17, 1, 128), (34, 2, 128), (64, 1, 128), (3, 3, 256)]


@pytest.mark.parametrize("qh,kvh,hd", HEADS)
@pytest.mark.parametrize("T,keys", [(1, 1), (1, 31), (1, 33), (1, 1000), (2, 2), (3, 64), (5, 700), (16, 16), (33, 257), (70, 70)])
def test_causal(T, keys, qh, kvh, hd):
    Case(T + keys + hd, T, keys, qh, kvh, hd).check(by_row=bool(T % 2))


@pytest.mark.parametrize("T,keys,qh,kvh,hd", [(1, 20000, 10, 2, 128), (2, 9000, 16, 2, 256), (300, 300, 10, 2, 128), (130, 1500, 16, 2, 256),
                                              (700, 700, 40, 8, 128), (1100, 1100, 16, 16, 128)])
@pytest.mark.parametrize("page", [0, 16, 24, 64])
def test_long(T, keys, qh, kvh, hd, page):
    Case(T + page, T, keys, qh, kvh, hd, cap=50.0 if page == 24 else 0.0, page=page).check()


@pytest.mark.parametrize("cap,slopes,scale,q_std", [(30.0, False, None, 3.0), (5.0, True, None, 4.0), (0.0, True, None, 1.0),
                                                    (0.0, False, -0.05, 1.0), (0.0, False, 0.0, 1.0), (50.0, False, 1.0, 2.0), (0.0, False, None, 20.0)])
@pytest.mark.parametrize("T,keys,qh,kvh,hd", [(1, 777, 10, 2, 128), (4, 500, 16, 2, 256), (90, 400, 10, 2, 128), (50, 130, 16, 2, 256)])
def test_caps_and_distance(T, keys, qh, kvh, hd, cap, slopes, scale, q_std):
    Case(T + keys, T, keys, qh, kvh, hd, cap=cap, slopes=slopes, scale=scale, q_std=q_std).check()


def documents(T, before, starts, given=0, window=0, padded=0):
    lo, hi = [], []
    for t in range(T):
        s = max(x for x in starts if x <= t)
        p = before + t
        lo.append(max(before + s, p + 1 - window if window else 0))
        hi.append(0 if t >= T - padded else max(p + 1, before + s + given))
    return lo, hi


@pytest.mark.parametrize("qh,kvh,hd", [(10, 2, 128), (16, 2, 256), (20, 1, 128)])
@pytest.mark.parametrize("T,before,starts,given,window,padded,shared", [
    (1, 400, [0], 0, 100, 0, False), (6, 300, [0, 2, 5], 0, 0, 1, True), (6, 300, [0, 2, 5], 0, 0, 0, False),
    (200, 0, [0, 3, 64, 65, 150], 0, 0, 0, False), (200, 333, [0, 40, 128], 30, 0, 17, True), (150, 31, [0, 77], 20, 16, 0, False),
    (64, 1000, [0, 32], 0, 0, 64, True), (97, 64, [0, 33, 34, 35], 1, 0, 60, True)])
def test_spans(T, before, starts, given, window, padded, shared, qh, kvh, hd):
    lo, hi = documents(T, before, starts, given, window, padded)
    c = Case(T + before, T, before + T, qh, kvh, hd, lo=lo, hi=hi, prefix=before if shared else 0, slopes=bool(given), cap=20.0 if window else 0.0)
    got = c.check()
    if padded:
        assert not got[T - padded:].any()


def test_rows_that_see_nothing_or_little():
    T, keys = 40, 300
    rng = np.random.default_rng(9)
    lo, hi = rng.integers(0, keys, T), rng.integers(0, keys + 50, T)
    lo[:6], hi[:6] = [5, 0, 299, 300, 7, 0], [5, 0, 300, 300, 3, 1]
    for prefix in (0, 1, 40, 1000):
        got = Case(1, T, keys, lo=lo, hi=hi, prefix=prefix, slopes=True, pos=rng.integers(0, 2 * keys, T)).check()
        if prefix == 0:
            assert not got[[0, 1, 3, 4]].any()
    for t in range(6):
        Case(2, 1, keys, lo=lo[t:t + 1], hi=hi[t:t + 1]).check()


@pytest.mark.parametrize("T,qh,kvh,hd", [(1, 10, 2, 128), (3, 16, 2, 256), (60, 10, 2, 128), (60, 16, 2, 256), (700, 40, 8, 128)])
@pytest.mark.parametrize("poison", [np.nan, np.inf, -np.inf])
def test_unseen_keys_have_no_part(T, qh, kvh, hd, poison):
    """infinities and NaN in K and V rows that some rows do not see: those rows are as if the rows were clean; the
    rows that see them are not finite there"""
    keys = 900
    lo = np.full(T, 100) if T < 10 else np.where(np.arange(T) < T // 2, 50, 300)
    c = Case(T, T, keys, qh, kvh, hd, lo=lo)
    k, v = c.k.copy(), c.v.copy()
    bad = [3, 40, 299 if T >= 10 else 99]  # seen by the first half of a chunk at most
    k[:, bad[0]] = poison
    v[:, bad, 5] = np.float16(poison)
    want, tol = c.exact()
    got = c.run(k=k, v=v).astype(np.float64)
    clean = np.arange(T) >= T // 2 if T >= 10 else np.ones(T, bool)
    assert np.all(np.abs(got - want)[clean] <= tol[clean])
    if T >= 10:
        assert not np.isfinite(got[c.seen()[0][:, bad[2]]][:, :, 5]).any()
        rest = np.arange(hd) != 5
        assert np.all(np.abs(got - want)[~clean][:, :, rest] <= tol[~clean][:, :, rest])


def test_keys_behind_kv_len_are_not_read():
    c = Case(4, 2, 500, hi=[700, 480], lo=[0, 10])
    short = Case(4, 2, 500, hi=[450, 450], lo=[0, 10])
    k, v = c.k.copy(), c.v.copy()
    k[:, 450:], v[:, 450:] = np.nan, np.nan
    want, tol = short.exact()
    got = c.run(k=k, v=v, kv_len=450).astype(np.float64)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("T", [1, 50])
def test_a_page_outside_the_cache_is_reported(T):
    c = Case(8, T, 400, page=32)
    pages = c.order.copy()
    pages[3] = c.n_pages
    pages[5] = 0xFFFFFFFF
    c.fill = np.float16(0)
    b = c.bind(pages=pages)
    mi.call("mi_attn_masked", *b["args"], stream())
    c.result(b)
    assert int(host(b["flag"], np.uint32)[0]) == mi.STATUS_BAD_PAGE
    no_flag = b["args"][:-1] + (None,)
    mi.call("mi_attn_masked", *no_flag, stream())
    sync()


def test_bf16_activations_round_to_bf16():
    for T in (1, 70):
        c = Case(5, T, 300)
        got = c.run(act=1)
        bits = got.astype(np.float32).view(np.uint32)
        assert not (bits & 0xFFFF).any()  # bf16 values
        want, tol = c.exact()
        assert np.all(np.abs(got.astype(np.float64) - want) <= tol + 2.0 ** -8 * np.abs(want))


def test_other_stream_and_replayed_graph():
    """a captured call reads spans, positions, pages and rows anew at every replay"""
    T = torch()
    side = T.cuda.Stream()
    with T.cuda.stream(side):
        c = Case(3, 1, 3000, cap=30.0)
        want, tol = c.exact()
        assert np.all(np.abs(c.run(st=side.cuda_stream).astype(np.float64) - want) <= tol)
    for rows, qh, kvh, hd in ((1, 10, 2, 128), (2, 16, 2, 256), (80, 10, 2, 128)):
        c = Case(6, rows, 1200, qh, kvh, hd, lo=np.zeros(rows), hi=np.ones(rows), pos=np.zeros(rows), slopes=True, page=64)
        b = c.bind()
        g = T.cuda.CUDAGraph()
        with T.cuda.graph(g):
            mi.call("mi_attn_masked", *b["args"], stream())
        for n in (40, 1200, 0, 700):
            c.hi = np.full(rows, n, np.uint32)
            c.lo = np.arange(rows, dtype=np.uint32) % 50
            c.pos = np.full(rows, max(n, 1) - 1, np.uint32)
            for name in ("lo", "hi", "pos"):
                b[name].copy_(dev(getattr(c, name)))
            b["out"][:-GUARD] = 0
            g.replay()
            want, tol = c.exact()
            assert np.all(np.abs(c.result(b).astype(np.float64) - want) <= tol)


@pytest.mark.parametrize("T,keys,qh,kvh,hd", [(400, 3000, 16, 2, 256), (40, 6000, 16, 2, 256), (25, 9000, 20, 4, 128), (300, 4000, 32, 8, 128)])
@pytest.mark.parametrize("page,cap,slopes,by_row", [(0, 0.0, False, False), (64, 30.0, True, False), (24, 0.0, True, True)])
def test_chunks_behind_a_long_text(T, keys, qh, kvh, hd, page, cap, slopes, by_row):
    """chunks whose keys are split into few and into many parts, with either width of a work-group"""
    before = keys - T
    lo, hi = documents(T, before, [0, T // 3, T // 2], given=9, padded=2)
    c = Case(T + keys, T, keys, qh, kvh, hd, cap=cap, slopes=slopes, page=page)
    c.check(by_row=by_row)
    c = Case(T + keys + 1, T, keys, qh, kvh, hd, cap=cap, slopes=slopes, page=page, lo=lo, hi=hi, prefix=before - 77)
    got = c.check(by_row=by_row)
    assert not got[T - 2:].any()


class FarCase(Case):
    """a cache whose last rows lie past 2^32 bytes, its first ones never written"""

    def place(self, x, by_row):
        T = torch()
        if self.page:  # head-major pages
            rows = self.n_pages * self.page
            j = np.arange(self.keys)
            at = self.order[j // self.page].astype(np.int64) * self.page + j % self.page
            strides = (self.hd, rows * self.hd)
        else:  # rows far apart
            at, strides = np.arange(self.keys, dtype=np.int64), (1 << 23, self.hd)
        c = T.empty(int(at.max() * strides[0] + (self.kvh - 1) * strides[1] + self.hd), dtype=T.int16, device="cuda")
        view = c.as_strided((int(at.max()) + 1, self.kvh, self.hd), (strides[0], strides[1], 1))
        view[T.from_numpy(at).cuda()] = T.from_numpy(np.ascontiguousarray(x.transpose(1, 0, 2)).view(np.int16)).cuda()
        return c, strides


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("T", [1, 50])
@pytest.mark.parametrize("page", [0, 64])
def test_offsets_past_32_bits(T, hd, page):
    c = FarCase(T + hd, T, 600, 8, 2, hd, page=page)
    if page:
        c.n_pages = 150000
        c.order = (c.n_pages - 1 - 997 * np.arange(10)).astype(np.uint32)
    c.check()
