"""mi_attn_tree against the definition in 64 bits.

Tolerance, per output: a score is off by at most ds = |scale| (2^-21 + head_dim 2^-23) sum|q k| (q in f16 high and low parts, sums in
fp32); a weight by that and by its f16 rounding, 2^-11 of it (weights under 2^-24 of 1/128 of the largest: 2^-32 each at most). The
weights' sum is taken before that rounding. So |out - exact| <= (2^-11 + 2.1 max ds + 2^-19) sum p|v| + keys 2^-32 max|v| + half a
step of f16."""
import numpy as np
import pytest

from mipkg import dev, empty, host, mi, ptr, stream, sync, torch

pytestmark = pytest.mark.gpu
NONE, GUARD = mi.NONE, 32


def tree(rng, n, wide=6):
    return [NONE] + [int(rng.integers(max(0, i - wide), i)) for i in range(1, n)]


def bits_of(parents):
    out = []
    for i, p in enumerate(parents):
        out.append(1 << i | (out[p] if p < i else 0))
    return out


class Case:
    """lengths: (cached, rows) of each sequence; trees: 'causal' (no masks), 'tree', 'random' bits, or a list of rows' bits"""

    def __init__(self, seed, lengths, qh=10, kvh=2, hd=128, page=16, trees="tree", scale=None, q_std=1.0, before=0, behind=0, kv_len=None,
                 words=None, act=0):
        rng = np.random.default_rng(seed)
        self.cached, self.rows = (np.array(x, np.int64) for x in zip(*lengths))
        self.qh, self.kvh, self.hd, self.page, self.act, self.before = qh, kvh, hd, page, act, before
        self.scale = hd ** -0.5 if scale is None else scale
        self.start = before + np.concatenate([[0], np.cumsum(self.rows)])
        self.T = int(self.start[-1]) + behind
        self.keys = self.cached + self.rows
        self.kv_len = kv_len or max(int(self.keys.max()), 1)
        self.q = (rng.standard_normal((self.T, qh, hd)) * q_std).astype(np.float32)
        self.k, self.v = ([rng.standard_normal((kvh, int(n), hd)).astype(np.float16) for n in self.keys] for _ in range(2))
        most = int(self.rows.max()) if len(self.rows) else 1
        self.words = 0 if trees == "causal" else words or max(1, -(-most // 32))
        self.seen_bits = []
        for b, n in enumerate(self.rows):
            if trees == "causal":
                self.seen_bits.append([(2 << i) - 1 for i in range(n)])
            elif trees == "tree":
                self.seen_bits.append(bits_of(tree(rng, n)) if n else [])
            elif trees == "random":
                self.seen_bits.append([int(rng.integers(0, 1 << 62)) & int(rng.integers(0, 1 << 62)) & ((1 << int(n)) - 1) for _ in range(n)])
            else:
                self.seen_bits.append(list(trees[b]))
        self.mask = None
        if self.words:
            self.mask = rng.integers(0, 1 << 32, (self.T, self.words)).astype(np.uint32)  # (of no sequence's rows: anything)
            for b, bits in enumerate(self.seen_bits):
                for i, x in enumerate(bits):
                    self.mask[self.start[b] + i] = [x >> 32 * w & 0xFFFFFFFF for w in range(self.words)]
        pages = [-(-int(n) // page) for n in self.keys] if page else []
        self.n_pages = sum(pages) + 3 if page else 0
        order = rng.permutation(max(self.n_pages, 1)).astype(np.uint32)
        self.stride = max(-(-self.kv_len // page), max(pages), 1) + 1 if page else self.kv_len + 2
        self.tables = np.full((len(lengths), self.stride), NONE, np.uint32) if page else None
        at = 0
        for b, n in enumerate(pages):
            self.tables[b, :n] = order[at:at + n]
            at += n
        self.cache_rows = self.n_pages * page if page else self.stride * len(lengths)
        self.fill = np.float16(np.nan)  # what the cache holds where no key is

    def at(self, b):
        j = np.arange(int(self.keys[b]))
        return self.tables[b, j // self.page].astype(np.int64) * self.page + j % self.page if self.page else b * self.stride + j

    def seen(self, b):
        n, c = int(self.rows[b]), int(self.cached[b])
        s = np.ones((n, c + n), bool)
        for i, x in enumerate(self.seen_bits[b]):
            s[i, c:] = [(x >> m) & 1 for m in range(n)]
        s[:, self.kv_len:] = False
        return s

    def exact(self):
        out, tol = np.zeros((self.T, self.qh, self.hd)), np.zeros((self.T, self.qh, self.hd))
        g = self.qh // self.kvh
        for b, n in enumerate(self.rows):
            if not n:
                continue
            rows, seen = slice(self.start[b], self.start[b] + n), self.seen(b)
            for h in range(self.qh):
                kd, vd = self.k[b][h // g].astype(np.float64), self.v[b][h // g].astype(np.float64)
                qd = self.q[rows, h].astype(np.float64)
                s = np.where(seen, qd @ kd.T * self.scale, -np.inf)
                ds = abs(self.scale) * (2.0 ** -21 + self.hd * 2.0 ** -23) * (np.abs(qd) @ np.abs(kd).T)
                m = s.max(1, keepdims=True)
                e = np.where(seen, np.exp(s - np.where(np.isfinite(m), m, 0)), 0)
                z = e.sum(1, keepdims=True)
                w = e / np.where(z > 0, z, 1)
                out[rows, h] = w @ vd
                near = np.where(w > 1e-12, ds, 0).max(1, keepdims=True)
                tol[rows, h] = (2.0 ** -11 + 2.1 * near + 2.0 ** -19) * (w @ np.abs(vd)) + kd.shape[0] * 2.0 ** -32 * np.abs(vd).max()
        return out, tol + 2.0 ** -11 * np.abs(out) + 2.0 ** -25

    def place(self, x, by_row):
        c = np.full((self.cache_rows, self.kvh, self.hd + 8) if by_row else (self.kvh, self.cache_rows, self.hd), self.fill, np.float16)
        for b in range(len(self.rows)):
            if by_row:
                c[self.at(b), :, :self.hd] = x[b].transpose(1, 0, 2)
            else:
                c[:, self.at(b)] = x[b]
        return dev(c.view(np.uint16)), ((self.kvh * (self.hd + 8), self.hd + 8) if by_row else (self.hd, self.cache_rows * self.hd))

    def bind(self, by_row=False, tables=None, k=None, v=None):
        T = torch()
        dk, (rs, hs) = self.place(self.k if k is None else k, by_row)
        dv, _ = self.place(self.v if v is None else v, by_row)
        keep = {"q": dev(self.q), "row_start": dev(self.start.astype(np.uint32)), "cached": dev(self.cached.astype(np.uint32)),
                "tables": dev(self.tables if tables is None else tables) if self.page else None, "mask": dev(self.mask)}
        sh = mi.AttnShape(self.qh, self.kvh, self.hd, self.hd, 0, (self.qh + 2 * self.kvh) * self.hd, self.qh * self.hd,
                          (self.qh + self.kvh) * self.hd, self.scale, 1e-6, self.act)
        batch = mi.AttnBatch(sequences=len(self.rows), kv_len=self.kv_len, table_stride=self.stride, page=self.page, n_pages=self.n_pages,
                             words=self.words, **{n: ptr(keep[n]) for n in ("row_start", "cached", "tables", "mask")})
        need = mi.lib().mi_attn_tree_ws(self.T, len(self.rows), mi.C.byref(sh))
        ws = T.full((need + GUARD,), 77, dtype=T.uint8, device="cuda")
        out = empty((self.T * self.qh * self.hd + GUARD,), np.uint16)
        out.fill_(1234)
        flag = dev(np.zeros(1, np.uint32))
        args = (ptr(keep["q"]), ptr(dk), ptr(dv), rs, hs, self.T, mi.C.byref(sh), mi.C.byref(batch), ptr(ws), need, ptr(out), ptr(flag))
        keep.update(k=dk, v=dv, sh=sh, batch=batch, ws=ws, out=out, flag=flag, need=need, args=args)
        return keep

    def result(self, b):
        sync()
        assert (b["ws"][b["need"]:] == 77).all()
        o = host(b["out"], np.uint16)
        assert (o[-GUARD:] == 1234).all()
        o = o[:-GUARD].reshape(self.T, self.qh, self.hd)
        assert (o[:self.before] == 1234).all() and (o[self.start[-1]:] == 1234).all()
        o = o.copy()
        o[:self.before], o[self.start[-1]:] = 0, 0
        return o.view(np.float16)

    def run(self, st=None, **kw):
        b = self.bind(**kw)
        mi.call("mi_attn_tree", *b["args"], st if st is not None else stream())
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
@pytest.mark.parametrize("lengths", [[(0, 1)], [(1, 1)], [(31, 1)], [(32, 1)], [(1000, 1)], [(700, 3)], [(0, 16)], [(33, 33)], [(97, 61)],
                                     [(5, 1), (0, 0), (130, 1), (64, 1), (0, 1)], [(40, 3), (0, 20), (333, 64), (0, 0), (9, 1), (31, 2)]])
@pytest.mark.parametrize("trees", ["causal", "tree"])
def test_small(lengths, qh, kvh, hd, trees):
    n = sum(a + b for a, b in lengths)
    Case(n + hd, lengths, qh, kvh, hd, page=(0, 16, 24, 64)[n % 4], trees=trees, before=n % 3, behind=n % 5).check(by_row=bool(n % 2))


@pytest.mark.parametrize("lengths,qh,kvh,hd", [
    ([(20000, 1)], 10, 2, 128), ([(9000, 2)], 16, 2, 256), ([(5000, 61)], 40, 8, 128), ([(6000, 60)], 16, 2, 256), ([(1500, 130)], 16, 2, 256),
    ([(700, 700)], 40, 8, 128), ([(3000, 12), (10, 12), (900, 12)], 10, 2, 128), ([(100 * i, 1) for i in range(30)], 10, 2, 128),
    ([(4000, 40), (100, 64), (2000, 7)], 32, 8, 128), ([(3000, 38)], 10, 2, 128), ([(2500, 51)], 40, 8, 128), ([(100, 51)], 10, 2, 128),
    ([(1000, 256)], 3, 3, 128), ([(600, 24)], 16, 2, 128), ([(50, 5)], 64, 1, 128)])
@pytest.mark.parametrize("page", [0, 16, 24, 64])
def test_long(lengths, qh, kvh, hd, page):
    Case(len(lengths) + page, lengths, qh, kvh, hd, page=page, trees="causal" if lengths[0][1] > 200 else "tree").check()


@pytest.mark.parametrize("n", [63, 64, 65, 130, 1024])
def test_many_sequences(n):
    rng = np.random.default_rng(n)
    Case(n, [(int(rng.integers(0, 90)), int(rng.integers(0, 4))) for _ in range(n)], behind=9).check()
    Case(n, [(int(rng.integers(0, 900)) if b % 50 == 3 else 0, 1) for b in range(n)], qh=4, kvh=1, page=0).check()


def test_one_long_sequence_among_many_short_ones():
    Case(1, [(30000, 1) if b == 77 else (b, 1) for b in range(300)], qh=8, kvh=8, page=64).check()
    Case(2, [(9000, 30) if b == 5 else (3 * b, 20) for b in range(40)], qh=8, kvh=4, page=64).check()
    # (so many rows that a work-group of the join takes several heads)
    Case(3, [(20000, 1) if b == 5 else (b, 50) for b in range(41)], qh=60, kvh=12, page=64).check()
    Case(4, [(9000, 2) if b == 7 else (0, 300) for b in range(11)], qh=12, kvh=2, hd=256, page=64).check()


@pytest.mark.parametrize("qh,kvh,hd", [(10, 2, 128), (16, 2, 256), (20, 1, 128)])
@pytest.mark.parametrize("rows", [1, 5, 31, 32, 33, 60])
@pytest.mark.parametrize("cached", [0, 7, 64, 2000])
def test_random_masks(rows, cached, qh, kvh, hd):
    """bits of any kind: rows that do not see themselves, that see later ones, that see nothing"""
    got = Case(rows + cached, [(cached, rows), (0, rows)], qh, kvh, hd, trees="random", page=24).check()
    empty_bits = [[0] * rows, [0] * rows]
    got = Case(3, [(cached, rows), (0, rows)], qh, kvh, hd, trees=empty_bits).check()
    assert not got[rows:].any() and (cached or not got.any())


def test_wide_masks():
    rng = np.random.default_rng(1)
    bits = [[int.from_bytes(rng.bytes(256), "little") & ((1 << 900) - 1) for _ in range(900)]]
    Case(1, [(100, 900)], trees=bits).check()
    Case(2, [(100, 500), (900, 3)], words=64).check()
    Case(3, [(50, 70)], words=1, trees=[[x & 0xFFFFFFFF for x in bits_of(tree(rng, 70))]]).check()  # (bits that no word holds: not seen)


@pytest.mark.parametrize("scale,q_std", [(-0.05, 1.0), (0.0, 1.0), (None, 20.0), (1.0, 2.0)])
@pytest.mark.parametrize("rows", [1, 40])
def test_scales(rows, scale, q_std):
    Case(rows, [(400, rows), (20, rows)], scale=scale, q_std=q_std).check()
    Case(rows, [(400, rows), (20, rows)], 16, 2, 256, scale=scale, q_std=q_std).check()


@pytest.mark.parametrize("rows,qh,kvh,hd", [(2, 10, 2, 128), (30, 10, 2, 128), (60, 16, 2, 256)])
@pytest.mark.parametrize("poison", [np.nan, np.inf, -np.inf])
def test_unseen_keys_have_no_part(rows, qh, kvh, hd, poison):
    """infinities and NaN in the K and V rows of nodes that no other node sees: only those nodes are not finite"""
    bits = [[1 << i | 1 for i in range(rows)], [1 << i | 1 for i in range(rows)]]
    c = Case(rows, [(300, rows), (0, rows)], qh, kvh, hd, trees=bits)
    want, tol = c.exact()
    k, v = [x.copy() for x in c.k], [x.copy() for x in c.v]
    k[0][:, 300 + rows - 1] = np.float16(poison)
    v[0][:, 300 + rows - 1, 5] = np.float16(poison)
    v[1][:, rows - 1, 9] = np.float16(poison)
    got = c.run(k=k, v=v).astype(np.float64)
    clean = np.ones(2 * rows, bool)
    clean[[rows - 1, 2 * rows - 1]] = False
    assert np.all(np.abs(got - want)[clean] <= tol[clean])
    assert not np.isfinite(got[2 * rows - 1, :, 9]).any()
    # and a cached one: every row of that sequence, no other sequence's
    k, v = [x.copy() for x in c.k], [x.copy() for x in c.v]
    v[0][:, 17, 5] = np.float16(poison)
    got = c.run(k=k, v=v).astype(np.float64)
    assert not np.isfinite(got[:rows, :, 5]).any()
    assert np.all(np.abs(got - want)[rows:] <= tol[rows:])


def test_a_row_that_sees_nothing_gives_zeros_whatever_its_q():
    for rows in (2, 30):
        c = Case(4, [(0, rows), (200, rows)], trees=[[0] + [1 << i for i in range(1, rows)], [1 << i for i in range(rows)]])
        c.q[0] = np.nan
        want, tol = Case.exact(c)
        got = c.run().astype(np.float64)
        assert not got[0].any()
        assert np.all(np.abs(got - want)[1:] <= tol[1:])


@pytest.mark.parametrize("rows", [1, 40])
def test_keys_behind_kv_len_are_not_read(rows):
    """(the cache holds none there: a page's entry would be none, a row NaN)"""
    c = Case(5, [(450, rows), (100, rows), (600, rows)], kv_len=460, page=64, trees="causal")
    c.tables[:, 8:] = NONE
    k, v = [x.copy() for x in c.k], [x.copy() for x in c.v]
    want, tol = c.exact()
    for b in range(3):
        k[b][:, 460:], v[b][:, 460:] = np.nan, np.nan
    order = c.tables.copy()
    c.tables[0, 7] = order[0, 7]

    def place(x, by_row):
        n = np.full((c.kvh, c.cache_rows, c.hd), np.nan, np.float16)
        for b in range(3):
            j = np.arange(min(int(c.keys[b]), 460))
            n[:, c.tables[b, j // 64].astype(np.int64) * 64 + j % 64] = x[b][:, :len(j)]
        return dev(n.view(np.uint16)), (c.hd, c.cache_rows * c.hd)

    c.place = place
    got = c.run(k=k, v=v).astype(np.float64)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("rows", [1, 50])
@pytest.mark.parametrize("page", [16, 24, 64])
def test_a_page_outside_the_cache_is_reported(rows, page):
    c = Case(8, [(300, rows), (0, 0), (100, rows)], page=page)
    c.fill = np.float16(0)
    tables = c.tables.copy()
    tables[1] = 0xFFFFFFF0  # (a sequence without rows)
    b = c.bind(tables=tables)
    mi.call("mi_attn_tree", *b["args"], stream())
    want, tol = c.exact()
    assert np.all(np.abs(c.result(b).astype(np.float64) - want) <= tol)
    assert int(host(b["flag"], np.uint32)[0]) == 0
    tables[0, 2], tables[2, 0] = c.n_pages, 0xFFFFFFFF
    b = c.bind(tables=tables)
    mi.call("mi_attn_tree", *b["args"], stream())
    c.result(b)
    assert int(host(b["flag"], np.uint32)[0]) == mi.STATUS_BAD_PAGE
    mi.call("mi_attn_tree", *b["args"][:-1], None, stream())
    sync()


@pytest.mark.parametrize("rows,cached,page", [(3, 100, 16), (3, 900, 64), (40, 900, 64)])
def test_sequences_that_overlap_are_refused(rows, cached, page):
    c = Case(9, [(cached, rows)] * 20, page=page)
    b = c.bind()
    b["row_start"].copy_(dev(np.where(np.arange(21) % 2, c.T, 0).astype(np.uint32)))
    mi.call("mi_attn_tree", *b["args"], stream())
    sync()
    assert int(host(b["flag"], np.uint32)[0]) == mi.STATUS_BAD_ROWS
    assert (host(b["out"], np.uint16) == 1234).all()


def test_bf16_activations_round_to_bf16():
    for rows in (1, 40):
        c = Case(5, [(300, rows), (0, rows)], act=1)
        got = c.run()
        assert not (got.astype(np.float32).view(np.uint32) & 0xFFFF).any()
        want, tol = c.exact()
        assert np.all(np.abs(got.astype(np.float64) - want) <= tol + 2.0 ** -8 * np.abs(want))


def test_other_stream_and_replayed_graph():
    """a captured call reads lengths, masks, tables and rows anew at every replay, with fewer rows too"""
    T = torch()
    side = T.cuda.Stream()
    with T.cuda.stream(side):
        c = Case(3, [(3000, 1), (10, 1)])
        want, tol = c.exact()
        assert np.all(np.abs(c.run(st=side.cuda_stream).astype(np.float64) - want) <= tol)
    for qh, kvh, hd, rows in ((10, 2, 128, 1), (16, 2, 256, 2), (10, 2, 128, 20), (16, 2, 256, 40)):
        c = Case(6, [(1200, rows), (900, rows), (1000, rows)], qh, kvh, hd, page=64, kv_len=1300)
        b = c.bind()
        g = T.cuda.CUDAGraph()
        with T.cuda.graph(g):
            mi.call("mi_attn_tree", *b["args"], stream())
        for n, lengths in enumerate([[(1200, rows), (900, rows), (1000, rows)], [(0, 1), (800, rows), (3, 0)], [(10, rows), (0, 0), (0, 0)],
                                     [(1100, 1), (1, 1), (500, rows)]]):
            o = Case(20 + n, lengths, qh, kvh, hd, page=64, kv_len=1300, behind=3 * rows - sum(r for _, r in lengths), words=c.words)
            o.n_pages, o.stride, o.cache_rows = c.n_pages, c.stride, c.cache_rows
            tables = np.full((3, c.stride), NONE, np.uint32)
            tables[:, :o.tables.shape[1]] = o.tables[:, :c.stride]
            o.tables = tables
            for name, a in (("q", o.q), ("row_start", o.start.astype(np.uint32)), ("cached", o.cached.astype(np.uint32)), ("tables", o.tables),
                            ("mask", o.mask)):
                b[name].copy_(dev(a))
            b["k"].copy_(o.place(o.k, False)[0])
            b["v"].copy_(o.place(o.v, False)[0])
            b["out"].fill_(1234)
            g.replay()
            want, tol = o.exact()
            assert np.all(np.abs(o.result(b).astype(np.float64) - want) <= tol), n
            assert int(host(b["flag"], np.uint32)[0]) == 0


def test_two_calls_at_once():
    T = torch()
    cases = [Case(30 + n, [(2000, 20), (300, 9)]) for n in range(2)]
    bound = [c.bind() for c in cases]
    sides = [T.cuda.Stream() for _ in cases]
    sync()
    for _ in range(3):
        for b, s in zip(bound, sides):
            mi.call("mi_attn_tree", *b["args"], s.cuda_stream)
    for c, b in zip(cases, bound):
        want, tol = c.exact()
        assert np.all(np.abs(c.result(b).astype(np.float64) - want) <= tol)


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("rows", [1, 50])
@pytest.mark.parametrize("page", [0, 64])
def test_offsets_past_32_bits(rows, hd, page):
    """a cache whose last rows lie past 2^32 bytes, its first ones never written"""
    T = torch()
    c = Case(rows + hd, [(500, rows), (90, rows)], 8, 2, hd, page=page)
    if page:
        c.n_pages = 150000
        c.tables = (c.n_pages - 1 - 997 * np.arange(c.tables.size)).reshape(c.tables.shape).astype(np.uint32)
        strides = (hd, c.n_pages * page * hd)
    else:
        strides = (1 << 23, hd)
        c.stride = 551

    def place(x, by_row):
        top = max(int(c.at(b).max()) for b in range(2))
        t = T.empty(top * strides[0] + (c.kvh - 1) * strides[1] + hd, dtype=T.int16, device="cuda")
        view = t.as_strided((top + 1, c.kvh, hd), (strides[0], strides[1], 1))
        for b in range(2):
            view[T.from_numpy(c.at(b)).cuda()] = T.from_numpy(np.ascontiguousarray(x[b].transpose(1, 0, 2)).view(np.int16)).cuda()
        return t, strides

    c.place = place
    c.check()


@pytest.mark.parametrize("rows,cached,hd", [(3, 100, 128), (20, 50, 128), (20, 900, 256)])
@pytest.mark.parametrize("starts", [(0, 1, 0, 1), (0, 1, 1, 0), (1, 0, 0, 1), (1, 0)])
def test_a_row_start_that_falls_is_refused(starts, rows, cached, hd):
    """few enough rows for the arrays, but two sequences of the same ones: no row is written"""
    c = Case(9, [(cached, rows)] + [(cached, 0)] * (len(starts) - 2), hd=hd)
    b = c.bind()
    b["row_start"].copy_(dev((np.array(starts) * rows).astype(np.uint32)))
    mi.call("mi_attn_tree", *b["args"], stream())
    sync()
    assert int(host(b["flag"], np.uint32)[0]) == mi.STATUS_BAD_ROWS
    assert (host(b["out"], np.uint16) == 1234).all()


@pytest.mark.parametrize("n,at", [(64, 64), (65, 64), (130, 70), (1024, 1023)])
def test_a_row_start_that_falls_far_behind_is_refused(n, at):
    c = Case(9, [(40, 1)] * n)
    b = c.bind()
    starts = c.start.astype(np.uint32)
    starts[at] = starts[at - 1] - 1
    b["row_start"].copy_(dev(starts))
    mi.call("mi_attn_tree", *b["args"], stream())
    sync()
    assert int(host(b["flag"], np.uint32)[0]) == mi.STATUS_BAD_ROWS
    assert (host(b["out"], np.uint16) == 1234).all()


def in_few_rows(c):
    """of a case whose sequences have at most 16 columns: the exact outputs, what the kernel that keeps its weights in two f16 halves may be
    off, and the outputs with each weight rounded to f16 once. A half is off by at most 2^-10 of what it holds, two halves by 2^-20; the
    difference that the exponential takes (up to 8) by 2^-22 and the exponential by 2^-23 of it, 2^-21 with the weights' sum's; the sums
    and the waves' join by 2^-19 of their terms. The other terms as above."""
    want, tol, once = c.exact()[0], np.zeros((c.T, c.qh, c.hd)), np.zeros((c.T, c.qh, c.hd))
    g = c.qh // c.kvh
    for b, n in enumerate(c.rows):
        rows, seen = slice(c.start[b], c.start[b] + n), c.seen(b)
        for h in range(c.qh):
            kd, vd, qd = c.k[b][h // g].astype(np.float64), c.v[b][h // g].astype(np.float64), c.q[rows, h].astype(np.float64)
            s = np.where(seen, qd @ kd.T * c.scale, -np.inf)
            ds = abs(c.scale) * (2.0 ** -21 + c.hd * 2.0 ** -23) * (np.abs(qd) @ np.abs(kd).T).max()
            e = np.exp(s - s.max(1, keepdims=True)) * 128  # (the reference is 2^7 below the largest score)
            z = e.sum(1, keepdims=True)
            tol[rows, h] = (2.0 ** -20 + 2.0 ** -21 + 2.1 * ds + 2.0 ** -19) * (e / z @ np.abs(vd)) + kd.shape[0] * 2.0 ** -32 * np.abs(vd).max()
            once[rows, h] = e.astype(np.float16).astype(np.float64) @ vd / z
    return want, tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -25, once


@pytest.mark.parametrize("qh,kvh,hd", [(10, 2, 128), (16, 2, 256), (7, 1, 128), (8, 8, 256)])
@pytest.mark.parametrize("lengths", [[(1, 1)], [(5, 1), (29, 1), (0, 2)], [(199, 1), (77, 1)]])
@pytest.mark.parametrize("page", [0, 16, 64])
def test_few_rows_keep_their_weights_in_two_halves(lengths, page, qh, kvh, hd):
    """values that cancel, near scores: the outputs are small beside sum p|v|, and their own rounding hides nothing of the weights'"""
    c = Case(page + hd, lengths, qh, kvh, hd, page=page, trees="causal", q_std=0.02)
    for v in c.v:
        n = v.shape[1] // 2
        v[:, n:2 * n] = -v[:, :n]
    want, tol, once = in_few_rows(c)
    assert np.any(np.abs(once - want) > 2 * tol)  # (one half would be seen)
    got = c.run().astype(np.float64)
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("rows", [1, 30])
@pytest.mark.parametrize("page", [0, 64])
def test_rows_so_far_apart_that_a_tile_passes_32_bits(rows, hd, page):
    """above 2^25 elements a row, where the many columns' tiles are not addressed from their first rows"""
    T = torch()
    c = Case(rows + hd, [(70, rows), (9, rows)], 8, 2, hd, page=page)
    strides = ((1 << 25) + 8, hd)

    def place(x, by_row):
        top = max(int(c.at(b).max()) for b in range(2))
        t = T.empty(top * strides[0] + (c.kvh - 1) * strides[1] + hd, dtype=T.int16, device="cuda")
        view = t.as_strided((top + 1, c.kvh, hd), (strides[0], strides[1], 1))
        for b in range(2):
            view[T.from_numpy(c.at(b)).cuda()] = T.from_numpy(np.ascontiguousarray(x[b].transpose(1, 0, 2)).view(np.int16)).cuda()
        return t, strides

    c.place = place
    c.check()


@pytest.mark.parametrize("lengths,qh,kvh,hd", [([(900, 61), (300, 40), (2000, 55)], 40, 8, 128), ([(5000, 60)], 16, 2, 256), ([(4000, 64)], 40, 8, 128),
                                               ([(3000, 1), (70, 1), (800, 1)], 16, 2, 256)])
def test_a_call_gives_the_same_bits_again(lengths, qh, kvh, hd):
    """whatever the workspace held before"""
    c = Case(7, lengths, qh, kvh, hd, page=64)
    b = c.bind()
    outs = []
    for fill in (0, 77, 255):
        b["ws"][:b["need"]] = fill
        b["out"].fill_(1234)
        mi.call("mi_attn_tree", *b["args"], stream())
        outs.append(c.result(b).view(np.uint16))
    assert np.array_equal(outs[0], outs[1]) and np.array_equal(outs[0], outs[2])


@pytest.mark.parametrize("page", [0, 64])
def test_tokens_and_a_stretch_of_a_prompt_in_one_call_and_in_two(page):
    lengths = [(100 * i, 1) for i in range(9)] + [(300, 90), (0, 40)]
    c = Case(11, lengths, 10, 2, 128, page=page, trees="causal")
    want, tol = c.check(), c.exact()[1]
    b = c.bind()
    L, n, T = mi.lib(), 9, c.T
    for first, count, rows in ((0, n, n), (n, 2, T)):
        off = 0 if page else first * c.stride * c.hd * 2
        batch = mi.AttnBatch(sequences=count, kv_len=c.kv_len, table_stride=c.stride, page=c.page, n_pages=c.n_pages, words=0, mask=None,
                             row_start=ptr(b["row_start"]) + 4 * first, cached=ptr(b["cached"]) + 4 * first,
                             tables=ptr(b["tables"]) + 4 * first * c.stride if page else None)
        assert L.mi_attn_tree_ws(rows, count, mi.C.byref(b["sh"])) <= b["need"]
        mi.call("mi_attn_tree", ptr(b["q"]), ptr(b["k"]) + off, ptr(b["v"]) + off, *b["args"][3:5], rows, mi.C.byref(b["sh"]),
                mi.C.byref(batch), *b["args"][8:], stream())
    got = c.result(b).astype(np.float64)
    assert np.all(np.abs(got - want) <= 2 * tol)
    assert int(host(b["flag"], np.uint32)[0]) == 0
