"""mi_beam_select and mi_kv_move.

A score is cum + x - m - log Z. Z is a sum of positive terms in 32 bits: at most vocab / 256 + 30 of them one after another (2^-24 each),
a term off by |x - m| 2^-22 of it (the exponent's two roundings) and an exponential's 2^-22. That holds for log Z, and the score rounds
once more. Candidates whose exact scores are closer than that may change places."""
import numpy as np
import pytest

from mipkg import dev, empty, host, mi, ptr, stream, sync, torch

pytestmark = pytest.mark.gpu
NONE, GUARD = mi.NONE, 16


class Beams:
    def __init__(self, seed, batch, beams, used, k, done=False, std=2.0, stride=0):
        rng = np.random.default_rng(seed)
        self.__dict__.update(batch=batch, beams=beams, used=used, k=k, stride=stride or used, eos=used // 2)
        self.x = (rng.standard_normal((batch * beams, self.stride)) * std).astype(np.float32)
        self.cum = rng.uniform(-9, -1, batch * beams).astype(np.float32)
        self.done = (rng.random(batch * beams) < 0.4).astype(np.uint32) if done else None

    def bind(self):
        d = {n: dev(getattr(self, n)) for n in ("x", "cum", "done")}
        for n, t in (("ids", np.uint32), ("from", np.uint32), ("scores", np.float32)):
            d[n] = empty((self.batch * self.k + GUARD,), t)
            d[n].fill_(99)
        need = mi.lib().mi_beam_select_ws(self.batch, self.beams, self.used, self.k)
        d["ws"], d["need"] = dev(np.full(need + GUARD, 77, np.uint8)), need
        d["args"] = (ptr(d["x"]), self.stride, ptr(d["cum"]), ptr(d["done"]), self.eos, self.batch, self.beams, self.used, self.k, ptr(d["ids"]),
                     ptr(d["from"]), ptr(d["scores"]), ptr(d["ws"]), need)
        return d

    def result(self, d):
        sync()
        assert (host(d["ws"], np.uint8)[d["need"]:] == 77).all()
        out = []
        for n, t in (("ids", np.uint32), ("from", np.uint32), ("scores", np.float32)):
            a = host(d[n], t)
            assert (a[-GUARD:] == 99).all()
            out.append(a[:-GUARD].reshape(self.batch, self.k))
        return out

    def run(self, st=None):
        d = self.bind()
        mi.call("mi_beam_select", *d["args"], stream() if st is None else st)
        return self.result(d)

    def check(self, got=None):
        ids, beams, scores = self.run() if got is None else got
        for b in range(self.batch):
            best, tol, lists = [], 0.0, {}
            for w in range(self.beams):
                r = b * self.beams + w
                cum = np.float64(self.cum[r])
                if self.done is not None and self.done[r]:
                    lists[w] = {self.eos: cum} if cum > -np.inf else {}
                    best += [(-cum, w, 0)] if cum > -np.inf else []
                    continue
                x = self.x[r, :self.used].astype(np.float64)
                lists[w] = {}
                if np.isnan(x).any() or (x == np.inf).any() or not (x > -np.inf).any() or not cum > -np.inf:
                    continue
                m = x.max()
                e = np.exp(x - m)
                s = cum + x - m - np.log(e.sum())
                with np.errstate(invalid="ignore"):
                    off = np.where(e > 0, e * np.abs(x - m), 0).sum() / e.sum()
                tol = max(tol, (self.used / 256 + 30) * 2.0 ** -24 + 2.0 ** -22 * (1 + off))
                order = np.lexsort((np.arange(self.used), -x))[:self.k]
                order = order[s[order] > -np.inf]
                lists[w] = {int(v): s[v] for v in order}
                best += [(-s[v], w, n) for n, v in enumerate(order)]
            best.sort()
            n = min(len(best), self.k)
            assert (ids[b, n:] == NONE).all() and (beams[b, n:] == NONE).all() and (scores[b, n:] == -np.inf).all()
            taken = {w: 0 for w in lists}
            for i in range(n):
                w, v = int(beams[b, i]), int(ids[b, i])
                assert list(lists[w])[taken[w]] == v  # a beam's own candidates in their order
                taken[w] += 1
                s = lists[w][v]
                slack = tol + 2.0 ** -23 * abs(s)
                assert abs(s + best[i][0]) <= 2 * slack and abs(scores[b, i] - s) <= slack
            assert np.all(np.diff(scores[b, :n]) <= 0)
        return ids, beams, scores


@pytest.mark.parametrize("batch,beams,used,k", [(1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 7, 64), (1, 4, 151936, 8), (16, 8, 1000, 16), (3, 64, 500, 64),
                                                (2, 5, 4099, 33), (129, 4, 2049, 5), (1, 1, 100000, 64), (40, 16, 300, 20), (3, 5, 20001, 64),
                                                (1, 64, 66001, 64), (128, 4, 1025, 9), (513, 1, 1500, 7)])
@pytest.mark.parametrize("done", [False, True])
def test_select(batch, beams, used, k, done):
    Beams(used + k, batch, beams, used, k, done, stride=used + 3 if beams == 5 else 0).check()


@pytest.mark.parametrize("used", [600, 5000])
def test_equal_scores_go_to_the_lower_beam_then_the_lower_token(used):
    c = Beams(1, 2, 4, used, 40)
    c.x[:] = np.round(c.x[0] * 2)  # equal rows, many equal logits
    c.cum[:] = -3.0
    ids, beams, _ = c.check()
    x = c.x[0, :used]
    want = sorted(((-x[v], w, v) for w in range(4) for v in range(used)))[:40]
    for b in range(2):
        assert [(int(w), int(v)) for w, v in zip(beams[b], ids[b])] == [(w, v) for _, w, v in want]


@pytest.mark.parametrize("used,k", [(2000, 64), (30000, 20), (30000, 1)])
@pytest.mark.parametrize("levels", [1, 2, 40])
def test_rows_of_few_different_logits(used, k, levels):
    """many tokens as good as the k-th best: of the lowest beams and tokens, whatever reads them"""
    c = Beams(used + levels, 2, 3, used, k, done=levels == 2)
    c.x[:] = np.random.default_rng(levels).integers(0, levels, c.x.shape) * np.float32(0.5)
    c.x[3] = c.x[4]
    c.cum[[3, 4]] = -2.0
    c.check()


@pytest.mark.parametrize("used", [900, 20000])
def test_beams_without_candidates(used):
    c = Beams(2, 3, 4, used, 12)
    c.cum[[1, 2, 3]] = -np.inf  # a text's first step: one beam lives
    c.x[4, 7] = np.nan
    c.x[5, 8] = np.inf
    c.x[6] = -np.inf
    c.x[7, 5:] = -np.inf  # a grammar that leaves five tokens
    c.cum[8:] = -np.inf  # nothing lives
    c.cum[9] = np.nan
    ids, beams, scores = c.check()
    assert (beams[0] == 0).all() and (beams[1, :5] == 3).all() and (ids[1, 5:] == NONE).all() and (ids[2] == NONE).all()
    c = Beams(3, 1, 4, used, 12)
    c.done = np.array([1, 0, 1, 1], np.uint32)
    c.cum = np.array([-1.0, -50.0, -np.inf, -2.0], np.float32)
    ids, beams, scores = c.check()
    assert list(beams[0, :2]) == [0, 3] and list(ids[0, :2]) == [c.eos] * 2 and (beams[0, 2:] == 1).all()


def test_captured_select_and_other_stream():
    T = torch()
    c = Beams(4, 2, 8, 5000, 16, done=True)
    d = c.bind()
    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g):
        mi.call("mi_beam_select", *d["args"], stream())
    for seed in (5, 6, 7):
        o = Beams(seed, 2, 8, 5000, 16, done=True)
        for n in ("x", "cum", "done"):
            d[n].copy_(dev(getattr(o, n)))
        g.replay()
        o.check(o.result(d))
    side = T.cuda.Stream()
    with T.cuda.stream(side):
        c.check(c.run(side.cuda_stream))


def move(k, v, rows, origin, to, by_row=False, flag=None, captured=False):
    """k, v [layers][kv_heads][rows][hd] uint16; what mi_kv_move leaves of them"""
    L, H, n, hd = k.shape
    dk, dv = (dev(np.ascontiguousarray(x.transpose(0, 2, 1, 3)) if by_row else x) for x in (k, v))
    strides = (H * hd, hd) if by_row else (hd, n * hd)
    df, dt = dev(np.asarray(origin, np.uint32)), dev(np.asarray(to, np.uint32))
    f = dev(np.zeros(1, np.uint32))
    groups, per = np.shape(to)
    mi.call("mi_kv_move", ptr(dk), ptr(dv), L, H * n * hd, *strides, H, hd, rows, ptr(df), ptr(dt), groups, per, ptr(f), stream())
    sync()
    assert int(host(f, np.uint32)[0]) == (flag or 0)
    out = [host(x, np.uint16).reshape((L, n, H, hd) if by_row else (L, H, n, hd)) for x in (dk, dv)]
    return [x.transpose(0, 2, 1, 3) if by_row else x for x in out]


def moved(x, rows, origin, to):
    y = x.copy()
    for a, b in zip(np.ravel(origin), np.ravel(to)):
        if b != NONE and a < rows and b < rows:
            y[:, :, b] = x[:, :, a]
    return y


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("groups,per", [(1, 1), (5, 3), (2, 16), (3, 17), (2, 33), (2, 64)])
@pytest.mark.parametrize("by_row", [False, True])
def test_moves_within_a_list_are_at_once(groups, per, hd, by_row):
    """each list permutes, closes up or copies rows of its own stretch"""
    rng = np.random.default_rng(groups * per + hd)
    n = groups * 80 + 3
    k, v = (rng.integers(0, 1 << 16, (3, 2, n, hd)).astype(np.uint16) for _ in range(2))
    origin, to = [], []
    for g in range(groups):
        f, t = 80 * g + rng.integers(0, 80, per), 80 * g + rng.permutation(80)[:per]
        if g % 3 == 1:
            f = rng.permutation(t)
        if g % 3 == 2:
            f, t = 80 * g + np.sort(rng.permutation(80)[:per]), 80 * g + np.arange(per)
        t = np.where(rng.random(per) < 0.2, NONE, t)
        origin.append(f)
        to.append(t)
    got = move(k, v, n, origin, to, by_row)
    for g, x in zip(got, (k, v)):
        assert np.array_equal(g, moved(x, n, origin, to))


def test_rows_outside_are_not_moved():
    rng = np.random.default_rng(1)
    k, v = (rng.integers(0, 1 << 16, (2, 3, 50, 128)).astype(np.uint16) for _ in range(2))
    origin, to = [[1, 48, 3, NONE], [5, 6, 7, 8]], [[10, 11, 45, 12], [13, NONE, 44, 14]]
    got = move(k, v, 45, origin, to, flag=mi.STATUS_BAD_PAGE)
    for g, x in zip(got, (k, v)):
        assert np.array_equal(g, moved(x, 45, origin, to))


def test_captured_moves_and_other_stream():
    """a captured move reads its lists anew, and the rows as the replay before left them"""
    T = torch()
    rng = np.random.default_rng(5)
    n, groups, per = 90, 3, 7
    k, v = (rng.integers(0, 1 << 16, (2, 3, n, 128)).astype(np.uint16) for _ in range(2))
    dk, dv = dev(k), dev(v)
    df, dt = (dev(np.zeros((groups, per), np.uint32)) for _ in range(2))

    def call(st):
        mi.call("mi_kv_move", ptr(dk), ptr(dv), 2, 3 * n * 128, 128, n * 128, 3, 128, n, ptr(df), ptr(dt), groups, per, None, st)

    def lists():
        f, t = ([30 * g + rng.permutation(30)[:per] for g in range(groups)] for _ in range(2))
        df.copy_(dev(np.array(f, np.uint32)))
        dt.copy_(dev(np.array(t, np.uint32)))
        return f, t

    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g):
        call(stream())
    side = T.cuda.Stream()
    for i in range(5):
        f, t = lists()
        sync()
        if i < 3:
            g.replay()
        else:
            call(side.cuda_stream)
        sync()
        k, v = moved(k, n, f, t), moved(v, n, f, t)
        assert np.array_equal(host(dk, np.uint16).reshape(k.shape), k) and np.array_equal(host(dv, np.uint16).reshape(v.shape), v)


@pytest.mark.parametrize("strides", [((1 << 32) + 8, 128, 128 * 40), (128 * 80, 128, (1 << 32) + 8), (128, 1 << 27, 0)])
def test_moves_past_32_bits(strides):
    """rows whose offsets pass 2^32 elements, by layers, by heads and by rows, the elements between them never written"""
    T = torch()
    L, H, n = (1 if strides[1] > 128 else 2), (1 if strides[1] > 128 else 2), 40
    rng = np.random.default_rng(6)
    k, v = (rng.integers(0, 1 << 16, (L, H, n, 128)).astype(np.uint16) for _ in range(2))
    f, t = [np.r_[39, 1, 38]], [np.r_[37, 39, 2]]
    views = []
    size = (L - 1) * strides[0] + (H - 1) * strides[2] + (n - 1) * strides[1] + 128
    for x in (k, v):
        d = T.empty(size, dtype=T.int16, device="cuda").as_strided((L, H, n, 128), (strides[0], strides[2], strides[1], 1))
        d.copy_(dev(x).reshape(x.shape))
        views.append(d)
    df, dt = dev(np.array(f, np.uint32)), dev(np.array(t, np.uint32))
    mi.call("mi_kv_move", ptr(views[0]), ptr(views[1]), L, strides[0], strides[1], strides[2], H, 128, n, ptr(df), ptr(dt), 1, 3, None, stream())
    sync()
    for d, x in zip(views, (k, v)):
        assert np.array_equal(host(d.contiguous(), np.uint16).reshape(x.shape), moved(x, n, f, t))
