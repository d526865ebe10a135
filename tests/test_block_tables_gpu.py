"""mi_block_tables against the plan made request by request and row by row on the host: whole numbers, equal."""
import numpy as np
import pytest

from mipkg import dev, empty, host, mi, ptr, stream, sync, torch

pytestmark = pytest.mark.gpu
NONE, GUARD = mi.NONE, 16


def plan_of(c):
    """the plan on the host: (outputs, flag)"""
    B, page, R = len(c["cached"]), c["page"], c["rows"]
    o = {"tables": c["tables"].copy(), "ring": c["ring"].copy(), "held_out": np.array(c["held"], np.uint32),
         "ring_at_out": np.array(c["ring_at"], np.uint32), "row_start": np.zeros(B + 1, np.uint32),
         "seq": np.full(R, NONE, np.uint32), "slot": np.full(R, NONE, np.uint32), "pos": np.zeros(R, np.uint32),
         "mask": np.zeros((R, c["words"]), np.uint32)}
    head, count = (int(x) for x in c["ring_at"])
    n = len(c["ring"])
    need = [-(-(int(k) + int(a)) // page) for k, a in zip(c["cached"], c["added"])]
    stride = c["tables"].shape[1]
    if (any(d > stride or int(h) > stride or int(h) * page < int(k) for d, h, k in zip(need, c["held"], c["cached"])) or
            sum(int(a) for a in c["added"]) > R or head >= n or count > n or
            (c["parent"] is not None and any(int(a) > 32 * c["words"] for a in c["added"]))):
        return o, mi.STATUS_BAD_ROWS
    if sum(max(d - int(h), 0) for d, h in zip(need, c["held"])) > count:
        return o, mi.STATUS_NO_PAGES
    flag, taken, back, t = 0, 0, [], 0
    for b in range(B):
        held = int(c["held"][b])
        for i in range(held, need[b]):
            o["tables"][b, i] = c["ring"][(head + taken) % n]
            taken += 1
        back += list(c["tables"][b, need[b]:held])
        o["held_out"][b] = need[b]
        bits = []
        for i in range(int(c["added"][b])):
            key = int(c["cached"][b]) + i
            pg = int(o["tables"][b, key // page])
            if pg >= c["n_pages"]:
                flag = mi.STATUS_BAD_PAGE
            o["seq"][t], o["pos"][t] = b, key
            o["slot"][t] = pg * page + key % page if pg < c["n_pages"] else NONE
            if c["parent"] is not None:
                up = int(c["parent"][int(o["row_start"][b]) + i])
                if up >= i and up != NONE:
                    flag = mi.STATUS_BAD_ROWS
                bits.append({i} | (bits[up] if up < i else set()))
                o["pos"][t] = int(c["cached"][b]) + len(bits[i]) - 1
                for x in bits[i]:
                    o["mask"][t, x // 32] |= np.uint32(1 << x % 32)
            t += 1
        o["row_start"][b + 1] = t
    for i, pg in enumerate(back):
        o["ring"][(head + count + i) % n] = pg
    o["ring_at_out"][:] = (head + taken) % n, count - taken + len(back)
    return o, flag


def make(seed, lengths, page, tree=False, spare=3, extra=0, parent=None):
    """lengths: (cached, added, pages held beyond the cached keys') of each request"""
    rng = np.random.default_rng(seed)
    cached, added, more = (np.array(x, np.uint32) for x in zip(*lengths))
    held = (-(-cached.astype(np.int64) // page) + more).astype(np.uint32)
    need = -(-(cached.astype(np.int64) + added) // page)
    stride = int(max(need.max(), held.max(), 1)) + 2
    free = int(np.maximum(need - held, 0).sum()) + spare
    total = int(held.sum()) + free
    order = rng.permutation(total).astype(np.uint32)
    tables, at = np.full((len(lengths), stride), NONE, np.uint32), 0
    for b, h in enumerate(held):
        tables[b, :h] = order[at:at + h]
        at += int(h)
    ring = np.full(total, NONE, np.uint32)
    head = int(rng.integers(total))
    ring[(head + np.arange(free)) % total] = order[at:]
    words = max(1, -(-int(added.max()) // 32)) if tree else 0
    if tree and parent is None:
        parent = np.concatenate([[NONE] + [int(rng.integers(max(0, i - 6), i)) if rng.random() < 0.95 else NONE for i in range(1, a)]
                                 for a in added if a] or [[]])
    rows = max(int(added.sum()) + extra, 1)
    if tree:
        parent = np.concatenate([np.asarray(parent, np.uint32), np.zeros(rows - len(parent), np.uint32)])
    return {"cached": cached, "added": added, "held": held, "tables": tables, "ring": ring, "ring_at": np.array([head, free], np.uint32),
            "page": page, "rows": rows, "words": words, "n_pages": total, "parent": parent if tree else None}


class Bound:
    def __init__(self, c, in_place=False):
        self.c, B = c, len(c["cached"])
        self.t = {k: dev(np.asarray(c[k], np.uint32)) for k in ("cached", "added", "held", "tables", "ring", "ring_at")}
        self.t["parent"] = dev(c["parent"]) if c["parent"] is not None else None
        sizes = {"held_out": B, "ring_at_out": 2, "row_start": B + 1, "seq": c["rows"], "slot": c["rows"], "pos": c["rows"],
                 "mask": c["rows"] * c["words"]}
        for k, n in sizes.items():
            self.t[k] = empty((n + GUARD,), np.uint32)
            self.t[k].fill_(1234)
        if in_place:
            self.t["held_out"], self.t["ring_at_out"] = self.t["held"], self.t["ring_at"]
        self.t["flag"] = dev(np.zeros(1, np.uint32))
        self.sizes = sizes
        self.in_place = in_place
        need = mi.lib().mi_block_tables_ws(B)
        self.ws = dev(np.full(need + 64, 77, np.uint8))
        self.need = need
        self.struct = mi.BlockPlan(requests=B, rows=c["rows"], page=c["page"], n_pages=c["n_pages"], table_stride=c["tables"].shape[1],
                                   ring_len=len(c["ring"]), words=c["words"],
                                   **{k: ptr(self.t[k]) for k in ("cached", "added", "held", "held_out", "tables", "ring", "ring_at",
                                                                  "ring_at_out", "parent", "row_start", "seq", "slot", "pos", "flag")},
                                   mask=ptr(self.t["mask"]) if c["words"] else None)

    def call(self, st=None):
        mi.call("mi_block_tables", mi.C.byref(self.struct), ptr(self.ws), self.need, stream() if st is None else st)

    def got(self):
        sync()
        assert (host(self.ws, np.uint8)[self.need:] == 77).all()
        o = {"tables": host(self.t["tables"], np.uint32).reshape(self.c["tables"].shape), "ring": host(self.t["ring"], np.uint32)}
        for k, n in self.sizes.items():
            a = host(self.t[k], np.uint32)
            if not (self.in_place and k in ("held_out", "ring_at_out")):
                assert (a[n:] == 1234).all(), k
            o[k] = a[:n]
        o["mask"] = o["mask"].reshape(self.c["rows"], self.c["words"])
        return o, int(host(self.t["flag"], np.uint32)[0])


def check(c, **kw):
    b = Bound(c, **kw)
    b.call()
    got, flag = b.got()
    want, wflag = plan_of(c)
    for k in want:
        assert np.array_equal(got[k], want[k]), k
    assert flag == wflag
    return want


@pytest.mark.parametrize("page", [1, 16, 24, 64])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("lengths", [
    [(0, 1, 0)], [(0, 0, 0)], [(0, 0, 5)], [(63, 1, 0)], [(64, 1, 0)], [(64, 1, 2)], [(65, 70, 0)], [(5, 3, 0), (0, 0, 4), (17, 61, 1), (0, 9, 0)],
    [(1000, 33, 0), (31, 32, 9), (0, 64, 0), (0, 0, 0), (48, 1, 0)]])
def test_small(lengths, tree, page):
    check(make(len(lengths) + page, lengths, page, tree, extra=5))
    check(make(len(lengths) + page, lengths, page, tree), in_place=True)


@pytest.mark.parametrize("n,most,tree", [(1024, 3, False), (1024, 4, True), (700, 90, False), (300, 60, True), (63, 2000, False), (65, 900, True),
                                         (64, 64, True), (1, 65535, False)])
def test_many(n, most, tree):
    """up to the most requests and rows; above 4096 rows in launches of their own"""
    rng = np.random.default_rng(n + most)
    lengths = [(int(rng.integers(0, 3000)), int(rng.integers(0, most + 1)) if n > 1 else most, int(rng.integers(0, 4))) for _ in range(n)]
    while sum(a for _, a, _ in lengths) > 65535:
        lengths.pop()
    c = make(n, lengths, 16, tree, extra=300 if n > 1 else 0)
    assert c["rows"] <= 65535
    check(c)


def test_a_chain_of_two_thousand_nodes_and_a_star():
    n = 2048
    chain = [NONE] + list(range(n - 1))
    check(make(1, [(100, n, 0), (7, n, 0), (0, 3, 0)], 64, True, parent=chain + [NONE] + [0] * (n - 1) + [NONE, NONE, 1]))


def test_parents_that_are_not_below_their_children_count_as_none():
    c = make(2, [(10, 5, 0), (3, 4, 0)], 16, True, parent=[NONE, 0, 2, 9, 1, 0, 0, 1, 4000000000])
    want = check(c)
    assert list(want["pos"]) == [10, 11, 10, 10, 12, 3, 4, 5, 3]


@pytest.mark.parametrize("what", ["pages", "stride", "held", "rows", "words", "head", "count", "wrapped"])
def test_a_step_that_does_not_fit_changes_nothing(what):
    c = make(3, [(40, 30, 0), (100, 50, 0), (0, 0, 6), (16, 4, 1)], 16, True, spare=0, extra=2)
    if what == "pages":
        c["ring_at"][1] -= 1
    elif what == "stride":
        c["tables"] = np.ascontiguousarray(c["tables"][:, :9])
    elif what == "held":
        c["held"][1] = 6
    elif what == "rows":
        c["rows"] = int(c["added"].sum()) - 1
        c["parent"] = c["parent"][:c["rows"]]
    elif what == "words":
        c["words"] = 1
    elif what == "head":
        c["ring_at"][0] = len(c["ring"])
    elif what == "count":
        c["ring_at"][1] = len(c["ring"]) + 1
    elif what == "wrapped":  # keys past 2^32
        c["cached"][1], c["added"][1] = 0xFFFFFFF0, 40
    b = Bound(c)
    b.call()
    got, flag = b.got()
    assert flag == (mi.STATUS_NO_PAGES if what == "pages" else mi.STATUS_BAD_ROWS)
    assert not got["row_start"].any() and (got["slot"] == NONE).all() and (got["seq"] == NONE).all() and not got["mask"].any()
    assert np.array_equal(got["tables"], c["tables"]) and np.array_equal(got["ring"], c["ring"])
    assert np.array_equal(got["held_out"], c["held"]) and np.array_equal(got["ring_at_out"], c["ring_at"])


def test_pages_outside_the_cache_give_no_slot():
    c = make(4, [(40, 30, 0), (5, 3, 0)], 16)
    c["tables"][0, 2] = c["n_pages"]
    c["ring"][(int(c["ring_at"][0]) + 1) % len(c["ring"])] = 0xFFFFFFF0
    want = check(c)
    assert (want["slot"] == NONE).any()


def test_replayed_steps_go_on_from_one_another():
    """a captured step with its state in place: sequences grow, are done, and their pages come back"""
    T = torch()
    rng = np.random.default_rng(5)
    c = make(6, [(0, 30, 0), (100, 10, 0), (55, 12, 2), (0, 1, 0)], 16, True, spare=20, extra=60)
    b = Bound(c, in_place=True)
    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g):
        b.call()
    for step in range(6):
        if step:
            c["cached"] = np.where(c["added"] > 0, c["cached"] + rng.integers(1, np.maximum(c["added"], 1) + 1), 0).astype(np.uint32)
            c["added"] = rng.integers(1, 20, 4).astype(np.uint32)
            if step % 2:
                c["cached"][step % 4] = c["added"][step % 4] = 0
            for k in ("cached", "added"):
                b.t[k].copy_(dev(c[k]))
            c["parent"][:] = np.concatenate([[NONE] + [int(rng.integers(i)) for i in range(1, a)] for a in c["added"] if a] +
                                            [np.zeros(c["rows"] - int(c["added"].sum()))])
            b.t["parent"].copy_(dev(c["parent"]))
        g.replay()
        got, flag = b.got()
        want, wflag = plan_of(c)
        assert flag == wflag == 0
        for k in want:
            assert np.array_equal(got[k], want[k]), (step, k)
        owned = [p for t, h in zip(got["tables"], got["held_out"]) for p in t[:h]]
        head, count = got["ring_at_out"]
        owned += list(got["ring"][(int(head) + np.arange(count)) % len(got["ring"])])
        assert sorted(owned) == list(range(c["n_pages"]))  # no page is lost, none is held twice
        c["tables"], c["ring"], c["held"], c["ring_at"] = got["tables"], got["ring"], got["held_out"], got["ring_at_out"]
    side = T.cuda.Stream()
    with T.cuda.stream(side):
        check(make(7, [(3, 9, 1)] * 40, 16))
