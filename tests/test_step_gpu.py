"""The entries of a step of several sequences one after another, as a program decodes with trees of drafts and with beams. Every
stage is held to its definition on what the stage before left on the device, and what the accepted rows leave in the cache to a
decoding without trees."""
import numpy as np
import pytest

from mipkg import dev, empty, host, mi, ptr, stream, sync, torch
from test_attn_tree_gpu import Case
from test_block_tables_gpu import Bound, plan_of
from test_rope_gpu import Rows, table

pytestmark = pytest.mark.gpu
NONE = mi.NONE
QH, KVH, HD, PAGE, LEN = 10, 2, 128, 16, 600


class Text:
    """What a model would say: the q||k||v row of a token at a position, and the token behind it, by hashing."""

    def __init__(self, seed):
        self.seed = seed

    def row(self, token, pos):
        return np.random.default_rng([self.seed, int(token), int(pos)]).standard_normal((QH + 2 * KVH) * HD).astype(np.float32)

    def next(self, token, pos):
        return int(np.random.default_rng([self.seed, 77, int(token), int(pos)]).integers(0, 5))


def step_plan(cached, added, tables, held, ring, ring_at, n_pages, parent):
    words = 0 if parent is None else max(1, -(-int(added.max()) // 32))
    return {"cached": cached, "added": added, "held": held, "tables": tables, "ring": ring, "ring_at": ring_at, "page": PAGE,
            "rows": int(added.sum()) + 4, "words": words, "n_pages": n_pages,
            "parent": None if parent is None else np.concatenate([parent, np.zeros(4)]).astype(np.uint32)}


def test_trees_of_drafts_decode_as_one_token_at_a_time_does():
    rng = np.random.default_rng(1)
    B, n_pages = 4, 200
    texts = [Text(b) for b in range(B)]
    rope = table(mi.Rope(rot_dim=HD, theta=1e4, scaling=mi.ROPE_LINEAR, factor=2.0), 0, LEN).copy()
    ring = rng.permutation(n_pages).astype(np.uint32)
    state = {"cached": np.zeros(B, np.uint32), "tables": np.full((B, 40), NONE, np.uint32), "held": np.zeros(B, np.uint32), "ring": ring,
             "ring_at": np.array([150, n_pages], np.uint32)}
    cache = [dev(np.zeros((KVH, n_pages * PAGE, HD), np.uint16)) for _ in range(2)]
    told = [[0] for _ in range(B)]  # the tokens so far, the last one not yet in the cache
    prompts = [37, 1, 16, 90]
    for b in range(B):
        told[b] = [int(x) for x in rng.integers(0, 5, prompts[b])]
        told[b].append(texts[b].next(told[b][-1], prompts[b] - 1))
    accepted = 0
    for step in range(6):
        # what each sequence adds: its prompt, then a tree over the next token with some right drafts in it
        tokens, parents = [], []
        for b in range(B):
            if step == 0:
                tokens.append(told[b][:-1])
                parents.append(None)
                continue
            tok, par, best, p = [told[b][-1]], [NONE], 0, int(state["cached"][b])
            for i in range(1, int(rng.integers(2, 41))):
                up = best if rng.random() < 0.4 else int(rng.integers(i))
                tok.append(int(rng.integers(0, 5)) if rng.random() < 0.5 else texts[b].next(tok[up], p + depth(par, up)))
                par.append(up)
                if tok[-1] == texts[b].next(tok[up], p + depth(par, up)):
                    best = i
            tokens.append(tok)
            parents.append(par)
        added = np.array([len(t) for t in tokens], np.uint32)
        c = step_plan(state["cached"], added, state["tables"], state["held"], state["ring"], state["ring_at"], n_pages,
                      None if step == 0 else np.concatenate(parents))
        plan = Bound(c)
        plan.call()
        # the rows at the plan's positions into the plan's slots, on the device
        r = Rows(step, c["rows"], QH, KVH, HD, HD, norm=False, cache=n_pages * PAGE)
        pos = [int(state["cached"][b]) + (depth(parents[b], i) if step else i) for b in range(B) for i in range(added[b])]
        r.x = np.stack([texts[b].row(t, p) for (b, t), p in zip([(b, t) for b in range(B) for t in tokens[b]], pos)] +
                       [np.ones((QH + 2 * KVH) * HD, np.float32)] * 4)
        r.rope, r.len = rope, LEN
        rb = r.bind()
        rargs = list(rb["args"])
        rargs[4], rargs[6], rargs[15], rargs[16] = ptr(plan.t["pos"]), ptr(plan.t["slot"]), ptr(cache[0]), ptr(cache[1])
        mi.call("mi_rope_rows", *rargs, stream())
        # the attention over the plan's sequences
        sh = mi.AttnShape(QH, KVH, HD, HD, 0, (QH + 2 * KVH) * HD, QH * HD, (QH + KVH) * HD, HD ** -0.5, 1e-6, 0)
        batch = mi.AttnBatch(sequences=B, kv_len=LEN, row_start=ptr(plan.t["row_start"]), cached=ptr(plan.t["cached"]),
                             tables=ptr(plan.t["tables"]), table_stride=40, page=PAGE, n_pages=n_pages,
                             mask=ptr(plan.t["mask"]) if step else None, words=c["words"])
        need = mi.lib().mi_attn_tree_ws(c["rows"], B, mi.C.byref(sh))
        ws = torch().empty(need, dtype=torch().uint8, device="cuda")
        out = empty((c["rows"], QH, HD), np.uint16)
        out.fill_(1234)
        mi.call("mi_attn_tree", ptr(rb["q"]), ptr(cache[0]), ptr(cache[1]), HD, n_pages * PAGE * HD, c["rows"], mi.C.byref(sh),
                mi.C.byref(batch), ptr(ws), need, ptr(out), None, stream())
        got, flag = plan.got()
        want, _ = plan_of(c)
        assert flag == 0 and all(np.array_equal(got[k], want[k]) for k in want)
        assert list(got["pos"][:len(pos)]) == pos
        T = int(added.sum())
        q = host(rb["q"], np.float32)[:c["rows"] * QH * HD].reshape(c["rows"], QH, HD)
        r.pos = got["pos"]
        wq, tq = r.exact()[:2]
        assert np.all(np.abs(q - wq)[:T] <= tq[:T])
        a = Case(step, [(int(k), int(n)) for k, n in zip(state["cached"], added)], QH, KVH, HD, page=PAGE, behind=4, kv_len=LEN,
                 trees="causal" if step == 0 else [[bits(parents[b], i) for i in range(added[b])] for b in range(B)])
        a.tables, a.q = got["tables"], q
        ck, cv = (host(x, np.uint16).view(np.float16).reshape(KVH, n_pages * PAGE, HD) for x in cache)
        a.k, a.v = ([x[:, a.at(b)] for b in range(B)] for x in (ck, cv))
        wo, to = a.exact()
        o = host(out, np.uint16).reshape(c["rows"], QH, HD)
        assert (o[T:] == 1234).all()
        assert np.all(np.abs(o.view(np.float16).astype(np.float64) - wo)[:T] <= to[:T])
        # what stays: the accepted nodes' rows close up behind node 0
        origin, to_rows, new = np.zeros((B, 40), np.uint32), np.full((B, 40), NONE, np.uint32), state["cached"].copy()
        for b in range(B):
            first = int(got["row_start"][b])
            if step == 0:
                new[b] += added[b]
                continue
            says = [texts[b].next(t, p) for t, p in zip(tokens[b], got["pos"][first:])]
            path, nxt = mi.accept_tree(says, tokens[b], parents[b])
            told[b] += [tokens[b][i] for i in path] + [nxt]
            accepted += len(path)
            for i, node in enumerate(path):
                key = int(state["cached"][b]) + 1 + i
                origin[b, i], to_rows[b, i] = got["slot"][first + node], got["tables"][b, key // PAGE] * PAGE + key % PAGE
            new[b] += 1 + len(path)
        df, dt = dev(origin), dev(to_rows)
        mi.call("mi_kv_move", ptr(cache[0]), ptr(cache[1]), 1, 0, HD, n_pages * PAGE * HD, KVH, HD, n_pages * PAGE, ptr(df), ptr(dt), B, 40,
                None, stream())
        sync()
        state = {"cached": new, "tables": got["tables"], "held": got["held_out"], "ring": got["ring"], "ring_at": got["ring_at_out"]}
    assert accepted > 5
    # the cache is that of the same tokens one after another at their positions
    for b in range(B):
        n = int(state["cached"][b])
        assert n == len(told[b]) - 1
        for p in range(prompts[b] - 1, n):
            assert told[b][p + 1] == texts[b].next(told[b][p], p)
        r = Rows(0, n, QH, KVH, HD, HD, norm=False, cache=LEN)
        r.x = np.stack([texts[b].row(t, p) for p, t in enumerate(told[b][:n])])
        r.pos, r.slot, r.rope, r.len = np.arange(n, dtype=np.uint32), np.arange(n, dtype=np.uint32), rope, LEN
        _, k, v, _ = r.run()
        at = state["tables"][b, np.arange(n) // PAGE].astype(np.int64) * PAGE + np.arange(n) % PAGE
        for x, y in zip(cache, (k, v)):
            assert np.array_equal(host(x, np.uint16).reshape(KVH, n_pages * PAGE, HD)[:, at], y[:, :n])


def depth(parents, i):
    n = 0
    while parents[i] != NONE:
        i, n = parents[i], n + 1
    return n


def bits(parents, i):
    x = 1 << i
    while parents[i] != NONE:
        i = parents[i]
        x |= 1 << i
    return x


def test_beams_move_their_states():
    """beams over a cache: each step the best continuations are selected and the beams' last pages change places"""
    rng = np.random.default_rng(2)
    W, V, n, steps = 4, 50, 64, 12
    k, v = (dev(rng.integers(0, 1 << 15, (2, KVH, n, HD)).astype(np.uint16)) for _ in range(2))
    logits = rng.standard_normal((steps, W, V)).astype(np.float32)
    cum = np.array([0.0] + [-np.inf] * (W - 1), np.float32)
    d = {"ids": empty((W,), np.uint32), "from": empty((W,), np.uint32), "scores": empty((W,), np.float32)}
    need = mi.lib().mi_beam_select_ws(1, W, V, W)
    ws = torch().empty(need, dtype=torch().uint8, device="cuda")
    history, best = [[] for _ in range(W)], [((), 0.0, 0)]
    rows = np.arange(W * 16).reshape(W, 16)  # beam w's rows of the cache
    held = host(k, np.uint16).reshape(2, KVH, n, HD)[:, :, :W * 16].copy()
    for s in range(steps):
        dl, dc = dev(logits[s]), dev(cum)
        mi.call("mi_beam_select", ptr(dl), V, ptr(dc), None, 0, 1, W, V, W, ptr(d["ids"]), ptr(d["from"]), ptr(d["scores"]), ptr(ws), need,
                stream())
        sync()
        ids, whence, cum = host(d["ids"], np.uint32), host(d["from"], np.uint32), host(d["scores"], np.float32).copy()
        lp = logits[s].astype(np.float64)
        lp = lp - np.log(np.exp(lp).sum(1, keepdims=True))
        best = sorted(((seq + (t,), sc + lp[w, t], w) for seq, sc, w in best for t in range(V)), key=lambda x: -x[1])[:W]
        history = [history[w] + [int(t)] for w, t in zip(whence, ids)]
        assert [list(x[0]) for x in best] == history
        assert np.all(np.abs(cum - np.array([x[1] for x in best])) < (s + 1) * 2.0 ** -17)
        best = [(x[0], x[1], w) for w, x in enumerate(best)]
        # list i: row i of every beam
        df, dt = dev(rows[whence].T.astype(np.uint32)), dev(rows.T.astype(np.uint32))
        mi.call("mi_kv_move", ptr(k), ptr(v), 2, KVH * n * HD, HD, n * HD, KVH, HD, n, ptr(df), ptr(dt), 16, W, None, stream())
        held = held.reshape(2, KVH, W, 16, HD)[:, :, whence].reshape(2, KVH, W * 16, HD)
        sync()
        assert np.array_equal(host(k, np.uint16).reshape(2, KVH, n, HD)[:, :, :W * 16], held)
