"""The entries of a step of several sequences, without a GPU: refusals, workspaces, and the host's acceptance of a tree."""
import numpy as np
import pytest

from mipkg import mi

ARG, SHAPE = -1, -2
P = 1 << 20  # a pointer that no refused call follows


def test_block_tables_refusals():
    L = mi.lib()
    arrays = ("cached", "added", "held", "held_out", "tables", "ring", "ring_at", "ring_at_out", "row_start", "seq", "slot", "pos")
    base = dict(requests=4, rows=40, page=16, n_pages=100, table_stride=20, ring_len=100, words=0, parent=None, mask=None, flag=None,
                **{a: P for a in arrays})

    def call(ws=P, nb=1 << 20, **kw):
        p = mi.BlockPlan(**dict(base, **kw))
        return L.mi_block_tables(mi.C.byref(p), ws, nb, None)

    for a in arrays:
        for bad in (None, P + 2):
            assert call(**{a: bad}) == ARG, a
            assert b"block_tables" in L.mi_last_error()
    for kw in ({"page": 0}, {"n_pages": 0}, {"table_stride": 0}, {"ring_len": 0}, {"parent": P}, {"mask": P}, {"words": 1}, {"parent": P, "mask": P},
               {"parent": P, "mask": P, "words": 65}, {"parent": P + 1, "mask": P, "words": 1}, {"flag": P + 2}, {"ws": None}, {"ws": P + 2},
               {"nb": L.mi_block_tables_ws(4) - 1}):
        assert call(**kw) == ARG, kw
    for kw in ({"requests": 0}, {"requests": 1025}, {"rows": 0}, {"rows": 65536}, {"page": 1 << 31, "n_pages": 3}, {"ring_len": (1 << 31) + 1},
               {"table_stride": (1 << 21) + 1}, {"page": (1 << 20) + 1, "n_pages": 9}):
        assert call(**kw) == SHAPE, kw
    assert L.mi_block_tables(None, P, 1 << 20, None) == ARG
    assert L.mi_block_tables_ws(0) == L.mi_block_tables_ws(1025) == 0 < L.mi_block_tables_ws(1)


def test_rope_table_refusals():
    L = mi.lib()

    def call(pos0=0, n=10, table=P, **kw):
        r = mi.Rope(**dict(dict(rot_dim=64, theta=1e4, scaling=mi.ROPE_YARN, factor=4.0, original=4096, low=1.0, high=32.0), **kw))
        return L.mi_rope_table(mi.C.byref(r), pos0, n, table, None)

    nan = float("nan")
    bad = np.array([1.0] * 31 + [0.0], np.float32)
    half = np.full(32, 0.5, np.float32)  # with a factor of 1e-6: a frequency of 2e6, above 2^20
    for kw in ({"table": None}, {"table": P + 2}, {"theta": 1.0}, {"theta": nan}, {"scaling": 5}, {"factor": 0.0}, {"factor": nan}, {"original": 0},
               {"low": 0.0}, {"high": 1.0}, {"high": nan}, {"attention": -1.0}, {"attention": nan}, {"divisors": bad.ctypes.data},
               {"factor": 1e-6, "scaling": mi.ROPE_LINEAR, "theta": 1.5, "divisors": half.ctypes.data}):
        assert call(**kw) == ARG, kw
        assert b"rope_table" in L.mi_last_error()
    for kw in ({"rot_dim": 0}, {"rot_dim": 12}, {"rot_dim": 264}, {"n": 0}, {"n": (1 << 24) + 1}, {"pos0": (1 << 31) - 9}):
        assert call(**kw) == SHAPE, kw


def shape(**kw):
    s = mi.AttnShape(10, 2, 128, 128, 0, 1792, 1280, 1536, 0.1, 1e-6, 0)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def test_rope_rows_refusals():
    L = mi.lib()

    def call(x=P, kind=0, stride=1792, T=4, pos=P, pos0=0, slots=P, rows=100, sh=shape(), paired=0, qn=P, kn=P, rope=P, n=50, q=P, k=P, v=P, flag=None):
        return L.mi_rope_rows(x, kind, stride, T, pos, pos0, slots, rows, mi.C.byref(sh), paired, qn, kn, rope, n, q, k, v, 128, 12800, flag, None)

    for kw in ({"x": None}, {"rope": None}, {"q": None}, {"k": None}, {"v": None}, {"kind": 2}, {"paired": 2}, {"stride": 1791}, {"x": P + 2},
               {"x": P + 1, "kind": 1}, {"pos": P + 2}, {"slots": P + 1}, {"qn": P + 2}, {"kn": P + 2}, {"rope": P + 2}, {"q": P + 2}, {"k": P + 1},
               {"v": P + 1}, {"flag": P + 2}, {"sh": shape(act=2)}):
        assert call(**kw) == ARG, kw
        assert b"rope_rows" in L.mi_last_error()
    for kw in ({"T": 0}, {"T": 65536}, {"rows": 0}, {"n": 0}, {"sh": shape(head_dim=64)}, {"sh": shape(gated=1)}, {"sh": shape(k_off=0)},
               {"sh": shape(rot_dim=136)}, {"sh": shape(rot_dim=0)}, {"sh": shape(rot_dim=12)}, {"sh": shape(kv_heads=0)},
               {"pos": None, "pos0": 0xFFFFFFFE}):
        assert call(**kw) == SHAPE, kw
    wide = mi.AttnShape(1024, 512, 128, 128, 0, 2048 * 128, 1024 * 128, 1536 * 128, 0.1, 1e-6, 0)  # (a launch of more than 2^32 threads)
    assert call(sh=wide, T=65535, stride=2048 * 128) == SHAPE
    assert L.mi_rope_rows(P, 0, 1792, 4, P, 0, P, 100, None, 0, P, P, P, 50, P, P, P, 128, 12800, None, None) == ARG


def test_attn_tree_refusals():
    L = mi.lib()
    base = dict(sequences=3, kv_len=500, row_start=P, cached=P, tables=P, table_stride=8, page=64, n_pages=40, mask=P, words=2)

    def call(q=P, k=P, v=P, rs=128, hs=12800, T=9, sh=shape(), ws=P, nb=1 << 30, out=P, flag=None, **kw):
        b = mi.AttnBatch(**dict(base, **kw))
        return L.mi_attn_tree(q, k, v, rs, hs, T, mi.C.byref(sh), mi.C.byref(b), ws, nb, out, flag, None)

    for kw in ({"q": None}, {"k": None}, {"v": None}, {"out": None}, {"row_start": None}, {"cached": None}, {"sh": shape(act=2)}, {"page": 0},
               {"n_pages": 0}, {"table_stride": 7}, {"words": 0}, {"words": 65}, {"mask": None}, {"rs": 4}, {"hs": 4}, {"k": P + 8}, {"v": P + 2},
               {"q": P + 2}, {"out": P + 1}, {"row_start": P + 2}, {"cached": P + 1}, {"tables": P + 2}, {"mask": P + 2}, {"flag": P + 1},
               {"ws": None}, {"ws": P + 8}, {"nb": 100}, {"tables": None, "table_stride": 499}):
        assert call(**kw) == ARG, kw
        assert b"attn_tree" in L.mi_last_error()
    for kw in ({"sh": shape(head_dim=64)}, {"sh": shape(q_heads=11)}, {"sh": shape(kv_heads=0)}, {"sh": shape(gated=1)}, {"T": 0}, {"T": 65536},
               {"kv_len": 0}, {"kv_len": (1 << 30) + 1, "table_stride": 1 << 28}, {"sequences": 0}, {"sequences": 1025},
               {"page": 1 << 31, "n_pages": 3}, {"tables": None, "table_stride": 1 << 31}, {"sh": shape(q_heads=130)}):
        assert call(**kw) == SHAPE, kw


@pytest.mark.parametrize("qh,kvh,hd", [(40, 8, 128), (16, 2, 256), (64, 1, 128), (8, 8, 256), (1024, 1024, 128), (20, 1, 128)])
def test_tree_workspace_never_falls(qh, kvh, hd):
    L = mi.lib()
    sh = shape(q_heads=qh, kv_heads=kvh, head_dim=hd)
    sizes = [L.mi_attn_tree_ws(T, 1, mi.C.byref(sh)) for T in (1, 2, 3, 4, 5, 12, 13, 16, 17, 64, 65, 500, 65535)]
    assert sizes[0] > 0 and sizes == sorted(sizes) and sizes[-1] < 400e6
    assert all(L.mi_attn_tree_ws(500, n, mi.C.byref(sh)) == sizes[-2] for n in (2, 7, 500, 1024))
    assert L.mi_attn_tree_ws(0, 1, mi.C.byref(sh)) == L.mi_attn_tree_ws(1, 0, mi.C.byref(sh)) == L.mi_attn_tree_ws(1, 1025, mi.C.byref(sh)) == 0


def test_beam_select_refusals():
    L = mi.lib()

    def call(x=P, stride=1000, cum=P, done=None, batch=2, beams=4, used=1000, k=8, ids=P, whence=P, scores=P, ws=P, nb=1 << 24):
        return L.mi_beam_select(x, stride, cum, done, 0, batch, beams, used, k, ids, whence, scores, ws, nb, None)

    for kw in ({"x": None}, {"x": P + 2}, {"cum": None}, {"cum": P + 1}, {"done": P + 2}, {"ids": None}, {"ids": P + 2}, {"whence": None}, {"whence": P + 1},
               {"scores": None}, {"scores": P + 2}, {"stride": 999}, {"ws": None}, {"ws": P + 8}, {"nb": L.mi_beam_select_ws(2, 4, 1000, 8) - 1}):
        assert call(**kw) == ARG, kw
        assert b"beam_select" in L.mi_last_error()
    for kw in ({"batch": 0}, {"beams": 0}, {"beams": 65}, {"batch": 65536}, {"batch": 16384}, {"used": 0}, {"used": (1 << 23) + 1, "stride": 1 << 24}, {"k": 0},
               {"k": 65}):
        assert call(**kw) == SHAPE, kw
    assert L.mi_beam_select_ws(0, 1, 10, 1) == L.mi_beam_select_ws(1, 65, 10, 1) == L.mi_beam_select_ws(1, 1, 10, 65) == 0


def test_kv_move_refusals():
    L = mi.lib()

    def call(k=P, v=P, layers=2, ls=25600, rs=128, hs=12800, heads=2, hd=128, rows=100, origin=P, to=P, groups=3, per=8, flag=None):
        return L.mi_kv_move(k, v, layers, ls, rs, hs, heads, hd, rows, origin, to, groups, per, flag, None)

    for kw in ({"k": None}, {"v": None}, {"origin": None}, {"to": None}, {"k": P + 8}, {"v": P + 2}, {"origin": P + 2}, {"to": P + 1}, {"flag": P + 2}, {"ls": 4},
               {"rs": 4}, {"hs": 4}):
        assert call(**kw) == ARG, kw
        assert b"kv_move" in L.mi_last_error()
    for kw in ({"hd": 64}, {"layers": 0}, {"layers": 65536}, {"heads": 0}, {"heads": 65536}, {"rows": 0}, {"groups": 0}, {"per": 0}, {"per": 65}):
        assert call(**kw) == SHAPE, kw


def test_accept_tree():
    none = mi.NONE
    #        0 -> 1, 2;  1 -> 3;  2 -> 4, 5;  5 -> 6
    parent = [none, 0, 0, 1, 2, 2, 5]
    tokens = [9, 11, 12, 13, 14, 15, 16]
    cases = {(12, 0, 15, 0, 0, 16, 77): ([2, 5, 6], 77), (11, 13, 0, 14, 0, 0, 0): ([1, 3], 14), (50, 1, 2, 3, 4, 5, 6): ([], 50),
             (12, 0, 14, 0, 8, 0, 0): ([2, 4], 8)}
    for argmax, (path, nxt) in cases.items():
        got, n = mi.accept_tree(argmax, tokens, parent)
        assert list(got) == path and n == nxt
    # equal drafts of one parent: the first
    got, n = mi.accept_tree([5, 1, 2, 3], [0, 5, 5, 1], [none, 0, 0, 1])
    assert list(got) == [1, 3] and n == 3
    nxt = mi.u32(77)  # (no node: nothing is read)
    assert mi.lib().mi_accept_tree(None, None, None, 0, None, mi.C.byref(nxt)) == 0 and nxt.value == 77
    got, n = mi.accept_tree([7], [0], [none])
    assert list(got) == [] and n == 7
    # a chain is accepted as mi_accept_greedy has it
    rng = np.random.default_rng(1)
    for _ in range(50):
        k = int(rng.integers(1, 8))
        argmax, drafts = rng.integers(0, 2, k + 1), rng.integers(0, 2, k)
        got, n = mi.accept_tree(argmax, [0, *drafts], [none, *range(k)])
        assert (len(got), n) == mi.accept_greedy(argmax, drafts) and list(got) == list(range(1, len(got) + 1))


def test_accept_tree_takes_arrays_of_one_size():
    none = mi.NONE
    for argmax, tokens, parent in (([1, 2, 3], [5, 6], [none, 0, 1]), ([1, 2, 3], [5, 6, 7], [none, 0]), ([1], [], [none]), ([], [1], [none])):
        with pytest.raises(ValueError, match="accept_tree"):
            mi.accept_tree(argmax, tokens, parent)
    path, _ = mi.accept_tree([], [], [])
    assert path.size == 0
