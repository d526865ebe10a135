"""mi_rope_table and mi_rope_rows against their definitions in more bits.

Tolerances. Table: the angle p f is off by 4 roundings of 64 bits (f's power and its scaling, the product, its reduction), 2^-51 of it,
and the value by that, 2^-46 (the series, and up to seven turns of 64 bits) and one rounding to 32 bits. Rows: the norm's factor is off by half of the sum's ten
roundings, a quotient, a root, a reciprocal and two products, ten of 2^-24; a turn adds two: 2^-20 (|x cos| + |y sin|) holds them, and k
rounds to f16."""
import numpy as np
import pytest

from mipkg import dev, empty, host, mi, ptr, stream, sync, torch

pytestmark = pytest.mark.gpu
NONE, GUARD = mi.NONE, 32
LD = np.longdouble
PI = LD("3.14159265358979323846264338327950288")


def frequencies(r, theta, scaling=0, factor=1.0, original=0, low=0.0, high=0.0, divisors=None):
    theta, factor, low, high = (LD(np.float32(x)) for x in (theta, factor, low, high))
    i = np.arange(r // 2).astype(LD)
    if scaling == mi.ROPE_BASE:
        theta = theta * factor ** (LD(r) / LD(r - 2))
    f = theta ** (-2 * i / r)
    if divisors is not None:
        f = f / np.asarray(divisors, np.float32).astype(LD)
    if scaling == mi.ROPE_LINEAR:
        f = f / factor
    elif scaling == mi.ROPE_WAVELENGTH:
        part = np.clip((original * f / (2 * PI) - low) / (high - low), 0, 1)
        f = part * f + (1 - part) * f / factor
    elif scaling == mi.ROPE_YARN:
        a, b = (r * np.log(original / (t * 2 * PI)) / (2 * np.log(theta)) for t in (high, low))
        a, b = max(np.floor(a), 0), min(np.ceil(b), r - 1)
        part = 1 - np.clip((i - a) / max(b - a, LD(np.float64(0.001))), 0, 1)
        f = part * f + (1 - part) * f / factor
    return f


def table(rope, pos0, n):
    t = empty((n * rope.rot_dim + GUARD,), np.float32)
    t.fill_(5.0)
    mi.call("mi_rope_table", mi.C.byref(rope), pos0, n, ptr(t), stream())
    sync()
    a = host(t, np.float32)
    assert (a[n * rope.rot_dim:] == 5.0).all()
    return a[:n * rope.rot_dim].reshape(n, 2, rope.rot_dim // 2)


def check_table(rope, pos0, n, much=1.0, **kw):
    got = table(rope, pos0, n)
    angle = (pos0 + np.arange(n)).astype(LD)[:, None] * frequencies(rope.rot_dim, rope.theta, rope.scaling, **kw)
    for k, fn in enumerate((np.cos, np.sin)):
        want = fn(angle) * LD(much)
        tol = 2.0 ** -24 * np.abs(want) + (2.0 ** -51 * angle + 2.0 ** -46) * much * 1.01
        assert np.all(np.abs(got[:, k] - want) <= tol), np.max(np.abs(got[:, k] - want) / tol)


@pytest.mark.parametrize("r", [8, 32, 96, 128, 256])
@pytest.mark.parametrize("pos0,n", [(0, 1), (0, 777), (100000, 333), ((1 << 24) - 100, 100), (12345, 1)])
def test_table(r, pos0, n):
    check_table(mi.Rope(rot_dim=r, theta=1e6), pos0, n)
    check_table(mi.Rope(rot_dim=r, theta=10000.0), pos0, n)


@pytest.mark.parametrize("r,theta", [(64, 10000.0), (128, 500000.0), (128, 1e6)])
@pytest.mark.parametrize("scaling,factor,low,high", [
    (mi.ROPE_LINEAR, 4.0, 0, 0), (mi.ROPE_BASE, 8.0, 0, 0), (mi.ROPE_WAVELENGTH, 8.0, 1.0, 4.0), (mi.ROPE_WAVELENGTH, 32.0, 1.0, 4.0),
    (mi.ROPE_YARN, 4.0, 1.0, 32.0), (mi.ROPE_YARN, 40.0, 1.0, 32.0), (mi.ROPE_YARN, 1.0, 1.0, 32.0), (mi.ROPE_YARN, 0.5, 1.0, 32.0)])
def test_scaled(r, theta, scaling, factor, low, high):
    much = 0.1 * np.log(factor) + 1 if scaling == mi.ROPE_YARN and factor > 1 else 1.0
    for attention in (0.0, 0.75):
        rope = mi.Rope(rot_dim=r, theta=theta, scaling=scaling, factor=factor, original=4096, low=low, high=high, attention=attention)
        check_table(rope, 30000, 500, much=attention or much, factor=factor, original=4096, low=low, high=high)


def test_divisors():
    d = np.linspace(1.0, 30.0, 48).astype(np.float32)
    rope = mi.Rope(rot_dim=96, theta=10000.0, attention=1.19, divisors=d.ctypes.data)
    check_table(rope, 5000, 300, much=float(np.float32(1.19)), divisors=d)


class Rows:
    def __init__(self, seed, T, qh=10, kvh=2, hd=128, rot=128, paired=False, f16=False, norm=True, pad=0, cache=None, act=0):
        rng = np.random.default_rng(seed)
        self.__dict__.update(T=T, qh=qh, kvh=kvh, hd=hd, rot=rot, paired=paired, f16=f16, pad=pad, act=act)
        self.n = (qh + 2 * kvh) * hd
        self.x = (rng.standard_normal((T, self.n + pad)) * 2).astype(np.float16 if f16 else np.float32)
        self.qn, self.kn = (rng.normal(1, 0.1, hd).astype(np.float32) if norm else None for _ in range(2))
        self.len = 500
        a = np.arange(self.len)[:, None] * 1e4 ** (-2.0 * np.arange(rot // 2) / rot)
        self.rope = np.stack([np.cos(a), np.sin(a)], 1).astype(np.float32)
        self.cache = cache or T + 9
        self.pos = rng.integers(0, self.len, T).astype(np.uint32)
        self.slot = rng.permutation(self.cache)[:T].astype(np.uint32)
        self.pos0 = 0

    def run(self, st=None, by_row=False):
        b = self.bind(by_row)
        mi.call("mi_rope_rows", *b["args"], stream() if st is None else st)
        return self.result(b)

    def bind(self, by_row=False):
        T = torch()
        rs, hs = (self.kvh * (self.hd + 8), self.hd + 8) if by_row else (self.hd, self.cache * self.hd)
        self.by_row = by_row
        q = empty((self.T * self.qh * self.hd + GUARD,), np.float32)
        q.fill_(7.0)
        size = self.cache * self.kvh * (self.hd + (8 if by_row else 0)) + GUARD
        k, v = (T.full((size,), 77, dtype=T.int16, device="cuda") for _ in range(2))
        sh = mi.AttnShape(self.qh, self.kvh, self.hd, self.rot, 0, self.n, self.qh * self.hd, (self.qh + self.kvh) * self.hd, 0.1, 1e-5, self.act)
        d = {n: dev(getattr(self, n)) for n in ("qn", "kn", "rope", "pos", "slot")}
        d["x"] = dev(self.x.view(np.uint16) if self.f16 else self.x)
        flag = dev(np.zeros(1, np.uint32))
        args = (ptr(d["x"]), mi.OUT_F16 if self.f16 else mi.OUT_F32, self.n + self.pad, self.T, ptr(d["pos"]), self.pos0, ptr(d["slot"]),
                self.cache, mi.C.byref(sh), int(self.paired), ptr(d["qn"]), ptr(d["kn"]), ptr(d["rope"]), self.len, ptr(q), ptr(k), ptr(v),
                rs, hs, ptr(flag))
        return dict(d, q=q, k=k, v=v, flag=flag, sh=sh, args=args)

    def result(self, b):
        sync()
        q = host(b["q"], np.float32)
        assert (q[self.T * self.qh * self.hd:] == 7.0).all()
        out = []
        for n in ("k", "v"):
            a = host(b[n], np.uint16)
            assert (a[-GUARD:] == 77).all()
            a = a[:-GUARD]
            if self.by_row:
                a = a.reshape(self.cache, self.kvh, self.hd + 8)
                assert (a[:, :, self.hd:] == 77).all()
                a = a[:, :, :self.hd].transpose(1, 0, 2)
            out.append(a.reshape(self.kvh, self.cache, self.hd))
        return q[:self.T * self.qh * self.hd].reshape(self.T, self.qh, self.hd), out[0], out[1], int(host(b["flag"], np.uint32)[0])

    def exact(self):
        """q, k [T][heads][hd] with their tolerances in 32 bits, v"""
        x = self.x[:, :self.n].astype(np.float64).reshape(self.T, -1, self.hd)
        pos = self.pos.astype(np.int64) if self.pos is not None else self.pos0 + np.arange(self.T)
        cs = self.rope[np.minimum(pos, self.len - 1)].astype(np.float64)[:, None]
        half, res = self.rot // 2, []
        for part, w in ((x[:, :self.qh], self.qn), (x[:, self.qh:self.qh + self.kvh], self.kn)):
            if w is not None:
                part = part / np.sqrt((part ** 2).mean(2, keepdims=True) + np.float64(np.float32(1e-5))) * w.astype(np.float64)
            a, b = (np.arange(half) * 2, np.arange(half) * 2 + 1) if self.paired else (np.arange(half), np.arange(half) + half)
            out, tol = part.copy(), 2.0 ** -20 * np.abs(part)
            c, s = cs[:, :, 0], cs[:, :, 1]
            out[:, :, a] = part[:, :, a] * c - part[:, :, b] * s
            out[:, :, b] = part[:, :, b] * c + part[:, :, a] * s
            tol[:, :, a] = 2.0 ** -20 * (np.abs(part[:, :, a] * c) + np.abs(part[:, :, b] * s))
            tol[:, :, b] = 2.0 ** -20 * (np.abs(part[:, :, b] * c) + np.abs(part[:, :, a] * s))
            res += [out, tol]
        return (*res, x[:, self.qh + self.kvh:])

    def check(self, got, live=None):
        q, ck, cv, _ = got
        live = np.ones(self.T, bool) if live is None else live
        wq, tq, wk, tk, wv = self.exact()
        assert np.all(np.abs(q - wq) <= tq)
        written = np.zeros(self.cache, bool)
        eps = 2.0 ** -8 + 2.0 ** -11 if self.act else 2.0 ** -11
        for t in np.nonzero(live)[0]:
            row = int(self.slot[t]) if self.slot is not None else self.pos0 + t if self.pos is None else int(self.pos[t])
            written[row] = True
            gk, gv = (c[:, row].view(np.float16).astype(np.float64) for c in (ck, cv))
            assert np.all(np.abs(gk - wk[t]) <= tk[t] + eps * np.abs(wk[t]) + 2.0 ** -24)
            assert np.all(np.abs(gv - wv[t]) <= eps * np.abs(wv[t]) + 2.0 ** -25)
        assert (ck[:, ~written] == 77).all() and (cv[:, ~written] == 77).all()


@pytest.mark.parametrize("qh,kvh,hd,rot", [(10, 2, 128, 128), (16, 2, 256, 64), (3, 3, 128, 96), (1, 1, 256, 256), (17, 1, 128, 8), (24, 4, 256, 248)])
@pytest.mark.parametrize("T", [1, 3, 70])
@pytest.mark.parametrize("paired", [False, True])
@pytest.mark.parametrize("f16,norm", [(False, True), (True, False), (True, True)])
def test_rows(T, qh, kvh, hd, rot, paired, f16, norm):
    c = Rows(T + rot, T, qh, kvh, hd, rot, paired, f16, norm, pad=5 if T == 3 else 0)
    got = c.run(by_row=bool(T % 2))
    c.check(got)
    assert got[3] == 0


@pytest.mark.parametrize("paired", [False, True])
def test_positions_and_rows_that_are_none_or_outside(paired):
    c = Rows(5, 40, paired=paired)
    c.slot[[3, 39]] = NONE
    live = c.slot != NONE
    got = c.run()
    c.check(got, live)
    assert got[3] == 0
    c = Rows(6, 40, paired=paired)
    c.slot[7] = c.cache
    live = np.arange(40) != 7
    got = c.run()
    c.check(got, live)
    assert got[3] == mi.STATUS_BAD_PAGE
    c = Rows(7, 40, paired=paired)
    c.pos[11] = c.len
    got = c.run()
    q = got[0].copy()
    assert (q[11] == 7.0).all()
    q[11] = c.exact()[0][11]
    c.check((q, *got[1:]), np.arange(40) != 11)
    assert got[3] == 0xDEAD0002


def test_given_positions_and_slots_may_be_left_out():
    c = Rows(8, 33, cache=100)
    c.pos, c.pos0 = None, 44
    c.check(c.run())
    c.slot = None
    c.check(c.run())
    c = Rows(9, 20, cache=500)
    c.pos = np.random.default_rng(1).permutation(500)[:20].astype(np.uint32)
    c.slot = None
    c.check(c.run())


def test_bf16_activations():
    c = Rows(10, 30, act=1)
    got = c.run()
    c.check(got)
    assert not (got[1][:, c.slot].view(np.float16).astype(np.float32).view(np.uint32) & 0xFFFF).any()


def test_table_then_rows_is_the_rows_entry_of_a_prompt_up_to_its_roundings():
    """the same rows through mi_attn_prep_rows, which rounds to f16 before and behind the norm: each of its q is within those
    roundings, 2^-11 of the norm's weight and input, of the one here"""
    T, qh, kvh, hd = 50, 10, 2, 128
    c = Rows(11, T, qh, kvh, hd, cache=T)
    c.pos, c.slot, c.pos0 = None, None, 0
    c.rope = table(mi.Rope(rot_dim=128, theta=1e4), 0, c.len).copy()
    b = c.bind()
    mi.call("mi_rope_rows", *b["args"], stream())
    mine = c.result(b)
    b2 = c.bind()
    mi.call("mi_attn_prep_rows", ptr(b2["x"]), T, 0, mi.C.byref(b2["sh"]), ptr(b2["qn"]), ptr(b2["kn"]), ptr(b2["rope"]), ptr(b2["q"]),
            ptr(b2["k"]), ptr(b2["v"]), c.hd, c.cache * c.hd, None, 0, stream())
    other = c.result(b2)
    tol = c.exact()[1] * 2.0 ** 20 * 2.0 ** -9 + 2.0 ** -20
    assert np.all(np.abs(mine[0] - other[0]) <= tol)
    assert np.array_equal(mine[2], other[2])


def test_captured_and_other_stream():
    T = torch()
    c = Rows(12, 30, f16=True)
    b = c.bind()
    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g):
        mi.call("mi_rope_rows", *b["args"], stream())
    rng = np.random.default_rng(3)
    for _ in range(3):
        c.pos, c.slot = rng.integers(0, c.len, 30).astype(np.uint32), rng.permutation(c.cache)[:30].astype(np.uint32)
        for n in ("pos", "slot"):
            b[n].copy_(dev(getattr(c, n)))
        b["k"].fill_(77)
        b["v"].fill_(77)
        g.replay()
        c.check(c.result(b))
    side = T.cuda.Stream()
    with T.cuda.stream(side):
        c.check(c.run(side.cuda_stream))


def test_tables_captured_and_on_another_stream():
    """the frequencies are read when the call is made"""
    T = torch()
    d = np.linspace(1.0, 9.0, 32).astype(np.float32)
    rope = mi.Rope(rot_dim=64, theta=10000.0, divisors=d.ctypes.data)
    outs = [T.zeros(100 * 64, dtype=T.float32, device="cuda") for _ in range(3)]
    mi.call("mi_rope_table", mi.C.byref(rope), 70, 100, ptr(outs[0]), stream())
    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g):
        mi.call("mi_rope_table", mi.C.byref(rope), 70, 100, ptr(outs[1]), stream())
    side = T.cuda.Stream()
    mi.call("mi_rope_table", mi.C.byref(rope), 70, 100, ptr(outs[2]), side.cuda_stream)
    d[:] = 3.0
    rope.theta = 5.0
    for _ in range(3):
        outs[1].zero_()
        g.replay()
        sync()
        assert T.equal(outs[0], outs[1]) and T.equal(outs[0], outs[2])


@pytest.mark.parametrize("by_row", [False, True])
def test_rows_past_32_bits(by_row):
    """cache rows whose offsets pass 2^32 elements, by heads or by rows"""
    T = torch()
    c = Rows(13, 3, kvh=2, cache=41)
    b = c.bind()
    rs, hs = (1 << 27, 128) if by_row else (128, (1 << 32) + 8)
    caches = [T.empty(40 * rs + hs + 128, dtype=T.int16, device="cuda").as_strided((2, 41, 128), (hs, rs, 1)) for _ in range(2)]
    for x in caches:
        x.fill_(77)
    c.slot = np.array([40, 3, 39], np.uint32)
    b["slot"].copy_(dev(c.slot))
    mi.call("mi_rope_rows", *b["args"][:15], ptr(caches[0]), ptr(caches[1]), rs, hs, ptr(b["flag"]), stream())
    for n, x in zip("kv", caches):
        b[n][:-GUARD] = x.reshape(-1)
    c.check(c.result(b))


def check_far_table(rope, pos0, n, **kw):
    """as check_table, with what two roundings of 64 bits leave of the angle (the frequency's and the product's): 2^-52 of it"""
    got = table(rope, pos0, n)
    angle = (pos0 + np.arange(n)).astype(LD)[:, None] * frequencies(rope.rot_dim, rope.theta, rope.scaling, **kw)
    for k, fn in enumerate((np.cos, np.sin)):
        want = fn(angle)
        tol = 2.0 ** -24 * np.abs(want) + 1.01 * (2.0 ** -52 * angle + 2.0 ** -46)
        assert np.all(np.abs(got[:, k] - want) <= tol), np.max(np.abs(got[:, k] - want) / tol)


@pytest.mark.parametrize("r", [24, 96, 128, 248, 256])
@pytest.mark.parametrize("theta", [1.5, 10000.0, 1e6, 1e30])
@pytest.mark.parametrize("pos0", [0, 1 << 24, 1 << 28, (1 << 31) - 999])
def test_table_of_far_positions(r, theta, pos0):
    check_far_table(mi.Rope(rot_dim=r, theta=theta), pos0, 999)


@pytest.mark.parametrize("r", [24, 64, 248])
@pytest.mark.parametrize("scaling,factor,low,high", [
    (mi.ROPE_LINEAR, 40.0, 0, 0), (mi.ROPE_LINEAR, 0.3, 0, 0), (mi.ROPE_BASE, 8.0, 0, 0), (mi.ROPE_WAVELENGTH, 32.0, 1.0, 4.0),
    (mi.ROPE_YARN, 40.0, 1.0, 32.0)])
@pytest.mark.parametrize("pos0", [1 << 20, (1 << 31) - 300])
def test_scaled_table_of_far_positions(r, scaling, factor, low, high, pos0):
    rope = mi.Rope(rot_dim=r, theta=1e6, scaling=scaling, factor=factor, original=4096, low=low, high=high, attention=1.0)
    check_far_table(rope, pos0, 300, factor=factor, original=4096, low=low, high=high)


def test_table_of_frequencies_above_one():
    """up to the most that is allowed, 2^20 a position"""
    d = np.geomspace(2.0 ** -20, 3.0, 120).astype(np.float32)
    for pos0 in (0, 100000, 1 << 24):
        check_far_table(mi.Rope(rot_dim=240, theta=1e6, divisors=d.ctypes.data), pos0, 200, divisors=d)
