"""The linear in 8-bit integers (mi_quant_rows_i8, mi_gemm_w8a8, mi_linear_w8a8) against its definition.

The scale max|x| / 127 and the quotient x / scale are fp32 divisions, which numpy rounds as the library
does, so scales and integers are equal bit for bit. The int32 sum is exact; an output takes one rounding to
fp32 and two fp32 products, 3 * 2^-24 of its value, and for f16 half a step more (2^-11, or half of the
smallest subnormal, 2^-25)."""
import numpy as np
import pytest

from mipkg import dev, empty, host, mi, ptr, stream, sync, torch

pytestmark = pytest.mark.gpu

GUARD = 64


def tile(q):
    """int8 [rows][K] -> mi_i8w_index's layout, rows padded to 16 with zeros"""
    M, K = q.shape
    p = np.zeros(((M + 15) // 16 * 16, K), np.int8)
    p[:M] = q
    return np.ascontiguousarray(p.reshape(-1, 16, K // 64, 2, 4, 8).transpose(0, 2, 4, 1, 3, 5)).reshape(-1)


def untile(t, M, K):
    a = t.reshape(-1, K // 64, 4, 16, 2, 8).transpose(0, 3, 1, 4, 2, 5)
    return np.ascontiguousarray(a).reshape(-1, K)


def quantised(x):
    xf = x.astype(np.float32)
    s = np.abs(xf).max(1) / np.float32(127)
    s[~np.isfinite(xf).all(1)] = np.nan
    with np.errstate(all="ignore"):
        q = np.rint(xf / s[:, None])
    q[~(s > 0)] = 0
    return q.astype(np.int8), s.astype(np.float32)


def rows(rng, M, K):
    x = rng.standard_normal((M, K)).astype(np.float16)
    x[rng.random((M, K)) < 0.01] *= 30  # some large channels
    return x


def strided(x, stride):
    buf = np.full((x.shape[0], stride), np.float16(7), np.float16)
    buf[:, :x.shape[1]] = x
    return dev(buf.view(np.uint16))


def weights(rng, N, K):
    return rng.integers(-127, 128, (N, K)).astype(np.int8), (rng.uniform(0.5, 1.5, N) / (73 * K ** 0.5)).astype(np.float32)


def call_linear(x, w, ws, kind, *, x_stride=None, out_stride=None, st=None):
    M, K = x.shape
    N = w.shape[0]
    x_stride, out_stride = x_stride or K, out_stride or N
    dx, dw, dws = strided(x, x_stride), dev(tile(w)), dev(ws)
    need = mi.lib().mi_linear_w8a8_ws(M, K)
    T = torch()
    scratch = T.full((need + GUARD,), 77, dtype=T.uint8, device="cuda")
    out = empty((M * out_stride + GUARD,), np.float32 if kind == mi.OUT_F32 else np.uint16)
    out.fill_(5)
    mi.call("mi_linear_w8a8", ptr(dx), x_stride, ptr(dw), ptr(dws), ptr(scratch), need, ptr(out), kind, out_stride, M, K, N,
            st if st is not None else stream())
    sync()
    assert (scratch[need:] == 77).all()
    flat = out.cpu().numpy()
    body = flat[:M * out_stride].reshape(M, out_stride)
    assert (flat[M * out_stride:] == 5).all() and (body[:, N:] == 5).all()  # nothing behind the rows or the matrix
    got = np.ascontiguousarray(body[:, :N])
    return got if kind == mi.OUT_F32 else got.view(np.float16)


def check(got, x, w, ws, kind):
    q, s = quantised(x)
    want = (q.astype(np.int64) @ w.T.astype(np.int64)) * s.astype(np.float64)[:, None] * ws.astype(np.float64)
    fine = np.isfinite(s)
    assert np.isnan(got[~fine].astype(np.float64)).all()
    got, want = got[fine].astype(np.float64), want[fine]
    tol = 3.01 * 2.0 ** -24 * np.abs(want) + 2.0 ** -149
    if kind == mi.OUT_F16:
        tol = tol + 2.0 ** -11 * np.abs(want) * (1 + 2.0 ** -20) + 2.0 ** -25
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / np.maximum(np.abs(want), 1e-30))


SHAPES = [(1, 64, 16), (1, 5120, 512), (2, 128, 48), (3, 17408, 80), (5, 448, 1040), (8, 1024, 256), (13, 5120, 272),
          (16, 192, 16), (17, 320, 64), (31, 1088, 144), (33, 4096, 528), (64, 64, 256), (65, 704, 272), (100, 2048, 1024),
          (129, 512, 400), (200, 1152, 2064), (257, 640, 784), (333, 1024, 512), (515, 256, 1296)]


@pytest.mark.parametrize("M,K", sorted({(m, k) for m, k, _ in SHAPES}))
def test_quantised_rows_bit_for_bit(M, K):
    rng = np.random.default_rng(M * 7 + K)
    x = rows(rng, M, K)
    if M > 4:
        x[1] = 0
        x[2, K // 2] = np.inf
        x[3, 0] = np.nan
        x[4] = np.float16(6e-8) * rng.integers(-3, 4, K)  # subnormals
    dx = strided(x, K + 24)
    nb = (M + 15) // 16 * 16 * K
    q, s = empty((nb + GUARD,), np.int8), empty((M + 4,), np.float32)
    q.fill_(99)
    s.fill_(3)
    mi.call("mi_quant_rows_i8", ptr(dx), K + 24, M, K, ptr(q), ptr(s), stream())
    sync()
    wq, wsc = quantised(x)
    hq, hs = host(q, np.int8), host(s, np.float32)
    assert (hq[nb:] == 99).all() and (hs[M:] == 3).all()
    assert np.array_equal(hs[:M], wsc, equal_nan=True)
    full = untile(hq[:nb], M, K)
    assert np.array_equal(full[:M], wq)
    assert not full[M:].any()
    L = mi.lib()
    for m, k in ((0, 0), (M - 1, K - 1), (M // 2, K // 3)):
        assert hq[L.mi_i8w_index(K, k, m)] == wq[m, k]


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear_against_the_definition(M, K, N, kind):
    rng = np.random.default_rng(M + K + N)
    x = rows(rng, M, K)
    if M > 4:
        x[M // 2] = 0
        x[M - 1, 5] = np.nan
    w, ws = weights(rng, N, K)
    print(f"linear_w8a8 M={M} K={K} N={N} kind={kind}", flush=True)
    got = call_linear(x, w, ws, kind, x_stride=K + 8 * (M % 3), out_stride=N + M % 5)
    check(got, x, w, ws, kind)


def test_largest_sums_do_not_overflow():
    K, N, M = 131072, 32, 3
    x = np.ones((M, K), np.float16)
    x[1] = -1
    w = np.full((N, K), 127, np.int8)
    w[1] = -127
    ws = np.full(N, 2.0 ** -20, np.float32)
    check(call_linear(x, w, ws, 0), x, w, ws, 0)


@pytest.mark.parametrize("K,N", [(1024, 272), (5120, 528)])
def test_a_row_is_the_same_among_others(K, N):
    """the sums are integers: a row's bits depend neither on the rows beside it nor on the kernel"""
    rng = np.random.default_rng(K)
    x, (w, ws) = rows(rng, 300, K), weights(rng, N, K)
    whole = call_linear(x, w, ws, 0)
    for r0, r1 in ((0, 1), (17, 20), (33, 46), (100, 130), (200, 300)):
        assert np.array_equal(call_linear(x[r0:r1], w, ws, 0), whole[r0:r1])


@pytest.mark.parametrize("M", [1, 7, 40, 300])
def test_the_parts_are_the_whole(M):
    K, N = 1536, 400
    rng = np.random.default_rng(M)
    x, (w, ws) = rows(rng, M, K), weights(rng, N, K)
    whole = call_linear(x, w, ws, 1)
    dx, dw, dws = strided(x, K), dev(tile(w)), dev(ws)
    q, s = empty(((M + 15) // 16 * 16 * K,), np.int8), empty((M,), np.float32)
    out = empty((M, N), np.uint16)
    mi.call("mi_quant_rows_i8", ptr(dx), K, M, K, ptr(q), ptr(s), stream())
    mi.call("mi_gemm_w8a8", ptr(q), ptr(s), ptr(dw), ptr(dws), ptr(out), mi.OUT_F16, N, M, K, N, stream())
    sync()
    assert np.array_equal(host(out, np.uint16), whole.view(np.uint16))


def test_other_stream_and_replayed_graph():
    T = torch()
    K, N = 2048, 512
    rng = np.random.default_rng(3)
    w, ws = weights(rng, N, K)
    side = T.cuda.Stream()
    with T.cuda.stream(side):
        for M in (1, 20):
            x = rows(rng, M, K)
            check(call_linear(x, w, ws, 0, st=side.cuda_stream), x, w, ws, 0)
    for M in (1, 12, 150):
        dx, dw, dws = dev(rows(rng, M, K).view(np.uint16)), dev(tile(w)), dev(ws)
        need = mi.lib().mi_linear_w8a8_ws(M, K)
        scratch, out = T.empty(need, dtype=T.uint8, device="cuda"), empty((M, N), np.float32)
        g = T.cuda.CUDAGraph()
        with T.cuda.graph(g):
            mi.call("mi_linear_w8a8", ptr(dx), K, ptr(dw), ptr(dws), ptr(scratch), need, ptr(out), 0, N, M, K, N, stream())
        for _ in range(3):
            x = rows(rng, M, K)
            dx.copy_(dev(x.view(np.uint16)))
            out.zero_()
            g.replay()
            sync()
            check(host(out, np.float32).reshape(M, N), x, w, ws, 0)


# sizes that between them take every shape of the product's work-groups, each with rows, columns or chunks that end
# inside one
WIDE = [(9, 2112, 5136), (27, 1088, 6160), (33, 5184, 7184), (61, 1088, 10256), (515, 8256, 80), (250, 64, 4112), (131, 2112, 10256),
        (333, 5184, 5136), (390, 576, 7184), (131, 64, 20496), (515, 1088, 7184), (1021, 64, 10256), (131, 2112, 34832),
        (1500, 192, 10256), (2045, 448, 7184), (500, 1088, 34848), (500, 1600, 45520)]


@pytest.mark.parametrize("M,K,N", WIDE)
def test_wide_products_are_the_exact_sums(M, K, N):
    """outputs compared bit for bit: the sums are integers below 2^53, so a product in fp64 is exact, and the two fp32
    products that follow round alike"""
    T = torch()
    rng = np.random.default_rng(M + K + N)
    q = rng.integers(-127, 128, (M, K)).astype(np.int8)
    w = rng.integers(-127, 128, (N, K)).astype(np.int8)
    qs, ws = dev(rng.uniform(0.01, 0.02, M).astype(np.float32)), dev(rng.uniform(0.01, 0.02, N).astype(np.float32))
    dq, dw = dev(tile(q)), dev(tile(w))
    stride = N + 5
    out = T.full((M * stride + GUARD,), 5.0, dtype=T.float32, device="cuda")
    print(f"gemm_w8a8 M={M} K={K} N={N}", flush=True)
    mi.call("mi_gemm_w8a8", ptr(dq), ptr(qs), ptr(dw), ptr(ws), ptr(out), mi.OUT_F32, stride, M, K, N, stream())
    sync()
    sums = T.mm(T.from_numpy(q).cuda().double(), T.from_numpy(w).cuda().double().t().contiguous())
    want = (sums.float() * qs[:, None]) * ws
    body = out[:M * stride].view(M, stride)
    assert T.equal(body[:, :N], want)
    assert (body[:, N:] == 5).all() and (out[M * stride:] == 5).all()


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("K,N", [(64, 16), (320, 7184), (448, 4112), (5120, 7168), (17408, 80), (32768, 48), (32832, 48)])
def test_a_single_row(K, N, kind):
    rng = np.random.default_rng(K + N)
    w, ws = weights(rng, N, K)
    for special in (None, 0, np.inf, np.nan, 65504):
        x = rows(rng, 1, K)
        if special == 0:
            x[:] = 0
        elif special is not None:
            x[0, K - 1] = special
        got = call_linear(x, w, ws, kind, x_stride=K + 8)
        if special in (0, None, 65504):
            assert np.isfinite(got).all()
        check(got, x, w, ws, kind)
