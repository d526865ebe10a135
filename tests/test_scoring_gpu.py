"""The scoring entries one after another, as a program scores packed texts: q||k||v in 8-bit integers, mi_attn_prep_rows
into the paged cache, attention inside each document behind a shared prompt, the o linear, the head and the log
probabilities. Every stage is held to its definition on what the stage before left on the device."""
import numpy as np
import pytest

from mipkg import dev, empty, host, mi, ptr, stream, sync, torch
from test_attn_masked_gpu import Case
from test_linear_w8a8_gpu import check as check_linear, rows, tile, weights
from test_logprobs_gpu import check_row

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,before,starts", [(1, 130, [0]), (45, 70, [0, 11, 12, 40])])
def test_packed_texts(T, before, starts):
    H, QH, KVH, HD, V, PAGE = 640, 10, 2, 128, 2064, 32
    rng = np.random.default_rng(T)
    keys, st = before + T, stream()
    n = (QH + 2 * KVH) * HD
    w = {"qkv": weights(rng, n, H), "o": weights(rng, H, QH * HD), "head": weights(rng, V, H)}
    dw = {k: (dev(tile(a)), dev(s)) for k, (a, s) in w.items()}
    lo = np.array([before + max(s for s in starts if s <= t) for t in range(T)], np.uint32)
    c = Case(T, T, keys, QH, KVH, HD, lo=lo, prefix=before, cap=30.0, page=PAGE)
    x = rows(rng, T, H)
    c.fill = np.float16(0)
    b = c.bind()  # the cache with the prompt's keys; the chunk's own rows are written below
    rope = np.zeros((keys, 2, HD // 2), np.float32)
    ang = np.arange(keys)[:, None] * (1e4 ** (-np.arange(HD // 2) / (HD // 2)))
    rope[:, 0], rope[:, 1] = np.cos(ang), np.sin(ang)
    drope, dx = dev(rope), dev(x.view(np.uint16))
    L, T_ = mi.lib(), torch()
    scratch = T_.empty(max(L.mi_linear_w8a8_ws(T, H), L.mi_linear_w8a8_ws(T, QH * HD)), dtype=T_.uint8, device="cuda")
    qkv, q = empty((T, n), np.float32), empty((T, QH, HD), np.float32)
    o, logits = empty((T, H), np.uint16), empty((T, V), np.float32)
    tokens = rng.integers(0, V, T)
    dt = dev(tokens.astype(np.uint32))
    lp, rank, en = empty((T,), np.float32), empty((T,), np.uint32), empty((T,), np.float32)
    ids, tl = empty((T, 5), np.uint32), empty((T, 5), np.float32)
    lws = T_.empty(max(L.mi_logprobs_ws(T, V, 5), 1), dtype=T_.uint8, device="cuda")

    def linear(name, src, K, out, kind, N):
        mi.call("mi_linear_w8a8", ptr(src), K, ptr(dw[name][0]), ptr(dw[name][1]), ptr(scratch), scratch.numel(), ptr(out), kind, N,
                T, K, N, st)

    attn_args = (ptr(q),) + b["args"][1:]
    rs, hs = attn_args[3], attn_args[4]
    linear("qkv", dx, H, qkv, mi.OUT_F32, n)
    mi.call("mi_attn_prep_rows", ptr(qkv), T, before, mi.C.byref(b["sh"]), None, None, ptr(drope), ptr(q), ptr(b["k"]), ptr(b["v"]), rs, hs,
            ptr(b["pages"]), PAGE, st)
    mi.call("mi_attn_masked", *attn_args, st)
    linear("o", b["out"], QH * HD, o, mi.OUT_F16, H)
    linear("head", o, H, logits, mi.OUT_F32, V)
    mi.call("mi_logprobs", ptr(logits), V, ptr(dt), T, V, 5, ptr(lp), ptr(rank), ptr(en), ptr(ids), ptr(tl), ptr(lws), lws.numel(), st)
    sync()

    check_linear(host(qkv, np.float32), x, *w["qkv"], mi.OUT_F32)
    at = c.order[np.arange(keys) // PAGE].astype(np.int64) * PAGE + np.arange(keys) % PAGE
    c.q = host(q, np.float32)
    c.k, c.v = (host(b[name], np.uint16).view(np.float16).reshape(KVH, -1, HD)[:, at] for name in ("k", "v"))
    want, tol = c.exact()
    a16 = c.result(b)
    assert np.all(np.abs(a16.astype(np.float64) - want) <= tol)
    check_linear(host(o, np.uint16).view(np.float16), a16.reshape(T, QH * HD), *w["o"], mi.OUT_F16)
    check_linear(host(logits, np.float32), host(o, np.uint16).view(np.float16), *w["head"], mi.OUT_F32)
    got = {"lp": host(lp, np.float32), "rank": host(rank, np.uint32), "entropy": host(en, np.float32), "ids": host(ids, np.uint32),
           "top": host(tl, np.float32)}
    lg = host(logits, np.float32)
    for t in range(T):
        check_row(lg[t], int(tokens[t]), 5, got, t)
