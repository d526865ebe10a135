"""Refusals and workspace sizes of the scoring entries (mi_linear_w8a8, mi_logprobs, mi_attn_masked): no GPU."""
import pytest

from mipkg import mi

ARG, SHAPE = -1, -2
P = 1 << 20  # a pointer that no refused call follows


def test_linear_refusals():
    L = mi.lib()

    def linear(x=P, xs=1024, w=P, wsc=P, ws=P, nb=1 << 30, out=P, kind=0, os_=256, M=8, K=1024, N=256):
        return L.mi_linear_w8a8(x, xs, w, wsc, ws, nb, out, kind, os_, M, K, N, None)

    for kw in ({"x": None}, {"w": None}, {"wsc": None}, {"ws": None}, {"out": None}, {"x": P + 2}, {"w": P + 8}, {"ws": P + 4},
               {"out": P + 2}, {"out": P + 1, "kind": 1}, {"xs": 1020}, {"xs": 1028}, {"os_": 255}, {"kind": 2}, {"wsc": P + 2},
               {"nb": L.mi_linear_w8a8_ws(8, 1024) - 1}):
        assert linear(**kw) == ARG, kw
        assert b"linear_w8a8" in L.mi_last_error()
    for kw in ({"M": 0}, {"K": 0}, {"N": 0}, {"K": 1000, "xs": 1000}, {"N": 250}, {"K": 131136, "xs": 131136}, {"M": (1 << 20) + 1},
               {"N": (1 << 22) + 16, "os_": 1 << 23}):
        assert linear(**kw) == SHAPE, kw


def test_quantiser_and_product_refusals():
    L = mi.lib()
    for args in ((None, 64, 1, 64, P, P), (P, 64, 1, 64, None, P), (P, 64, 1, 64, P, None), (P, 64, 1, 64, P + 8, P), (P, 56, 1, 64, P, P),
                 (P, 64, 1, 64, P, P + 2)):
        assert L.mi_quant_rows_i8(*args, None) == ARG, args
    for args in ((P, 64, 0, 64, P, P), (P, 64, 1, 32, P, P), (P, 0, 1, 0, P, P)):
        assert L.mi_quant_rows_i8(*args, None) == SHAPE, args

    def product(q=P, s=P, w=P, wsc=P, out=P, kind=1, os_=64, M=2, K=64, N=64):
        return L.mi_gemm_w8a8(q, s, w, wsc, out, kind, os_, M, K, N, None)

    for kw in ({"q": None}, {"s": None}, {"w": None}, {"wsc": None}, {"out": None}, {"q": P + 8}, {"s": P + 1}, {"os_": 63}, {"kind": 9}):
        assert product(**kw) == ARG, kw
    for kw in ({"M": 0}, {"K": 96}, {"N": 72, "os_": 72}):
        assert product(**kw) == SHAPE, kw


def test_linear_workspace_holds_the_rows_and_their_scales():
    L = mi.lib()
    for M in (1, 15, 16, 17, 2048):
        for K in (64, 5120, 131072):
            assert L.mi_linear_w8a8_ws(M, K) >= (M + 15) // 16 * 16 * K + 4 * M


def test_logprobs_refusals():
    L = mi.lib()

    def logprobs(x=P, stride=1000, tokens=P, M=2, used=1000, top=5, lp=P, rank=P, en=P, ids=P, tl=P, ws=P, nb=1 << 30):
        return L.mi_logprobs(x, stride, tokens, M, used, top, lp, rank, en, ids, tl, ws, nb, None)

    for kw in ({"x": None}, {"x": P + 2}, {"stride": 999}, {"tokens": None}, {"tokens": None, "lp": None}, {"ids": None}, {"tl": None},
               {"top": 0}, {"top": 0, "ids": None}, {"lp": None, "rank": None, "en": None, "top": 0, "ids": None, "tl": None}):
        assert logprobs(**kw) == ARG, kw
        assert b"logprobs" in L.mi_last_error()
    for kw in ({"M": 0}, {"M": 65536}, {"used": 0}, {"used": (1 << 23) + 1, "stride": 1 << 24}, {"top": 65}):
        assert logprobs(**kw) == SHAPE, kw
    need = L.mi_logprobs_ws(1, 151936, 20)
    assert need > 0
    for kw in ({"ws": None}, {"ws": P + 8}, {"nb": need - 1}):
        assert logprobs(M=1, used=151936, stride=151936, top=20, **kw) == ARG, kw


def test_logprobs_workspace():
    L = mi.lib()
    assert L.mi_logprobs_ws(0, 10, 1) == 0 and L.mi_logprobs_ws(1, 0, 1) == 0
    for M in (1, 7, 333, 2048, 65535):
        for used in (1, 1000, 151936, 1 << 23):
            assert L.mi_logprobs_ws(M, used, 64) <= 64 << 20
            assert L.mi_logprobs_ws(M, used, 64) >= L.mi_logprobs_ws(M, used, 0)


def shape(qh=40, kvh=8, hd=128, gated=0, act=0):
    return mi.AttnShape(qh, kvh, hd, hd, gated, (qh + 2 * kvh) * hd, qh * hd, (qh + kvh) * hd, hd ** -0.5, 1e-6, act)


def test_attention_refusals():
    L = mi.lib()

    def attn(q=P, k=P, v=P, rs=128, hs=1 << 20, pages=None, page=0, n_pages=0, kv_len=1000, T=1, sh=None, mask=None, ws=P, nb=1 << 30,
             out=P, sh_ref=True, mask_ref=True):
        sh, mask = sh or shape(), mask or mi.AttnMask()
        return L.mi_attn_masked(q, k, v, rs, hs, pages, page, n_pages, kv_len, T, mi.C.byref(sh) if sh_ref else None,
                                mi.C.byref(mask) if mask_ref else None, ws, nb, out, None, None)

    need = L.mi_attn_masked_ws(1, 1000, mi.C.byref(shape()))
    assert need > 0
    for kw in ({"q": None}, {"k": None}, {"v": None}, {"out": None}, {"sh_ref": False}, {"mask_ref": False}, {"k": P + 8}, {"v": P + 2},
               {"q": P + 2}, {"out": P + 1}, {"rs": 132}, {"hs": (1 << 20) + 4}, {"pages": P, "page": 0, "n_pages": 5},
               {"pages": P, "page": 64, "n_pages": 0}, {"ws": None}, {"ws": P + 4}, {"nb": need - 1}, {"sh": shape(act=2)},
               {"mask": mi.AttnMask(cap=-1.0)}, {"mask": mi.AttnMask(cap=float("nan"))}, {"mask": mi.AttnMask(cap=float("inf"))}, {"mask": mi.AttnMask(cap=1e-30)}):
        assert attn(**kw) == ARG, kw
        assert b"attn_masked" in L.mi_last_error()
    for kw in ({"T": 0}, {"T": 65536}, {"kv_len": 0}, {"kv_len": (1 << 30) + 1}, {"sh": shape(hd=64)}, {"sh": shape(40, 7)}, {"sh": shape(40, 0)},
               {"sh": shape(130, 2)}, {"sh": shape(0, 2)}, {"sh": shape(gated=1)}, {"pages": P, "page": 1 << 20, "n_pages": 1 << 13}):
        assert attn(**kw) == SHAPE, kw


def test_attention_workspace_grows_with_rows_and_keys_within_bounds():
    L = mi.lib()
    for qh, kvh, hd in ((40, 8, 128), (16, 2, 256), (64, 1, 128), (1, 1, 128), (1024, 1024, 128)):
        sh = mi.C.byref(shape(qh, kvh, hd))
        assert L.mi_attn_masked_ws(0, 5, sh) == 0 and L.mi_attn_masked_ws(1, 0, sh) == 0
        for T in (1, 2, 3, 7, 64, 500, 2048, 65535):
            sizes = [L.mi_attn_masked_ws(T, n, sh) for n in (1, 100, 1000, 10000, 131072)]
            assert sizes == sorted(sizes) and sizes[-1] <= 1 << 30, (qh, kvh, hd, T, sizes)
    assert L.mi_attn_masked_ws(1, 100, mi.C.byref(shape(hd=64))) == 0
