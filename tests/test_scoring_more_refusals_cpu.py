"""More of what the scoring entries refuse before anything is launched: no GPU."""
import pytest

from mipkg import mi
from test_scoring_cpu import ARG, SHAPE, P, shape


@pytest.mark.parametrize("name", ["tokens", "logprob", "rank", "entropy", "top_ids", "top_logprobs"])
def test_misaligned_arrays_of_log_probabilities(name):
    L = mi.lib()
    a = dict(tokens=P, logprob=P, rank=P, entropy=P, top_ids=P, top_logprobs=P)
    for by in (1, 2):
        a[name] = P + by
        assert L.mi_logprobs(P, 1000, a["tokens"], 600, 1000, 5, a["logprob"], a["rank"], a["entropy"], a["top_ids"], a["top_logprobs"],
                             P, 1 << 30, None) == ARG
        assert b"misaligned" in L.mi_last_error()


@pytest.mark.parametrize("name", ["lo", "hi", "pos", "slopes", "pages", "flag"])
def test_misaligned_arrays_of_attention(name):
    L = mi.lib()
    for by in (1, 2):
        mask = mi.AttnMask(**({name: P + by} if name in ("lo", "hi", "pos", "slopes") else {}))
        pages, flag = (P + by if name == n else P for n in ("pages", "flag"))
        sh = shape()
        assert L.mi_attn_masked(P, P, P, 128, 1 << 20, pages, 64, 100, 1000, 1, mi.C.byref(sh), mi.C.byref(mask), P, 1 << 30, P, flag,
                                None) == ARG
        assert b"misaligned" in L.mi_last_error()


@pytest.mark.parametrize("T,pos0", [(1, 1 << 31), (2, (1 << 31) - 1), (65535, 0xFFFFFFFF), (1, 0xFFFFFFFF)])
def test_positions_past_31_bits(T, pos0):
    L = mi.lib()
    sh, mask = shape(), mi.AttnMask(pos0=pos0)
    assert L.mi_attn_masked(P, P, P, 128, 1 << 20, None, 0, 0, 1000, T, mi.C.byref(sh), mi.C.byref(mask), P, 1 << 30, P, None, None) == SHAPE
    assert b"positions" in L.mi_last_error()
