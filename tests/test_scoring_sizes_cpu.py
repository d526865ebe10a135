"""The workspace sizes of the scoring entries over all that a program may ask: no GPU."""
from mipkg import mi

HEADS = [(40, 8, 128), (32, 8, 128), (16, 16, 128), (16, 2, 256), (24, 4, 256), (10, 2, 128), (1, 1, 128), (64, 1, 256), (1024, 1024, 128)]


def shape(qh, kvh, hd):
    return mi.C.byref(mi.AttnShape(qh, kvh, hd, hd, 0, (qh + 2 * kvh) * hd, qh * hd, (qh + kvh) * hd, hd ** -0.5, 1e-6, 0))


def test_sizes_that_the_calls_refuse():
    L = mi.lib()
    for n in (0, (1 << 23) + 1, 0xFFFFFC00, 0xFFFFFC01, 0xFFFFFFFF):
        assert L.mi_logprobs_ws(1, n, 5) == 0
    for M in (0, 65536, 0xFFFFFFFF):
        assert L.mi_logprobs_ws(M, 1000, 5) == 0
    for heads in HEADS:
        for T in (0, 65536, 1 << 31, 0xFFFFFFC0, 0xFFFFFFF5, 0xFFFFFFFF):
            assert L.mi_attn_masked_ws(T, 1000, shape(*heads)) == 0
        for n in (0, (1 << 30) + 1, 0xFFFFFFE0, 0xFFFFFFFF):
            for T in (1, 20, 2048):
                assert L.mi_attn_masked_ws(T, n, shape(*heads)) == 0
    assert L.mi_attn_masked_ws(1, 1000, None) == 0


def test_attention_workspace_never_falls():
    """a workspace that was asked for the largest call serves the smaller ones"""
    L = mi.lib()
    rows = sorted(set(list(range(1, 80)) + [int(80 * 1.13 ** i) for i in range(55)] + [777, 1000, 2048, 65535]))
    keys = sorted(set(list(range(1, 300, 7)) + [int(300 * 1.17 ** i) for i in range(97)] + [3406, 3503, 8000, 131072, 1 << 30]))
    assert rows[-1] == 65535 and keys[-1] == 1 << 30
    for heads in HEADS:
        size = [[L.mi_attn_masked_ws(T, n, shape(*heads)) for n in keys] for T in rows]
        assert all(r == sorted(r) for r in size), heads
        assert all(list(c) == sorted(c) for c in zip(*size)), heads
        assert size[-1][-1] <= (1 << 18) * (heads[2] + 4) * 4
