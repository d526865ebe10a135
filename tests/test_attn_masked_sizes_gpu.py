"""mi_attn_masked's workspace: one that was asked for the largest call serves the smaller ones."""
import numpy as np
import pytest

from mipkg import mi, ptr, stream, torch
from test_attn_masked_gpu import GUARD, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qh,kvh,hd", [(40, 8, 128), (16, 16, 128), (16, 2, 256)])
def test_one_workspace_for_all_smaller_calls(qh, kvh, hd):
    """asked once for the largest chunk and the longest cache; each call may use no more than that"""
    T = torch()
    big = Case(1, 700, 1600, qh, kvh, hd)
    sh = big.shape()
    need = mi.lib().mi_attn_masked_ws(700, 1600, mi.C.byref(sh))
    ws = T.full((need + GUARD,), 77, dtype=T.uint8, device="cuda")
    for rows, keys in ((1, 1600), (2, 900), (3, 1600), (4, 1600), (20, 1600), (60, 1000), (130, 1500), (300, 1600), (500, 700), (700, 1600)):
        for with_lo in (False, True):
            c = Case(rows, rows, keys, qh, kvh, hd, lo=np.full(rows, 40) if with_lo else None)
            b = c.bind()
            mi.call("mi_attn_masked", *b["args"][:12], ptr(ws), need, *b["args"][14:], stream())
            want, tol = c.exact()
            assert np.all(np.abs(c.result(b).astype(np.float64) - want) <= tol), (rows, keys)
    assert (ws[need:] == 77).all()
