"""mi_attn_masked's scores over the range that it accepts: caps from small to far above the scores, and scores far below zero.
The tolerances are test_attn_masked_gpu.py's, but for the cap's part, which does not grow with the cap: 2^-21 of one up to 256,
of larger ones 2^-20 of the score."""
import numpy as np
import pytest

from test_attn_masked_gpu import Case

pytestmark = pytest.mark.gpu


class Capped(Case):
    """The oracle's scores capped by tanh in 64 bits. With E = e^(2 |x| / cap) and u = 2^-24, the kernels' second term 2 / (E + 1) is off
    by E / (E + 1) 2 u (the exponential), u (the sum) and 2 u (the reciprocal) of itself: as a part of the cap 2 * 3 u at most and
    with the other roundings 8 u; where |x| / cap >= 1/4 and E >= 1 0.76 * 4.3 u and with them 4 u, 16 u of the score, which is
    0.24 cap at least. A cap only shrinks the error that the score has from its sum."""

    def exact(self):
        seen, p = self.seen()
        out, tol = np.zeros((self.T, self.qh, self.hd)), np.zeros((self.T, self.qh, self.hd))
        group = self.qh // self.kvh
        for h in range(self.qh):
            kd, vd, qd = self.k[h // group].astype(np.float64), self.v[h // group].astype(np.float64), self.q[:, h].astype(np.float64)
            s = self.cap * np.tanh(qd @ kd.T * self.scale / self.cap)
            ds = abs(self.scale) * (2.0 ** -21 + self.hd * 2.0 ** -23) * (np.abs(qd) @ np.abs(kd).T)
            ds = ds + (2.0 ** -21 * self.cap if self.cap <= 256 else 2.0 ** -20 * np.abs(s))
            m = np.where(seen, s, -np.inf).max(1, keepdims=True)
            e = np.exp(np.where(seen, s - m, -np.inf))
            w = e / e.sum(1, keepdims=True)
            out[:, h] = w @ vd
            near = np.where(w > 1e-12, ds, 0).max(1, keepdims=True)
            tol[:, h] = (2.0 ** -11 + 2.1 * near + 2.0 ** -19) * (w @ np.abs(vd)) + self.keys * 2.0 ** -32 * np.abs(vd).max()
        return out, tol + 2.0 ** -11 * np.abs(out) + 2.0 ** -25


@pytest.mark.parametrize("cap", [1e-3, 0.5, 2.0, 30.0, 128.0, 200.0, 256.0, 257.0, 1e3, 1e5, 1e6, 1e8, 1e20, 1e30])
@pytest.mark.parametrize("T,keys,qh,kvh,hd,page", [(1, 777, 10, 2, 128, 0), (2, 500, 16, 2, 256, 24), (90, 400, 10, 2, 128, 0), (50, 130, 16, 2, 256, 64),
                                                   (700, 700, 40, 8, 128, 64), (130, 1500, 16, 2, 256, 0)])
def test_caps(T, keys, qh, kvh, hd, page, cap):
    Capped(T + keys, T, keys, qh, kvh, hd, cap=cap, q_std=4.0, page=page).check()


@pytest.mark.parametrize("cap", [1e3, 1e6])
@pytest.mark.parametrize("T,keys,qh,kvh,hd", [(1, 300, 10, 2, 128), (90, 400, 10, 2, 128), (50, 130, 16, 2, 256)])
def test_caps_near_large_scores(T, keys, qh, kvh, hd, cap):
    """scores up to and past the cap, where the tanh bends and where it is 1"""
    Capped(T + keys, T, keys, qh, kvh, hd, cap=cap, q_std=cap / 2).check()


@pytest.mark.parametrize("T,keys,qh,kvh,hd", [(1, 300, 10, 2, 128), (1, 5000, 10, 2, 128), (90, 400, 10, 2, 128), (50, 130, 16, 2, 256),
                                              (20, 4020, 40, 8, 128)])
def test_scores_far_below_zero(T, keys, qh, kvh, hd):
    """a bias that takes every key that a row sees below -1e30: the nearest one has it all"""
    hi = np.arange(T) + keys - T - 20
    c = Case(T + keys, T, keys, qh, kvh, hd, hi=hi, pos=hi + 19, slopes=True)
    c.slopes[:] = np.float32(1e30)
    got = c.run().astype(np.float64)
    assert np.array_equal(got, np.repeat(c.v[:, hi - 1].transpose(1, 0, 2), qh // kvh, axis=1).astype(np.float64))
