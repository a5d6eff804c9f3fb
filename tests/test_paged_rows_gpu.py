"""Attention over pages held to each output element by itself: rows of thousands of
positions, whose results are small, no less than rows of one.

Tolerance.  The result is o = sum w_j v_j; weights off by factors 1 + e_j move it by
sum w_j e_j (v_j - o), at most max|e| times twice W = sum w_j |v_j|.  With u = 2^-24
and N(0, 1) data: a score is a sum of hd products whose partial sums grow like a
random walk, roundings of rms u/sqrt(3) of them each, hd / sqrt(2) of which over
sqrt(hd) are 0.4 sqrt(hd) u (6.5 u at 256); q in two halves 1 u; scaling, and the
exponential's argument, of scores up to 5 in base 2, 5 u; the exponential 2 u, a weight
in two halves 2 u: about 10 u rms for one e_j, which are independent, so that the
sum's rms is below 10 u W.  Sums of weights and products add roundings of a sum
that grows to W: sqrt(n / 3) u for n in one run of at most 2500 additions,
29 u, of which a fifth remains where runs are joined of dozens of shorter ones.
64 u W is five times the larger of both; there are 10^5 elements a case, for which five
sigma are exceeded once in ten million."""
from __future__ import annotations

import numpy as np
import pytest

from test_paged_gpu import _attend, _step

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _check_rows(bh, dev, s, **kw):
    got = _attend(bh, dev, s, **kw)[0].astype(np.float64)
    k, v = (c.cpu().numpy().astype(np.float64) for c in (s["k"], s["v"]))
    n_q, n_kv, hd = s["q"].shape[1], k.shape[2], k.shape[3]
    group, page = n_q // n_kv, k.shape[1]
    worst = 0.0
    for r, n in enumerate(s["lens"]):
        at = s["table"][r, :-(-int(n) // page)]
        kr, vr = (c[at].reshape(-1, n_kv, hd)[:n] for c in (k, v))
        a, b = int(s["start"][r]), int(s["start"][r + 1])
        sees = n - (b - a) + 1 + np.arange(b - a)
        behind = np.arange(n)[None, :] >= sees[:, None]
        for h in range(n_q):
            x = s["q"][a:b, h].astype(np.float64) @ kr[:, h // group].T / np.sqrt(hd)
            x[behind] = -np.inf
            w = np.exp(x - x.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            vh = vr[:, h // group]
            worst = max(worst, (np.abs(got[a:b, h] - w @ vh) / (w @ np.abs(vh))).max())
    end = int(s["start"][-1])
    assert (got[end:] == 5.25).all()
    print("of sum w|v|: %.1f u" % (worst / U), flush=True)
    assert worst <= 64 * U


HEADS = [(24, 4, 256), (32, 8, 128), (16, 2, 64), (12, 3, 80)]


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n_q,n_kv,hd", HEADS)
def test_decode_rows(bh, dev, n_q, n_kv, hd, f16):
    rng = np.random.default_rng(hd)
    lens = [1, 2, 17, 64, 129, 700, 2049, 9001]
    s = _step(rng, dev, lens, [1] * len(lens), 16, n_q, n_kv, hd, f16, pad=2)
    _check_rows(bh, dev, s)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("new", [[8, 3, 5], [150, 1, 33], [200]])
@pytest.mark.parametrize("n_q,n_kv,hd", HEADS)
def test_drafts_and_prompts_rows(bh, dev, new, n_q, n_kv, hd, f16):
    rng = np.random.default_rng(hd + len(new))
    lens = [n + e for n, e in zip(new, (2500, 40, 0))]
    s = _step(rng, dev, lens, new, 48, n_q, n_kv, hd, f16, pad=1)
    _check_rows(bh, dev, s)
