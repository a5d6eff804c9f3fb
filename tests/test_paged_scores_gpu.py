"""Attention over pages where scores are large: the weights stay finite and what
they are known to be.

u = 2^-24.  Equal values v at n positions: the result is v, whatever the weights
are; numerator and denominator are sums of n terms of one sign, (n + 8) u each at
worst, and a weight against an f16 cache has 22 bits in its two halves (4 u)."""
from __future__ import annotations

import numpy as np
import pytest

from test_paged_gpu import _attend, _step

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n_q,n_kv,hd", [(24, 4, 256), (32, 8, 128), (8, 2, 64), (6, 2, 96)])
@pytest.mark.parametrize("new", [[1, 1], [3, 5], [40, 1]])
@pytest.mark.parametrize("offset", [1.4e7, -1.4e7, 3e7, 1e9])
def test_scores_far_from_zero(bh, dev, offset, new, n_q, n_kv, hd, f16):
    """All scores of a row near one large number, where neighbouring f32 are 1, 2, 64
    apart: the running maximum moves by whole steps, and no weight may pass the
    range of its type."""
    import torch
    rng = np.random.default_rng(int(abs(offset)) % 1000 + hd + sum(new))
    lens = [700, 130]
    s = _step(rng, dev, lens, new, 16, n_q, n_kv, hd, f16)
    # q.k / sqrt(hd) = offset + N(0, 3^2), but for the rounding
    s["q"] *= 3.0
    s["q"][:, :, 0] = offset * np.sqrt(hd) / 4096.0
    s["k"][..., 0] = 4096.0
    row = _row(rng, n_kv, hd)
    s["v"][:] = torch.from_numpy(row).to(dev).to(s["v"].dtype)
    got = _attend(bh, dev, s)[0]
    want = np.repeat(row, n_q // n_kv, 0)[None]
    tol = (2 * max(lens) + 24) * U
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol * np.abs(want)).all(), np.abs(got / want - 1).max()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n_q,n_kv,hd,new", [(24, 4, 256, 1), (24, 4, 256, 4), (32, 8, 128, 3),
                                             (8, 8, 64, 2)])
@pytest.mark.parametrize("offset", [1.4e7, -1.4e7])
def test_long_runs_far_from_zero(bh, dev, offset, n_q, n_kv, hd, new, f16):
    """The same where a few rows' positions are split among waves: enough of them that
    each takes many steps in a row."""
    import torch
    rng = np.random.default_rng(hd + new)
    lens = [int(n) for n in rng.integers(6000, 12000, 8)] + [int(n) for n in rng.integers(1, 900, 8)]
    s = _step(rng, dev, lens, [min(n, new) for n in lens], 32, n_q, n_kv, hd, f16)
    s["q"] *= 3.0
    s["q"][:, :, 0] = offset * np.sqrt(hd) / 4096.0
    s["k"][..., 0] = 4096.0
    row = _row(rng, n_kv, hd)
    s["v"][:] = torch.from_numpy(row).to(dev).to(s["v"].dtype)
    got = _attend(bh, dev, s)[0]
    want = np.repeat(row, n_q // n_kv, 0)[None]
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= (2 * max(lens) + 24) * U * np.abs(want)).all()


def _row(rng, n_kv, hd):
    """Values that both cache types hold exactly, none of them 0."""
    return (rng.integers(1, 64, (n_kv, hd)) * rng.choice([-1.0, 1.0], (n_kv, hd)) / 8).astype(
        np.float32)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n_q,n_kv,hd", [(12, 2, 256), (16, 2, 64), (3, 1, 16)])
@pytest.mark.parametrize("new", [1, 9, 80])
@pytest.mark.parametrize("size", [0, 16, 1024, 2 ** 14, 2 ** 18])
def test_known_distance(bh, dev, size, new, n_q, n_kv, hd, f16):
    """Scores that are exact: `size` + 1 at some positions, `size` at others, 0 - or
    50 less - elsewhere.  Powers of two make every product and sum exact, so that a
    weight is off by the score's f32 in base 2 alone: size * log2(e) rounded, and
    log2(e) itself, 1.3 u each of it, twice for two scores: a factor of
    (1 +- 4 u |size|), besides 64 u for exponentials and sums of n <= 300 terms."""
    import torch
    rng = np.random.default_rng(size % 97 + hd + new)
    n = 300
    s = _step(rng, dev, [n], [new], 16, n_q, n_kv, hd, f16)
    root = int(np.sqrt(hd))
    # scores: q0 k0 + q1 k1 with q0 = sqrt(hd) / 4 (k0 in quarters), q1 = sqrt(hd) 2^6
    score = np.where(rng.random(n) < 0.3, 1.0, 0.0)
    score[rng.random(n) < 0.3] = -50.0
    score[0] = 1.0
    s["q"][:] = 0.0
    s["q"][:, :, 0], s["q"][:, :, 1] = root / 4.0, root * 64.0
    k = np.zeros((n, n_kv, hd), np.float32)
    k[:, :, 0] = 4.0 * score[:, None]
    k[:, :, 1] = size / 64.0
    v = (rng.integers(-64, 65, (n, n_kv, hd)) / 8).astype(np.float32)
    for p in range(n):
        at = int(s["table"][0, p // 16]), p % 16
        s["k"][at] = torch.from_numpy(k[p]).to(dev).to(s["k"].dtype)
        s["v"][at] = torch.from_numpy(v[p]).to(dev).to(s["v"].dtype)
    got = _attend(bh, dev, s)[0]
    for t in range(new):
        sees = n - new + t + 1
        w = np.exp(score[:sees] - 1.0)
        w /= w.sum()
        for h in range(n_q):
            vh = v[:sees, h // (n_q // n_kv)].astype(np.float64)
            want = w @ vh
            tol = (4 * size + 64 + sees) * U * (w @ np.abs(vh - want) + w @ np.abs(vh))
            assert (np.abs(got[t, h] - want) <= tol).all(), (t, h)
