"""Each row of attention over pages stands for itself: what a query does not see, and
what the queries and heads beside it hold, changes no bit of its result."""
from __future__ import annotations

import numpy as np
import pytest

from test_paged_gpu import _attend, _step, _t

pytestmark = pytest.mark.gpu

HEADS = [(24, 4, 256), (32, 8, 128), (8, 2, 64), (6, 2, 96)]
NEW = [[1, 1, 1], [5, 3, 1], [90, 1, 40]]


def _bits(x):
    return x.view(np.uint32)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n_q,n_kv,hd", HEADS)
@pytest.mark.parametrize("new", NEW)
def test_other_queries_change_nothing(bh, dev, new, n_q, n_kv, hd, f16):
    """Rows of one tile share a wave's running maxima: one of them that grows, or is
    not finite, leaves the others as they are."""
    rng = np.random.default_rng(hd)
    s = _step(rng, dev, [700, 60, 2333], new, 16, n_q, n_kv, hd, f16)
    clean = _attend(bh, dev, s)[0]
    q = s["q"]
    other = rng.random(clean.shape[:2]) < 0.2
    for value in (None, np.nan, np.inf, -np.inf):
        s["q"] = q.copy()
        s["q"][other] = s["q"][other] * 4.0 if value is None else value
        got = _attend(bh, dev, s)[0]
        assert np.array_equal(_bits(got[~other]), _bits(clean[~other])), value
        assert value is None or np.isnan(got[other]).all()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n_q,n_kv,hd", HEADS)
@pytest.mark.parametrize("new", [3, 16, 90])
def test_later_keys_change_nothing(bh, dev, new, n_q, n_kv, hd, f16):
    """The rows of the last new tokens, which the ones before do not see, as large
    numbers: the last queries' maxima jump at the end."""
    rng = np.random.default_rng(hd + new)
    n, hide = 1500, 2
    s = _step(rng, dev, [n], [new], 16, n_q, n_kv, hd, f16)
    clean = _attend(bh, dev, s)[0]
    for p in range(n - hide, n):
        at = int(s["table"][0, p // 16]), p % 16
        s["k"][at] = _t(rng.standard_normal((n_kv, hd)).astype(np.float32) * 30, dev)
        s["v"][at] = _t(rng.standard_normal((n_kv, hd)).astype(np.float32) * 30, dev)
    got = _attend(bh, dev, s)[0]
    assert np.array_equal(_bits(got[:new - hide]), _bits(clean[:new - hide]))
    assert np.isfinite(got).all() and (got[new - hide:] != clean[new - hide:]).any()
