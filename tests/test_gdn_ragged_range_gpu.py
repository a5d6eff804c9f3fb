"""The delta rule of prompts whose values differ by many powers of ten: over the state's
rows, over the tokens, and between the state and what comes after it.

An output is held to the scale of what it is made of, |m| |q| / sqrt(s) of the state after
its token, a state to its own, row by row where rows differ, else the head's largest.
Tolerance: the recurrence rounds a state three times a token, at random 3 2^-24 sqrt(n),
and a dot of 128 12 times: 4e-6, 1e-5 as in test_gdn_ragged_gpu.py.  By chunks an operand
has besides an absolute error of up to 2^-39 of the largest of what shares its unit (half a
step of 2^-24 where that is 2^14 to 2^15).  A sum of 64 products of two such, of which the
outputs are at least 2^-18 of the largest that it could be, is then off by 8 sqrt(2) 2^-39 /
sqrt(3) 2^18 = 2.5e-6 at random, and the deltas, sums of their own, by as much again."""
from __future__ import annotations

import numpy as np
import pytest

from test_gdn_ragged_gpu import _case, _run, _views

pytestmark = pytest.mark.gpu

TOL = 1.5e-5


def _want(c):
    """attn, state of the slots written, |m| |q| / sqrt(s) of each (token, head, row)."""
    q, k, v = (x.astype(np.float64) for x in _views(c))
    gate, beta = c["gate"].astype(np.float64), c["beta"].astype(np.float64)
    h_v, s = c["h_v"], c["s"]
    head = np.arange(h_v) % c["h_k"]
    pool = c["pool"][:, :h_v * s * s].reshape(-1, h_v, s, s).astype(np.float64)
    attn, scale, states = np.zeros(v.shape), np.zeros(v.shape), {}
    for r in range(len(c["src"])):
        m = pool[c["src"][r]].copy() if c["src"][r] >= 0 else np.zeros(pool.shape[1:])
        for t in range(c["start"][r], c["start"][r + 1]):
            m *= np.exp(gate[t])[:, None, None]
            delta = (v[t] - (m @ k[t, head][:, :, None])[:, :, 0]) * beta[t][:, None]
            m += delta[:, :, None] * k[t, head][:, None, :]
            attn[t] = (m @ q[t, head][:, :, None])[:, :, 0] / np.sqrt(s)
            scale[t] = np.sqrt((m * m).sum(2) * (q[t, head] ** 2).sum(1)[:, None] / s)
        if c["start"][r + 1] > c["start"][r] and c["dst"][r] >= 0:
            states[int(c["dst"][r])] = m
    return attn, states, scale


def _check(bh, dev, c, by_row=False, **kw):
    attn, pool, _ = _run(bh, dev, c, **kw)
    want, states, scale = _want(c)
    n = int(c["start"][-1])
    if not by_row:
        scale = np.broadcast_to(scale.max(2, keepdims=True), scale.shape)
    off = np.abs(attn[:n] - want[:n])
    zero = scale[:n] == 0
    assert np.all(off[zero] == 0)
    worst = (off[~zero] / scale[:n][~zero]).max(initial=0)
    assert worst < TOL, worst
    h_v, s = c["h_v"], c["s"]
    for slot, m in states.items():
        got = pool[slot, :h_v * s * s].reshape(m.shape)
        size = np.abs(m).max(2 if by_row else (1, 2), keepdims=True)
        size = np.where(size == 0, 1, size)  # (nothing but 0 is then near it)
        worst = (np.abs(got - m) / size).max()
        assert worst < TOL, (slot, worst)
    return attn, pool


def _v(c):
    h_k, h_v, s = c["h_k"], c["h_v"], c["s"]
    return c["rows"][:, 2 * h_k * s:(2 * h_k + h_v) * s].reshape(len(c["rows"]), h_v, s)


def _parts(c):
    c = {k: v.copy() if isinstance(v, np.ndarray) else v for k, v in c.items()}
    return c, c["pool"].reshape(len(c["pool"]), c["h_v"], c["s"], c["s"])


def _set_v(c, v):
    h_k, h_v, s = c["h_k"], c["h_v"], c["s"]
    c["rows"][:, 2 * h_k * s:(2 * h_k + h_v) * s] = v.reshape(len(v), -1)


@pytest.mark.parametrize("s", [128, 64])
@pytest.mark.parametrize("fresh", [[], [0]])
@pytest.mark.parametrize("what", ["three large", "three small", "each"])
def test_rows_of_any_scale(bh, dev, s, fresh, what):
    """A state row's results have the precision of that row's own values."""
    c, pool = _parts(_case([150, 2, 64], 1, 2, s, decay=-0.05, fresh=fresh))
    by = np.ones(s, np.float32)
    if what == "each":
        by[:] = np.float32(10.0) ** np.random.default_rng(s).permutation(np.linspace(-9, 9, s))
    else:
        by[[0, 1, s - 3]] = 1e5 if what == "three large" else 1e-7
    _set_v(c, _v(c) * by)
    pool *= by[:, None]
    _check(bh, dev, c, by_row=True)


@pytest.mark.parametrize("s", [128, 64])
@pytest.mark.parametrize("size", [1e3, 1e6, 1e9, 1e30])
@pytest.mark.parametrize("row", [None, 3])
def test_a_large_value_reaches_no_earlier_token(bh, dev, s, size, row):
    for fresh in ([], [1]):
        c, _ = _parts(_case([3, 200, 70], 2, 4, s, fresh=fresh))
        v = _v(c).copy()
        at = 3 + 100  # in the second chunk of the second request, v-head 1
        v[at, 1, slice(None) if row is None else row] *= np.float32(size)
        clean, _, _ = _run(bh, dev, c)
        _set_v(c, v)
        attn, _ = _check(bh, dev, c)
        others = np.ones(attn.shape, bool)
        others[at:203, 1] = False
        assert np.abs(attn - clean)[others].max() <= 2 * TOL * np.abs(clean[others]).max()
        others[3:203, 1] = False
        assert np.array_equal(attn[others], clean[others])


@pytest.mark.parametrize("s", [128, 64])
@pytest.mark.parametrize("new", [[64], [150], [50, 100]])
@pytest.mark.parametrize("size", [1e3, 1e6, 1e9])
@pytest.mark.parametrize("what", ["state", "first values", "state, no q"])
def test_what_decays_leaves_no_error(bh, dev, s, new, size, what):
    c, pool = _parts(_case(new, 1, 2, s, decay=-2.0 if what.startswith("state") else -1.0))
    if what.startswith("state"):
        pool *= np.float32(size)
        if what != "state":
            c["rows"][:, :s] = 0
    else:
        v = _v(c).copy()
        for a in c["start"][:-1]:
            v[a:a + 20] *= np.float32(size)
        _set_v(c, v)
    _check(bh, dev, c)


@pytest.mark.parametrize("s", [128, 64])
@pytest.mark.parametrize("beta", [0.0, 1e-3, 1e-6, 1e-9, 1e-20])
@pytest.mark.parametrize("fresh", [[], [0]])
def test_small_steps_before_large_ones(bh, dev, s, beta, fresh):
    c, _ = _parts(_case([200, 70], 1, 2, s, fresh=fresh))
    c["beta"][:100] = beta
    c["beta"][100:, 1] = 1.0
    _check(bh, dev, c)


@pytest.mark.parametrize("s", [128, 64])
def test_nothing_at_first(bh, dev, s):
    """Values, keys and queries of exactly 0, of some tokens and of all."""
    for what in range(4):
        c, _ = _parts(_case([100, 64], 1, 2, s, fresh=[0]))
        v = _v(c).copy()
        if what == 0:
            v[:10] = 0
        elif what == 1:
            v[:] = 0
        elif what == 2:
            c["rows"][20:50, s:2 * s] = 0
        else:
            c["rows"][20:50, :s] = 0
        _set_v(c, v)
        _check(bh, dev, c)


@pytest.mark.parametrize("s", [128, 64])
def test_a_chunk_that_grows_among_others(bh, dev, s):
    """Gates above 0 in one chunk of four, values far apart in another."""
    c, _ = _parts(_case([256, 130], 2, 4, s))
    c["gate"][70:75, 1] = 0.3
    v = _v(c).copy()
    v[150, 2] *= np.float32(1e8)
    v[256 + 65, 0] *= np.float32(1e8)
    _set_v(c, v)
    _check(bh, dev, c)
    _check(bh, dev, c, max_new=256)


def test_wide_ranges_of_the_models_heads(bh, dev):
    """Requests in halves of heads and in whole ones, with values far apart in some chunks."""
    for new in ([200], [70, 130, 300], [60] * 8):
        c, _ = _parts(_case(new, 16, 48, 128))
        v = _v(c).copy()
        rng = np.random.default_rng(len(new))
        for _ in range(40):
            v[rng.integers(0, len(v)), rng.integers(0, 48)] *= np.float32(10.0 ** rng.uniform(4, 12))
        _set_v(c, v)
        _check(bh, dev, c)
