"""The gated delta rule of many requests at once against 64 bits.

Tolerance, relative to the largest value, 1e-5 as bh_gdn_step is held to: with u =
2^-24 a token adds about 3 u |m| to a row (decay, delta, sum), at random, and decays
never enlarge it: 3 u sqrt(n) = 4e-6 after 500 tokens; a dot of 128 adds (8 + 4) u of
its terms."""
from __future__ import annotations

import numpy as np
import pytest

import batchdata as bd
from conftest import rel_err

pytestmark = pytest.mark.gpu

TOL = 1e-5


def _t(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def _case(new, h_k, h_v, s, seed=0, inplace=False, fresh=(), drop=(), rows_pad=0, slot_pad=0,
          decay=None, alike=0.0, beta_one=False):
    rng = np.random.default_rng(seed + 1000 * len(new) + h_v + s)
    n, reqs = int(np.sum(new)) + 2, len(new)
    rows = rng.standard_normal((n, (2 * h_k + h_v) * s + rows_pad)).astype(np.float32)
    for part in range(2 * h_k):
        x = rows[:, part * s:(part + 1) * s]
        if part >= h_k and alike:
            x[:] = alike * rng.standard_normal(s) + (1 - alike) * x
        x /= np.sqrt((x * x).sum(1, keepdims=True))
    gate = -np.exp(rng.uniform(-6.5, 0.5, (n, h_v))).astype(np.float32)
    if decay is not None:
        gate[:] = decay
    beta = (1 / (1 + np.exp(-rng.standard_normal((n, h_v))))).astype(np.float32)
    if beta_one:
        beta[:] = 1.0
    n_slots = 2 * reqs + 1
    pool = (0.3 * rng.standard_normal((n_slots, h_v * s * s + slot_pad))).astype(np.float32)
    order = rng.permutation(n_slots).astype(np.int32)
    src, dst = order[:reqs].copy(), order[reqs:2 * reqs].copy()
    if inplace:
        dst = src.copy()
    src[list(fresh)] = -1
    dst[list(drop)] = -1
    return dict(rows=rows, gate=gate, beta=beta, pool=pool, start=bd.offsets(new), src=src,
                dst=dst, h_k=h_k, h_v=h_v, s=s)


def _views(c):
    n, a, b, s = len(c["rows"]), c["h_k"] * c["s"], c["h_v"] * c["s"], c["s"]
    r = c["rows"]
    return (r[:, :a].reshape(n, -1, s), r[:, a:2 * a].reshape(n, -1, s),
            r[:, 2 * a:2 * a + b].reshape(n, -1, s))


def _run(bh, dev, c, again=0, **kw):
    import torch
    h_k, h_v, s = c["h_k"], c["h_v"], c["s"]
    n, a, b = len(c["rows"]), h_k * s, h_v * s
    rows, pool = _t(c["rows"], dev), _t(c["pool"], dev)
    q, k, v = (rows[:, i:j].unflatten(1, (-1, s)) for i, j in ((0, a), (a, 2 * a),
                                                               (2 * a, 2 * a + b)))
    state = pool[:, :h_v * s * s].unflatten(1, (h_v, s, s))
    attn = torch.full((n, h_v, s), -7.0, device=dev)
    args = bh.make_gdn_ragged_args(q, k, v, _t(c["gate"], dev), _t(c["beta"], dev), state,
                                   _t(c["start"], dev), _t(c["src"], dev), _t(c["dst"], dev),
                                   attn=attn, **kw)
    bh.gdn_ragged(args)
    torch.cuda.synchronize()
    return attn.cpu().numpy(), pool.cpu().numpy(), args


def _check(bh, dev, c, tol=TOL, **kw):
    h_v, s = c["h_v"], c["s"]
    m = h_v * s * s
    q, k, v = _views(c)
    want, state = bd.gdn(q, k, v, c["gate"], c["beta"], c["pool"][:, :m].reshape(-1, h_v, s, s),
                         c["start"], c["src"], c["dst"],
                         np.full((len(q), h_v, s), -7.0))
    attn, pool, _ = _run(bh, dev, c, **kw)
    n = int(c["start"][-1])
    assert np.all(attn[n:] == -7.0)
    if n:
        assert rel_err(attn[:n], want[:n]) < tol
    got = pool[:, :m].reshape(state.shape)
    written = {int(d) for d, a, b in zip(c["dst"], c["start"], c["start"][1:])
               if 0 <= d < len(pool) and b > a}
    for i in range(len(pool)):
        if i in written:
            assert rel_err(got[i], state[i]) < tol, i
        else:  # bit for bit
            assert np.array_equal(pool[i], c["pool"][i]), i
    assert np.array_equal(pool[:, m:], c["pool"][:, m:])


HEADS = [(2, 6, 128), (1, 1, 128), (2, 3, 128), (2, 4, 64), (3, 3, 64), (2, 2, 32), (1, 2, 80),
         (1, 1, 7), (1, 1, 256)]


@pytest.mark.parametrize("h_k,h_v,s", HEADS)
@pytest.mark.parametrize("inplace", [False, True])
def test_gdn_ragged_matches(bh, dev, h_k, h_v, s, inplace):
    for new in ([1], [1, 1, 1, 1], [0, 2, 1, 0, 5, 33], [64], [63, 1, 65]):
        print(h_k, h_v, s, new, flush=True)
        _check(bh, dev, _case(new, h_k, h_v, s, inplace=inplace))
        _check(bh, dev, _case(new, h_k, h_v, s, seed=1, inplace=inplace, fresh=[0],
                              drop=[len(new) - 1]), max_new=max(new))


@pytest.mark.parametrize("new", [[127], [128], [129], [191, 1], [192, 0, 1, 193], [130, 131, 2, 256],
                                 [300, 1, 1, 128, 64]])
@pytest.mark.parametrize("s", [128, 64])
def test_gdn_ragged_prompts(bh, dev, new, s):
    for h_k, h_v in ((1, 3), (2, 2)):
        print(new, h_k, h_v, flush=True)
        _check(bh, dev, _case(new, h_k, h_v, s, fresh=[0]))
        _check(bh, dev, _case(new, h_k, h_v, s, seed=1, inplace=True), max_new=max(new))
    # a hint that is too low costs time only
    _check(bh, dev, _case(new, 1, 2, s, seed=2), max_new=1)


@pytest.mark.parametrize("kw", [dict(decay=0.0, alike=0.95, beta_one=True), dict(decay=-30.0),
                                dict(decay=-np.inf), dict(decay=-1e-4, alike=0.5),
                                dict(decay=-3.0, beta_one=True)])
def test_gdn_ragged_hard_prompts(bh, dev, kw):
    """Keys nearly alike with whole steps and no decay, decays that underflow."""
    _check(bh, dev, _case([200, 1, 140], 1, 2, 128, **kw))


def test_gdn_ragged_scales(bh, dev):
    """States and values of any size: large, tiny, and both in one state."""
    for size, rows in ((1e6, None), (1e-12, None), (1e5, 3)):
        c = _case([150, 2], 1, 2, 128, decay=-0.05)
        v = c["rows"][:, 256:]
        if rows is None:
            v *= size
            c["pool"] *= size
        else:  # a few rows far larger than the others
            v[:, :rows] *= size
        _check(bh, dev, c)


@pytest.mark.parametrize("rows_pad,slot_pad", [(4, 0), (1, 0), (0, 4), (0, 3)])
def test_gdn_ragged_strides(bh, dev, rows_pad, slot_pad):
    _check(bh, dev, _case([1, 140, 3], 1, 2, 128, rows_pad=rows_pad, slot_pad=slot_pad))


@pytest.mark.parametrize("n_req", [65, 300])
def test_gdn_ragged_many_requests(bh, dev, n_req):
    rng = np.random.default_rng(n_req)
    new = rng.integers(0, 3, n_req)
    new[[7, n_req - 1]] = 150, 129
    _check(bh, dev, _case(list(new), 1, 1, 128, inplace=True))
    _check(bh, dev, _case([1] * n_req, 1, 2, 64))


def test_gdn_ragged_model_heads(bh, dev):
    _check(bh, dev, _case([1] * 6, 16, 48, 128, inplace=True), max_new=1)
    _check(bh, dev, _case([1, 130, 2], 16, 48, 128))


def test_gdn_ragged_bad_slots_and_offsets(bh, dev):
    import torch
    c = _case([2, 3, 1], 1, 2, 128)
    c["src"], c["dst"] = np.array([1, 99, 2], np.int32), np.array([70, 3, -2 ** 31], np.int32)
    bad = torch.full((1,), -1, dtype=torch.int32, device=dev)
    _check(bh, dev, c, bad_slot=bad)
    assert bad.item() in (99, 70)
    for new in ([2, 3, 1], [2, 200, 140]):
        n = sum(new)
        for start in ([0, 2, 2 ** 30, n], [0, n, 2, n], [-5, 2, 5, n], [3, 3, 3, 6]):
            c = _case(new, 1, 2, 128)
            c["start"] = np.array(start, np.int32)
            attn, pool, _ = _run(bh, dev, c)
            assert attn.shape == (n + 2, 2, 128)


def test_gdn_ragged_matches_one_sequence(bh, dev):
    """What bh_gdn_step gives for each request by itself."""
    import torch
    c = _case([5, 1, 150], 2, 6, 128)
    attn, pool, _ = _run(bh, dev, c)
    q, k, v = _views(c)
    for r in range(3):
        a, b = c["start"][r], c["start"][r + 1]
        st = _t(c["pool"][c["src"][r]].reshape(6, 128, 128), dev)
        one = bh.gdn_step(*(_t(x[a:b], dev) for x in (q, k, v, c["gate"], c["beta"])), st)
        torch.cuda.synchronize()
        assert rel_err(attn[a:b], one.cpu().numpy()) < 2 * TOL
        assert rel_err(pool[c["dst"][r]], st.cpu().numpy().reshape(-1)) < 2 * TOL


def test_gdn_ragged_nan_stays_in_its_request(bh, dev):
    for new in ([2, 3, 1], [140, 150, 1]):
        c = _case(new, 1, 2, 128)
        clean, clean_pool, _ = _run(bh, dev, c)
        c["rows"] = c["rows"].copy()
        c["rows"][new[0], 130] = np.nan  # of a key of the second request
        attn, pool, _ = _run(bh, dev, c)
        a, b = c["start"][1], c["start"][2]
        assert np.isnan(attn[b - 1]).all()
        keep = np.r_[0:a, b:len(attn)]
        assert np.array_equal(attn[keep], clean[keep])
        for i in range(len(pool)):
            if i != c["dst"][1]:
                assert np.array_equal(pool[i], clean_pool[i])


def test_gdn_ragged_chunk_is_its_tokens(bh, dev):
    """A chunk of tokens equals its tokens one by one, state by state."""
    new = [140, 131]
    c = _case(new, 1, 2, 128, inplace=True)
    attn, pool, _ = _run(bh, dev, c)
    import torch
    h_v, s = 2, 128
    rows, p = _t(c["rows"], dev), _t(c["pool"], dev)
    q, k, v = rows[:, :128].unflatten(1, (1, s)), rows[:, 128:256].unflatten(1, (1, s)), \
        rows[:, 256:].unflatten(1, (2, s))
    state = p.unflatten(1, (h_v, s, s))
    out = torch.zeros((len(rows), h_v, s), device=dev)
    gate, beta, slots = _t(c["gate"], dev), _t(c["beta"], dev), _t(c["src"], dev)
    one = _t(np.array([0, 1, 2], np.int32), dev)
    for t in range(131):
        at = torch.tensor([t, 140 + t], device=dev)
        args = bh.make_gdn_ragged_args(q[at], k[at], v[at], gate[at], beta[at], state, one, slots,
                                       slots, max_new=1)
        out[at] = bh.gdn_ragged(args)
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    both = np.r_[0:131, 140:271]
    assert rel_err(attn[both], got[both]) < 2 * TOL
    assert rel_err(pool[c["dst"][1]], p.cpu().numpy()[c["dst"][1]]) < 2 * TOL
