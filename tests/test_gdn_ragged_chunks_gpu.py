"""The delta rule of many requests where prompts go by chunks: about the length from
which they do, and each way the chunks' blocks are shared out (a head's state rows in one
block or in two, by how many prompts there are).

Tolerance as in test_gdn_ragged_gpu.py, 1e-5 of the largest value: an operand of a
chunk's products keeps 22 bits of each value, 2^-23 of it, where a token by token sum
rounds to 2^-24, and a chunk's 64 tokens are one sum of products in f32 instead of 64
roundings of the state."""
from __future__ import annotations

import numpy as np
import pytest

from test_gdn_ragged_gpu import _case, _check, _run, _t

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [[47], [48], [49], [63, 48], [64, 47, 65], [95, 1, 96, 0, 97],
                                 [48, 31, 32, 33, 111]])
def test_lengths_from_which_chunks_begin(bh, dev, new):
    for h_k, h_v in ((1, 3), (2, 2)):
        print(new, h_k, h_v, flush=True)
        _check(bh, dev, _case(new, h_k, h_v, 128, fresh=[0]))
        _check(bh, dev, _case(new, h_k, h_v, 128, seed=1, inplace=True, drop=[0]),
               max_new=max(new))


# of 256 compute units: all heads in two blocks, the longest's, none
@pytest.mark.parametrize("new", [[70], [1, 200, 90], [50, 130, 64], [66, 60, 100, 129], [50] * 6])
def test_shares_of_the_models_heads(bh, dev, new):
    _check(bh, dev, _case(new, 16, 48, 128, fresh=[len(new) - 1]))


@pytest.mark.parametrize("reqs", [63, 64, 65, 100, 300])
def test_many_prompts(bh, dev, reqs):
    """More prompts than a wave has lanes, and lengths that are alike."""
    rng = np.random.default_rng(reqs)
    new = 48 + 20 * rng.integers(0, 3, reqs)
    new[rng.integers(0, reqs, reqs // 4)] = 3
    _check(bh, dev, _case(list(new), 1, 1, 128))


def test_workspace_of_ones_own(bh, dev):
    """The same bits in the library's scratch, in a workspace, in one with a garbage past
    and at any hint that lets prompts go by chunks."""
    import torch
    c = _case([60, 1, 200, 7], 2, 6, 128)
    attn, pool, args = _run(bh, dev, c)
    need = bh.gdn_ragged_workspace(args)
    assert need > 0
    for fill in (0, 255):
        ws = torch.full((need,), fill, dtype=torch.uint8, device=dev)
        got, got_pool, _ = _run(bh, dev, c, workspace=ws, max_new=200)
        assert np.array_equal(attn, got) and np.array_equal(pool, got_pool)
    small = torch.empty(need - 4, dtype=torch.uint8, device=dev)
    with pytest.raises(bh.BonsaiError, match="workspace"):
        _run(bh, dev, c, workspace=small)


def test_two_streams_with_workspaces(bh, dev):
    """Calls on two streams at once, a workspace each, are each other's no concern."""
    import torch
    cases = [_case([300, 1, 64], 2, 6, 128, seed=i) for i in range(2)]
    want, runs = [], []
    for c in cases:
        want.append(_run(bh, dev, c)[:2])
        h_k, h_v, s = c["h_k"], c["h_v"], c["s"]
        rows, pool = _t(c["rows"], dev), _t(c["pool"], dev)
        q, k, v = (rows[:, i:j].unflatten(1, (-1, s)) for i, j in (
            (0, h_k * s), (h_k * s, 2 * h_k * s), (2 * h_k * s, (2 * h_k + h_v) * s)))
        fixed = [_t(c[n], dev) for n in ("gate", "beta", "start", "src", "dst")]

        def make(ws=None):
            return bh.make_gdn_ragged_args(q, k, v, *fixed[:2], pool.unflatten(1, (h_v, s, s)),
                                           *fixed[2:], attn=attn, workspace=ws)
        attn = torch.full((len(rows), h_v, s), -7.0, device=dev)
        ws = torch.empty(bh.gdn_ragged_workspace(make()), dtype=torch.uint8, device=dev)
        runs.append((make(ws), torch.cuda.Stream(), attn, pool))
    torch.cuda.synchronize()
    for _ in range(3):  # (the slots read are not those written)
        for args, st, _, _ in runs:
            bh.gdn_ragged(args, stream=st)
    torch.cuda.synchronize()
    for (attn, pool), (_, _, got, got_pool) in zip(want, runs):
        assert np.array_equal(attn, got.cpu().numpy())
        assert np.array_equal(pool, got_pool.cpu().numpy())


def test_captured_and_replayed_with_other_lengths(bh, dev):
    """One graph over steps of other lengths and slots; the eager call's bits."""
    import torch
    n_tok, h_k, h_v, s = 320, 2, 6, 128
    c = _case([n_tok - 2], h_k, h_v, s)
    rows, pool = _t(c["rows"], dev), _t(np.repeat(c["pool"][:1], 9, 0), dev)
    q, k, v = (rows[:, i:j].unflatten(1, (-1, s)) for i, j in (
        (0, 256), (256, 512), (512, 512 + 6 * s)))
    gate, beta = _t(c["gate"], dev), _t(c["beta"], dev)
    start, src, dst = (torch.zeros(n, dtype=torch.int32, device=dev) for n in (5, 4, 4))
    attn = torch.empty((n_tok, h_v, s), device=dev)

    def make(pool, attn, ws=None):
        return bh.make_gdn_ragged_args(q, k, v, gate, beta, pool.unflatten(1, (h_v, s, s)), start,
                                       src, dst, attn=attn, workspace=ws)
    ws = torch.empty(bh.gdn_ragged_workspace(make(pool, attn)), dtype=torch.uint8, device=dev)
    st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        bh.gdn_ragged(make(pool, attn, ws), stream=st)
    other, other_attn = pool.clone(), attn.clone()
    for new in ([1, 1, 1, 1], [300, 0, 1, 2], [47, 48, 64, 100], [0, 0, 0, 0], [9, 200, 1, 50]):
        start.copy_(torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32))
        order = torch.randperm(9, generator=torch.Generator().manual_seed(sum(new)))
        src.copy_(order[:4].int())
        dst.copy_(order[4:8].int())
        attn.fill_(-7.0)
        other_attn.fill_(-7.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        bh.gdn_ragged(make(other, other_attn))
        torch.cuda.synchronize()
        assert torch.equal(attn, other_attn) and torch.equal(pool, other), new


@pytest.mark.parametrize("what", ["v", "k", "q", "gate", "beta", "inf v", "inf k", "state"])
def test_a_value_that_is_not_finite_reaches_no_earlier_token(bh, dev, what):
    """As the recurrence has it: outputs of the tokens before are as without it, those
    after are not finite where the formula's are not."""
    import batchdata as bd
    from test_gdn_ragged_gpu import _views
    from conftest import rel_err
    c = _case([3, 200, 70], 2, 4, 128)
    at = 3 + 100  # in the second chunk of the second request
    bad = np.inf if what.startswith("inf") else np.nan
    for name in ("rows", "gate", "beta", "pool"):
        c[name] = c[name].copy()
    if what.endswith("v"):
        c["rows"][at, 4 * 128 + 128 + 9] = bad  # v-head 1, row 9
    elif what.endswith("k"):
        c["rows"][at, 2 * 128 + 17] = bad
    elif what == "q":
        c["rows"][at, 17] = bad
    elif what == "state":
        c["pool"][c["src"][1], 5 * 128 + 3] = bad  # v-head 0, row 5
    else:
        c[what][at, 1] = bad
    q, k, v = _views(c)
    with np.errstate(all="ignore"):
        want, state = bd.gdn(q, k, v, c["gate"], c["beta"], c["pool"].reshape(-1, 4, 128, 128),
                             c["start"], c["src"], c["dst"], np.full(v.shape, -7.0))
    for kw in ({}, dict(max_new=1)):  # by chunks and token by token
        attn, pool, _ = _run(bh, dev, c, **kw)
        for got, ref in ((attn, want), (pool.reshape(state.shape)[c["dst"]], state[c["dst"]])):
            fine = np.isfinite(ref)  # (q reaches no state)
            assert fine.any() and (what == "q" or not fine.all()), what
            assert np.array_equal(np.isfinite(got), fine), what
            assert rel_err(got[fine], ref[fine]) < 1e-5, what


@pytest.mark.parametrize("gate", [0.02, 0.5, 3.0])
def test_states_that_grow(bh, dev, gate):
    """Gates above 0, to where a state passes what f32 holds."""
    c = _case([130, 1, 60], 1, 2, 128, decay=gate)
    if gate < 3:
        c["beta"] *= 0.1
        _check(bh, dev, c, tol=1e-5)
    else:
        with np.errstate(all="ignore"):
            attn, pool, _ = _run(bh, dev, c)
        assert np.isfinite(attn[:20]).all() and not np.isfinite(attn[129]).any()


@pytest.mark.parametrize("new", [[47], [48, 1], [63, 64, 65], [130, 0, 3, 257], [50] * 70])
@pytest.mark.parametrize("h_k,h_v", [(1, 3), (8, 16), (3, 2)])
def test_heads_of_64(bh, dev, new, h_k, h_v):
    print(new[:4], h_k, h_v, flush=True)
    _check(bh, dev, _case(new, h_k, h_v, 64, fresh=[0]))
    _check(bh, dev, _case(new, h_k, h_v, 64, seed=1, inplace=True, slot_pad=4), max_new=max(new))


@pytest.mark.parametrize("decay", [0.0, -30.0, -np.inf, -0.3])
def test_heads_of_64_with_hard_decays(bh, dev, decay):
    _check(bh, dev, _case([200, 1, 140], 1, 2, 64, decay=decay, alike=0.9, beta_one=True))
