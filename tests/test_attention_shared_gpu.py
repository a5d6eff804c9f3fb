"""Attention of requests that share a prefix: against 64 bits (test_paged_gpu's
tolerance, whose argument holds: one more join of two sums adds a rounding), and
against bh_attention_paged on the same arguments."""
from __future__ import annotations

import numpy as np
import pytest

import pageddata as pd
from conftest import rel_err

pytestmark = pytest.mark.gpu

TOL = 1e-5


def _t(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def _case(groups, *, page=16, n_head=4, n_kv=2, hd=64, f16=True, by_head=False, seed=0,
          same_pages=True, spare_tokens=2, own_width=None):
    """groups: a list of (shared positions, [(own positions, new tokens) ...]); the
    shared ones are whole pages, or the pages are the requests' own copies."""
    rng = np.random.default_rng(seed + 17 * hd + sum(g[0] for g in groups))
    lens, new, shared, start, group = [], [], [], [0], []
    for g, (s, reqs) in enumerate(groups):
        shared.append(s)
        start.append(start[-1] + len(reqs))
        for own, n in reqs:
            lens.append(s + own), new.append(n), group.append(g)
    have = [-(-n // page) for n in lens]
    width = max(have + [1]) + 1
    n_pages = sum(have) + 3
    order = rng.permutation(n_pages).astype(np.int32)
    table, at = np.full((len(lens), width), -1, np.int32), 0
    for r, h in enumerate(have):
        table[r, :h] = order[at:at + h]
        at += h
    dt = np.float16 if f16 else np.float32
    k, v = (rng.standard_normal((n_pages, page, n_kv, hd)).astype(dt) for _ in range(2))
    for g, (s, reqs) in enumerate(groups):
        first = start[g]
        for r in range(first + 1, first + len(reqs)):
            full = s // page
            if same_pages:
                table[r, :full] = table[first, :full]
            for b in range(full if same_pages else 0, -(-s // page)):
                n = min(page, s - b * page)
                k[table[r, b], :n] = k[table[first, b], :n]
                v[table[r, b], :n] = v[table[first, b], :n]
    q_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    n_tok = int(q_start[-1]) + spare_tokens
    q = rng.standard_normal((n_tok, n_head, hd)).astype(np.float32)
    return dict(q=q, k=k, v=v, table=table, q_start=q_start, kv_len=np.array(lens, np.int32),
                group=np.array(group, np.int32), group_start=np.array(start, np.int32),
                shared=np.array(shared, np.int32), by_head=by_head)


def _cache(bh, dev, c):
    k, v = (_t(c[n].transpose(0, 2, 1, 3), dev).transpose(1, 2) if c["by_head"] else _t(c[n], dev)
            for n in ("k", "v"))
    return bh.make_paged_cache(k, v)


def _args(bh, dev, c, cache=None, **kw):
    import torch
    q = _t(c["q"], dev)
    out = torch.full_like(q, -7.0)
    return bh.make_attention_shared_args(
        _cache(bh, dev, c) if cache is None else cache, q, _t(c["q_start"], dev),
        _t(c["kv_len"], dev), _t(c["table"], dev), _t(c["group"], dev), _t(c["group_start"], dev),
        _t(c["shared"], dev), out=out, **kw)


def _run(bh, dev, c, **kw):
    import torch
    out = bh.attention_shared(_args(bh, dev, c, **kw))
    torch.cuda.synchronize()
    return out.cpu().numpy()


def _paged(bh, dev, c, **kw):
    import torch
    q = _t(c["q"], dev)
    a = bh.make_attention_paged_args(_cache(bh, dev, c), q, _t(c["q_start"], dev),
                                     _t(c["kv_len"], dev), _t(c["table"], dev),
                                     out=torch.full_like(q, -7.0), **kw)
    out = bh.attention_paged(a)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def _want(c):
    out = np.full(c["q"].shape, -7.0)
    return pd.attention(c["q"], c["k"], c["v"], c["q_start"], c["kv_len"], c["table"], out)


def _check(bh, dev, c, **kw):
    got, want = _run(bh, dev, c, **kw), _want(c)
    n = int(c["q_start"][-1])
    assert np.all(got[n:] == -7.0)
    assert rel_err(got[:n], want[:n]) < TOL
    for r in range(len(c["kv_len"])):  # of each request by itself too
        a, b = c["q_start"][r], c["q_start"][r + 1]
        if b > a:
            assert rel_err(got[a:b], want[a:b]) < TOL, r
    return got


BEAMS = [(64, [(5, 1)] * 4), (200, [(1, 1), (30, 1), (64, 1)])]
HEADS = [(4, 2, 64), (24, 4, 256), (8, 2, 128), (3, 1, 64), (8, 8, 128), (4, 4, 256), (32, 1, 64)]


@pytest.mark.parametrize("n_head,n_kv,hd", HEADS)
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("same", [True, False])
def test_shared_beams(bh, dev, n_head, n_kv, hd, f16, same):
    c = _case(BEAMS, n_head=n_head, n_kv=n_kv, hd=hd, f16=f16, same_pages=same, by_head=same)
    print(n_head, n_kv, hd, f16, flush=True)
    _check(bh, dev, c)
    _check(bh, dev, c, max_new=1, max_group_new=4)
    _check(bh, dev, c, max_new=1, max_group_new=1)  # a hint that is too low


@pytest.mark.parametrize("page", [1, 7, 16, 48, 64])
@pytest.mark.parametrize("f16", [True, False])
def test_shared_lengths(bh, dev, page, f16):
    for groups in (
            [(0, [(1, 1)])], [(1, [(1, 1)])], [(1, [(1, 1), (2, 2)])], [(15, [(1, 1)] * 3)],
            [(33, [(3, 2), (1, 1)]), (0, [(9, 4)]), (128, [(40, 3), (2, 1), (1, 0)])],
            [(1000, [(1, 1)] * 2 + [(130, 5)])], [(257, [(64, 1)] * 9), (64, [(65, 1)])]):
        print(page, groups, flush=True)
        _check(bh, dev, _case(groups, page=page, f16=f16, same_pages=page != 7))
        _check(bh, dev, _case(groups, page=page, f16=f16, same_pages=page != 7, hd=256),
               max_new=5, max_group_new=9)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_shared_many_rows(bh, dev, f16, hd):
    """Groups of more than 64 rows a kv head; prompts behind a prefix; both beside
    decoders of their own."""
    for groups in ([(400, [(3, 1)] * 40)], [(300, [(70, 70), (1, 1), (33, 33)])],
                   [(96, [(20, 1)] * 20), (0, [(50, 1)]), (130, [(200, 150), (4, 1)])]):
        print(hd, f16, groups[0][0], flush=True)
        _check(bh, dev, _case(groups, n_head=8, n_kv=2, hd=hd, f16=f16))


def test_shared_long(bh, dev):
    """A long prefix in hundreds of parts."""
    c = _case([(9000, [(100, 1)] * 3)], n_head=6, n_kv=1, hd=128)
    got = _check(bh, dev, c, max_new=1, max_group_new=3)
    assert rel_err(got, _paged(bh, dev, c, max_new=1)) < 2 * TOL


def test_shared_is_only_a_hint(bh, dev):
    """What does not fit a group is by itself: results are bh_attention_paged's."""
    base = _case([(64, [(5, 2), (7, 1)]), (48, [(9, 1)] * 3)], same_pages=True)
    n = int(base["q_start"][-1])
    for name, change in (
            ("no group", dict(group=[-1, 5, 0, 1, 1])),
            ("not among its group", dict(group=[1, 0, 0, 0, 1])),
            ("shorter than the prefix", dict(kv_len=[66, 64, 57, 48, 57])),
            ("half of it shared", dict(shared=[31, 0])),
            ("below 0", dict(shared=[-4, -2 ** 31])),
            ("none", dict(group_start=[0, 0, 0])),
            ("a group of nobody", dict(group_start=[2, 2, 5]))):
        c = dict(base)
        for key, val in change.items():
            c[key] = np.array(val, np.int32)
        got, want = _run(bh, dev, c), _want(c)
        print(name, flush=True)
        assert rel_err(got[:n], want[:n]) < TOL, name
        assert np.all(got[n:] == -7.0)


def test_shared_first_request_without_tokens(bh, dev):
    """The prefix is read through the first request's pages, refused or not."""
    c = _case([(64, [(5, 0), (7, 1), (1, 1)])])
    c["kv_len"][0] = 0
    _check(bh, dev, c)


def test_shared_rows_that_see_nothing(bh, dev):
    c = _case([(32, [(1, 1), (4, 1)])])
    c["kv_len"] = np.array([0, 36], np.int32)
    got = _run(bh, dev, c)
    assert np.all(got[0] == 0.0) and rel_err(got[1:2], _want(c)[1:2]) < TOL
    c["table"][:, :] = -1  # pages outside the pool are left out
    import torch
    bad = torch.zeros(1, dtype=torch.int32, device=dev)
    got = _run(bh, dev, c, bad_page=bad)
    assert np.all(got[:2] == 0.0) and bad.item() == -1


@pytest.mark.parametrize("f16", [True, False])
def test_shared_masked_values_do_not_reach(bh, dev, f16):
    """NaN and infinities behind a request's end and in other groups' pages."""
    c = _case([(40, [(5, 1), (21, 3)]), (16, [(3, 1)])], f16=f16, same_pages=False, spare_tokens=0)
    want = _want(c)
    page = c["k"].shape[1]
    seen = np.zeros(c["k"].shape[:2], bool)
    for r, n in enumerate(c["kv_len"]):
        for p in range(n):
            seen[c["table"][r, p // page], p % page] = True
    for name in ("k", "v"):
        c[name] = c[name].copy()
        c[name][~seen] = np.nan
    assert rel_err(_run(bh, dev, c), want) < TOL
    # an infinite value of the prefix makes its group's rows not finite, and no others
    c["v"][c["table"][0, 0], 3] = np.inf
    if True:
        c["v"][c["table"][1, 0], 3] = np.inf
    got = _run(bh, dev, c)
    assert not np.isfinite(got[:4]).any() and np.isfinite(got[4:]).all()


def test_shared_scores_of_minus_infinity(bh, dev):
    """Keys that mask a whole prefix, or all that a row sees."""
    c = _case([(32, [(4, 1), (4, 1)])], n_head=2, n_kv=2, spare_tokens=0, f16=False)
    c["q"][:] = np.abs(c["q"])
    c["k"] = c["k"].copy()
    for b in range(2):
        c["k"][c["table"][0, b]] = -np.inf
    got = _run(bh, dev, c)
    assert rel_err(got, _want(c)) < TOL
    c["k"][:] = -np.inf
    assert np.isnan(_run(bh, dev, c)).all()


def test_shared_garbage_offsets_stay_in_bounds(bh, dev):
    base = _case([(64, [(5, 2), (7, 1)]), (48, [(9, 1)] * 3)], spare_tokens=0)
    n = len(base["q"])
    for key, val in (("q_start", [0, 2, 1, 3, 2 ** 30, n]), ("q_start", [n, 5, 4, 3, 2, 1]),
                     ("q_start", [0, 0, n, 0, n, 0]), ("q_start", [-5, -2, 3, 4, 5, 9]),
                     ("group_start", [3, 1, 5]), ("group_start", [-9, 2 ** 30, 1]),
                     ("group_start", [0, 5, 5]), ("group", [0, 1, 0, 1, 0]),
                     ("shared", [2 ** 31 - 1, 2 ** 31 - 1]), ("kv_len", [2 ** 31 - 1, -4, 0, 1, 2])):
        for hints in ({}, dict(max_new=1, max_group_new=1)):
            c = dict(base)
            c[key] = np.array(val, np.int32)
            print(key, val, flush=True)
            assert _run(bh, dev, c, **hints).shape == base["q"].shape


def test_shared_other_layouts_run_as_paged(bh, dev):
    """Head sizes and strides off the matrix cores."""
    for hd in (80, 40):
        _check(bh, dev, _case(BEAMS, hd=hd))
    c = _case(BEAMS, hd=64)
    c["k"], c["v"] = (np.concatenate([a, a[..., :3]], -1) for a in (c["k"], c["v"]))
    k, v = _t(c["k"], dev)[..., :64], _t(c["v"], dev)[..., :64]
    cache = bh.make_paged_cache(k, v)
    c["k"], c["v"] = c["k"][..., :64], c["v"][..., :64]
    _check(bh, dev, c, cache=cache)


def test_shared_workspace_and_bits(bh, dev):
    """The same bits from call to call; a workspace of the bytes named is enough."""
    import torch
    c = _case([(500, [(9, 1)] * 5), (100, [(3, 1)])], n_head=24, n_kv=4, hd=256)
    got = _run(bh, dev, c, max_new=1, max_group_new=5)
    a = _args(bh, dev, c, max_new=1, max_group_new=5)
    need = bh.attention_shared_workspace(a)
    buf = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device=dev)
    for _ in range(3):
        again = _run(bh, dev, c, max_new=1, max_group_new=5, workspace=buf[:need])
        assert np.array_equal(again, got)
    assert bool((buf[need:] == 0xA5).all())
    with pytest.raises(bh.BonsaiError, match="needed on a 16-byte boundary"):
        _run(bh, dev, c, max_new=1, max_group_new=5, workspace=buf[:need - 16])
