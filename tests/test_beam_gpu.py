"""Beam search's selection and the reordering of its storage.

A score's tolerance.  exp2 of the hardware and its f32 argument (x - m) inv_temp log2 e
put a term of S off by about |z| 2^-23 + 2^-22 of itself, z = 15 for what weighs little:
below 2e-6 of log Z; the result is rounded to f32, 2^-24 of itself."""
from __future__ import annotations

import numpy as np
import pytest

import batchdata as bd

pytestmark = pytest.mark.gpu


def _t(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def _select(bh, dev, x, score, width, n_best, inv_temp=1.0, pad=0, skip=0, **kw):
    import torch
    rows, vocab = x.shape
    buf = torch.full((rows * (vocab + pad) + skip,), 99.0, device=dev)  # after a row: large logits
    wide = buf[skip:].view(rows, vocab + pad)
    wide[:, :vocab] = _t(x, dev)
    args = bh.make_beam_select_args(wide[:, :vocab], _t(score, dev), width, n_best, inv_temp, **kw)
    got = bh.beam_select(args)
    torch.cuda.synchronize()
    return [g.cpu().numpy() for g in got]


def _check(bh, dev, x, score, width, n_best, inv_temp=1.0, exact=False, **kw):
    parent, token, out = _select(bh, dev, x, score, width, n_best, inv_temp, **kw)
    token = token.view(np.uint32)
    for g, (s, rows, toks) in enumerate(bd.continuations(x, score, width, inv_temp)):
        n = min(n_best, len(s))
        tol = 2e-6 + np.abs(s[:n]) * 2.0 ** -24
        assert np.all(np.abs(out[g, :n] - s[:n]) <= tol), (g, out[g, :n] - s[:n])
        if exact:
            assert np.array_equal(parent[g, :n], rows[:n]) and np.array_equal(token[g, :n], toks[:n])
        else:  # nearer than the tolerance either order will do
            near = 4 * n_best + 64
            at = {(r, t): i for i, (r, t) in enumerate(zip(rows[:near].tolist(),
                                                           toks[:near].tolist()))}
            mine = [at[p, t] for p, t in zip(parent[g, :n].tolist(), token[g, :n].tolist())]
            assert len(set(mine)) == n and np.all(np.abs(s[mine] - s[:n]) <= 4e-6)
        assert np.all(parent[g, n:] == -1) and np.all(token[g, n:] == 0xffffffff)
        assert np.all(out[g, n:] == -np.inf)


def _logits(rng, rows, vocab):
    x = (2.5 * rng.standard_normal((rows, vocab))).astype(np.float32)
    at = rng.integers(0, vocab, (rows, 6))
    x[np.arange(rows)[:, None], at] = 8 + 6 * rng.random((rows, 6))
    return x


@pytest.mark.parametrize("groups,width,n_best,vocab", [
    (1, 1, 1, 1), (1, 1, 1, 5), (1, 4, 8, 100), (3, 2, 4, 4096), (2, 5, 10, 4097), (1, 1, 32, 33),
    (7, 3, 1, 1000), (1, 32, 32, 5000), (1, 8, 16, 248320), (40, 8, 16, 9000), (300, 4, 8, 700),
    (2, 16, 32, 30011), (1, 2, 2, 2), (5, 32, 32, 32)])
def test_select_matches(bh, dev, groups, width, n_best, vocab):
    rng = np.random.default_rng(groups + 10 * width + vocab)
    x = _logits(rng, groups * width, vocab)
    score = (-20 * rng.random(groups * width)).astype(np.float32)
    for inv_temp, pad, skip in ((1.0, 0, 0), (1 / 0.7, 3, 1)):
        print(groups, width, n_best, vocab, pad, flush=True)
        _check(bh, dev, x, score, width, n_best, inv_temp, pad=pad, skip=skip)


@pytest.mark.parametrize("vocab", [50, 5000, 70001])
@pytest.mark.parametrize("pad", [0, 1])
def test_select_ties_go_to_the_lowest(bh, dev, vocab, pad):
    """Equal beams: by row, then by token.  (Rows of one bit pattern have one log Z.)"""
    width, n_best = 6, 24
    for kind in ("all", "few", "rows"):
        rng = np.random.default_rng(vocab)
        row = np.zeros(vocab, np.float32) if kind == "all" else \
            np.round(rng.standard_normal(vocab)).astype(np.float32)
        x = np.tile(row, (2 * width, 1))
        score = np.full(2 * width, -3.25, np.float32)
        if kind == "rows":
            score[1::2] = -3.5
        print(kind, vocab, flush=True)
        _check(bh, dev, x, score, width, n_best, exact=True, pad=pad)


def test_select_near_scores_keep_their_order(bh, dev):
    """Scores nearer than a step of f32 at their size are still told apart."""
    rng = np.random.default_rng(2)
    row = (0.01 * rng.standard_normal(300)).astype(np.float32)
    x = np.tile(row, (4, 1))
    score = np.array([-1000.0, -1000.0, -1000.0001, -1000.00006], np.float32)
    x[1] = np.roll(row, 7)
    _check(bh, dev, x, score, 4, 32)
    one = row.copy()
    one[:4] = [9.0, np.nextafter(np.float32(9.0), np.float32(10)), 9.0, 8.9999999]
    _check(bh, dev, one[None], np.array([-5e4], np.float32), 1, 4, exact=True)


def test_select_beams_without_continuations(bh, dev):
    rng = np.random.default_rng(3)
    x = _logits(rng, 12, 9000)
    score = (-rng.random(12)).astype(np.float32)
    score[1:4] = -np.inf         # the first step: one beam
    score[4], score[5] = np.nan, np.inf
    x[6, 17] = np.nan
    x[7, 8999] = np.inf
    score[8:] = -np.inf          # none at all
    _check(bh, dev, x, score, 4, 8)
    # fewer continuations than wanted: banned tokens
    x = np.full((4, 5000), -np.inf, np.float32)
    x[0, [3, 4999]], x[2, 7] = [1.0, 0.5], -2.0
    _check(bh, dev, x, np.zeros(4, np.float32), 4, 8, exact=True)
    _check(bh, dev, x[1:2], np.zeros(1, np.float32), 1, 3, exact=True)


def test_select_banned_and_large(bh, dev):
    rng = np.random.default_rng(4)
    x = _logits(rng, 8, 20000)
    x[:, rng.integers(0, 20000, 3000)] = -np.inf
    _check(bh, dev, x, np.zeros(8, np.float32), 4, 8)
    _check(bh, dev, (x * np.float32(1e30)).astype(np.float32), np.zeros(8, np.float32), 4, 4)
    _check(bh, dev, x, np.full(8, -3e38, np.float32), 4, 4)


def test_select_in_place_and_workspace(bh, dev):
    import torch
    rng = np.random.default_rng(5)
    x = _logits(rng, 8, 40000)
    score = (-rng.random(8)).astype(np.float32)
    want = _select(bh, dev, x, score, 4, 4)
    s = _t(score, dev)
    args = bh.make_beam_select_args(_t(x, dev), s, 4, 4, score_out=s)
    args.workspace_bytes = bh.beam_select_workspace(args)
    ws = torch.zeros(args.workspace_bytes, dtype=torch.uint8, device=dev)
    args = bh.make_beam_select_args(_t(x, dev), s, 4, 4, score_out=s, workspace=ws)
    got = bh.beam_select(args)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert np.array_equal(a.cpu().numpy().reshape(-1), b.reshape(-1))
    short = bh.make_beam_select_args(_t(x, dev), s, 4, 4, workspace=ws[:-16])
    with pytest.raises(bh.BonsaiError, match="needed on a 16-byte boundary"):
        bh.beam_select(short)


# ---------------------------------------------------------------------------
# storage
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("groups,width,columns", [(1, 1, 1), (1, 4, 3), (5, 8, 64), (3, 32, 65),
                                                  (2, 31, 700), (70, 2, 5)])
def test_reorder_matches_loop(bh, dev, groups, width, columns):
    import torch
    rng = np.random.default_rng(groups * width + columns)
    n = groups * width
    for kind in ("random", "one", "same", "swap", "none", "beyond"):
        base = (np.arange(groups) * width)[:, None]
        parent = base + rng.integers(0, width, (groups, width))
        if kind == "one":
            parent = base + np.full((groups, width), width - 1)
        elif kind == "same":
            parent = base + np.arange(width)[None]
        elif kind == "swap":
            parent = base + rng.permutation(width)[None]
        elif kind == "none":
            parent[rng.random(parent.shape) < 0.4] = -1
        elif kind == "beyond":
            parent = rng.integers(-3, n + 3, (groups, width))
        wide = np.full((groups, width + 3), -9, np.int32)
        wide[:, :width] = parent
        table = rng.integers(-1, 1000, (n, columns)).astype(np.int32)
        slots = rng.permutation(2 * n).astype(np.int32)
        want = bd.reorder(parent, table, slots[:n], slots[n:], width)
        tt = [_t(a, dev) for a in (table, np.full(n, 7, np.int32), np.zeros(n, np.int32),
                                   slots[:n], slots[n:])]
        for with_slots in (True, False):
            d = [a.clone() for a in tt]
            kw = dict(src_slot=d[2], dst_slot=d[3], spare_slot=d[4]) if with_slots else {}
            args = bh.make_beam_reorder_args(_t(wide, dev)[:, :width], d[0], copy_from=d[1], **kw)
            bh.beam_reorder(args)
            torch.cuda.synchronize()
            for i, (g, w) in enumerate(zip(d, want)):
                if with_slots or i < 2:
                    assert np.array_equal(g.cpu().numpy(), w), (kind, i)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("page,heads,hd,by_head,pad", [
    (16, 4, 256, False, 0), (16, 2, 64, True, 0), (5, 3, 80, False, 0), (1, 1, 8, False, 0),
    (7, 2, 7, False, 0), (16, 2, 64, False, 3), (64, 1, 128, True, 8)])
def test_copy_matches_loop(bh, dev, f16, page, heads, hd, by_head, pad):
    import torch
    rng = np.random.default_rng(page + heads + hd)
    reqs, width = 9, 6
    n_pages = reqs * width + 2
    dt = np.float16 if f16 else np.float32
    shape = (n_pages, heads, page, hd + pad) if by_head else (n_pages, page, heads, hd + pad)
    raw = [rng.standard_normal(shape).astype(dt) for _ in range(2)]
    table = rng.permutation(n_pages)[:reqs * width].reshape(reqs, width).astype(np.int32)
    table[:, 0] = table[0, 0]       # a page that all share
    table[4, 2] = -1                # pages outside the pool
    table[1, 3] = n_pages
    copy = np.array([-1, 0, 0, -1, 3, 99, -5, 0, 3], np.int32)
    most = width * page
    end = np.array([most, most, page + 1, 3, most, most, most, 2 * page, 10 ** 9], np.int32)
    for begin in (None, np.array([0, 1, page, 0, -7, 0, 0, 2 * page, 3], np.int32)):
        views = [_t(a, dev) for a in raw]
        kv = [(a.transpose(1, 2) if by_head else a)[..., :hd] for a in views]
        cache = bh.make_paged_cache(*kv)
        args = bh.make_kv_copy_args(cache, _t(table, dev), _t(copy, dev),
                                    None if begin is None else _t(begin, dev), _t(end, dev))
        bh.kv_copy_paged(args)
        torch.cuda.synchronize()
        plain = [(a.transpose(0, 2, 1, 3) if by_head else a) for a in raw]
        b = np.zeros(reqs, np.int32) if begin is None else begin
        want = bd.copy_pages(*plain, table, copy, b, end)
        for got, w, p in zip(views, want, plain):
            g = got.cpu().numpy()
            g = g.transpose(0, 2, 1, 3) if by_head else g
            assert np.array_equal(g[..., :hd], w[..., :hd])
            assert np.array_equal(g[..., hd:], p[..., hd:])  # what lies between the rows
