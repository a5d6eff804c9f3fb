"""Log probabilities, entropy and top alternatives against 64-bit arithmetic.

Tolerances.  u = 2^-24.  A log probability is z_tok - log Z with z = (x - max)
inv_temp: two f32 roundings of z (2 u |z|), the f32 inv_temp (u |z|), a sum of
exponentials each off by a few u (and by |z| u through its argument, where e^z
|z| <= 0.37), its logarithm's rounding and the last subtraction: below
4 u |z| + 8 u (1 + log Z') with Z' relative to the maximum.  The entropy adds
sum p |z| (4 u) <= 4 u (H + log Z')."""
from __future__ import annotations

import numpy as np
import pytest

import pageddata as pd

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _t(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def _run(bh, dev, x, tokens, n_top, inv_temp, pad=0, shift=0, **kw):
    """x in rows `pad` floats apart, beginning `shift` floats into a buffer."""
    import torch
    rows, vocab = x.shape
    buf = torch.full((rows * (vocab + pad) + shift + 4,), float("nan"), device=dev)
    xt = buf[shift:shift + rows * (vocab + pad)].view(rows, vocab + pad)[:, :vocab]
    xt.copy_(_t(x, dev))
    args = bh.make_token_logprobs_args(xt, _t(tokens.astype(np.int32), dev), n_top, inv_temp, **kw)
    got = bh.token_logprobs(args)
    torch.cuda.synchronize()
    return [None if g is None else g.cpu().numpy() for g in got], args


def _close(got, want, tol, what):
    got, want = got.astype(np.float64), np.asarray(want)
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)]), what
    err = np.abs(got[fin] - want[fin])
    tol = np.broadcast_to(tol, want.shape)[fin]
    assert (err <= tol).all(), (what, err.max(), (err / tol).max())


def _check(bh, dev, x, tokens, n_top, inv_temp=1.0, **kw):
    got, args = _run(bh, dev, x, tokens, n_top, inv_temp, **kw)
    inv32 = float(np.float32(inv_temp))
    lp, ent, ids, top = pd.logprobs(x, tokens, n_top, inv32)
    with np.errstate(all="ignore"):
        z = x.astype(np.float64) * inv32
        z -= z.max(1, keepdims=True)
        log_z = np.log(np.exp(z).sum(1))
        base = np.where(np.isfinite(log_z), 8 * U * (1 + log_z), 1.0)
    zt = np.where(np.isfinite(lp), -lp, 0.0)
    _close(got[0], lp, 4 * U * zt + base, "logprob")
    h = np.where(np.isfinite(ent), ent, 0.0)
    _close(got[1], ent, 8 * U * (h + 1) + 4 * base, "entropy")
    if n_top:
        assert np.array_equal(got[2], ids)
        _close(got[3], top, 4 * U * np.where(np.isfinite(top), -top, 0.0) + base[:, None], "top")
    return got


def _logits(rng, rows, vocab, coarse=True):
    x = rng.standard_normal((rows, vocab)) * 2.5
    if coarse:
        x = np.round(x * 16) / 16
    for r in range(rows):
        at = rng.integers(0, vocab, min(6, vocab))
        x[r, at] = 8 + np.round(6 * rng.random(len(at)) * 4) / 4
    return x.astype(np.float32), rng.integers(0, vocab, rows)


@pytest.mark.parametrize("rows,vocab", [
    (1, 1), (3, 2), (2, 31), (5, 64), (1, 255), (4, 257), (7, 1000), (3, 4095), (2, 4097),
    (1, 8193), (33, 16384), (300, 1025), (1, 32003), (61, 32003), (600, 20001), (1, 248320),
    (8, 248320), (70, 100003), (2100, 513),
])
def test_sizes(bh, dev, rows, vocab):
    rng = np.random.default_rng(rows * 7 + vocab)
    x, tok = _logits(rng, rows, vocab)
    for n_top, inv_temp in ((min(20, vocab), 1.0), (0, 1 / 0.7), (min(5, vocab), 0.35)):
        print(rows, vocab, n_top, flush=True)
        _check(bh, dev, x, tok, n_top, inv_temp)


@pytest.mark.parametrize("rows", [2, 700])
@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (3, 2), (29, 3), (4, 0)])
def test_strides_and_alignment(bh, dev, rows, pad, shift):
    rng = np.random.default_rng(pad)
    x, tok = _logits(rng, rows, 5003)
    _check(bh, dev, x, tok, 7, pad=pad, shift=shift)


@pytest.mark.parametrize("n_top", [1, 2, 8, 31, 32])
@pytest.mark.parametrize("rows,vocab", [(1, 40), (2, 70000), (520, 9001)])
def test_ties_go_to_the_lowest_id(bh, dev, n_top, rows, vocab):
    rng = np.random.default_rng(n_top)
    tok = rng.integers(0, vocab, rows)
    # all alike; three values only; zeros of both signs; a rising and a falling row
    x = np.zeros((rows, vocab), np.float32)
    _check(bh, dev, x, tok, n_top)
    _check(bh, dev, rng.integers(0, 3, (rows, vocab)).astype(np.float32), tok, n_top)
    x[:, ::2] = -0.0
    _check(bh, dev, x, tok, n_top)
    x[:] = np.arange(vocab) / 64.0
    _check(bh, dev, x, tok, n_top)
    _check(bh, dev, np.ascontiguousarray(x[:, ::-1]), tok, n_top)


@pytest.mark.parametrize("vocab", [50, 5000, 100000])
@pytest.mark.parametrize("rows", [6, 600])
def test_masked_and_infinite(bh, dev, rows, vocab):
    rng = np.random.default_rng(vocab)
    x, tok = _logits(rng, rows, vocab)
    low = np.finfo(np.float32).min
    x[0, :] = -np.inf              # nothing left
    x[1, :] = -np.inf
    x[1, vocab // 2] = 3.0         # one token left
    x[2, vocab // 3:] = low        # masked by the type's lowest value
    x[3, :] = low                  # all of it: uniform
    x[4, ::3] = -np.inf
    x[5, 7] = np.nan
    if rows > 7:
        x[6, 9] = np.inf
        x[7, :] = np.nan
    tok[1], tok[4] = vocab // 2, 3
    with np.errstate(all="ignore"):
        _check(bh, dev, x, tok, 20)


def test_confident_rows(bh, dev):
    """One token far above the rest: entropies near 0 keep their digits to
    8 u absolute, log probabilities near 0 too."""
    rng = np.random.default_rng(3)
    x, tok = _logits(rng, 16, 50000, coarse=False)
    for r in range(16):
        x[r, 77 + r] = 14.0 + 3 * r
        tok[r] = 77 + r
    _check(bh, dev, x, tok, 10)
    _check(bh, dev, x, tok, 10, 20.0)


@pytest.mark.parametrize("rows", [3, 600])
def test_bad_tokens(bh, dev, rows):
    import torch
    rng = np.random.default_rng(4)
    x, tok = _logits(rng, rows, 5000)
    word = torch.full((1,), -5, dtype=torch.int32, device=dev)
    _check(bh, dev, x, tok, 3, bad_id=word)
    assert word.item() == -5
    tok[1] = 5000
    _check(bh, dev, x, tok, 3, bad_id=word)
    assert word.item() == 5000
    tok[1] = 0xFFFFFFFF
    got, _ = _run(bh, dev, x, tok.astype(np.uint32).view(np.int32), 3, 1.0, bad_id=word)
    assert np.isnan(got[0][1]) and np.isfinite(got[1]).all() and word.item() == -1


@pytest.mark.parametrize("rows,vocab", [(5, 30000), (600, 3000), (2, 50)])
def test_parts_asked_for(bh, dev, rows, vocab):
    """Without tokens, without alternatives; own workspaces; the same bits."""
    import torch
    rng = np.random.default_rng(5)
    x, tok = _logits(rng, rows, vocab)
    full, args = _run(bh, dev, x, tok, 6, 1.0)
    need = bh.token_logprobs_workspace(args)
    ws = torch.empty(max(16, need), dtype=torch.uint8, device=dev)
    again, _ = _run(bh, dev, x, tok, 6, 1.0, workspace=ws)
    for a, b in zip(full, again):
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
    if need:
        with pytest.raises(bh.BonsaiError, match="workspace"):
            _run(bh, dev, x, tok, 6, 1.0, workspace=ws[:need - 16])
    xt = _t(x, dev)
    args = bh.make_token_logprobs_args(xt, n_top=6)
    lp, ent, ids, top = bh.token_logprobs(args)
    assert lp is None
    assert np.array_equal(ids.cpu().numpy(), full[2])
    assert np.array_equal(ent.cpu().numpy(), full[1])
    args = bh.make_token_logprobs_args(xt, _t(tok.astype(np.int32), dev))
    lp, ent, ids, top = bh.token_logprobs(args)
    assert ids is None and np.allclose(lp.cpu().numpy(), full[0], rtol=0, atol=1e-5)
    # uint32 ids as the rest of the library takes them
    args = bh.make_token_logprobs_args(xt, _t(tok.astype(np.int32), dev).view(torch.uint32), 6)
    assert np.array_equal(bh.token_logprobs(args)[2].cpu().numpy(), full[2])


def test_graph_replays(bh, dev):
    import torch
    rng = np.random.default_rng(6)
    xs = [_logits(rng, 9, 70000) for _ in range(3)]
    x, tok = _t(xs[0][0], dev), _t(xs[0][1].astype(np.int32), dev)
    args = bh.make_token_logprobs_args(x, tok, 12)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    bh.token_logprobs(args, stream=st)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        bh.token_logprobs(args, stream=st)
    for a, b in xs + xs[:1]:
        x.copy_(_t(a, dev)), tok.copy_(_t(b.astype(np.int32), dev))
        for t in args.results:
            t.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in args.results]
        bh.token_logprobs(args)
        torch.cuda.synchronize()
        for p, q in zip(got, args.results):
            assert torch.equal(p, q)
        assert np.array_equal(got[2].cpu().numpy(), pd.logprobs(a, b, 12, 1.0)[2])
