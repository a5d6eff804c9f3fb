"""A serving step over a paged cache on the GPU: the plan against a loop over
requests (exact), the append bit for bit, attention against 64-bit arithmetic,
and a whole step, eager and captured.

Attention's tolerance.  The result is a mean of v with weights w = softmax(s).
With u = 2^-24, a score is off by at most ds = (hd + 8) u sum|q_d k_d| / sqrt(hd)
(hd products and sums in f32; operands split into two halves of f16 carry 22
bits, 2^-23 each, which the 8 covers), the weights by a factor e^(2 ds), and the
sum over n positions adds (n + 8) u.  Those are worst cases; a random walk over
hd terms gives sqrt(hd) for hd.  For N(0, 1) data and hd = 256 that is ds =
(16 + 8) u * 10 = 1.4e-5, of which the difference to the mean's matters, times
|v - o| ~ 1 weighted by w: below 1e-5 of the largest output for every shape
here.  1e-5 is what bh_attention is held to as well."""
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


# ---------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------

def _run_plan(bh, dev, cached, new, table, free, n_free, page, n_tok, inplace=False):
    import torch
    i32 = np.int32
    n_req = len(cached)
    d = [_t(np.asarray(a, i32), dev) for a in (cached, new, table, free, [n_free])]
    z = lambda *s: torch.full(s, -77, dtype=torch.int32, device=dev)  # noqa: E731
    out = dict(kv_len=z(n_req), q_start=z(n_req + 1), slots=z(n_tok), pos=z(n_tok, 4),
               n_free_out=None if inplace else z(1), n_refused=z(1))
    args = bh.make_paged_plan_args(*d, page, **out)
    bh.paged_plan(args)
    torch.cuda.synchronize()
    left = d[4] if inplace else out["n_free_out"]
    got = [out["kv_len"], out["q_start"], out["slots"], out["pos"], d[2], d[3], left,
           out["n_refused"]]
    return [g.cpu().numpy() for g in got], args


def _check_plan(bh, dev, cached, new, table, free, n_free, page, n_tok, **kw):
    want = pd.plan(cached, new, np.asarray(table, np.int32), np.asarray(free, np.int32), n_free,
                   page, n_tok)
    got, args = _run_plan(bh, dev, cached, new, table, free, n_free, page, n_tok, **kw)
    names = ("kv_len", "q_start", "slots", "pos", "table", "free", "n_free", "refused")
    for n, g, w in zip(names, got, want):
        assert np.array_equal(g.reshape(-1), np.asarray(w).reshape(-1)), n
    return args


def _random_plan(rng, n_req, page, width, n_tok, tight):
    cached = rng.integers(0, width * page + 1, n_req)
    cached[rng.random(n_req) < 0.2] = 0
    new = rng.integers(0, 4, n_req)
    new[rng.random(n_req) < 0.1] = rng.integers(0, width * page + 3)
    new[rng.random(n_req) < 0.15] = -1
    have = -(-cached // page)
    table = np.full((n_req, width), -1, np.int32)
    n_pages = int(have.sum()) + max(4, n_req * 2) + 1
    order = rng.permutation(n_pages).astype(np.int32)
    at = 0
    for i in range(n_req):
        table[i, :have[i]] = order[at:at + have[i]]
        at += have[i]
    n_free = (n_pages - at) // (6 if tight else 1)
    free = np.full(n_pages, -1, np.int32)
    free[:n_free] = order[at:at + n_free]
    return cached, new, table, free, n_free


@pytest.mark.parametrize("n_req,page,width,n_tok,tight", [
    (1, 16, 4, 1, False), (1, 1, 1, 3, False), (3, 16, 8, 8, False), (64, 16, 20, 200, False),
    (64, 7, 20, 150, True), (65, 100, 3, 400, True), (300, 16, 9, 250, True),
    (1000, 33, 5, 4000, False), (1024, 16, 4, 2000, True), (1025, 16, 4, 3000, False),
    (4095, 2, 6, 9000, False), (4096, 16, 2, 9000, True), (17, 128, 40, 20000, False),
])
def test_plan_matches_loop(bh, dev, n_req, page, width, n_tok, tight):
    for seed in range(3):
        rng = np.random.default_rng(1000 * n_req + seed)
        print(n_req, page, seed, flush=True)
        _check_plan(bh, dev, *_random_plan(rng, n_req, page, width, n_tok, tight), page, n_tok,
                    inplace=seed == 1)


def test_plan_edges(bh, dev):
    import torch
    none = np.full((2, 3), -1, np.int32)
    free = np.arange(6)
    # nothing to do; no room for tokens; the whole stack; past it by one
    _check_plan(bh, dev, [0, 0], [0, 0], none, free, 6, 4, 5)
    _check_plan(bh, dev, [0, 0], [1, 1], none, free, 6, 4, 0)
    _check_plan(bh, dev, [0, 0], [12, 12], none, free, 6, 4, 24)
    _check_plan(bh, dev, [0, 0], [12, 12], none, free, 5, 4, 24)
    # longer than the table; a later short one still fits
    _check_plan(bh, dev, [0, 0], [13, 2], none, free, 6, 4, 24)
    _check_plan(bh, dev, [2 ** 31 - 1, 0], [2 ** 31 - 1, 2], none, free, 6, 4, 24)
    # lengths and counts that no program should pass: clipped, in bounds
    _check_plan(bh, dev, [-5, 0], [3, 1], none, free, 6, 4, 24)
    _check_plan(bh, dev, [0, 0], [3, 1], none, free, -3, 4, 24)
    _check_plan(bh, dev, [0, 0], [3, 1], none, free, 99, 4, 24)
    # a stack that overflows on release: the pages past it are dropped
    full = np.array([[8, 9, 7], [1, 2, 3]], np.int32)
    _check_plan(bh, dev, [12, 5], [-1, 1], full, free, 5, 4, 4)
    # a release longer than its table row, a page outside the pool
    _check_plan(bh, dev, [40, 5], [-1, 1], full, np.full(12, -1), 0, 4, 4)
    _check_plan(bh, dev, [3, 5], [1, 1], np.array([[99, 1, 1], [-4, 0, 0]]), free, 6, 4, 4)
    # no requests at all
    i32 = dict(dtype=torch.int32, device=dev)
    slots, start = torch.zeros(4, **i32), torch.full((1,), 9, **i32)
    args = bh.make_paged_plan_args(torch.zeros(0, **i32), torch.zeros(0, **i32),
                                   torch.zeros((0, 3), **i32), torch.zeros(5, **i32),
                                   torch.tensor([2], **i32), 4, kv_len=torch.zeros(0, **i32),
                                   q_start=start, slots=slots)
    bh.paged_plan(args)
    assert start.item() == 0 and slots.tolist() == [-1] * 4


def test_plan_again_gives_the_same(bh, dev):
    import torch
    rng = np.random.default_rng(5)
    cached, new, table, free, n_free = _random_plan(rng, 200, 16, 10, 300, True)
    got, args = _run_plan(bh, dev, cached, new, table, free, n_free, 16, 300)
    for _ in range(3):
        bh.paged_plan(args)
    torch.cuda.synchronize()
    again = [t.cpu().numpy() for t in (args.tensors[5], args.tensors[6], args.tensors[7],
                                       args.tensors[8], args.tensors[2], args.tensors[3])]
    for a, b in zip(got, again):
        assert np.array_equal(a, b)


# ---------------------------------------------------------------------------
# store
# ---------------------------------------------------------------------------

def _pool(dev, n_pages, page, n_kv, hd, f16, layout, fill=None, rng=None):
    """K and V [page][position][head][dim] in a layout; random or constant."""
    import torch
    dt = torch.float16 if f16 else torch.float32

    def make():
        if layout == "rows":
            t = torch.empty((n_pages, page, n_kv, hd), dtype=dt, device=dev)
        elif layout == "heads":
            t = torch.empty((n_pages, n_kv, page, hd), dtype=dt, device=dev).transpose(1, 2)
        else:  # rows wider than their heads, by an odd number of elements
            t = torch.empty((n_pages, page, n_kv, hd + 3), dtype=dt, device=dev)[..., :hd]
        return t
    if layout == "both":  # K and V of a page side by side
        t = torch.empty((n_pages, 2, page, n_kv, hd), dtype=dt, device=dev)
        k, v = t[:, 0], t[:, 1]
    else:
        k, v = make(), make()
    for c in (k, v):
        if fill is not None:
            c.fill_(fill)
        else:
            c.copy_(_t(rng.standard_normal((n_pages, page, n_kv, hd), np.float32), dev))
    return k, v


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("layout", ["rows", "heads", "both", "odd"])
@pytest.mark.parametrize("n_tok,page,n_kv,hd", [(1, 16, 4, 256), (37, 5, 3, 80), (200, 64, 8, 128),
                                                (9, 1, 1, 7), (70, 16, 2, 64)])
def test_store_paged_bits(bh, dev, oracle, f16, layout, n_tok, page, n_kv, hd):
    import torch
    rng = np.random.default_rng(n_tok + hd)
    n_pages = 2 * n_tok // page + 3
    k_cache, v_cache = _pool(dev, n_pages, page, n_kv, hd, f16, layout, fill=7.0)
    cache = bh.make_paged_cache(k_cache, v_cache)
    slots = rng.permutation(n_pages * page)[:n_tok].astype(np.int32)
    slots[rng.random(n_tok) < 0.1] = -1
    if n_tok > 2:
        slots[1], slots[2] = n_pages * page, np.iinfo(np.int32).max
    k, v = (rng.standard_normal((n_tok, n_kv * hd)).astype(np.float32) for _ in range(2))
    special = np.array([np.nan, np.inf, -np.inf, -0.0, 1e6, 65519.9, 65520.0, 6e-8, 2.9e-8, 1e-9],
                       np.float32)
    k.reshape(-1)[:min(10, k.size)] = special[:min(10, k.size)]
    bh.kv_store_paged(cache, _t(k, dev), _t(v, dev), _t(slots, dev))
    torch.cuda.synchronize()
    for rows, got in ((k, k_cache), (v, v_cache)):
        want = np.full((n_pages * page, n_kv * hd), 7.0, np.float16 if f16 else np.float32)
        ok = (slots >= 0) & (slots < n_pages * page)
        with np.errstate(over="ignore"):
            want[slots[ok]] = rows[ok].astype(want.dtype)
        g = got.contiguous().cpu().numpy().reshape(want.shape)
        bits = np.uint16 if f16 else np.uint32
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(g), nan)
        assert np.array_equal(g.view(bits)[~nan], want.view(bits)[~nan])


@pytest.mark.parametrize("f16", [False, True])
def test_store_paged_is_kv_store(bh, dev, f16):
    """One page after the other: the bits that bh_kv_store writes, NaN too."""
    import torch
    n, page = 48, 16
    k, v = (torch.randn((n, 1024), device=dev, generator=torch.Generator(dev).manual_seed(i))
            for i in (1, 2))
    k[3, :4] = torch.tensor([float("nan"), float("inf"), -0.0, 1e5], device=dev)
    k[4, 5] = torch.tensor([0xFFC12345 - 2 ** 32], dtype=torch.int32, device=dev).view(
        torch.float32)[0]
    dt = torch.float16 if f16 else torch.float32
    flat = [torch.zeros((n, 1024), dtype=dt, device=dev) for _ in range(2)]
    bh.kv_store(k, v, *flat, 0)
    pool = [torch.zeros((3, page, 4, 256), dtype=dt, device=dev) for _ in range(2)]
    bh.kv_store_paged(bh.make_paged_cache(*pool), k, v,
                      torch.arange(n, dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    bits = torch.int16 if f16 else torch.int32
    for a, b in zip(flat, pool):
        assert torch.equal(a.view(bits).reshape(-1), b.view(bits).reshape(-1))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _step(rng, dev, lens, new, page, n_q, n_kv, hd, f16, layout="rows", pad=0, fill=None,
          q_scale=1.0, width=None):
    table, n_pages = pd.pages(rng, lens, page, width)
    k, v = _pool(dev, n_pages, page, n_kv, hd, f16, layout, rng=rng)
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = (rng.standard_normal((int(start[-1]) + pad, n_q, hd)) * q_scale).astype(np.float32)
    return dict(table=table, k=k, v=v, start=start, q=q, lens=np.asarray(lens, np.int32),
                max_new=int(max(list(new) + [0])))


def _attend(bh, dev, s, **kw):
    import torch
    out = torch.full(s["q"].shape, 5.25, device=dev)
    args = bh.make_attention_paged_args(
        bh.make_paged_cache(s["k"], s["v"]), _t(s["q"], dev), _t(s["start"], dev),
        _t(s["lens"], dev), _t(s["table"], dev), out=out,
        **{"max_new": s["max_new"], **kw})
    bh.attention_paged(args)
    torch.cuda.synchronize()
    return out.cpu().numpy(), args


def _want(s):
    k, v = (c.float().cpu().numpy() for c in (s["k"], s["v"]))
    return pd.attention(s["q"], k, v, s["start"], s["lens"], s["table"],
                        np.full(s["q"].shape, 5.25))


def _check(bh, dev, s, tol=TOL, **kw):
    got, _ = _attend(bh, dev, s, **kw)
    want = _want(s)
    err = rel_err(got, want.astype(np.float32))
    print("rel err", err, flush=True)
    assert err <= tol
    end = int(s["start"][-1])
    assert (got[end:] == 5.25).all()
    return got


HEADS = [(24, 4, 256), (32, 8, 128), (16, 2, 64), (3, 3, 256), (24, 1, 128), (40, 2, 64)]


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n_q,n_kv,hd", HEADS)
def test_decode_ragged(bh, dev, n_q, n_kv, hd, f16):
    rng = np.random.default_rng(hd + n_q)
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 100, 127, 128, 129, 1000, 2049]
    s = _step(rng, dev, lens, [1] * len(lens), 16, n_q, n_kv, hd, f16, pad=3)
    _check(bh, dev, s)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n_q,n_kv,hd", [(24, 4, 256), (32, 8, 128), (4, 4, 64)])
@pytest.mark.parametrize("layout", ["rows", "heads", "both", "odd"])
@pytest.mark.parametrize("page", [1, 7, 48, 300])
def test_layouts_and_pages(bh, dev, n_q, n_kv, hd, f16, layout, page):
    rng = np.random.default_rng(page)
    s = _step(rng, dev, [5, 333, 64], [1, 3, 2], page, n_q, n_kv, hd, f16, layout, pad=1)
    _check(bh, dev, s)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("new", [[2, 8, 1, 5], [16, 3], [40, 1, 1], [1, 130, 2], [257]])
@pytest.mark.parametrize("n_q,n_kv,hd", [(24, 4, 256), (32, 8, 128), (8, 8, 64)])
def test_several_new_tokens(bh, dev, new, n_q, n_kv, hd, f16):
    rng = np.random.default_rng(sum(new))
    lens = [n + int(x) for n, x in zip(new, rng.integers(0, 400, len(new)))]
    lens[0] = new[0]  # a prompt from its beginning
    s = _step(rng, dev, lens, new, 16, n_q, n_kv, hd, f16)
    _check(bh, dev, s)


@pytest.mark.parametrize("n_q,n_kv,hd", [(6, 2, 80), (5, 5, 1), (4, 2, 512), (7, 1, 200),
                                         (2, 1, 65)])
@pytest.mark.parametrize("f16", [True, False])
def test_any_head_size(bh, dev, n_q, n_kv, hd, f16):
    rng = np.random.default_rng(hd)
    s = _step(rng, dev, [1, 70, 19], [1, 2, 1], 8, n_q, n_kv, hd, f16, pad=2)
    _check(bh, dev, s)


@pytest.mark.parametrize("hd", [256, 128, 64, 40])
@pytest.mark.parametrize("f16", [True, False])
def test_empty_and_short(bh, dev, hd, f16):
    """Requests without tokens, without a cache, with fewer positions than
    tokens (the first queries see nothing: zeros)."""
    rng = np.random.default_rng(hd)
    lens, new = [0, 10, 3, 0, 50], [0, 0, 5, 2, 1]
    s = _step(rng, dev, lens, new, 16, 8, 2, hd, f16, pad=4, width=5)
    got = _check(bh, dev, s)
    assert (got[:2] == 0).all() and (got[5:7] == 0).all() and (got[2] != 0).all()


@pytest.mark.parametrize("hd", [256, 64, 40])
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("new", [[1, 4, 1], [20, 2, 70]])
def test_what_is_masked_may_hold_anything(bh, dev, hd, f16, new):
    """NaN and infinities behind each request's last position, in pages of no
    request, and in the rows of later new tokens for the earlier ones."""
    import torch
    rng = np.random.default_rng(hd)
    lens = [77, 33, 128 + 70]
    s = _step(rng, dev, lens, new, 16, 12, 2, hd, f16)
    bad = [float("nan"), float("inf"), -float("inf")]
    used = torch.zeros(s["k"].shape[:2], dtype=torch.bool, device=dev)
    for r, n in enumerate(lens):
        for p in range(n):
            used[s["table"][r, p // 16], p % 16] = True
    for c in (s["k"], s["v"]):
        for i, b in enumerate(bad):
            m = ~used
            m[:, [j for j in range(16) if j % 3 != i]] = False
            c[m] = b
    clean = _attend(bh, dev, s)[0]
    assert np.isfinite(clean).all()
    assert rel_err(clean, _want(s).astype(np.float32)) <= TOL
    # the last new token of each request: only its own row may change
    for r, n in enumerate(lens):
        p = n - 1
        s["v"][int(s["table"][r, p // 16]), p % 16, :, ::2] = bad[r]
        s["k"][int(s["table"][r, p // 16]), p % 16, 1] = bad[(r + 1) % 3]
    got = _attend(bh, dev, s)[0]
    for r in range(3):
        a, b = s["start"][r], s["start"][r + 1]
        assert np.array_equal(got[a:b - 1], clean[a:b - 1]), r
        assert not np.isfinite(got[b - 1, :6, ::2]).any()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("hd,n_q", [(256, 24), (128, 24), (96, 8)])
def test_bad_pages(bh, dev, hd, f16, n_q):
    """Table entries outside the pool leave their positions out."""
    import torch
    rng = np.random.default_rng(3)
    lens, new = [200, 90, 40, 64], [1, 3, 1, 64]
    s = _step(rng, dev, lens, new, 16, n_q, 4, hd, f16)
    n_pages = s["k"].shape[0]
    s["table"][0, 3], s["table"][0, 12] = -1, n_pages
    s["table"][1, 0], s["table"][1, 5] = np.iinfo(np.int32).max, np.iinfo(np.int32).min
    s["table"][2, :] = -9  # nothing left: zeros
    s["table"][3, 1] = n_pages + 5
    word = torch.full((1,), 12345, dtype=torch.int32, device=dev)
    got = _check(bh, dev, s, bad_page=word)
    assert (got[4] == 0).all()
    assert word.item() in (-1, n_pages, np.iinfo(np.int32).max, np.iinfo(np.int32).min, -9,
                           n_pages + 5)
    word.fill_(12345)
    s = _step(rng, dev, lens, new, 16, n_q, 4, hd, f16)
    _check(bh, dev, s, bad_page=word)
    assert word.item() == 12345


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n_q,n_kv,hd", [(24, 4, 256), (8, 8, 64)])
def test_long_cache_alone_and_among_short(bh, dev, n_q, n_kv, hd, f16):
    rng = np.random.default_rng(8)
    for lens in ([20000], [3, 9001, 1, 700]):
        s = _step(rng, dev, lens, [1] * len(lens), 16, n_q, n_kv, hd, f16)
        _check(bh, dev, s)


@pytest.mark.parametrize("n_req", [257, 1500])
def test_many_requests(bh, dev, n_req):
    rng = np.random.default_rng(n_req)
    lens = rng.integers(0, 60, n_req)
    new = np.minimum(rng.integers(0, 3, n_req), lens)
    s = _step(rng, dev, lens, new, 16, 8, 2, 64, True, pad=9)
    _check(bh, dev, s)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("scale,tol", [(30.0, None), (1e-3, TOL), (1e4, None)])
def test_score_ranges(bh, dev, f16, scale, tol):
    """Peaked and flat attention.  Scores of size S = max|s| carry an error of
    about 24 u S (see the module's text), which the weights take as a factor:
    the tolerance grows with it, by S / 10 over TOL for N(0, 1) data."""
    rng = np.random.default_rng(11)
    s = _step(rng, dev, [500, 70], [1, 9], 16, 24, 4, 256, f16, q_scale=scale)
    top = 5.0 * scale  # N(0, scale^2) scores
    _check(bh, dev, s, tol=tol or max(TOL, 2 * 24 * 2.0 ** -24 * top))


@pytest.mark.parametrize("f16", [True, False])
def test_value_ranges(bh, dev, f16):
    """Tiny and huge values, equal keys (uniform weights: a mean)."""
    rng = np.random.default_rng(12)
    for vs, ks in ((1e-4, 1.0), (6e4 if f16 else 3e30, 1.0), (1.0, 0.0)):
        s = _step(rng, dev, [400, 35], [1, 4], 16, 24, 4, 256, f16)
        s["v"].copy_(s["v"].clamp(-0.99, 0.99) * vs)
        s["k"].mul_(ks)
        _check(bh, dev, s)


def test_infinite_and_nan_keys_seen(bh, dev):
    """A key of -inf against a positive query weighs nothing; a row whose every
    score is -inf, or with a NaN, is NaN, as the softmax of 64 bits has it."""
    for f16 in (True, False):
        for hd in (256, 96):
            rng = np.random.default_rng(13)
            s = _step(rng, dev, [40, 3, 20], [1, 1, 2], 16, 6, 1, hd, f16)
            s["q"][:] = np.abs(s["q"]) + 0.1
            s["k"][int(s["table"][0, 0]), 5, 0, 3] = -float("inf")
            for p in range(3):
                s["k"][int(s["table"][1, 0]), p, 0, 3] = -float("inf")
            s["k"][int(s["table"][2, 1]), 2, 0, 7] = float("nan")  # position 18: row 0 of it too
            got = _check(bh, dev, s)
            assert np.isfinite(got[0]).all() and np.isnan(got[1:]).all()


def test_max_new_changes_nothing_it_should_not(bh, dev):
    """max_new steers the layout of the work; 0 and too small a value are
    right as well."""
    rng = np.random.default_rng(14)
    s = _step(rng, dev, [300, 80, 5], [70, 1, 3], 16, 24, 4, 256, True)
    for m in (70, 0, 1, 4, 4096):
        _check(bh, dev, s, max_new=m)


def test_same_bits_again_and_own_workspace(bh, dev):
    import torch
    rng = np.random.default_rng(15)
    s = _step(rng, dev, [3000, 80, 700], [1, 8, 60], 16, 24, 4, 256, True)
    first, args = _attend(bh, dev, s)
    need = bh.attention_paged_workspace(args)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    for kw in ({}, {"workspace": ws}):
        got, _ = _attend(bh, dev, s, **kw)
        assert np.array_equal(got.view(np.uint32), first.view(np.uint32))
    if need:
        with pytest.raises(bh.BonsaiError, match="workspace"):
            _attend(bh, dev, s, workspace=ws[:need - 16])
        with pytest.raises(bh.BonsaiError, match="workspace"):
            _attend(bh, dev, s, workspace=torch.empty(need + 16, dtype=torch.uint8,
                                                      device=dev)[1:need + 1])


def test_two_streams_with_their_own_workspaces(bh, dev):
    import torch
    steps, outs, calls = [], [], []
    for i in range(2):
        rng = np.random.default_rng(20 + i)
        s = _step(rng, dev, [9000 + 500 * i, 300], [1, 2], 16, 24, 4, 256, True)
        d = [_t(s[n], dev) for n in ("q", "start", "lens", "table")]
        args = bh.make_attention_paged_args(bh.make_paged_cache(s["k"], s["v"]), *d, max_new=2)
        n = bh.attention_paged_workspace(args)
        ws = torch.empty(max(n, 16), dtype=torch.uint8, device=dev)
        args = bh.make_attention_paged_args(bh.make_paged_cache(s["k"], s["v"]), *d, max_new=2,
                                            workspace=ws)
        steps.append(s)
        calls.append(args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for st, c in zip(streams, calls):
            bh.attention_paged(c, stream=st)
    torch.cuda.synchronize()
    for s, c in zip(steps, calls):
        assert rel_err(c.out_tensor.cpu().numpy(), _want(s).astype(np.float32)) <= TOL


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n_q,n_kv,hd", [(6, 1, 256), (24, 1, 128), (3, 1, 64)])
def test_one_head_in_hundreds_of_parts(bh, dev, n_q, n_kv, hd, f16):
    """A single row tile that every worker has a part of."""
    rng = np.random.default_rng(31)
    _check(bh, dev, _step(rng, dev, [40000], [1], 64, n_q, n_kv, hd, f16))


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n_q,n_kv,hd", [(24, 4, 256), (32, 8, 128), (8, 8, 64)])
def test_prompts_beside_decoders_replayed(bh, dev, n_q, n_kv, hd, f16):
    """Both forms of a step in one graph, their tiles cut and joined, replayed over
    other lengths: prompts alone, decoders alone, nothing at all."""
    import torch
    rng = np.random.default_rng(32)
    s = _step(rng, dev, [1500, 900, 2600, 40], [130, 1, 61, 5], 32, n_q, n_kv, hd, f16, pad=3)
    d = {n: _t(s[n], dev) for n in ("q", "start", "lens", "table")}
    out = torch.empty(s["q"].shape, device=dev)

    def make(workspace=None):
        return bh.make_attention_paged_args(
            bh.make_paged_cache(s["k"], s["v"]), d["q"], d["start"], d["lens"], d["table"],
            out=out, max_new=200, workspace=workspace)
    ws = torch.empty(max(16, bh.attention_paged_workspace(make())), dtype=torch.uint8, device=dev)
    args, st = make(ws), torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        bh.attention_paged(args, stream=st)
    for start, lens in (([0, 130, 131, 192, 197], [1500, 900, 2600, 40]),
                        ([0, 200, 200, 200, 200], [700, 0, 2600, 17]),
                        ([0, 0, 0, 0, 0], [1500, 900, 2600, 40]),
                        ([0, 1, 2, 3, 4], [1500, 900, 1, 40]),
                        ([0, 90, 91, 197, 198], [1311, 1, 2600, 3])):
        s["start"], s["lens"] = np.array(start, np.int32), np.array(lens, np.int32)
        d["start"].copy_(_t(s["start"], dev))
        d["lens"].copy_(_t(s["lens"], dev))
        out.fill_(5.25)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = out.cpu().numpy()
        assert rel_err(got, _want(s).astype(np.float32)) <= TOL
        assert (got[start[-1]:] == 5.25).all()
        out.fill_(5.25)
        bh.attention_paged(make())
        torch.cuda.synchronize()
        assert np.array_equal(got.view(np.uint32), out.cpu().numpy().view(np.uint32))


def test_strange_offsets_stay_in_bounds(bh, dev):
    """Offsets past the tokens and lengths past the table are clipped."""
    import torch
    rng = np.random.default_rng(16)
    s = _step(rng, dev, [30, 40], [1, 1], 16, 24, 4, 256, True)
    s["start"] = np.array([-5, 1, 1 << 30], np.int32)
    s["lens"] = np.array([30, 1 << 30], np.int32)
    got, _ = _attend(bh, dev, s)
    s["start"], s["lens"] = np.array([0, 1, 2], np.int32), np.array([30, 48], np.int32)
    assert rel_err(got, _want(s).astype(np.float32)) <= TOL
    s["lens"] = np.array([-4, 48], np.int32)
    assert (_attend(bh, dev, s)[0][0] == 0).all()


def test_overlapping_offsets_stay_in_bounds(bh, dev):
    """Offsets that go back and forth ask for far more row tiles than tokens that
    do not overlap have: nothing is written past the workspace or the output."""
    import torch
    rng = np.random.default_rng(18)
    for max_new in (1, 40):
        s = _step(rng, dev, [600] * 64, [1] * 64, 16, 24, 4, 256, True, pad=2)
        s["start"] = np.array([0, 60] * 32 + [0], np.int32)
        d = [_t(s[n], dev) for n in ("q", "start", "lens", "table")]
        out = torch.full((70, 24, 256), 5.25, device=dev)
        args = bh.make_attention_paged_args(bh.make_paged_cache(s["k"], s["v"]), *d, out=out[2:68],
                                            max_new=max_new)
        need = bh.attention_paged_workspace(args)
        ws = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device=dev)
        args = bh.make_attention_paged_args(bh.make_paged_cache(s["k"], s["v"]), *d, out=out[2:68],
                                            max_new=max_new, workspace=ws[:need])
        bh.attention_paged(args)
        torch.cuda.synchronize()
        assert (ws[need:] == 0x5A).all()
        assert (out[:2] == 5.25).all() and (out[62:] == 5.25).all()


@pytest.mark.parametrize("hd", [256, 128, 64])
@pytest.mark.parametrize("new", [[1], [3], [40]])
def test_infinite_keys_and_padding_rows(bh, dev, hd, new):
    """An infinite key that every row sees, in steps where nothing is masked; the
    rows that fill up a tile of 16 belong to nobody."""
    rng = np.random.default_rng(19)
    s = _step(rng, dev, [700], new, 16, 5, 1, hd, True)
    s["q"][:] = np.abs(s["q"]) + 0.1
    for p in (3, 100, 333):
        s["k"][int(s["table"][0, p // 16]), p % 16, 0, 2] = -float("inf")
    got = _check(bh, dev, s)
    assert np.isfinite(got).all()


def test_offsets_past_32_bits(bh, dev):
    """A pool of over 2^32 bytes and 2^31 elements, a request in its last pages."""
    import torch
    n_pages, page = (1 << 31) // (256 * 256) + 40, 256
    k, v = (torch.empty((n_pages, page, 1, 256), dtype=torch.float16, device=dev)
            for _ in range(2))
    rng = np.random.default_rng(17)
    table = np.array([[n_pages - 1, n_pages - 7, 0]], np.int32)
    for c in (k, v):
        for p in table[0]:
            c[int(p)] = _t(rng.standard_normal((page, 1, 256), np.float32), dev)
    rows = _t(rng.standard_normal((2, 256), np.float32), dev)
    bh.kv_store_paged(bh.make_paged_cache(k, v), rows, rows,
                      _t(np.array([(n_pages - 7) * page + 9, 3], np.int32), dev))
    small_k, small_v = (c[torch.from_numpy(table[0].astype(np.int64)).to(dev)] for c in (k, v))
    assert torch.equal(small_k[1, 9, 0], rows[0].half())
    assert torch.equal(small_v[2, 3, 0], rows[1].half())
    s = dict(table=table, k=k, v=v, start=np.array([0, 2], np.int32),
             lens=np.array([700], np.int32), max_new=2,
             q=rng.standard_normal((2, 6, 256)).astype(np.float32))
    got, _ = _attend(bh, dev, s)
    want = _want({**s, "k": small_k, "v": small_v, "table": np.array([[0, 1, 2]], np.int32)})
    assert rel_err(got, want.astype(np.float32)) <= TOL


def test_python_checks(bh, dev):
    import torch
    k = torch.zeros((4, 16, 2, 64), device=dev, dtype=torch.float16)
    cache = bh.make_paged_cache(k, k.clone())
    q = torch.zeros((2, 4, 64), device=dev)
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
    ok = dict(q=q, q_start=i(3), kv_len=i(2), block_table=i(2, 4))
    for bad in (dict(q=q.double()), dict(q=q[:, :, :32]), dict(q=q.transpose(0, 1)),
                dict(q_start=i(2)), dict(kv_len=i(2).long()), dict(block_table=i(8)),
                dict(block_table=i(2, 4).cpu()), dict(block_table=i(2, 8)[:, ::2])):
        with pytest.raises(ValueError):
            bh.make_attention_paged_args(cache, **{**ok, **bad})
    with pytest.raises(ValueError):
        bh.kv_store_paged(cache, torch.zeros((2, 127), device=dev), torch.zeros((2, 128),
                                                                               device=dev), i(2))
    with pytest.raises(TypeError):
        bh.make_paged_cache(k.double(), k.double())


# ---------------------------------------------------------------------------
# a step as it would be used
# ---------------------------------------------------------------------------

class Engine:
    """A small server's step: plan, rotation at the planned positions, append,
    attention, logits, log probabilities, on buffers that stay."""

    def __init__(self, bh, dev, n_req=6, n_tok=12, page=4, width=12, n_pages=40, f16=True):
        import torch
        self.bh, self.n_q, self.n_kv, self.hd, self.vocab = bh, 8, 2, 64, 1000
        z = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
        self.cached, self.new = z(n_req), z(n_req)
        self.table = torch.full((n_req, width), -1, dtype=torch.int32, device=dev)
        self.free = torch.arange(n_pages, dtype=torch.int32, device=dev)
        self.n_free = torch.tensor([n_pages], dtype=torch.int32, device=dev)
        self.kv_len, self.q_start, self.slots = z(n_req), z(n_req + 1), z(n_tok)
        self.pos, self.refused = z(n_tok, 4), z(1)
        g = torch.Generator(dev).manual_seed(4)
        dt = torch.float16 if f16 else torch.float32
        self.k, self.v = (torch.full((n_pages, page, self.n_kv, self.hd), float("nan"), dtype=dt,
                                     device=dev) for _ in range(2))
        self.q_in = torch.randn((n_tok, self.n_q, self.hd), device=dev, generator=g)
        self.k_in = torch.randn((n_tok, self.n_kv, self.hd), device=dev, generator=g)
        self.v_in = torch.randn((n_tok, self.n_kv * self.hd), device=dev, generator=g)
        self.q, self.kr = torch.empty_like(self.q_in), torch.empty_like(self.k_in)
        self.out = torch.zeros_like(self.q)
        self.w = torch.ones(self.hd, device=dev)
        self.head = torch.randn((self.n_q * self.hd, self.vocab), device=dev, generator=g) * 0.1
        self.logits = torch.zeros((n_tok, self.vocab), device=dev)
        self.tokens = z(n_tok)
        self.plan = bh.make_paged_plan_args(
            self.cached, self.new, self.table, self.free, self.n_free, page, kv_len=self.kv_len,
            q_start=self.q_start, slots=self.slots, pos=self.pos, n_refused=self.refused)
        self.qk = bh.make_qk_args(self.q_in, self.q, self.k_in, self.kr, self.w, self.w, self.pos,
                                  n_tok, self.n_q, self.n_kv, head_dim=self.hd, n_dims=32,
                                  sections=(8, 4, 4, 0))
        self.cache = bh.make_paged_cache(self.k, self.v)
        self.attn = bh.make_attention_paged_args(self.cache, self.q, self.q_start, self.kv_len,
                                                 self.table, out=self.out)
        self.lp = bh.make_token_logprobs_args(self.logits, self.tokens, n_top=4)

    def step(self, stream=None):
        import torch
        bh = self.bh
        bh.paged_plan(self.plan, stream=stream)
        bh.qk_norm_rope(self.qk, stream=stream)
        bh.kv_store_paged(self.cache, self.kr.view(len(self.slots), -1), self.v_in, self.slots,
                          stream=stream)
        bh.attention_paged(self.attn, stream=stream)
        torch.mm(self.out.view(len(self.slots), -1), self.head, out=self.logits)
        bh.token_logprobs(self.lp, stream=stream)
        self.cached.copy_(self.kv_len)

    def results(self):
        return [t.clone() for t in (self.kv_len, self.q_start, self.slots, self.table, self.out,
                                    self.logits, *self.lp.results)]


STEPS = [  # new tokens of the six requests, step by step
    [5, 3, 0, 0, 1, 0], [1, 1, 4, 0, 1, 0], [1, 1, 1, 7, 1, 0], [1, -1, 1, 1, 1, 0],
    [1, 6, 1, 1, -1, 0], [-1, 1, 1, 1, 2, 3], [4, 1, 1, 1, 1, 1],
]


def _drive(e, new, inputs):
    import torch
    e.new.copy_(torch.tensor(new, dtype=torch.int32))
    e.q_in.copy_(inputs[0]), e.k_in.copy_(inputs[1]), e.v_in.copy_(inputs[2])
    e.tokens.copy_(inputs[3])


def _inputs(e, dev):
    import torch
    g = torch.Generator(dev).manual_seed(9)
    return [(torch.randn(e.q_in.shape, device=dev, generator=g),
             torch.randn(e.k_in.shape, device=dev, generator=g),
             torch.randn(e.v_in.shape, device=dev, generator=g),
             torch.randint(0, e.vocab, e.tokens.shape, device=dev, generator=g).int())
            for _ in STEPS]


@pytest.mark.parametrize("f16", [True, False])
def test_steps_against_plain_caches(bh, dev, f16):
    """Requests come, grow, are released and come again; each keeps a plain list
    of its k and v rows on the host.  The pool starts as NaN, and pages return
    with what the requests before left in them."""
    import torch
    e = Engine(bh, dev, f16=f16)
    rows = [([], []) for _ in range(6)]
    for new, x in zip(STEPS, _inputs(e, dev)):
        _drive(e, new, x)
        e.step()
        torch.cuda.synchronize()
        assert e.refused.item() == 0
        start, q = e.q_start.cpu().numpy(), e.q.cpu().numpy().astype(np.float64)
        kr, vr = e.kr.cpu().numpy(), e.v_in.view(-1, e.n_kv, e.hd).cpu().numpy()
        dt = np.float16 if f16 else np.float32
        out = e.out.cpu().numpy()
        for r, n in enumerate(new):
            if n < 0:
                rows[r] = ([], [])
                n = 0
            assert start[r + 1] - start[r] == n
            for t in range(start[r], start[r + 1]):
                rows[r][0].append(kr[t].astype(dt).astype(np.float64))
                rows[r][1].append(vr[t].astype(dt).astype(np.float64))
                k, v = np.array(rows[r][0]), np.array(rows[r][1])
                for h in range(e.n_q):
                    s = k[:, h // 4] @ q[t, h] / np.sqrt(e.hd)
                    w = np.exp(s - s.max())
                    want = (w[:, None] * v[:, h // 4]).sum(0) / w.sum()
                    assert np.abs(out[t, h] - want).max() <= TOL * max(1, np.abs(want).max())
            assert e.kv_len[r].item() == len(rows[r][0])
        # log probabilities of what the step's head gives
        lp, ent, ids, top = pd.logprobs(e.logits.cpu().numpy(), e.tokens.cpu().numpy(), 4, 1.0)
        got = [t.cpu().numpy() for t in e.lp.results]
        assert np.abs(got[0] - lp).max() < 1e-5 and np.abs(got[1] - ent).max() < 1e-5
        assert np.array_equal(got[2], ids) and np.abs(got[3] - top).max() < 1e-5


def test_captured_step_replays(bh, dev):
    """One graph of the whole step, replayed over steps whose lengths differ,
    with eager work between; the eager engine's results, bit for bit."""
    import torch
    eager, graphed = Engine(bh, dev), Engine(bh, dev)
    xs = _inputs(eager, dev)
    warm = Engine(bh, dev)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        _drive(warm, STEPS[0], xs[0])
        warm.step(stream=st)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        graphed.step(stream=st)
    torch.cuda.synchronize()
    for i, (new, x) in enumerate(zip(STEPS, xs)):
        _drive(eager, new, x)
        eager.step()
        torch.cuda.synchronize()
        want = eager.results()
        _drive(graphed, new, x)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        end = int(want[1][-1])
        for n, (a, b) in enumerate(zip(graphed.results(), want)):
            if a.dim() and a.shape[0] == len(eager.slots) and n > 3:
                a, b = a[:end], b[:end]
            assert torch.equal(a, b), (i, n)
