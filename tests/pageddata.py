"""A serving step over a paged cache in plain numpy: the plan as a loop over
requests, attention and log probabilities in 64 bits.  Inputs for their tests."""
from __future__ import annotations

import numpy as np


def plan(cached, new, table, free, n_free, page, n_tok):
    """(kv_len, q_start, slots, pos, table, free, n_free, refused), one request
    and one page at a time, as include/bonsai_hip_serve.h describes it."""
    table, free = table.copy(), free.copy()
    n_req, width = table.shape
    n_pages = len(free)
    n_free = min(max(int(n_free), 0), n_pages)
    cached = [max(int(c), 0) for c in cached]
    for i in range(n_req):
        if new[i] < 0:
            for b in range(min(-(-cached[i] // page), width)):
                if n_free < n_pages:
                    free[n_free] = table[i, b]
                    n_free += 1
    stack, pages, toks, refused = n_free, 0, 0, 0
    kv_len, start, slots, pos = [], [0], [], []
    for i in range(n_req):
        n, length = int(new[i]), 0
        if n >= 0:
            have = -(-cached[i] // page)
            need = -(-(cached[i] + n) // page) - have
            ok = cached[i] + n <= width * page
            if ok:
                pages += need
                toks += n
                ok = not (need > 0 and pages > stack) and not (n > 0 and toks > n_tok)
            if ok:
                for b in range(have, have + need):
                    n_free -= 1
                    table[i, b] = free[n_free]
                length = cached[i] + n
                for p in range(cached[i], length):
                    at = int(table[i, p // page])
                    slots.append(at * page + p % page if 0 <= at < n_pages else -1)
                    pos.append([p] * 4)
            else:
                refused += 1
                n = 0
        else:
            n = 0
        kv_len.append(length)
        start.append(start[-1] + n)
    while len(slots) < n_tok:
        slots.append(-1)
        pos.append([0] * 4)
    i32 = np.int32
    return (np.array(kv_len, i32), np.array(start, i32), np.array(slots, i32),
            np.array(pos, i32).reshape(n_tok, 4), table, free, n_free, refused)


def attention(q, k, v, start, kv_len, table, out):
    """out [n_tok, n_head, hd] in 64 bits; k, v [page, position, head, dim]."""
    out = out.astype(np.float64)
    n_pages, page, n_kv, hd = k.shape
    group = q.shape[1] // n_kv
    for r, length in enumerate(kv_len):
        a, b = int(start[r]), int(start[r + 1])
        pages = table[r, :-(-int(length) // page)]
        good = (pages >= 0) & (pages < n_pages)
        at = np.where(good, pages, 0)
        kr = k[at].reshape(-1, n_kv, hd)[:length].astype(np.float64)
        vr = v[at].reshape(-1, n_kv, hd)[:length].astype(np.float64)
        there = np.repeat(good, page)[:length]
        for t in range(a, b):
            p = int(length) - (b - a) + (t - a)
            sees = np.nonzero(there[:max(p + 1, 0)])[0]
            for h in range(q.shape[1]):
                if len(sees) == 0:
                    out[t, h] = 0.0
                    continue
                with np.errstate(invalid="ignore"):
                    s = kr[sees, h // group] @ q[t, h].astype(np.float64) / np.sqrt(hd)
                    w = np.exp(s - s.max())
                    out[t, h] = (w[:, None] * vr[sees, h // group]).sum(0) / w.sum()
    return out


def logprobs(x, tokens, n_top, inv_temp):
    """(logprob, entropy, top ids, top logprobs) in 64 bits."""
    z = x.astype(np.float64) * inv_temp
    with np.errstate(all="ignore"):
        top = z.max(1, keepdims=True)
        z = z - top  # against the maximum first: log Z is lost beside a row of -3e38
        e = np.exp(z)
        p = z - np.log(e.sum(1, keepdims=True))
        pr = np.exp(p)
        entropy = -np.where(pr > 0, pr * np.where(pr > 0, p, 0), 0.0).sum(1)
    bad = ~np.isfinite(top[:, 0])
    p[bad] = np.nan
    entropy[bad] = np.nan
    order = np.where(np.isnan(x), -np.inf, x)
    # NaN below -inf, then by id
    rank = np.lexsort((np.broadcast_to(np.arange(x.shape[1]), x.shape), np.isnan(x), -order))
    ids = rank[:, :n_top]
    rows = np.arange(len(x))
    in_row = tokens < x.shape[1]
    lp = np.where(in_row, p[rows, np.where(in_row, tokens, 0)], np.nan)
    return lp, entropy, ids, np.take_along_axis(p, ids, 1)


def pages(rng, lens, page, width=None, spare=3):
    """(table [n_req, width] of shuffled pages, -1 behind; pages in the pool)."""
    have = [-(-int(n) // page) for n in lens]
    width = max(have + [1]) if width is None else width
    total = sum(have)
    order = rng.permutation(total + spare).astype(np.int32)
    table = np.full((len(lens), width), -1, np.int32)
    at = 0
    for r, h in enumerate(have):
        table[r, :h] = order[at:at + h]
        at += h
    return table, total + spare
