"""The recurrent layers of many requests and beam search in plain numpy, 64 bits, one
request, token and beam at a time, as include/bonsai_hip_batch.h describes them."""
from __future__ import annotations

import numpy as np


def slot(i, n_slots):
    return int(i) if 0 <= i < n_slots else -1


def conv(x, w, state, start, src, dst, out, l2_dim=0, head_dim=0, eps=1e-6):
    """(out, state, bound): outputs, the slots (f32, exact), and how far rounding may
    move an output.  The k products and sums of a channel are f32, each off by half a
    step of what it holds, at most sum |w x| 2^-24: (2 k + 1) of them; silu moves that by
    at most 1.1 and adds 8 steps of its own (exponential, reciprocal, products).  A norm's
    relative error is at most that of its largest part; scaling adds 4 steps."""
    out, state, old = out.astype(np.float64), state.copy(), state.copy()
    bound = np.zeros_like(out)
    k, n_slots = w.shape[1], len(state)
    u = 2.0 ** -24
    for r in range(len(src)):
        a, b = int(start[r]), int(start[r + 1])
        if a >= b:
            continue
        s = slot(src[r], n_slots)
        past = old[s].T if s >= 0 else np.zeros((k - 1, w.shape[0]), np.float32)
        line = np.concatenate([past, x[a:b]])
        for t in range(a, b):
            win = line[t - a:t - a + k].T.astype(np.float64)
            acc = (win * w).sum(1)
            y = acc / (1.0 + np.exp(-acc))
            e = 1.1 * (2 * k + 1) * u * np.abs(win * w).sum(1) + 8 * u * np.abs(y)
            for g in range(0, l2_dim, head_dim or 1):
                z = y[g:g + head_dim]
                norm = max(np.sqrt((z * z).sum()), eps)
                off = np.sqrt((e[g:g + head_dim] ** 2).sum()) / norm
                y[g:g + head_dim] = z / norm
                e[g:g + head_dim] = e[g:g + head_dim] / norm + np.abs(z / norm) * (off + 4 * u)
            out[t], bound[t] = y, e
        d = slot(dst[r], n_slots)
        if d >= 0 and k > 1:
            state[d] = line[len(line) - k + 1:].T
    return out, state, bound


def gdn(q, k, v, gate, beta, state, start, src, dst, attn):
    """(attn, state) in 64 bits."""
    attn, old = attn.astype(np.float64), state.astype(np.float64)
    new = old.copy()
    h_k, h_v, s = q.shape[1], v.shape[1], q.shape[2]
    head = np.arange(h_v) % h_k
    q, k, v, gate, beta = (a.astype(np.float64) for a in (q, k, v, gate, beta))
    for r in range(len(src)):
        a, b = int(start[r]), int(start[r + 1])
        if a >= b:
            continue
        f = slot(src[r], len(state))
        m = old[f].copy() if f >= 0 else np.zeros_like(old[0])
        for t in range(a, b):
            m *= np.exp(gate[t])[:, None, None]
            delta = (v[t] - np.einsum("hji,hi->hj", m, k[t, head])) * beta[t][:, None]
            m += delta[:, :, None] * k[t, head][:, None, :]
            attn[t] = np.einsum("hji,hi->hj", m, q[t, head]) / np.sqrt(s)
        d = slot(dst[r], len(state))
        if d >= 0:
            new[d] = m
    return attn, new


def continuations(x, score, width, inv_temp):
    """Of each group, (score, row, token) of all continuations, best first; a row's own
    in the order of its logits, which a score of -3e38 would swallow in 64 bits too."""
    groups = []
    with np.errstate(all="ignore"):
        for g in range(0, len(x), width):
            rows, toks, scores, logits = [], [], [], []
            for r in range(g, g + width):
                z = x[r].astype(np.float64)
                m = z.max() if not np.isnan(z).any() else np.nan
                if not np.isfinite(m) or not np.isfinite(score[r]):
                    continue
                z = (z - m) * np.float64(np.float32(inv_temp))
                s = float(score[r]) + (z - np.log(np.exp(z).sum()))
                t = np.nonzero(s > -np.inf)[0]
                rows.append(np.full(len(t), r)), toks.append(t), scores.append(s[t])
                logits.append(x[r][t])
            if not rows:
                groups.append((np.zeros(0), np.zeros(0, int), np.zeros(0, int)))
                continue
            rows, toks, scores = map(np.concatenate, (rows, toks, scores))
            order = np.lexsort((toks, -np.concatenate(logits), rows, -scores))
            groups.append((scores[order], rows[order], toks[order]))
    return groups


def reorder(parent, table, dst, spare, width):
    """(table, copy_from, src, dst, spare): one group and one beam at a time."""
    table, old = table.copy(), table.copy()
    n = len(table)
    copy, src = np.full(n, -1, np.int32), np.zeros(n, np.int32)
    for g in range(0, n, width):
        ps = [int(p) if g <= p < g + width else -1 for p in parent[g // width]]
        heir = {}
        for i, p in enumerate(ps):
            if p >= 0:
                heir.setdefault(p, i)
        free = iter(r for r in range(g, g + width) if r not in heir)
        for i, p in enumerate(ps):
            if p >= 0 and heir[p] == i:
                table[g + i] = old[p]
            else:
                table[g + i] = old[next(free)]
                copy[g + i] = g + heir[p] if p >= 0 else -1
            src[g + i] = dst[p if p >= 0 else g + i]
    return table, copy, src, spare.copy(), dst.copy()


def copy_pages(k, v, table, copy, begin, end):
    """K and V [page][position][head][dim] after the copies."""
    n_pages, page = k.shape[:2]
    k, v = k.copy(), v.copy()
    k0, v0 = k.copy(), v.copy()
    for i, of in enumerate(copy):
        if not 0 <= of < len(copy):
            continue
        for p in range(max(int(begin[i]), 0), min(max(int(end[i]), 0), table.shape[1] * page)):
            to, fr = int(table[i, p // page]), int(table[of, p // page])
            if 0 <= to < n_pages and 0 <= fr < n_pages and to != fr:
                k[to, p % page], v[to, p % page] = k0[fr, p % page], v0[fr, p % page]
    return k, v


def offsets(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
