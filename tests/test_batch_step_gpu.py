"""Beam search of a small hybrid model, the calls in a row as a server makes them: plan,
conv, delta rule, append, attention over the shared prompt, selection, reordering, copies;
against numpy in 64 bits beam by beam, and captured once and replayed.

Tolerances, of the largest value: the conv's 1e-6 (see batchdata.conv) goes into the
delta rule, which is held to 1e-5 by itself, so 2e-5; attention sums at most 80 values
over f16 keys that are the same on both sides, 2^-21 a weight (its hi + lo halves and its
exponential): 1e-5."""
from __future__ import annotations

import numpy as np
import pytest

import batchdata as bd
from conftest import rel_err

pytestmark = pytest.mark.gpu

GROUPS, WIDTH, PAGE, SHARED = 2, 4, 16, [32, 48]
ROWS, H_K, H_V, S, TAPS = GROUPS * WIDTH, 2, 4, 128, 4
CH, L2 = (2 * H_K + H_V) * S, 2 * H_K * S
Q_HEADS, HEADS, HD, VOCAB, STEPS = 6, 2, 64, 1000, 20


class Beams:
    """The buffers of a server of ROWS beams; x, gate, .. are a step's inputs."""

    def __init__(self, bh, dev):
        import torch
        self.bh, rng = bh, np.random.default_rng(5)
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)
        f = lambda *shape: t(rng.standard_normal(shape).astype(np.float32))
        z = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=dev)
        self.w, self.conv_state = f(CH, TAPS) * 0.5, f(2 * ROWS, CH, TAPS - 1)
        self.state = f(2 * ROWS, H_V, S, S) * 0.2
        # groups' first pages are the same; the rest come from the stack
        width, pages = 8, 64
        table = np.full((ROWS, width), -1, np.int32)
        at = 0
        for g, n in enumerate(SHARED):
            table[g * WIDTH:(g + 1) * WIDTH, :n // PAGE] = np.arange(at, at + n // PAGE)
            at += n // PAGE
        self.k, self.v = (t(rng.standard_normal((pages, PAGE, HEADS, HD)).astype(np.float16))
                          for _ in range(2))
        free = np.full(pages, -1, np.int32)  # a stack as large as the pool
        free[:pages - at] = np.arange(at, pages)
        self.table, self.free = t(table), t(free)
        self.n_free = t(np.array([pages - at], np.int32))
        cached = np.repeat(SHARED, WIDTH).astype(np.int32)
        self.cached, self.begin = t(cached), t(cached)
        self.one, self.kv_len, self.q_start = z(ROWS) + 1, z(ROWS), z(ROWS + 1)
        self.slots = z(ROWS)
        order = rng.permutation(2 * ROWS).astype(np.int32)
        self.dst, self.spare = t(order[:ROWS]), t(order[ROWS:])
        self.src, self.copy_from = self.spare.clone(), z(ROWS)
        self.group = t(np.repeat(np.arange(GROUPS), WIDTH).astype(np.int32))
        self.group_start = t(np.arange(0, ROWS + 1, WIDTH, dtype=np.int32))
        self.shared = t(np.array(SHARED, np.int32))
        self.score = t(np.where(np.arange(ROWS) % WIDTH == 0, 0, -np.inf).astype(np.float32))
        self.x, self.gate, self.beta = f(ROWS, CH), -f(ROWS, H_V).abs(), f(ROWS, H_V).sigmoid()
        self.q = f(ROWS, Q_HEADS, HD)
        self.k_new, self.v_new = f(ROWS, HEADS * HD), f(ROWS, HEADS * HD)
        self.logits = f(ROWS, VOCAB)
        cache = bh.make_paged_cache(self.k, self.v)
        self.cache = cache
        self.plan = bh.make_paged_plan_args(
            self.cached, self.one, self.table, self.free, self.n_free, PAGE,
            kv_len=self.kv_len, q_start=self.q_start, slots=self.slots)
        self.conv = bh.make_conv_ragged_args(self.x, self.w, self.conv_state, self.q_start,
                                             self.src, self.dst, l2_dim=L2, head_dim=S, max_new=1)
        c, n = self.conv.out_tensor, H_K * S
        self.gdn = bh.make_gdn_ragged_args(
            c[:, :n].unflatten(1, (H_K, S)), c[:, n:2 * n].unflatten(1, (H_K, S)),
            c[:, 2 * n:].unflatten(1, (H_V, S)), self.gate, self.beta, self.state, self.q_start,
            self.src, self.dst, max_new=1)
        def shared(ws=None):
            return bh.make_attention_shared_args(
                cache, self.q, self.q_start, self.kv_len, self.table, self.group,
                self.group_start, self.shared, out=self.out, max_new=1, max_group_new=WIDTH,
                workspace=ws)
        self.out = torch.zeros_like(self.q)
        own = torch.empty(bh.attention_shared_workspace(shared()), dtype=torch.uint8, device=dev)
        self.attn = shared(own)

        def select(ws=None):
            return bh.make_beam_select_args(self.logits, self.score, WIDTH, WIDTH,
                                            score_out=self.score, parent=self.parent,
                                            token=self.token, workspace=ws)
        self.parent, self.token = z(GROUPS, WIDTH), z(GROUPS, WIDTH)
        own = torch.empty(bh.beam_select_workspace(select()), dtype=torch.uint8, device=dev)
        self.select = select(own)
        self.reorder = bh.make_beam_reorder_args(
            self.parent, self.table, copy_from=self.copy_from, src_slot=self.src,
            dst_slot=self.dst, spare_slot=self.spare)
        self.copy = bh.make_kv_copy_args(cache, self.table, self.copy_from, self.begin,
                                         self.kv_len)

    def step(self, stream=None):
        bh = self.bh
        bh.paged_plan(self.plan, stream)
        bh.conv1d_silu_ragged(self.conv, stream)
        bh.gdn_ragged(self.gdn, stream)
        bh.kv_store_paged(self.cache, self.k_new, self.v_new, self.slots, stream)
        bh.attention_shared(self.attn, stream)
        bh.beam_select(self.select, stream)
        bh.beam_reorder(self.reorder, stream)
        bh.kv_copy_paged(self.copy, stream)

    def inputs(self, i, dev):
        import torch
        g = torch.Generator().manual_seed(100 + i)
        for t in (self.x, self.q, self.k_new, self.v_new, self.logits):
            t.copy_(torch.randn(t.shape, generator=g))
        self.logits.mul_(2.0)
        self.gate.copy_(-torch.rand(self.gate.shape, generator=g))
        self.beta.copy_(torch.rand(self.beta.shape, generator=g))
        if i:
            self.cached.add_(1)

    def results(self):
        return [t.clone() for t in (self.conv.out_tensor, self.gdn.attn_tensor, self.out,
                                    self.parent, self.token, self.score, self.table,
                                    self.copy_from, self.src, self.dst, self.spare, self.kv_len)]


def test_beams_against_numpy(bh, dev):
    import torch
    b = Beams(bh, dev)
    np_ = lambda t: t.cpu().numpy()
    src = np_(b.src)
    window, m = np_(b.conv_state)[src], np_(b.state)[src].astype(np.float64)
    table = np_(b.table)
    past = [[np_(c)[table[r, :SHARED[r // WIDTH] // PAGE]].reshape(-1, HEADS, HD).astype(np.float64)
             for c in (b.k, b.v)] for r in range(ROWS)]
    w, one, rows = np_(b.w), np.arange(ROWS + 1, dtype=np.int32), np.arange(ROWS, dtype=np.int32)
    for i in range(STEPS):
        b.inputs(i, dev)
        score = np_(b.score).copy()
        b.step()
        torch.cuda.synchronize()
        conv, attn, out, parent, token, got_score = map(np_, b.results()[:6])
        want, window, _ = bd.conv(np_(b.x), w, window, one, rows, rows, np.zeros((ROWS, CH)),
                                  l2_dim=L2, head_dim=S)
        assert rel_err(conv, want) < 2e-6, i
        n = H_K * S
        want, m = bd.gdn(want[:, :n].reshape(ROWS, H_K, S), want[:, n:2 * n].reshape(ROWS, H_K, S),
                         want[:, 2 * n:].reshape(ROWS, H_V, S), np_(b.gate), np_(b.beta), m, one,
                         rows, rows, np.zeros((ROWS, H_V, S)))
        assert rel_err(attn, want) < 2e-5, i
        new = [np_(t).astype(np.float16).astype(np.float64).reshape(ROWS, HEADS, HD)
               for t in (b.k_new, b.v_new)]
        past = [[np.concatenate([p, x[r:r + 1]]) for p, x in zip(past[r], new)]
                for r in range(ROWS)]
        want = np.zeros((ROWS, Q_HEADS, HD))
        for r, (k, v) in enumerate(past):
            for h in range(Q_HEADS):
                z = k[:, h // 3] @ np_(b.q)[r, h].astype(np.float64) / np.sqrt(HD)
                e = np.exp(z - z.max())
                want[r, h] = e @ v[:, h // 3] / e.sum()
        assert rel_err(out, want) < 1e-5, i
        for g, (s, of, toks) in enumerate(bd.continuations(np_(b.logits), score, WIDTH, 1.0)):
            assert np.array_equal(parent[g], of[:WIDTH]), i
            assert np.array_equal(token[g], toks[:WIDTH]), i
            assert np.all(np.abs(got_score[g * WIDTH:][:WIDTH] - s[:WIDTH]) <= 2e-6 + np.abs(s[:WIDTH]) * 2.0 ** -24)
        of = parent.reshape(-1)
        window, m = window[of], m[of]
        past = [[c.copy() for c in past[r]] for r in of]
    # the cache that the tables name is the beams' own
    table, k, v = np_(b.table), np_(b.k), np_(b.v)
    for r in range(ROWS):
        n = len(past[r][0])
        for cache, want in ((k, past[r][0]), (v, past[r][1])):
            got = cache[table[r, :-(-n // PAGE)]].reshape(-1, HEADS, HD)[:n]
            assert np.array_equal(got.astype(np.float64), want), r


def test_step_captured_and_replayed(bh, dev):
    """The eager engine's results, bit for bit, eager work between the replays."""
    import torch
    eager, graphed, warm = (Beams(bh, dev) for _ in range(3))
    st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        warm.inputs(0, dev)
        warm.step(st)
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        graphed.step(st)
    torch.cuda.synchronize()
    for i in range(STEPS):
        eager.inputs(i, dev)
        eager.step()
        torch.cuda.synchronize()
        want = eager.results()
        graphed.inputs(i, dev)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for n, (a, b) in enumerate(zip(graphed.results(), want)):
            assert torch.equal(a, b), (i, n)
    assert torch.equal(eager.k, graphed.k) and torch.equal(eager.v, graphed.v)
    assert torch.equal(eager.state[eager.src.long()], graphed.state[graphed.src.long()])
