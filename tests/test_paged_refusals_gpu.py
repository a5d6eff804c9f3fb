"""Steps of a small server whose pool and token slots run out: refused requests keep
their pages and rows and are sent again."""
from __future__ import annotations

import numpy as np
import pytest

from test_paged_gpu import TOL, Engine, _drive, _inputs

pytestmark = pytest.mark.gpu


class Server(Engine):
    """Carries a refused request over: its length stays what it was."""

    def step(self, stream=None):
        import torch
        before = self.cached.clone()
        super().step(stream)
        self.cached.copy_(torch.where((self.kv_len > 0) | (self.new < 0), self.kv_len, before))


STEPS = [  # new tokens of the six requests; pages of 4, 14 of them, 12 tokens a step
    [5, 3, 0, 0, 1, 0], [1, 1, 7, 0, 1, 0], [1, 1, 1, 9, 0, 0], [1, 1, 1, 1, 9, 0],
    [1, 1, 1, 1, 8, 0], [1, 1, 1, 1, 1, 2], [1, 1, 1, 1, 1, 2], [-1, 1, 1, 1, 1, 2],
    [0, -1, 1, 1, 1, 2], [3, 2, 1, 1, -1, 1],
]
REFUSED = [[], [], [], [4], [], [5], [1, 3, 5], [4, 5], [], []]


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("graphed", [False, True])
def test_steps_with_refusals(bh, dev, graphed, f16):
    import torch
    e = Server(bh, dev, n_pages=14, f16=f16)
    xs = _inputs(e, dev) * 2
    if graphed:
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            Server(bh, dev, n_pages=14, f16=f16).step(stream=st)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            e.step(stream=st)
        torch.cuda.synchronize()
    rows = [([], []) for _ in range(6)]
    dt = np.float16 if f16 else np.float32
    for new, x, refused in zip(STEPS, xs, REFUSED):
        _drive(e, new, x)
        torch.cuda.synchronize()
        g.replay() if graphed else e.step()
        torch.cuda.synchronize()
        assert e.refused.item() == len(refused)
        start, kv_len = e.q_start.cpu().numpy(), e.kv_len.cpu().numpy()
        q, out = e.q.cpu().numpy().astype(np.float64), e.out.cpu().numpy()
        kr, vr = e.kr.cpu().numpy(), e.v_in.view(-1, e.n_kv, e.hd).cpu().numpy()
        for r, n in enumerate(new):
            if n < 0:
                rows[r] = ([], [])
                n = 0
            if r in refused:
                assert kv_len[r] == 0 and n > 0
                n = 0
            else:
                assert kv_len[r] == len(rows[r][0]) + n
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
        # no page is lost or held twice
        cached, table = e.cached.cpu().numpy(), e.table.cpu().numpy()
        assert cached.tolist() == [len(k) for k, _ in rows]
        held = [int(p) for r in range(6) for p in table[r, :-(-cached[r] // 4)]]
        held += e.free.cpu().tolist()[:e.n_free.item()]
        assert sorted(held) == list(range(14))
