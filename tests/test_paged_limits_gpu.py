"""The paged calls where counts are largest: the plan over the largest pool that its
indexes hold, attention with offsets that ask for more than there is."""
from __future__ import annotations

import numpy as np
import pytest

from test_paged_gpu import TOL, _attend, _step, _want
from conftest import rel_err

pytestmark = pytest.mark.gpu


def test_plan_releases_the_largest_pool(bh, dev):
    """One request gives back 2^31 - 1 pages of one position: the last round of the
    block's threads ends past 2^31."""
    import torch
    n = (1 << 31) - 1
    i32 = dict(dtype=torch.int32, device=dev)
    table = torch.arange(n, **i32).view(1, n)
    free = torch.full((n,), -1, **i32)
    one = lambda x: torch.tensor([x], **i32)  # noqa: E731
    out = dict(kv_len=one(-7), q_start=torch.full((2,), -7, **i32),
               slots=torch.full((129,), -7, **i32), n_free_out=one(-7), n_refused=one(-7))
    args = bh.make_paged_plan_args(one(n), one(-1), table, free, one(0), 1, **out)
    print("releasing", n, flush=True)
    bh.paged_plan(args)
    torch.cuda.synchronize()
    assert out["n_free_out"].item() == n and out["n_refused"].item() == 0
    assert out["kv_len"].item() == 0 and out["q_start"].tolist() == [0, 0]
    assert (out["slots"] == -1).all()
    assert torch.equal(free, table[0])


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n_req,max_new", [(64, 1), (64, 4), (64, 40), (1000, 1), (1000, 40)])
def test_offsets_that_ask_for_too_much(bh, dev, n_req, max_new, f16):
    """Offsets that go back and forth between 0 and n_tok would have every other
    request attend all tokens: work, tiles and counts without a bound.  Such a call does
    nothing; the next one, whose offsets are in order, is as it should be."""
    rng = np.random.default_rng(n_req + max_new)
    lens = [300] * n_req
    s = _step(rng, dev, lens, [1] * 40 + [0] * (n_req - 40), 16, 8, 2, 64, f16, pad=2)
    start = s["start"]
    s["start"] = np.array([0, 40] * (n_req // 2) + [0], np.int32)
    assert (_attend(bh, dev, s, max_new=max_new)[0] == 5.25).all()
    s["start"] = np.array([0, 40] * (n_req // 2) + [40], np.int32)  # back only within
    assert (_attend(bh, dev, s, max_new=max_new)[0] == 5.25).all()
    s["start"] = start
    got = _attend(bh, dev, s, max_new=max_new)[0]
    assert rel_err(got, _want(s).astype(np.float32)) <= TOL
