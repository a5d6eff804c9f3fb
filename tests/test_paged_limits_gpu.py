"""The plan at the largest pool that its indexes hold."""
from __future__ import annotations

import pytest

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
