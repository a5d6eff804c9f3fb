"""A conv of one tap has no state, so no slot of it is bad: whatever the slots are, outputs
are those of the formula and nothing is noted.  Tolerance: batchdata.conv's bound."""
from __future__ import annotations

import numpy as np
import pytest

import batchdata as bd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("slots", [0, 3, -1, 2 ** 31 - 1])
@pytest.mark.parametrize("ch,l2_dim,head_dim", [(33, 0, 0), (64, 32, 16)])
def test_one_tap(bh, dev, ch, l2_dim, head_dim, slots):
    import torch
    rng = np.random.default_rng(ch + l2_dim)
    new = [1, 0, 5, 2]
    start = bd.offsets(new)
    n = int(start[-1])
    x, w = (rng.standard_normal(s).astype(np.float32) for s in ((n + 1, ch), (ch, 1)))
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)
    src = np.full(4, slots, np.int32)
    bad = torch.full((1,), -7, dtype=torch.int32, device=dev)
    args = bh.make_conv_ragged_args(t(x), t(w), None, t(start), t(src), t(src), l2_dim=l2_dim,
                                    head_dim=head_dim, bad_slot=bad,
                                    out=torch.full((n + 1, ch), -7.0, device=dev))
    out = bh.conv1d_silu_ragged(args)
    torch.cuda.synchronize()
    assert bad.item() == -7
    want, _, bound = bd.conv(x, w, np.zeros((4, ch, 0), np.float32), start, src, src,
                             np.full((n + 1, ch), -7.0), l2_dim, head_dim)
    got = out.cpu().numpy()
    assert np.all(got[n:] == -7.0)
    assert np.all(np.abs(got[:n] - want[:n]) <= bound[:n])
