"""Attention over a shared prefix under offsets that leave a group without tokens while
one of its requests has some: where a group's prefix lies is written by every call, so
that nothing which a workspace held before is taken for it."""
from __future__ import annotations

import numpy as np
import pytest

from test_attention_shared_gpu import _args, _case, _check

pytestmark = pytest.mark.gpu


def _records(ws, n_group):
    """What the workspace begins with: a group's launch, first tile, first token, tokens."""
    import torch
    return ws[:16 * n_group].view(torch.int32).reshape(n_group, 4).cpu().numpy()


# offsets, and the tokens of the two groups (requests 0, 1 and 2, 3, 4)
OFFSETS = [
    ([0, 2, 0, 1, 2, 3], [0, 3]),    # request 0 has 2 tokens, its group 0 - 0
    ([5, 7, 3, 4, 5, 6], [0, 3]),    # 3 - 5
    ([0, 1, 2, 6, 3, 2], [2, 0]),    # request 2 has 4, its group 2 - 2
    ([4, 6, 2, 5, 3, 2], [0, 0]),    # both
    ([0, None, 0, None, 0, None], [0, 0]),  # more than the call has: nothing is done
]


@pytest.mark.parametrize("fill", [0xFF, 0x7F, 0x01])
@pytest.mark.parametrize("columns", [0, 20000])  # one form for all requests, and two
@pytest.mark.parametrize("nth", range(len(OFFSETS)))
def test_groups_without_tokens(bh, dev, nth, columns, fill):
    import torch
    offsets, tokens = OFFSETS[nth]
    new = 40 if columns else 2  # (two forms: of requests of more than 64 rows)
    c = _case([(64, [(64, new), (67, 1)]), (48, [(69, 1)] * 3)], n_head=8, n_kv=2, hd=128)
    c["table"] = np.concatenate([c["table"], np.full((5, columns), -1, np.int32)], 1)
    c["q"] = np.concatenate([c["q"], c["q"][:4]])
    good = dict(c)
    offsets = [len(c["q"]) if o is None else o for o in offsets]
    c["q_start"] = np.array(offsets, np.int32)
    print(offsets, columns, fill, flush=True)
    ws = torch.empty(bh.attention_shared_workspace(_args(bh, dev, c)), dtype=torch.uint8, device=dev)
    ws.fill_(fill)
    args = _args(bh, dev, c, workspace=ws)
    out = bh.attention_shared(args)
    torch.cuda.synchronize()
    for g, (launch, base, q0, n) in enumerate(_records(ws, 2)):
        assert launch in (0, 1) and n == tokens[g], (g, launch, n)
        assert 0 <= base and 0 <= q0 <= len(c["q"])
    # rows of no request stay as they were
    named = np.zeros(len(c["q"]), bool)
    for a, b in zip(offsets, offsets[1:]):
        named[a:max(b, a)] = True
    assert bool((out.cpu().numpy()[~named] == -7.0).all())
    # and the same workspace serves the next call
    _check(bh, dev, good, workspace=ws)
