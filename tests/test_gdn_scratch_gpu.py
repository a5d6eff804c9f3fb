"""bh_gdn_step's and bh_gdn_ragged's prompts on two streams at once, both in the library's
scratch, which is each one's own: the bits of the calls by themselves."""
from __future__ import annotations

import numpy as np
import pytest

from test_gdn_ragged_gpu import _case, _t, _views

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("h_k,h_v", [(2, 6), (16, 48)])
def test_a_prompt_of_one_sequence_beside_a_batch(bh, dev, h_k, h_v):
    import torch
    s = 128
    one, many = _case([513], h_k, h_v, s), _case([300, 1, 64, 200], h_k, h_v, s, seed=1)

    def parts(c):
        rows = _t(c["rows"], dev)
        q, k, v = (rows[:, i:j].unflatten(1, (-1, s)) for i, j in (
            (0, h_k * s), (h_k * s, 2 * h_k * s), (2 * h_k * s, (2 * h_k + h_v) * s)))
        return q, k, v, _t(c["gate"], dev), _t(c["beta"], dev)

    step = [_t(x, dev) for x in (*_views(one), one["gate"], one["beta"])]
    state = _t(one["pool"][0].reshape(h_v, s, s), dev)
    pool = _t(many["pool"], dev)
    attn = torch.full((len(many["rows"]), h_v, s), -7.0, device=dev)
    args = bh.make_gdn_ragged_args(*parts(many), pool.unflatten(1, (h_v, s, s)),
                                   *(_t(many[n], dev) for n in ("start", "src", "dst")), attn=attn)
    streams = [torch.cuda.Stream() for _ in range(2)]
    rounds = 6

    def run(together):
        states = [state.clone() for _ in range(rounds)]
        outs = [torch.empty_like(step[2]) for _ in range(rounds)]
        attn.fill_(-7.0)
        torch.cuda.synchronize()
        for i in range(rounds):
            bh.gdn_step(*step, states[i], attn=outs[i], stream=streams[0])
            if not together:
                torch.cuda.synchronize()
            bh.gdn_ragged(args, stream=streams[1])  # (the slots read are not those written)
            if not together:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return [x.cpu().numpy() for x in (*states, *outs, attn, pool)]

    want = run(False)
    for _ in range(3):
        print("together", flush=True)
        for a, b in zip(run(True), want):
            assert np.array_equal(a, b)
