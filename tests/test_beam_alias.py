"""bh_beam_reorder's parents and its outputs: parents that lie in an output are refused,
whichever it is and wherever they begin (on the CPU: pointers are compared, never read)."""
from __future__ import annotations

import numpy as np
import pytest

import batchdata as bd
from test_batch import P, _refused, _reorder

# two groups of 4 beams, rows of 4 words 4 or 100 words apart; tables of 9 columns
OUTPUTS = {"block_table": 72, "copy_from": 8, "src_slot": 8, "dst_slot": 8, "spare_slot": 8}


@pytest.mark.parametrize("name", OUTPUTS)
@pytest.mark.parametrize("stride", [4, 100])
def test_parents_in_an_output(bh, name, stride):
    words = OUTPUTS[name]
    last = stride + 4  # words from the first parent to behind the last
    for at in {0, 3, last - 1, stride, stride + 1, 1 - words, -1, -4}:
        if -words < at < 4 or stride - words < at < last:
            _refused(bh, "bh_beam_reorder", _reorder(bh, parent_stride=stride,
                                                     **{name: P + 4 * at}), "ARG", "not be an output")


def _meets(parent, stride, width, n_group, out, n):
    own = {parent + 4 * (g * stride + i) for g in range(n_group) for i in range(width)}
    return any(out + 4 * i in own for i in range(n))


@pytest.mark.parametrize("n_group,width,stride", [(1, 4, 4), (2, 4, 30), (3, 2, 9), (3, 1, 1)])
def test_every_place_of_copy_from(bh, n_group, width, stride):
    n = n_group * width
    for at in range(-n - 3, (n_group - 1) * stride + width + 3):
        if _meets(P, stride, width, n_group, P + 4 * at, n):
            args = _reorder(bh, parent=P, parent_stride=stride, n_group=n_group, width=width,
                            copy_from=P + 4 * at, block_table=P << 8, src_slot=None,
                            dst_slot=None, spare_slot=None, table_width=1)
            _refused(bh, "bh_beam_reorder", args, "ARG", "not be an output")


@pytest.mark.gpu
@pytest.mark.parametrize("begin", [4, 20])
def test_outputs_between_the_rows_of_parents(bh, dev, begin):
    """Words of the same allocation that are no parents may be outputs."""
    import torch
    n_group, width, stride = 2, 4, 48
    rng = np.random.default_rng(begin)
    parent = np.array([[1, 1, 0, 2], [7, 4, 4, 4]], np.int32)
    table = rng.permutation(72).astype(np.int32).reshape(8, 9)
    slots = rng.permutation(16).astype(np.int32)
    buf = torch.full((stride + width,), -9, dtype=torch.int32, device=dev)
    rows = torch.as_strided(buf, (n_group, width), (stride, 1))
    rows.copy_(torch.from_numpy(parent))
    arrays = [buf[begin + 8 * i:begin + 8 * i + 8] for i in range(3)]  # copy_from, dst, src
    arrays[1].copy_(torch.from_numpy(slots[:8]))
    spare = torch.from_numpy(slots[8:].copy()).to(dev)
    pages = torch.from_numpy(table).to(dev)
    bh.beam_reorder(bh.make_beam_reorder_args(rows, pages, copy_from=arrays[0], dst_slot=arrays[1],
                                              src_slot=arrays[2], spare_slot=spare))
    torch.cuda.synchronize()
    want = bd.reorder(parent, table, slots[:8], slots[8:], width)
    for got, ref in zip((pages, arrays[0], arrays[2], arrays[1], spare), want):
        assert np.array_equal(got.cpu().numpy(), ref)
    assert np.array_equal(rows.cpu().numpy(), parent)
