"""Alternatives of rows with NaN logits: NaN stands below every number, of equal
ones the lowest id first, and every place of top_ids is an id of the row.  Sizes
whose last tile ends inside one of a thread's pieces, so that places behind the
row stand beside the NaN in the same lanes."""
from __future__ import annotations

import numpy as np
import pytest

from test_logprobs_gpu import _check, _logits

pytestmark = pytest.mark.gpu


def _rows(rng, vocab, n_top):
    """NaN alone, or beside a few numbers and infinities."""
    x, tok = _logits(rng, 9, vocab)
    few = rng.permutation(vocab)
    x[0, :] = np.nan
    x[1, few[3:]] = np.nan
    x[2, few[n_top:]] = np.nan          # exactly as many numbers as are asked for
    x[3, few[n_top - 1:]] = np.nan      # one fewer
    x[4, ::2], x[4, 1::2] = np.nan, -np.inf
    x[5, :] = np.nan
    x[5, few[:5]] = -np.inf
    x[5, few[5]] = 1.5
    x[6, :] = np.nan
    x[6, few[:2]] = np.inf
    x[6, few[2:4]] = -np.inf
    x[7, :vocab // 2] = np.nan
    x[8, vocab // 2:] = np.nan
    return x, tok


@pytest.mark.parametrize("n_top", [1, 5, 20, 32])
@pytest.mark.parametrize("vocab", [40, 1000, 2040, 3050, 4056, 4095, 7100, 8152, 20400, 101000])
def test_nan_rows(bh, dev, vocab, n_top):
    rng = np.random.default_rng(vocab + n_top)
    x, tok = _rows(rng, vocab, n_top)
    for pad, shift in ((0, 0), (3, 1)):
        print(vocab, n_top, pad, flush=True)
        with np.errstate(all="ignore"):
            got = _check(bh, dev, x, tok, n_top, pad=pad, shift=shift)
        assert (got[2].view(np.uint32) < vocab).all()


def test_nan_rows_many(bh, dev):
    """Rows enough for one block a row."""
    rng = np.random.default_rng(1)
    x, tok = _rows(rng, 11200, 20)
    x, tok = np.tile(x, (70, 1)), np.tile(tok, 70)
    with np.errstate(all="ignore"):
        _check(bh, dev, x, tok, 20)
