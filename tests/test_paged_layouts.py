"""Layouts of a paged pool, on the CPU: those whose rows share memory are refused
before the device is touched, the others are not."""
from __future__ import annotations

import ctypes
import itertools

import numpy as np
import pytest

P = 1 << 20


def _cache(bh, n, strides, hd):
    n_pages, page, n_kv = n
    return bh.PagedCache(P, P, bh.BH_KV_F16, n_pages, page, n_kv, hd, *strides)


def _overlaps(n, strides, hd):
    at = [sum(i * s for i, s in zip(ix, strides))
          for ix in itertools.product(*map(range, n))]
    at = np.sort(np.array(at))
    return bool((np.diff(at) < hd).any())


def _status(bh, cache):
    """Of an append of no tokens: the layout's checks alone."""
    return bh.lib().bh_kv_store_paged(ctypes.byref(cache), None, None, None, 0, None)


SHARED = [  # pages, positions, heads; strides of the same
    ((8, 16, 4), (16 * 1024, 256, 256)),      # positions and heads alike
    ((8, 16, 4), (1, 1024, 256)),             # pages an element apart
    ((8, 16, 4), (1024, 1024, 256)),          # pages as far apart as positions
    ((8, 16, 4), (16 * 1024, 1023, 256)),     # a position inside the last head before it
    ((8, 16, 4), (16 * 1024, 256, 16 * 255)),  # head by head, a row short
    ((8, 1, 4), (1023, 0, 256)),
    ((1, 16, 4), (0, 512, 256)),
    ((8, 16, 1), (15 * 256, 256, 0)),
]

APART = [
    ((8, 16, 4), (16 * 1024, 1024, 256)),     # rows of heads
    ((8, 16, 4), (16 * 1024, 256, 16 * 256)),  # head by head
    ((8, 16, 4), (32 * 1024, 1024, 256)),     # K and V of a page side by side
    ((8, 16, 4), (32 * 1024, 2048, 256)),     # of a position
    ((8, 16, 4), (16 * 1036, 1036, 259)),     # rows a few elements wider than heads
    ((8, 16, 4), (256, 8 * 1024, 8 * 256)),   # pages innermost
    ((1, 16, 4), (0, 1024, 256)),             # strides of single entries don't matter
    ((8, 1, 4), (1024, 0, 256)),
    ((8, 16, 1), (16 * 256, 256, 0)),
    ((1, 1, 1), (0, 0, 0)),
    ((8, 16, 4), (15 * 1024 + 4 * 256, 1024, 256)),
]


@pytest.mark.parametrize("n,strides", SHARED)
def test_rows_that_share_memory_are_refused(bh, n, strides):
    assert _overlaps(n, strides, 256)
    assert _status(bh, _cache(bh, n, strides, 256)) == bh.BH_ERR_SHAPE
    assert "rows overlap" in bh.last_error()


@pytest.mark.parametrize("n,strides", APART)
def test_rows_apart_are_taken(bh, n, strides):
    assert not _overlaps(n, strides, 256)
    assert _status(bh, _cache(bh, n, strides, 256)) == bh.BH_OK


def test_no_layout_that_overlaps_is_taken(bh):
    """All small strides against the places themselves."""
    hd, taken = 4, 0
    for n in ((2, 3, 2), (3, 2, 1), (1, 2, 3), (2, 1, 2)):
        for strides in itertools.product(range(0, 26, 2), repeat=3):
            if _status(bh, _cache(bh, n, strides, hd)) == bh.BH_OK:
                taken += 1
                assert not _overlaps(n, strides, hd), (n, strides)
    assert taken > 500
