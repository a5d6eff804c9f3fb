"""Counts past what the paged kernels' 32-bit indexes reach, on the CPU: refused
before the device is touched."""
from __future__ import annotations

import ctypes

import pytest

from test_paged import _attn, _cache

MOST_REQ = (1 << 31) - (1 << 16)


@pytest.mark.parametrize("hd", [256, 96])
@pytest.mark.parametrize("n_req", [MOST_REQ + 1, (1 << 31) - 257, (1 << 31) - 2])
def test_requests_past_the_index_are_refused(bh, n_req, hd):
    """A block's threads go through the requests 64 or 256 at a time: the index of the
    round after the last has to stand below 2^31 too."""
    c = _cache(bh, hd=hd, head_stride=hd, pos_stride=4 * hd, page_stride=64 * hd)
    a = _attn(bh, cache=c, n_req=n_req)
    assert bh.lib().bh_attention_paged(ctypes.byref(a), None) == bh.BH_ERR_SHAPE
    assert "overflow" in bh.last_error()
    assert bh.lib().bh_attention_paged_workspace(ctypes.byref(a)) == 0
