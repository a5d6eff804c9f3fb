"""Attention over a shared prefix in each of the forms that it chooses by rows and by the
positions that a table has room for: the same requests under tables of more columns, which
name no pages.  Tolerance as in test_attention_shared_gpu.py."""
from __future__ import annotations

import numpy as np
import pytest

from test_attention_shared_gpu import TOL, _case, _check, _run, _want
from conftest import rel_err

pytestmark = pytest.mark.gpu

# columns of 16 positions: some, more than small tiles are taken for, more than any but the
# forms of bh_attention_paged are
COLUMNS = [0, 700, 20000]


def _wider(c, columns):
    c = dict(c)
    c["table"] = np.concatenate(
        [c["table"], np.full((len(c["table"]), columns), -1, np.int32)], 1)
    return c


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n_head,n_kv,hd", [(8, 2, 64), (8, 2, 128), (12, 2, 256)])
@pytest.mark.parametrize("columns", COLUMNS)
def test_forms(bh, dev, f16, n_head, n_kv, hd, columns):
    for groups in ([(130, [(9, 1)] * 9)], [(100, [(3, 1)] * 40)],
                   [(64, [(70, 1)] * 6), (48, [(1, 2)] * 5), (0, [(30, 1)])],
                   [(300, [(70, 70), (1, 1), (33, 33)])],
                   [(96, [(20, 1)] * 30), (0, [(50, 1)]), (130, [(200, 150), (4, 1)])]):
        c = _wider(_case(groups, n_head=n_head, n_kv=n_kv, hd=hd, f16=f16), columns)
        print(columns, hd, f16, groups[0], flush=True)
        _check(bh, dev, c)
        new = [n for _, reqs in groups for _, n in reqs]
        most = max(sum(n for _, n in reqs) for _, reqs in groups)
        _check(bh, dev, c, max_new=max(new), max_group_new=most)


@pytest.mark.parametrize("columns", COLUMNS)
@pytest.mark.parametrize("f16", [True, False])
def test_masked_values_do_not_reach(bh, dev, columns, f16):
    """NaN behind the requests' ends; an infinite value of one group's prefix."""
    c = _case([(40, [(5, 1)] * 20), (16, [(3, 1)])], f16=f16, same_pages=False, spare_tokens=0,
              n_head=8, n_kv=2, hd=256)
    want, page = _want(c), c["k"].shape[1]
    seen = np.zeros(c["k"].shape[:2], bool)
    for r, n in enumerate(c["kv_len"]):
        for p in range(n):
            seen[c["table"][r, p // page], p % page] = True
    for name in ("k", "v"):
        c[name] = c[name].copy()
        c[name][~seen] = np.nan
    c = _wider(c, columns)
    assert rel_err(_run(bh, dev, c), want) < TOL
    c["v"][c["table"][:20, 0], 3] = np.inf
    got = _run(bh, dev, c)
    assert not np.isfinite(got[:20]).any() and np.isfinite(got[20:]).all()


@pytest.mark.parametrize("columns", COLUMNS)
def test_garbage_offsets_stay_in_bounds(bh, dev, columns):
    base = _wider(_case([(64, [(5, 20), (7, 30)]), (48, [(9, 9)] * 3)], spare_tokens=0, n_head=8,
                        n_kv=2, hd=128), columns)
    n = len(base["q"])
    for key, val in (("q_start", [0, 20, 10, 60, 2 ** 30, n]), ("q_start", [n, 50, 40, 30, 2, 1]),
                     ("q_start", [0, 0, n, 0, n, 0]), ("group_start", [3, 1, 5]),
                     ("group_start", [-9, 2 ** 30, 1]), ("group_start", [0, 5, 5]),
                     ("group", [0, 1, 0, 1, 0]), ("shared", [2 ** 31 - 1, 2 ** 31 - 1]),
                     ("kv_len", [2 ** 31 - 1, -4, 0, 1, 2])):
        c = dict(base)
        c[key] = np.array(val, np.int32)
        print(columns, key, val, flush=True)
        assert _run(bh, dev, c).shape == base["q"].shape


# Groups of long prefixes and few rows, where a tile's parts are whole runs of several units
# (with 256 compute units 2 to 7), short, odd, and none of a request's own among them.  The
# tolerance holds at these lengths too: of n positions with scores of unit variance the
# output and the part of the scores' errors that a mean leaves both go with 1 / sqrt(n).
LONG = [
    [(16384, [(100, 1)] * 7)],
    [(9001, [(30, 1)] * 10), (5003, [(333, 3)] * 4), (0, [(70, 1)])],
    [(30017, [(1, 1)] * 3)],
    [(9001, [(30, 1)] * 24)],
    [(12000, [(65, 1), (640, 2), (3, 1)]), (7999, [(1, 1), (63, 9)]), (33, [(700, 1)])],
]


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n_head,n_kv,hd,page", [(8, 2, 64, 16), (6, 2, 128, 7), (12, 2, 256, 16)])
@pytest.mark.parametrize("nth", range(len(LONG)))
def test_long_prefixes_of_few_rows(bh, dev, nth, n_head, n_kv, hd, page, f16):
    groups = LONG[nth]
    c = _case(groups, page=page, n_head=n_head, n_kv=n_kv, hd=hd, f16=f16)
    print(nth, hd, f16, flush=True)
    got = _check(bh, dev, c)
    new = [n for _, reqs in groups for _, n in reqs]
    most = max(sum(n for _, n in reqs) for _, reqs in groups)
    again = _check(bh, dev, c, max_new=max(new), max_group_new=most)
    assert np.array_equal(again, _run(bh, dev, c, max_new=max(new), max_group_new=most))
    assert np.array_equal(got, _run(bh, dev, c))


def test_long_prefix_under_garbage_offsets(bh, dev):
    base = _case([(9001, [(30, 1)] * 3), (4100, [(70, 5), (9, 2)])], n_head=8, n_kv=2, hd=128,
                 spare_tokens=0)
    n = len(base["q"])
    for key, val in (("q_start", [0, 3, 2, 3, 2 ** 30, n]), ("q_start", [n, 8, 6, 4, 2, 1]),
                     ("group_start", [3, 1, 5]), ("group_start", [-9, 2 ** 30, 1]),
                     ("group", [0, 1, 0, 1, 0]), ("shared", [2 ** 31 - 1, 2 ** 31 - 1]),
                     ("kv_len", [2 ** 31 - 1, -4, 0, 1, 2]), ("kv_len", [9031, 0, 9031, 4170, 4109])):
        c = dict(base)
        c[key] = np.array(val, np.int32)
        print(key, val, flush=True)
        assert _run(bh, dev, c).shape == base["q"].shape
