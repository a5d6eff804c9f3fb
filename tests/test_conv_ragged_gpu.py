"""The conv of many requests at once against 64 bits (bounds counted from the
roundings, in batchdata.conv), its slots bit for bit."""
from __future__ import annotations

import numpy as np
import pytest

import batchdata as bd

pytestmark = pytest.mark.gpu


def _t(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def _case(new, ch, k, seed=0, inplace=False, fresh=(), drop=(), pad=0, slot_pad=0):
    rng = np.random.default_rng(seed + 100 * len(new) + ch + k)
    n, reqs = int(np.sum(new)), len(new)
    wide = rng.standard_normal((n + 3, ch + pad)).astype(np.float32)
    w = (0.5 * rng.standard_normal((ch, k))).astype(np.float32)
    n_slots = 2 * reqs + 1
    pool = rng.standard_normal((n_slots, ch * (k - 1) + slot_pad)).astype(np.float32)
    order = rng.permutation(n_slots).astype(np.int32)
    src, dst = order[:reqs].copy(), order[reqs:2 * reqs].copy()
    if inplace:
        dst = src.copy()
    src[list(fresh)] = -1
    dst[list(drop)] = -1
    return wide, w, pool, bd.offsets(new), src, dst


def _run(bh, dev, case, ch, k, **kw):
    import torch
    wide, w, pool, start, src, dst = case
    x, p = _t(wide, dev), _t(pool, dev)
    state = p[:, :ch * (k - 1)].unflatten(1, (ch, k - 1)) if k > 1 else None
    out = torch.full((len(wide), ch), -7.0, device=dev)
    args = bh.make_conv_ragged_args(x[:, :ch], _t(w, dev), state, _t(start, dev), _t(src, dev),
                                    _t(dst, dev), out=out, **kw)
    bh.conv1d_silu_ragged(args)
    torch.cuda.synchronize()
    return out.cpu().numpy(), p.cpu().numpy(), args


def _check(bh, dev, case, ch, k, **kw):
    wide, w, pool, start, src, dst = case
    state = pool[:, :ch * (k - 1)].reshape(len(pool), ch, k - 1)
    lost = {n: v for n, v in kw.items() if n in ("l2_dim", "head_dim")}
    want, slots, bound = bd.conv(wide[:, :ch], w, state, start, src, dst,
                                 np.full((len(wide), ch), -7.0), **lost)
    got, p, _ = _run(bh, dev, case, ch, k, **kw)
    assert np.all(np.abs(got - want) <= bound)
    assert np.array_equal(p[:, :ch * (k - 1)].reshape(state.shape), slots)
    assert np.array_equal(p[:, ch * (k - 1):], pool[:, ch * (k - 1):])
    assert np.all(got[start[-1]:] == -7.0)


SHAPES = [  # channels, taps, L2 channels, head
    (1024, 4, 512, 128), (1280, 4, 512, 64), (2052, 4, 0, 0), (260, 4, 256, 256),
    (64, 4, 32, 8), (96, 4, 96, 16), (40, 4, 40, 20), (12, 4, 4, 4), (2050, 3, 0, 0),
    (70, 2, 21, 7), (33, 1, 0, 0), (130, 64, 128, 64), (1024, 4, 0, 0), (1152, 4, 1152, 32)]


@pytest.mark.parametrize("ch,k,l2,head", SHAPES)
@pytest.mark.parametrize("inplace", [False, True])
def test_conv_ragged_matches(bh, dev, ch, k, l2, head, inplace):
    for new in ([1], [1] * 7, [3, 1, 0, 8, 9, 2, 0, 17, 65], [0, 0, 5], [100]):
        print(ch, k, l2, new, flush=True)
        case = _case(new, ch, k, inplace=inplace, fresh=[0], drop=[len(new) - 1])
        _check(bh, dev, case, ch, k, l2_dim=l2, head_dim=head)


@pytest.mark.parametrize("pad,slot_pad", [(4, 0), (3, 0), (0, 5), (8, 4)])
def test_conv_ragged_strides(bh, dev, pad, slot_pad):
    case = _case([4, 0, 1, 30], 256, 4, pad=pad, slot_pad=slot_pad)
    _check(bh, dev, case, 256, 4, l2_dim=128, head_dim=128)


@pytest.mark.parametrize("n_req", [63, 64, 65, 700, 4097])
def test_conv_ragged_many_requests(bh, dev, n_req):
    rng = np.random.default_rng(n_req)
    new = rng.integers(0, 4, n_req)
    new[n_req // 2] = 40
    for ch, k in ((32, 4), (30, 3)):
        _check(bh, dev, _case(list(new), ch, k, inplace=True), ch, k)


def test_conv_ragged_bad_slots_and_offsets(bh, dev):
    import torch
    case = list(_case([2, 3, 1], 64, 4))
    case[4] = np.array([1, 99, 2], np.int32)
    case[5] = np.array([70, 3, 2 ** 31 - 1], np.int32)
    bad = torch.full((1,), -1, dtype=torch.int32, device=dev)
    _check(bh, dev, case, 64, 4, bad_slot=bad)
    assert bad.item() in (99, 70, 2 ** 31 - 1)
    # offsets that pass the rows, go down, or are below 0: in bounds, whatever comes out
    for start in ([0, 2, 2 ** 30, 6], [0, 5, 2, 6], [-5, 2, 5, 6], [3, 3, 3, 6]):
        case = list(_case([2, 3, 1], 64, 4))
        case[3] = np.array(start, np.int32)
        got, p, _ = _run(bh, dev, case, 64, 4)
        assert np.isfinite(got).all()


def test_conv_ragged_nan_stays_in_its_request(bh, dev):
    wide, w, pool, start, src, dst = _case([3, 4, 2], 128, 4)
    clean, _, _ = _run(bh, dev, (wide, w, pool, start, src, dst), 128, 4, l2_dim=128, head_dim=32)
    wide = wide.copy()
    wide[3, 40] = np.nan
    got, _, _ = _run(bh, dev, (wide, w, pool, start, src, dst), 128, 4, l2_dim=128, head_dim=32)
    hit = np.isnan(got)
    assert hit[3:7, 32:64].all() and hit.sum() == 4 * 32
    assert np.array_equal(got[~hit], clean[~hit])


def test_conv_ragged_matches_one_sequence(bh, dev):
    """The same bits as bh_conv1d_silu of each request by itself."""
    import torch
    new = [1, 12, 3]
    wide, w, pool, start, src, dst = _case(new, 1024, 4)
    got, p, _ = _run(bh, dev, (wide, w, pool, start, src, dst), 1024, 4)
    for r in range(3):
        st = _t(pool[src[r]].reshape(1024, 3), dev)
        one = bh.conv1d_silu(_t(wide[start[r]:start[r + 1]], dev), st, _t(w, dev))
        torch.cuda.synchronize()
        assert np.array_equal(one.cpu().numpy(), got[start[r]:start[r + 1]])
        assert np.array_equal(st.cpu().numpy().reshape(-1), p[dst[r]])
