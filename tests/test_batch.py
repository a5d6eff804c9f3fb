"""Refusals of the recurrent layers of many requests and of beam search, on the CPU:
every status comes back before the device is touched (the pointers are never read)."""
from __future__ import annotations

import ctypes
import math

import pytest

P = 1 << 20  # any aligned non-null address


def test_batch_header_symbols(bh):
    names = bh.header_symbols(bh.BATCH_HEADER_PATH)
    assert sorted(bh._BATCH_SIGNATURES) == names
    assert all(hasattr(bh.lib(), n) for n in names)


def _make(cls, fields, kw):
    args = cls()
    for name, value in {**fields, **kw}.items():
        setattr(args, name, value)
    return args


def _conv(bh, **kw):
    return _make(bh.ConvRaggedArgs, dict(
        x=P, w=P, state=P, out=2 * P, q_start=P, src_slot=P, dst_slot=P, n_tok=8, n_req=2, ch=256,
        k=4, l2_dim=128, head_dim=64, n_slots=4, x_stride=256, slot_stride=768, eps=1e-6), kw)


def _gdn(bh, **kw):
    return _make(bh.GdnRaggedArgs, dict(
        q=P, k=P, v=P, gate=P, beta=P, state=P, attn=P, q_start=P, src_slot=P, dst_slot=P,
        n_tok=8, n_req=2, h_k=2, h_v=4, s=128, n_slots=4, q_stride=256, k_stride=256,
        v_stride=512, slot_stride=4 * 128 * 128), kw)


def _cache(bh, **kw):
    return _make(bh.PagedCache, dict(
        k=P, v=P, kv_dtype=bh.BH_KV_F16, n_pages=8, page_size=16, n_kv=4, hd=256,
        page_stride=16 * 1024, pos_stride=1024, head_stride=256), kw)


def _shared(bh, paged=None, **kw):
    p = _make(bh.AttentionPagedArgs, dict(
        cache=_cache(bh), q=P, out=2 * P, q_start=P, kv_len=P, block_table=P, n_tok=8, n_req=2,
        n_head=24, table_width=4), paged or {})
    return _make(bh.AttentionSharedArgs, dict(
        paged=p, group=P, group_start=P, shared_len=P, n_group=1), kw)


def _select(bh, **kw):
    return _make(bh.BeamSelectArgs, dict(
        x=P, score=P, parent=P, token=P, score_out=2 * P, n_group=2, width=4, vocab=1000,
        row_stride=1000, n_best=8, inv_temp=1.0), kw)


def _reorder(bh, **kw):
    return _make(bh.BeamReorderArgs, dict(
        parent=P, block_table=2 * P, copy_from=3 * P, src_slot=4 * P, dst_slot=5 * P,
        spare_slot=6 * P, n_group=2, width=4, parent_stride=4, table_width=9), kw)


def _copy(bh, cache=None, **kw):
    return _make(bh.KvCopyArgs, dict(
        cache=_cache(bh, **(cache or {})), block_table=P, copy_from=P, begin=P, end=P, n_req=4,
        table_width=9), kw)


def _refused(bh, fn, args, status, text):
    assert getattr(bh.lib(), fn)(ctypes.byref(args), None) == getattr(bh, "BH_ERR_" + status)
    name = fn[3:]
    assert bh.last_error().startswith(name + ": ") and text in bh.last_error(), bh.last_error()
    if hasattr(bh.lib(), fn + "_workspace") and status != "HIP" and "workspace" not in text:
        assert getattr(bh.lib(), fn + "_workspace")(ctypes.byref(args)) == 0


ALL = ["bh_conv1d_silu_ragged", "bh_gdn_ragged", "bh_attention_shared", "bh_beam_select",
       "bh_beam_reorder", "bh_kv_copy_paged"]


@pytest.mark.parametrize("fn", ALL)
def test_null_args(bh, fn):
    assert getattr(bh.lib(), fn)(None, None) == bh.BH_ERR_ARG
    assert "null args" in bh.last_error()
    if hasattr(bh.lib(), fn + "_workspace"):
        assert getattr(bh.lib(), fn + "_workspace")(None) == 0


@pytest.mark.parametrize("fn,make,names", [
    ("bh_conv1d_silu_ragged", _conv, "x w state out q_start src_slot dst_slot"),
    ("bh_gdn_ragged", _gdn, "q k v gate beta state attn q_start src_slot dst_slot"),
    ("bh_attention_shared", _shared, "group group_start shared_len"),
    ("bh_beam_select", _select, "x score parent token score_out"),
    ("bh_beam_reorder", _reorder, "parent block_table copy_from"),
    ("bh_kv_copy_paged", _copy, "block_table copy_from end"),
])
def test_null_pointers(bh, fn, make, names):
    for name in names.split():
        _refused(bh, fn, make(bh, **{name: None}), "ARG", "null pointer")


@pytest.mark.parametrize("kw,status,text", [
    (dict(k=0), "SHAPE", "must be in 1..64"), (dict(k=65), "SHAPE", "must be in 1..64"),
    (dict(ch=0), "SHAPE", "ch must be"), (dict(l2_dim=257), "SHAPE", "is above ch or no multiple"),
    (dict(l2_dim=100), "SHAPE", "no multiple"), (dict(head_dim=0), "SHAPE", "no multiple"),
    (dict(x_stride=255), "SHAPE", "stride"), (dict(slot_stride=767), "SHAPE", "stride"),
    (dict(n_tok=1 << 32), "SHAPE", "overflow"), (dict(n_tok=(1 << 24)), "SHAPE", "overflow"),
    (dict(n_req=1 << 24), "SHAPE", "overflow"), (dict(n_slots=1 << 31), "SHAPE", "overflow"),
    (dict(slot_stride=1 << 61), "SHAPE", "overflow"), (dict(x_stride=1 << 60), "SHAPE", "overflow"),
    (dict(out=P), "ARG", "out must not be x"),
])
def test_conv_refusals(bh, kw, status, text):
    _refused(bh, "bh_conv1d_silu_ragged", _conv(bh, **kw), status, text)


@pytest.mark.parametrize("kw,status,text", [
    (dict(h_k=0), "SHAPE", "must be above 0"), (dict(h_v=0), "SHAPE", "must be above 0"),
    (dict(s=0), "SHAPE", "must be above 0"), (dict(s=1025), "SHAPE", "above 1024"),
    (dict(h_v=1 << 16), "SHAPE", "65535"), (dict(h_k=1 << 40), "SHAPE", "65535"),
    (dict(q_stride=255), "SHAPE", "stride"), (dict(k_stride=255), "SHAPE", "stride"),
    (dict(v_stride=511), "SHAPE", "stride"), (dict(slot_stride=65535), "SHAPE", "stride"),
    (dict(n_tok=1 << 31), "SHAPE", "overflow"), (dict(n_req=1 << 24), "SHAPE", "overflow"),
    (dict(n_req=1 << 18), "SHAPE", "overflow"), (dict(n_slots=1 << 31), "SHAPE", "overflow"),
    (dict(slot_stride=1 << 62), "SHAPE", "overflow"), (dict(v_stride=1 << 61), "SHAPE", "overflow"),
])
def test_gdn_refusals(bh, kw, status, text):
    _refused(bh, "bh_gdn_ragged", _gdn(bh, **kw), status, text)


@pytest.mark.parametrize("paged,kw,status,text", [
    (dict(n_head=23), {}, "SHAPE", "not a multiple"), (dict(out=P), {}, "ARG", "out must not be q"),
    (dict(table_width=0), {}, "SHAPE", "table_width"), (dict(q=None), {}, "ARG", "null pointer"),
    ({}, dict(n_group=1 << 31), "SHAPE", "overflow"),
    (dict(n_req=(1 << 31) - (1 << 16)), dict(n_group=1), "SHAPE", "overflow"),
])
def test_shared_refusals(bh, paged, kw, status, text):
    _refused(bh, "bh_attention_shared", _shared(bh, paged, **kw), status, text)


def test_shared_workspace_counts(bh):
    """Of fewer bytes than are needed the call is refused; none where none are used."""
    lib = bh.lib()
    a = _shared(bh)
    need = lib.bh_attention_shared_workspace(ctypes.byref(a))
    assert need > 0
    a.paged.workspace, a.paged.workspace_bytes = P, need - 1
    assert lib.bh_attention_shared(ctypes.byref(a), None) == bh.BH_ERR_SHAPE
    assert "16-byte boundary" in bh.last_error()
    a.paged.workspace, a.paged.workspace_bytes = P + 4, need + 64
    assert lib.bh_attention_shared(ctypes.byref(a), None) == bh.BH_ERR_SHAPE
    none = _shared(bh, n_group=0, group=None, group_start=None, shared_len=None)
    assert lib.bh_attention_shared_workspace(ctypes.byref(none)) == \
        lib.bh_attention_paged_workspace(ctypes.byref(none.paged))
    assert lib.bh_attention_shared_workspace(ctypes.byref(_shared(bh, dict(n_tok=0)))) == 0


@pytest.mark.parametrize("kw,status,text", [
    (dict(width=0), "SHAPE", "width"), (dict(width=33), "SHAPE", "width"),
    (dict(vocab=0), "SHAPE", "vocab"), (dict(vocab=1 << 31, row_stride=1 << 31), "SHAPE", "vocab"),
    (dict(row_stride=999), "SHAPE", "below vocab"), (dict(n_best=0), "SHAPE", "n_best"),
    (dict(n_best=33), "SHAPE", "n_best"), (dict(vocab=5, n_best=6), "SHAPE", "n_best"),
    (dict(n_group=1 << 20), "SHAPE", "overflow"), (dict(row_stride=1 << 60), "SHAPE", "overflow"),
    (dict(inv_temp=0.0), "ARG", "inv_temp"), (dict(inv_temp=-1.0), "ARG", "inv_temp"),
    (dict(inv_temp=math.inf), "ARG", "inv_temp"), (dict(inv_temp=math.nan), "ARG", "inv_temp"),
    (dict(x=P + 2), "ARG", "misaligned"), (dict(score_out=P), "ARG", "only where n_best is width"),
])
def test_select_refusals(bh, kw, status, text):
    _refused(bh, "bh_beam_select", _select(bh, **kw), status, text)


def test_select_workspace(bh):
    a = _select(bh)
    need = bh.lib().bh_beam_select_workspace(ctypes.byref(a))
    assert need > 0
    a.workspace, a.workspace_bytes = P, need - 1
    assert bh.lib().bh_beam_select(ctypes.byref(a), None) == bh.BH_ERR_SHAPE
    assert "16-byte boundary" in bh.last_error()


@pytest.mark.parametrize("kw,status,text", [
    (dict(width=0), "SHAPE", "width"), (dict(width=33, parent_stride=40), "SHAPE", "width"),
    (dict(parent_stride=3), "SHAPE", "below width"), (dict(table_width=0), "SHAPE", "table_width"),
    (dict(table_width=1 << 31), "SHAPE", "table_width"), (dict(n_group=1 << 26), "SHAPE", "overflow"),
    (dict(n_group=1 << 20, table_width=1 << 20), "SHAPE", "overflow"),
    (dict(src_slot=None), "ARG", "go together"), (dict(dst_slot=None), "ARG", "go together"),
    (dict(spare_slot=None), "ARG", "go together"), (dict(dst_slot=4 * P), "ARG", "must differ"),
    (dict(spare_slot=5 * P), "ARG", "must differ"), (dict(copy_from=P), "ARG", "not be an output"),
])
def test_reorder_refusals(bh, kw, status, text):
    _refused(bh, "bh_beam_reorder", _reorder(bh, **kw), status, text)


@pytest.mark.parametrize("cache,kw,status,text", [
    (dict(kv_dtype=9), {}, "ARG", "kv_dtype"), (dict(pos_stride=10), {}, "SHAPE", "overlap"),
    ({}, dict(table_width=0), "SHAPE", "table_width"),
    ({}, dict(table_width=1 << 28), "SHAPE", "table_width"),
    ({}, dict(n_req=1 << 24), "SHAPE", "overflow"),
])
def test_copy_refusals(bh, cache, kw, status, text):
    _refused(bh, "bh_kv_copy_paged", _copy(bh, cache, **kw), status, text)


def test_nothing_to_do(bh):
    """No requests, tokens or groups: done, whatever the pointers."""
    lib = bh.lib()
    none = dict(x=None, w=None, state=None, out=None, q_start=None, src_slot=None, dst_slot=None)
    for kw in (dict(n_tok=0), dict(n_req=0)):
        assert lib.bh_conv1d_silu_ragged(ctypes.byref(_conv(bh, **none, **kw)), None) == bh.BH_OK
        assert lib.bh_gdn_ragged(ctypes.byref(_gdn(bh, q=None, state=None, **kw)), None) == bh.BH_OK
        a = _shared(bh, dict(q=None, **kw), group=None)
        assert lib.bh_attention_shared(ctypes.byref(a), None) == bh.BH_OK
    assert lib.bh_beam_select(ctypes.byref(_select(bh, x=None, n_group=0)), None) == bh.BH_OK
    assert lib.bh_beam_reorder(ctypes.byref(_reorder(bh, parent=None, n_group=0)), None) == bh.BH_OK
    assert lib.bh_kv_copy_paged(ctypes.byref(_copy(bh, end=None, n_req=0)), None) == bh.BH_OK
