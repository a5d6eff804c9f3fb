"""Refusals of the paged serving calls, on the CPU: every status comes back
before the device is touched (the pointers are never read)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

P = 1 << 20  # any aligned non-null address


def test_serve_header_symbols(bh):
    names = bh.header_symbols(bh.SERVE_HEADER_PATH)
    assert len(names) == 6 and sorted(bh._SERVE_SIGNATURES) == names
    assert all(hasattr(bh.lib(), n) for n in names)


def _cache(bh, **kw):
    f = dict(k=P, v=P, kv_dtype=bh.BH_KV_F16, n_pages=8, page_size=16, n_kv=4, hd=256,
             page_stride=16 * 1024, pos_stride=1024, head_stride=256)
    f.update(kw)
    return bh.PagedCache(*f.values())


@pytest.mark.parametrize("kw,status,text", [
    (dict(kv_dtype=7), "ARG", "kv_dtype must be"),
    (dict(k=None), "ARG", "null cache"),
    (dict(v=P + 1), "ARG", "misaligned"),
    (dict(n_pages=0), "SHAPE", "must be above 0"),
    (dict(page_size=0), "SHAPE", "must be above 0"),
    (dict(n_kv=0), "SHAPE", "must be above 0"),
    (dict(hd=0), "SHAPE", "must be above 0"),
    (dict(n_pages=1 << 28), "SHAPE", "pass 2^31"),
    (dict(n_pages=1 << 40, page_size=1 << 40), "SHAPE", "pass 2^31"),
    (dict(page_stride=1 << 62), "SHAPE", "strides overflow"),
    (dict(head_stride=255), "SHAPE", "rows overlap"),
    (dict(pos_stride=10), "SHAPE", "rows overlap"),
    (dict(page_stride=0), "SHAPE", "rows overlap"),
])
def test_cache_refusals(bh, kw, status, text):
    c = _cache(bh, **kw)
    want = getattr(bh, "BH_ERR_" + status)
    assert bh.lib().bh_kv_store_paged(ctypes.byref(c), P, P, P, 1, None) == want
    assert bh.last_error().startswith("kv_store_paged: ") and text in bh.last_error()
    a = _attn(bh, cache=c)
    assert bh.lib().bh_attention_paged(ctypes.byref(a), None) == want
    assert bh.last_error().startswith("attention_paged: ") and text in bh.last_error()
    assert bh.lib().bh_attention_paged_workspace(ctypes.byref(a)) == 0


def test_store_refusals(bh):
    lib, c = bh.lib(), _cache(bh)
    ref = ctypes.byref(c)
    assert lib.bh_kv_store_paged(None, P, P, P, 1, None) == bh.BH_ERR_ARG
    for bad in ((None, P, P), (P, None, P), (P, P, None)):
        assert lib.bh_kv_store_paged(ref, *bad, 1, None) == bh.BH_ERR_ARG
    assert lib.bh_kv_store_paged(ref, P, P, P, 1 << 31, None) == bh.BH_ERR_SHAPE
    assert lib.bh_kv_store_paged(ref, None, None, None, 0, None) == bh.BH_OK


def _attn(bh, cache=None, **kw):
    f = dict(cache=cache or _cache(bh), q=P, out=2 * P, q_start=P, kv_len=P, block_table=P,
             bad_page=None, n_tok=3, n_req=2, n_head=24, table_width=4, max_new=1,
             workspace=None, workspace_bytes=0)
    f.update(kw)
    return bh.AttentionPagedArgs(*f.values())


@pytest.mark.parametrize("kw,status,text", [
    (dict(n_head=0), "SHAPE", "multiple of n_kv"),
    (dict(n_head=22), "SHAPE", "multiple of n_kv"),
    (dict(n_head=1 << 20), "SHAPE", "overflow"),
    (dict(n_tok=1 << 31), "SHAPE", "overflow"),
    (dict(n_req=1 << 31), "SHAPE", "overflow"),
    (dict(table_width=0), "SHAPE", "table_width"),
    (dict(table_width=1 << 27), "SHAPE", "table_width"),
    (dict(table_width=(1 << 27) - 4095), "SHAPE", "table_width"),
    (dict(q=None), "ARG", "null pointer"),
    (dict(out=None), "ARG", "null pointer"),
    (dict(q_start=None), "ARG", "null pointer"),
    (dict(kv_len=None), "ARG", "null pointer"),
    (dict(block_table=None), "ARG", "null pointer"),
    (dict(out=P), "ARG", "out must not be q"),
])
def test_attention_refusals(bh, kw, status, text):
    a = _attn(bh, **kw)
    assert bh.lib().bh_attention_paged(ctypes.byref(a), None) == getattr(bh, "BH_ERR_" + status)
    assert bh.last_error().startswith("attention_paged: ") and text in bh.last_error()


def test_attention_head_size_limit_and_empty(bh):
    a = _attn(bh, cache=_cache(bh, hd=520, head_stride=520, pos_stride=2080, page_stride=33280))
    assert bh.lib().bh_attention_paged(ctypes.byref(a), None) == bh.BH_ERR_SHAPE
    assert "hd 520 above 512" in bh.last_error()
    assert bh.lib().bh_attention_paged(None, None) == bh.BH_ERR_ARG
    assert bh.lib().bh_attention_paged_workspace(None) == 0
    for kw in (dict(n_tok=0), dict(n_req=0)):
        a = _attn(bh, q=None, out=None, q_start=None, kv_len=None, block_table=None, **kw)
        assert bh.lib().bh_attention_paged(ctypes.byref(a), None) == bh.BH_OK


def test_attention_refuses_more_than_a_grid_holds(bh):
    # the generic layout: a block a (token, head)
    odd = _cache(bh, hd=40, n_kv=1, head_stride=40, pos_stride=40, page_stride=640)
    a = _attn(bh, cache=odd, n_head=1, n_tok=1 << 24)
    assert bh.lib().bh_attention_paged(ctypes.byref(a), None) == bh.BH_ERR_SHAPE
    assert "size overflow" in bh.last_error()
    # a tile a (request, kv head) and more
    c = _cache(bh, hd=64, n_kv=64, head_stride=64, pos_stride=4096, page_stride=65536)
    a = _attn(bh, cache=c, n_head=64, n_tok=1 << 20, n_req=1 << 20)
    assert bh.lib().bh_attention_paged(ctypes.byref(a), None) == bh.BH_ERR_SHAPE
    assert "row tiles" in bh.last_error()


def _plan(bh, **kw):
    f = dict(cached=P, n_new=P, block_table=P, free_pages=P, n_free=P, kv_len=2 * P, q_start=P,
             slots=P, pos=P, n_free_out=P, n_refused=None, n_req=4, n_tok=8, table_width=4,
             page_size=16, n_pages=64)
    f.update(kw)
    return bh.PagedPlanArgs(*f.values())


@pytest.mark.parametrize("kw,status,text", [
    (dict(n_req=4097), "SHAPE", "n_req 4097 above 4096"),
    (dict(page_size=0), "SHAPE", "above 0"),
    (dict(n_pages=0), "SHAPE", "above 0"),
    (dict(table_width=0), "SHAPE", "above 0"),
    (dict(n_pages=1 << 27), "SHAPE", "n_pages * page_size"),
    (dict(table_width=1 << 27), "SHAPE", "table_width * page_size"),
    (dict(n_tok=1 << 31), "SHAPE", "n_tok"),
    (dict(kv_len=P), "ARG", "kv_len must not be cached"),
    (dict(pos=P + 4), "ARG", "aligned"),
] + [({n: None}, "ARG", "null pointer") for n in (
    "cached", "n_new", "block_table", "free_pages", "n_free", "kv_len", "q_start", "slots",
    "n_free_out")])
def test_plan_refusals(bh, kw, status, text):
    a = _plan(bh, **kw)
    assert bh.lib().bh_paged_plan(ctypes.byref(a), None) == getattr(bh, "BH_ERR_" + status)
    assert bh.last_error().startswith("paged_plan: ") and text in bh.last_error()


def _lp(bh, **kw):
    f = dict(x=P, tokens=P, logprob=P, entropy=P, top_ids=P, top_logprobs=P, bad_id=None,
             n_rows=2, vocab=100, row_stride=100, n_top=5, inv_temp=1.0, workspace=None,
             workspace_bytes=0)
    f.update(kw)
    return bh.TokenLogprobsArgs(*f.values())


@pytest.mark.parametrize("kw,status,text", [
    (dict(vocab=0), "SHAPE", "vocab"),
    (dict(vocab=1 << 31, row_stride=1 << 31), "SHAPE", "vocab"),
    (dict(row_stride=99), "SHAPE", "row_stride 99 below vocab 100"),
    (dict(n_rows=1 << 31), "SHAPE", "overflow"),
    (dict(row_stride=1 << 62), "SHAPE", "overflow"),
    (dict(n_top=33), "SHAPE", "n_top 33"),
    (dict(n_top=5, vocab=4), "SHAPE", "n_top 5"),
    (dict(inv_temp=0.0), "ARG", "inv_temp"),
    (dict(inv_temp=-1.0), "ARG", "inv_temp"),
    (dict(inv_temp=float("nan")), "ARG", "inv_temp"),
    (dict(inv_temp=float("inf")), "ARG", "inv_temp"),
    (dict(x=None), "ARG", "null pointer"),
    (dict(x=P + 2), "ARG", "misaligned x"),
    (dict(tokens=None), "ARG", "null pointer"),
    (dict(top_ids=None), "ARG", "null pointer"),
    (dict(top_logprobs=None), "ARG", "null pointer"),
])
def test_logprobs_refusals(bh, kw, status, text):
    a = _lp(bh, **kw)
    assert bh.lib().bh_token_logprobs(ctypes.byref(a), None) == getattr(bh, "BH_ERR_" + status)
    assert bh.last_error().startswith("token_logprobs: ") and text in bh.last_error()
    assert bh.lib().bh_token_logprobs_workspace(None) == 0


def test_logprobs_nothing_to_do(bh):
    lib = bh.lib()
    assert lib.bh_token_logprobs(None, None) == bh.BH_ERR_ARG
    a = _lp(bh, n_rows=0, x=None, tokens=None, top_ids=None, top_logprobs=None)
    assert lib.bh_token_logprobs(ctypes.byref(a), None) == bh.BH_OK
    a = _lp(bh, logprob=None, entropy=None, n_top=0)
    assert lib.bh_token_logprobs(ctypes.byref(a), None) == bh.BH_OK


def test_python_refuses_host_tensors(bh):
    import torch
    k = torch.zeros((4, 16, 2, 64))
    with pytest.raises(ValueError, match="one GPU"):
        bh.make_paged_cache(k, k)
    with pytest.raises(ValueError, match="alike"):
        bh.make_paged_cache(k, k[:, :, :, :32])
    with pytest.raises(ValueError, match="CUDA"):
        bh.make_token_logprobs_args(torch.zeros((2, 8)))
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        bh.make_paged_plan_args(i, i, i.view(4, 1), i, i[:1], 16, kv_len=i.clone(),
                                q_start=torch.zeros(5, dtype=torch.int32), slots=i)


def test_plan_model_by_hand():
    """The plain plan the GPU is checked against, on a step done by hand."""
    from pageddata import plan
    table = np.array([[7, 3, -1], [5, -1, -1], [4, 6, -1], [-1, -1, -1]], np.int32)
    free = np.array([0, 1, 2, -1, -1, -1, -1, -1], np.int32)
    # page 4: 8 cached + 1 needs a page; 3 + 1 needs none; request 2 (5 cached)
    # leaves two pages; a prompt of 9 needs three
    got = plan([8, 3, 5, 0], [1, 1, -1, 9], table, free, 3, 4, 12)
    assert got[0].tolist() == [9, 4, 0, 9] and got[1].tolist() == [0, 1, 2, 2, 11]
    # released 4, 6 lie on top: stack 0 1 2 4 6; request 0 takes 6, 3 takes 4 2 1
    assert got[4].tolist() == [[7, 3, 6], [5, -1, -1], [4, 6, -1], [4, 2, 1]]
    assert got[2].tolist() == [24, 23, 16, 17, 18, 19, 8, 9, 10, 11, 4, -1]
    assert got[3][:, 0].tolist() == [8, 3, 0, 1, 2, 3, 4, 5, 6, 7, 8, 0]
    assert got[6] == 1 and got[7] == 0 and got[5].tolist() == [0, 1, 2, 4, 6, -1, -1, -1]
    # one token slot too few: the prompt is refused
    got = plan([8, 3, 5, 0], [1, 1, -1, 9], table, free, 3, 4, 10)
    assert got[7] == 1 and got[0].tolist() == [9, 4, 0, 0] and got[6] == 4
