"""Python binding of the bonsai HIP library (ctypes over the C ABI).

The product is lib/libbonsai_hip.so with the C ABI of include/bonsai_hip.h;
this module only loads it and offers torch-tensor conveniences for tests and
benchmarks (torch provides device memory and streams; every computation runs
in the library's HIP kernels).  There is no CPU fallback: if the library is
missing, `lib()` raises.

The package directory name contains dashes, so import it by path:

    spec = importlib.util.spec_from_file_location(
        "bonsai_amd", "ternary-bonsai-inference_amd/__init__.py")
"""
from __future__ import annotations

import ctypes
import os
import re
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
LIB_PATH = PKG_DIR / "lib" / "libbonsai_hip.so"
HEADER_PATH = REPO_DIR / "include" / "bonsai_hip.h"
SERVE_HEADER_PATH = REPO_DIR / "include" / "bonsai_hip_serve.h"
BATCH_HEADER_PATH = REPO_DIR / "include" / "bonsai_hip_batch.h"

BH_OK = 0
BH_ERR_SHAPE = -1
BH_ERR_RANGE = -2
BH_ERR_HIP = -3
BH_ERR_ARG = -4

BH_SILU = 0
BH_SIGMOID = 1
BH_SOFTPLUS = 2
BH_SILU_MUL = 3
BH_SIGMOID_MUL = 4

BH_SOFTMAX_SAMPLER_NORM = 1  # bh_softmax_rows_ex flag

# Ternary-Bonsai-27B constants (reference src/gdev.rs:21-37, src/weights.rs:42-62)
N_EMBD = 5120
N_HEAD = 24
N_HEAD_KV = 4
HEAD_DIM = 256
N_ROT = 64
SECTIONS = (11, 11, 10, 0)
FREQ_BASE = 1e7
EPS = 1e-6
N_VOCAB = 248320
GDN_HV = 48
GDN_STATE = 128

_c_size = ctypes.c_size_t
_c_float = ctypes.c_float
_c_int = ctypes.c_int
_vp = ctypes.c_void_p


class BonsaiError(RuntimeError):
    """A non-zero status from the library, with bh_last_error()'s message."""

    def __init__(self, status: int, message: str):
        super().__init__(f"status {status}: {message}")
        self.status = status
        self.message = message


class GdnPrepArgs(ctypes.Structure):
    """bh_gdn_prep_args (include/bonsai_hip.h)."""

    _fields_ = [
        ("conv", _vp), ("conv_out", _vp), ("z", _vp), ("y", _vp), ("gated_out", _vp),
        ("alpha_raw", _vp), ("dt_bias", _vp), ("ssm_a", _vp), ("beta_raw", _vp),
        ("gate_out", _vp), ("beta_out", _vp),
        ("n_tok", _c_size), ("conv_dim", _c_size), ("l2_dim", _c_size), ("head_dim", _c_size),
        ("inner_dim", _c_size), ("n_v_head", _c_size), ("gate_mode", _c_int), ("eps", _c_float),
        ("conv_w", _vp), ("conv_state", _vp), ("conv_k", _c_size),
    ]


class QkNormRopeArgs(ctypes.Structure):
    """bh_qk_norm_rope_args (include/bonsai_hip.h)."""

    _fields_ = [
        ("q", _vp), ("q_out", _vp), ("gate_out", _vp), ("k", _vp), ("k_out", _vp),
        ("wq", _vp), ("wk", _vp), ("pos", _vp),
        ("n_tok", _c_size), ("n_q_head", _c_size), ("n_k_head", _c_size), ("head_dim", _c_size),
        ("q_head_stride", _c_size), ("n_dims", _c_size),
        ("sections", ctypes.c_int32 * 4), ("freq_base", _c_float), ("eps", _c_float),
    ]


_SIGNATURES = {
    "bh_last_error": (ctypes.c_char_p, []),
    "bh_version": (ctypes.c_char_p, []),
    "bh_scratch_retired_bytes": (ctypes.c_size_t, []),
    "bh_scratch_release": (_c_int, []),
    "bh_pq2_row_bytes": (_c_size, [_c_size]),
    "bh_rms_norm": (_c_int, [_vp, _vp, _c_size, _c_float, _vp, _vp]),
    "bh_rms_norm_rows": (_c_int, [_vp, _c_size, _vp, _c_size, _c_size, _c_float, _vp, _vp]),
    "bh_add_rms_norm_rows": (_c_int, [_vp, _vp, _c_size, _vp, _c_size, _c_size, _c_float, _vp,
                                      _vp, _vp]),
    "bh_l2_norm_rows": (_c_int, [_vp, _c_size, _c_size, _c_float, _vp, _vp]),
    "bh_silu_l2_norm_rows": (_c_int, [_vp, _c_size, _c_size, _c_float, _vp, _vp]),
    "bh_unary": (_c_int, [_c_int, _vp, _vp, _c_size, _vp, _vp]),
    "bh_gdn_gate_prep": (_c_int, [_vp, _vp, _vp, _vp, _c_size, _c_size, _vp, _vp, _vp]),
    "bh_gdn_prep_fused": (_c_int, [ctypes.POINTER(GdnPrepArgs), _vp]),
    "bh_softmax_rows": (_c_int, [_vp, _c_size, _c_size, _c_float, _vp, _vp]),
    "bh_softmax_rows_noalloc": (_c_int, [_vp, _c_size, _c_size, _c_float, _vp, _vp]),
    "bh_softmax_rows_ex": (_c_int, [_vp, _c_size, _c_size, _c_float, _c_int, _vp, _vp]),
    "bh_rope_imrope": (_c_int, [_vp, _c_size, _c_size, _c_size, _vp, _c_size,
                                ctypes.POINTER(ctypes.c_int32), _c_float, _vp]),
    "bh_qk_norm_rope": (_c_int, [ctypes.POINTER(QkNormRopeArgs), _vp]),
    "bh_pq2_embed_gather": (_c_int, [_vp, _c_size, _c_size, _vp, _c_size, _vp, _vp, _vp]),
    "bh_pq2_embed_gather_rms": (_c_int, [_vp, _c_size, _c_size, _vp, _c_size, _vp, _c_size,
                                         _c_float, _vp, _vp, _vp, _vp]),
    "bh_host_rms_norm": (_c_int, [_vp, _c_size, _vp, _c_float, _vp]),
    "bh_host_rms_norm_rows": (_c_int, [_vp, _c_size, _vp, _c_size, _c_size, _c_float, _vp]),
    "bh_host_l2_norm_rows": (_c_int, [_vp, _c_size, _c_size, _c_float, _vp]),
    "bh_host_map_inplace": (_c_int, [_vp, _c_size, _c_int]),
    "bh_host_softmax_rows": (_c_int, [_vp, _c_size, _c_size, _vp]),
    "bh_host_rope_imrope": (_c_int, [_vp, _c_size, ctypes.c_int64, ctypes.c_int64,
                                     ctypes.c_int64, ctypes.c_int64, _c_size,
                                     ctypes.POINTER(ctypes.c_int32), _c_float]),
    "bh_host_decode_pq2_0_row": (_c_int, [_vp, _c_size, _c_size, _vp]),
    "bh_host_batch_embed": (_c_int, [_vp, _c_size, _c_size, _c_size, _vp, _c_size, _vp]),
    "bh_conv1d_silu": (_c_int, [_vp, _vp, _vp, _c_size, _c_size, _c_size, _vp, _vp]),
    "bh_host_gdn_step": (_c_int, [_vp, _c_size, _vp, _c_size, _vp, _c_size, _vp, _c_size, _vp,
                                  _c_size, _vp, _c_size, _vp, _c_size]),
    "bh_kv_store": (_c_int, [_vp, _vp, _c_size, _c_size, _vp, _vp, _c_size, _c_int, _vp]),
    "bh_attention": (_c_int, [_vp, _c_size, _c_size, _vp, _vp, _c_int, _c_size, _c_size, _c_size,
                              _vp, _vp]),
    "bh_gdn_step": (_c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _c_size, _c_size, _c_size,
                             _c_size, _vp]),
    "bh_planar_packed_len": (_c_size, [_c_size, ctypes.c_uint]),
    "bh_kv_store_planar": (_c_int, [_vp, _vp, _c_size, _c_size, _c_size, ctypes.c_uint, _vp, _vp,
                                    _vp, _vp, _vp, _c_size, _vp]),
    "bh_attention_planar": (_c_int, [_vp, _c_size, _c_size, _vp, _vp, _vp, _vp, _vp,
                                     ctypes.c_uint, _c_size, _c_size, _c_size, _vp, _vp]),
    "bh_pq2_matvec_range": (_c_int, [_vp, _c_size, _c_size, ctypes.c_uint64, _c_size, _vp,
                                     _c_size, _vp, _c_size, _vp]),
    "bh_pq2_matmul_n": (_c_int, [_vp, _c_size, _c_size, ctypes.c_uint64, _c_size, _vp, _c_size,
                                 _c_size, _vp, _c_size, _vp]),
    "bh_host_dot_pq2_0_row": (_c_int, [_vp, _c_size, _c_size, ctypes.c_uint64, _vp, _c_size,
                                       _vp]),
    "bh_host_pq2_matvec_range": (_c_int, [_vp, _c_size, _c_size, ctypes.c_uint64, _c_size, _vp,
                                          _c_size, _vp, _c_size]),
    "bh_host_pq2_matmul_n": (_c_int, [_vp, _c_size, _c_size, ctypes.c_uint64, _c_size, _vp,
                                      _c_size, _c_size, _vp, _c_size]),
}

class PagedCache(ctypes.Structure):
    """bh_paged_cache (include/bonsai_hip_serve.h)."""

    _fields_ = [
        ("k", _vp), ("v", _vp), ("kv_dtype", _c_int),
        ("n_pages", _c_size), ("page_size", _c_size), ("n_kv", _c_size), ("hd", _c_size),
        ("page_stride", _c_size), ("pos_stride", _c_size), ("head_stride", _c_size),
    ]


class PagedPlanArgs(ctypes.Structure):
    """bh_paged_plan_args (include/bonsai_hip_serve.h)."""

    _fields_ = [
        ("cached", _vp), ("n_new", _vp), ("block_table", _vp), ("free_pages", _vp),
        ("n_free", _vp), ("kv_len", _vp), ("q_start", _vp), ("slots", _vp), ("pos", _vp),
        ("n_free_out", _vp), ("n_refused", _vp),
        ("n_req", _c_size), ("n_tok", _c_size), ("table_width", _c_size), ("page_size", _c_size),
        ("n_pages", _c_size),
    ]


class AttentionPagedArgs(ctypes.Structure):
    """bh_attention_paged_args (include/bonsai_hip_serve.h)."""

    _fields_ = [
        ("cache", PagedCache), ("q", _vp), ("out", _vp), ("q_start", _vp), ("kv_len", _vp),
        ("block_table", _vp), ("bad_page", _vp),
        ("n_tok", _c_size), ("n_req", _c_size), ("n_head", _c_size), ("table_width", _c_size),
        ("max_new", _c_size), ("workspace", _vp), ("workspace_bytes", _c_size),
    ]


class TokenLogprobsArgs(ctypes.Structure):
    """bh_token_logprobs_args (include/bonsai_hip_serve.h)."""

    _fields_ = [
        ("x", _vp), ("tokens", _vp), ("logprob", _vp), ("entropy", _vp), ("top_ids", _vp),
        ("top_logprobs", _vp), ("bad_id", _vp),
        ("n_rows", _c_size), ("vocab", _c_size), ("row_stride", _c_size), ("n_top", _c_size),
        ("inv_temp", _c_float), ("workspace", _vp), ("workspace_bytes", _c_size),
    ]


_SERVE_SIGNATURES = {
    "bh_paged_plan": (_c_int, [ctypes.POINTER(PagedPlanArgs), _vp]),
    "bh_kv_store_paged": (_c_int, [ctypes.POINTER(PagedCache), _vp, _vp, _vp, _c_size, _vp]),
    "bh_attention_paged": (_c_int, [ctypes.POINTER(AttentionPagedArgs), _vp]),
    "bh_attention_paged_workspace": (_c_size, [ctypes.POINTER(AttentionPagedArgs)]),
    "bh_token_logprobs": (_c_int, [ctypes.POINTER(TokenLogprobsArgs), _vp]),
    "bh_token_logprobs_workspace": (_c_size, [ctypes.POINTER(TokenLogprobsArgs)]),
}


class ConvRaggedArgs(ctypes.Structure):
    """bh_conv_ragged_args (include/bonsai_hip_batch.h)."""

    _fields_ = [
        ("x", _vp), ("w", _vp), ("state", _vp), ("out", _vp), ("q_start", _vp),
        ("src_slot", _vp), ("dst_slot", _vp), ("bad_slot", _vp),
        ("n_tok", _c_size), ("n_req", _c_size), ("ch", _c_size), ("k", _c_size),
        ("l2_dim", _c_size), ("head_dim", _c_size), ("n_slots", _c_size), ("x_stride", _c_size),
        ("slot_stride", _c_size), ("max_new", _c_size), ("eps", _c_float),
    ]


class GdnRaggedArgs(ctypes.Structure):
    """bh_gdn_ragged_args (include/bonsai_hip_batch.h)."""

    _fields_ = [
        ("q", _vp), ("k", _vp), ("v", _vp), ("gate", _vp), ("beta", _vp), ("state", _vp),
        ("attn", _vp), ("q_start", _vp), ("src_slot", _vp), ("dst_slot", _vp), ("bad_slot", _vp),
        ("n_tok", _c_size), ("n_req", _c_size), ("h_k", _c_size), ("h_v", _c_size),
        ("s", _c_size), ("n_slots", _c_size), ("q_stride", _c_size), ("k_stride", _c_size),
        ("v_stride", _c_size), ("slot_stride", _c_size), ("max_new", _c_size),
        ("workspace", _vp), ("workspace_bytes", _c_size),
    ]


class AttentionSharedArgs(ctypes.Structure):
    """bh_attention_shared_args (include/bonsai_hip_batch.h)."""

    _fields_ = [
        ("paged", AttentionPagedArgs), ("group", _vp), ("group_start", _vp), ("shared_len", _vp),
        ("n_group", _c_size), ("max_group_new", _c_size),
    ]


class BeamSelectArgs(ctypes.Structure):
    """bh_beam_select_args (include/bonsai_hip_batch.h)."""

    _fields_ = [
        ("x", _vp), ("score", _vp), ("parent", _vp), ("token", _vp), ("score_out", _vp),
        ("n_group", _c_size), ("width", _c_size), ("vocab", _c_size), ("row_stride", _c_size),
        ("n_best", _c_size), ("inv_temp", _c_float), ("workspace", _vp),
        ("workspace_bytes", _c_size),
    ]


class BeamReorderArgs(ctypes.Structure):
    """bh_beam_reorder_args (include/bonsai_hip_batch.h)."""

    _fields_ = [
        ("parent", _vp), ("block_table", _vp), ("copy_from", _vp), ("src_slot", _vp),
        ("dst_slot", _vp), ("spare_slot", _vp),
        ("n_group", _c_size), ("width", _c_size), ("parent_stride", _c_size),
        ("table_width", _c_size),
    ]


class KvCopyArgs(ctypes.Structure):
    """bh_kv_copy_args (include/bonsai_hip_batch.h)."""

    _fields_ = [
        ("cache", PagedCache), ("block_table", _vp), ("copy_from", _vp), ("begin", _vp),
        ("end", _vp), ("n_req", _c_size), ("table_width", _c_size),
    ]


_BATCH_SIGNATURES = {
    "bh_conv1d_silu_ragged": (_c_int, [ctypes.POINTER(ConvRaggedArgs), _vp]),
    "bh_gdn_ragged": (_c_int, [ctypes.POINTER(GdnRaggedArgs), _vp]),
    "bh_gdn_ragged_workspace": (_c_size, [ctypes.POINTER(GdnRaggedArgs)]),
    "bh_attention_shared": (_c_int, [ctypes.POINTER(AttentionSharedArgs), _vp]),
    "bh_attention_shared_workspace": (_c_size, [ctypes.POINTER(AttentionSharedArgs)]),
    "bh_beam_select": (_c_int, [ctypes.POINTER(BeamSelectArgs), _vp]),
    "bh_beam_select_workspace": (_c_size, [ctypes.POINTER(BeamSelectArgs)]),
    "bh_beam_reorder": (_c_int, [ctypes.POINTER(BeamReorderArgs), _vp]),
    "bh_kv_copy_paged": (_c_int, [ctypes.POINTER(KvCopyArgs), _vp]),
}

_LIB = None


def header_symbols(path: Path = HEADER_PATH) -> list[str]:
    """Every function name declared in a header (include/bonsai_hip.h)."""
    text = path.read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(bh_[a-z0-9_]+)\s*\(", text)))


def lib() -> ctypes.CDLL:
    """Load lib/libbonsai_hip.so (raises if it has not been built)."""
    global _LIB
    if _LIB is not None:
        return _LIB
    if not LIB_PATH.exists():
        raise FileNotFoundError(
            f"{LIB_PATH} is missing: run __graft_entry__.build() (hipcc for gfx950) first")
    try:  # share torch's HIP runtime when torch is present (same soname)
        import torch  # noqa: F401
    except ImportError:
        pass
    handle = ctypes.CDLL(str(LIB_PATH), mode=ctypes.RTLD_LOCAL)
    for name, (res, args) in {**_SIGNATURES, **_SERVE_SIGNATURES, **_BATCH_SIGNATURES}.items():
        fn = getattr(handle, name)
        fn.restype = res
        fn.argtypes = args
    _LIB = handle
    return handle


def last_error() -> str:
    return lib().bh_last_error().decode()


def check(status: int) -> None:
    if status != BH_OK:
        raise BonsaiError(status, last_error())


def pq2_row_bytes(ne0: int) -> int:
    return int(lib().bh_pq2_row_bytes(ne0))


# ---------------------------------------------------------------------------
# torch-tensor conveniences (device tensors, current torch stream)
# ---------------------------------------------------------------------------

def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(stream=None) -> int:
    import torch
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def _f32(t, name: str):
    import torch
    if t.dtype != torch.float32 or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 CUDA tensor")
    return t


def rms_norm_rows(x, w, eps: float = EPS, out=None, stream=None):
    import torch
    _f32(x, "x"), _f32(w, "w")
    out = torch.empty_like(x) if out is None else out
    check(lib().bh_rms_norm_rows(x.data_ptr(), x.numel(), w.data_ptr(), w.numel(), w.numel(),
                                 eps, out.data_ptr(), _stream(stream)))
    return out


def add_rms_norm_rows(x, residual, w, eps: float = EPS, sum_out=None, out=None, stream=None):
    import torch
    sum_out = torch.empty_like(x) if sum_out is None else sum_out
    out = torch.empty_like(x) if out is None else out
    check(lib().bh_add_rms_norm_rows(x.data_ptr(), residual.data_ptr(), x.numel(), w.data_ptr(),
                                     w.numel(), w.numel(), eps, sum_out.data_ptr(),
                                     out.data_ptr(), _stream(stream)))
    return sum_out, out


def l2_norm_rows(x, row_len: int, eps: float = EPS, out=None, silu_first=False, stream=None):
    import torch
    _f32(x, "x")
    out = torch.empty_like(x) if out is None else out
    fn = lib().bh_silu_l2_norm_rows if silu_first else lib().bh_l2_norm_rows
    check(fn(x.data_ptr(), x.numel(), row_len, eps, out.data_ptr(), _stream(stream)))
    return out


def unary(mode: int, a, b=None, out=None, stream=None):
    import torch
    out = torch.empty_like(a) if out is None else out
    check(lib().bh_unary(mode, a.data_ptr(), _ptr(b), a.numel(), out.data_ptr(),
                         _stream(stream)))
    return out


def softmax_rows(x, row_len: int, inv_temp: float = 1.0, out=None, stream=None,
                 noalloc: bool = False, sampler_norm: bool = False):
    """bh_softmax_rows; with noalloc=True bh_softmax_rows_noalloc (fixed
    library scratch, no device allocation by the library); with
    sampler_norm=True bh_softmax_rows_ex(BH_SOFTMAX_SAMPLER_NORM), the
    sampler's f64 normalisation (src/sampler.rs:118-126)."""
    import torch
    _f32(x, "x")
    if noalloc and sampler_norm:
        raise ValueError("softmax_rows: noalloc has no sampler normalisation")
    out = torch.empty_like(x) if out is None else out
    if sampler_norm:
        check(lib().bh_softmax_rows_ex(x.data_ptr(), x.numel(), row_len, inv_temp,
                                       BH_SOFTMAX_SAMPLER_NORM, out.data_ptr(), _stream(stream)))
        return out
    fn = lib().bh_softmax_rows_noalloc if noalloc else lib().bh_softmax_rows
    check(fn(x.data_ptr(), x.numel(), row_len, inv_temp, out.data_ptr(), _stream(stream)))
    return out


def gdn_gate_prep(alpha_raw, dt_bias, ssm_a, beta_raw, stream=None):
    import torch
    n_tok, n_head = alpha_raw.shape
    gate = torch.empty_like(alpha_raw)
    beta = torch.empty_like(beta_raw)
    check(lib().bh_gdn_gate_prep(alpha_raw.data_ptr(), dt_bias.data_ptr(), ssm_a.data_ptr(),
                                 beta_raw.data_ptr(), n_tok, n_head, gate.data_ptr(),
                                 beta.data_ptr(), _stream(stream)))
    return gate, beta


def make_gdn_args(conv=None, conv_out=None, z=None, y=None, gated_out=None, alpha_raw=None,
                  dt_bias=None, ssm_a=None, beta_raw=None, gate_out=None, beta_out=None,
                  n_tok=0, conv_dim=0, l2_dim=0, head_dim=GDN_STATE, inner_dim=0,
                  n_v_head=0, gate_mode=BH_SILU_MUL, eps=EPS, conv_w=None, conv_state=None,
                  conv_k=0) -> GdnPrepArgs:
    """With conv_w (and conv_state, conv_k), `conv` is the raw qkv and the
    causal conv1d runs in front of the SiLU (src/forward.rs:508-533)."""
    return GdnPrepArgs(_ptr(conv), _ptr(conv_out), _ptr(z), _ptr(y), _ptr(gated_out),
                       _ptr(alpha_raw), _ptr(dt_bias), _ptr(ssm_a), _ptr(beta_raw),
                       _ptr(gate_out), _ptr(beta_out), n_tok, conv_dim, l2_dim, head_dim,
                       inner_dim, n_v_head, gate_mode, eps, _ptr(conv_w), _ptr(conv_state),
                       conv_k if conv_w is not None else 0)


def gdn_prep_fused(args: GdnPrepArgs, stream=None) -> None:
    check(lib().bh_gdn_prep_fused(ctypes.byref(args), _stream(stream)))


def make_qk_args(q, q_out, k, k_out, wq, wk, pos, n_tok, n_q_head, n_k_head,
                 head_dim=HEAD_DIM, q_head_stride=None, n_dims=N_ROT, sections=SECTIONS,
                 freq_base=FREQ_BASE, eps=EPS, gate_out=None) -> QkNormRopeArgs:
    return QkNormRopeArgs(_ptr(q), _ptr(q_out), _ptr(gate_out), _ptr(k), _ptr(k_out), _ptr(wq),
                          _ptr(wk), _ptr(pos), n_tok, n_q_head, n_k_head, head_dim,
                          head_dim if q_head_stride is None else q_head_stride, n_dims,
                          (ctypes.c_int32 * 4)(*sections), freq_base, eps)


def qk_norm_rope(args: QkNormRopeArgs, stream=None) -> None:
    check(lib().bh_qk_norm_rope(ctypes.byref(args), _stream(stream)))


def rope_imrope(heads, pos, n_dims=N_ROT, sections=SECTIONS, freq_base=FREQ_BASE, stream=None):
    """In place on heads [n_tok, n_head, head_dim]; pos int32 [n_tok, 4]."""
    n_tok, n_head, head_dim = heads.shape
    sec = (ctypes.c_int32 * 4)(*sections)
    check(lib().bh_rope_imrope(heads.data_ptr(), n_tok, n_head, head_dim, pos.data_ptr(), n_dims,
                               sec, freq_base, _stream(stream)))
    return heads


def pq2_embed_gather(table, ne0: int, n_rows: int, ids, out=None, w=None, eps: float = EPS,
                     out_norm=None, bad_id=None, stream=None):
    """Gather ids from a packed PQ2_0 table (uint8 device tensor); with w, also
    returns the fused RMSNorm rows."""
    import torch
    n = ids.numel()
    out = torch.empty((n, ne0), dtype=torch.float32, device=ids.device) if out is None else out
    if w is None:
        check(lib().bh_pq2_embed_gather(table.data_ptr(), ne0, n_rows, ids.data_ptr(), n,
                                        out.data_ptr(), _ptr(bad_id), _stream(stream)))
        return out
    out_norm = torch.empty_like(out) if out_norm is None else out_norm
    check(lib().bh_pq2_embed_gather_rms(table.data_ptr(), ne0, n_rows, ids.data_ptr(), n,
                                        w.data_ptr(), w.numel(), eps, out.data_ptr(),
                                        out_norm.data_ptr(), _ptr(bad_id), _stream(stream)))
    return out, out_norm


def conv1d_silu(x, state, w, out=None, stream=None):
    """Causal conv1d + SiLU (src/forward.rs:508-533) over x [n_tok, ch] with
    the cache state [ch, k-1] (advanced in place) and taps w [ch, k]."""
    import torch
    n_tok, ch = x.shape
    k = w.shape[1]
    out = torch.empty_like(x) if out is None else out
    check(lib().bh_conv1d_silu(x.data_ptr(), _ptr(state), w.data_ptr(), n_tok, ch, k,
                               out.data_ptr(), _stream(stream)))
    return out


BH_KV_F32, BH_KV_F16 = 0, 1


def _kv_dtype(cache):
    import torch
    if cache.dtype == torch.float32:
        return BH_KV_F32
    if cache.dtype in (torch.float16, torch.int16, torch.uint16):
        return BH_KV_F16
    raise TypeError(f"KV cache dtype {cache.dtype}: f32 or 16-bit f16 storage")


def kv_store(k, v, k_cache, v_cache, pos0: int, stream=None):
    """AttnCache::append / append_f16 (src/forward.rs:90-95, 120-125): rows
    k, v [n_tok, n_kv_elems] f32 into the caches [cap, n_kv_elems] (f32, or
    16-bit tensors holding f16 bits) at positions pos0 .."""
    n_tok, elems = k.shape
    check(lib().bh_kv_store(k.data_ptr(), v.data_ptr(), n_tok, elems, k_cache.data_ptr(),
                            v_cache.data_ptr(), pos0, _kv_dtype(k_cache), _stream(stream)))


def attention(q, pos0: int, k_cache, v_cache, n_kv: int, out=None, stream=None):
    """The GQA block of full_attention_layer (src/forward.rs:282-375) for
    queries q [n_q, n_head, hd] at positions pos0 ..; caches [cap, n_kv*hd]."""
    import torch
    n_q, n_head, hd = q.shape
    out = torch.empty_like(q) if out is None else out
    check(lib().bh_attention(q.data_ptr(), n_q, pos0, k_cache.data_ptr(), v_cache.data_ptr(),
                             _kv_dtype(k_cache), n_head, n_kv, hd, out.data_ptr(),
                             _stream(stream)))
    return out


def _ptr(t):
    return None if t is None else t.data_ptr()


def kv_store_planar(k, v, pos0: int, n_kv: int, bits: int, kq, kn, vq=None, vn=None, v_f32=None,
                    stream=None):
    """AttnCache::append_k_quantized / append_v_quantized / append_v
    (src/forward.rs:99-140): rows k, v [n_tok, n_kv * 256] into the planar
    caches kq [cap, n_kv, plen] u8, kn [cap, n_kv] f32 (and vq / vn, or the
    f32 v_f32 [cap, n_kv * 256] when vq is None), in place."""
    n_tok = k.shape[0]
    check(lib().bh_kv_store_planar(k.data_ptr(), v.data_ptr(), n_tok, n_kv, 256, bits,
                                   kq.data_ptr(), kn.data_ptr(), _ptr(vq), _ptr(vn), _ptr(v_f32),
                                   pos0, _stream(stream)))


def attention_planar(q, pos0: int, kq, kn, n_kv: int, bits: int, vq=None, vn=None, v_f32=None,
                     out=None, stream=None):
    """The quantized-cache branches of full_attention_layer
    (src/forward.rs:296-349) for q [n_q, n_head, 256] at positions pos0 ..."""
    import torch
    n_q, n_head, hd = q.shape
    out = torch.empty_like(q) if out is None else out
    check(lib().bh_attention_planar(q.data_ptr(), n_q, pos0, kq.data_ptr(), kn.data_ptr(),
                                    _ptr(vq), _ptr(vn), _ptr(v_f32), bits, n_head, n_kv, hd,
                                    out.data_ptr(), _stream(stream)))
    return out


def gdn_step(q, k, v, gate, beta, state, attn=None, stream=None):
    """Gated delta-net recurrence (src/gdn.rs:17-77 per token) over device
    tensors q, k [n_tok, h_k, s], v [n_tok, h_v, s], gate, beta [n_tok, h_v];
    state [h_v, s, s] is advanced in place; returns attn [n_tok, h_v, s]."""
    import torch
    n_tok, h_k, s = q.shape
    h_v = v.shape[1]
    attn = torch.empty_like(v) if attn is None else attn
    check(lib().bh_gdn_step(q.data_ptr(), k.data_ptr(), v.data_ptr(), gate.data_ptr(),
                            beta.data_ptr(), state.data_ptr(), attn.data_ptr(), n_tok, h_k, h_v,
                            s, _stream(stream)))
    return attn


def pq2_matmul_n(payload, ne0: int, n_rows: int, x, base_row: int = 0, out=None, stream=None):
    """kernels::pq2_matmul_n (src/kernels.rs:340-423) on device tensors:
    payload uint8 (the tensor's whole PQ2_0 data), x [n_tok, ne0] f32 ->
    y [n_tok, n_rows]; a 1-D x runs pq2_matvec_range and returns y [n_rows]."""
    import torch
    if x.dim() == 1:
        y = torch.empty(n_rows, dtype=torch.float32, device=x.device) if out is None else out
        check(lib().bh_pq2_matvec_range(payload.data_ptr(), payload.numel(), ne0, base_row,
                                        n_rows, x.data_ptr(), x.numel(), y.data_ptr(),
                                        y.numel(), _stream(stream)))
        return y
    n_tok = x.shape[0]
    y = torch.empty((n_tok, n_rows), dtype=torch.float32, device=x.device) if out is None else out
    check(lib().bh_pq2_matmul_n(payload.data_ptr(), payload.numel(), ne0, base_row, n_rows,
                                x.data_ptr(), x.numel(), n_tok, y.data_ptr(), y.numel(),
                                _stream(stream)))
    return y


# ---------------------------------------------------------------------------
# a serving step over a paged cache (include/bonsai_hip_serve.h): argument
# blocks over device tensors, made once for buffers that stay, and the calls
# ---------------------------------------------------------------------------

BH_PAGED_MAX_REQ = 4096
BH_MAX_TOP = 32


def _dev_tensor(t, name: str, dtypes, device, shape=None):
    """t, checked: a contiguous tensor of one of dtypes on `device`."""
    if t.dtype not in dtypes or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of {dtypes[0]}, got {t.dtype}")
    if not t.is_cuda or t.get_device() != device.index:
        raise ValueError(f"{name} is on {t.device}, the call's tensors on {device}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t


def _ids_dtypes():
    import torch
    return (torch.int32, torch.uint32)


def _hold(args, device, *tensors):
    """args with the tensors whose addresses it holds, and their device."""
    args.tensors, args.device, args.index = tensors, device, device.index
    return args


_TORCH_STREAM = None  # torch's current device and raw current stream, looked up once


def _call(fn, args, stream):
    """fn(args, stream) on the device of args' tensors, whichever is current.
    (A stream object a call would cost as much as the launch.)"""
    global _TORCH_STREAM
    import torch
    if _TORCH_STREAM is None:
        _TORCH_STREAM = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
    device, raw = _TORCH_STREAM
    index = args.index
    if device() == index:
        status = fn(ctypes.byref(args), raw(index) if stream is None else stream.cuda_stream)
    else:
        with torch.cuda.device(index):
            status = fn(ctypes.byref(args), raw(index) if stream is None else stream.cuda_stream)
    if status != BH_OK:
        raise BonsaiError(status, last_error())


def make_paged_cache(k, v) -> PagedCache:
    """The pool k, v [n_pages, page_size, n_kv, hd] of f32 or f16 (or 16-bit
    integers holding f16 bits); any equal strides of the first three whose rows
    share no memory, so a transposed [n_pages, n_kv, page_size, hd] or one of
    two halves of an allocation will do (the calls refuse others)."""
    if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype:
        raise ValueError("k and v must be [n_pages, page_size, n_kv, hd], alike in shape, "
                         "strides and type")
    if not k.is_cuda or k.device != v.device:
        raise ValueError("k and v must be on one GPU")
    if k.stride(3) != 1 and k.shape[3] != 1:
        raise ValueError("a head's elements must lie side by side")
    n_pages, page_size, n_kv, hd = k.shape
    return _hold(PagedCache(k.data_ptr(), v.data_ptr(), _kv_dtype(k), n_pages, page_size, n_kv,
                            hd, k.stride(0), k.stride(1), k.stride(2)), k.device, k, v)


def make_paged_plan_args(cached, n_new, block_table, free_pages, n_free, page_size: int, *,
                         kv_len, q_start, slots, pos=None, n_free_out=None,
                         n_refused=None) -> PagedPlanArgs:
    """int32 tensors: cached, n_new, kv_len [n_req], block_table [n_req, width],
    free_pages [n_pages], n_free [1], q_start [n_req + 1], slots [n_tok],
    pos [n_tok, 4]; n_free_out [1] (None: n_free moves on in place),
    n_refused [1]."""
    import torch
    i32, dev = (torch.int32,), cached.device
    n_req, n_tok = cached.numel(), slots.numel()
    n_free_out = n_free if n_free_out is None else n_free_out
    if block_table.dim() != 2:
        raise ValueError("block_table must be [n_req, width]")
    _dev_tensor(cached, "cached", i32, dev, (n_req,))
    _dev_tensor(n_new, "n_new", i32, dev, (n_req,))
    _dev_tensor(block_table, "block_table", i32, dev, (n_req, block_table.shape[1]))
    _dev_tensor(free_pages, "free_pages", i32, dev, (free_pages.numel(),))
    _dev_tensor(kv_len, "kv_len", i32, dev, (n_req,))
    _dev_tensor(q_start, "q_start", i32, dev, (n_req + 1,))
    _dev_tensor(slots, "slots", i32, dev, (n_tok,))
    for name, word in (("n_free", n_free), ("n_free_out", n_free_out), ("n_refused", n_refused)):
        if word is not None:
            _dev_tensor(word, name, i32, dev)
            if word.numel() != 1:
                raise ValueError(f"{name} must be one word")
    if pos is not None:
        _dev_tensor(pos, "pos", i32, dev, (n_tok, 4))
    return _hold(
        PagedPlanArgs(_ptr(cached), _ptr(n_new), _ptr(block_table), _ptr(free_pages),
                      _ptr(n_free), _ptr(kv_len), _ptr(q_start), _ptr(slots), _ptr(pos),
                      _ptr(n_free_out), _ptr(n_refused), n_req, n_tok, block_table.shape[1],
                      page_size, free_pages.numel()),
        dev, cached, n_new, block_table, free_pages, n_free, kv_len, q_start, slots, pos,
        n_free_out, n_refused)


def paged_plan(args: PagedPlanArgs, stream=None) -> None:
    """A step's pages, offsets, slots and positions from the requests' lengths."""
    _call(lib().bh_paged_plan, args, stream)


def kv_store_paged(cache: PagedCache, k, v, slots, stream=None) -> None:
    """kv_store into pages: rows k, v [n_tok, n_kv * hd] f32 to the positions
    slots int32 [n_tok] of the cache (page * page_size + offset; below 0: none)."""
    import torch
    n_tok, index, f32 = slots.numel(), cache.index, torch.float32
    shape = (n_tok, cache.n_kv * cache.hd)
    if not (slots.dtype is torch.int32 and k.dtype is f32 and v.dtype is f32
            and k.shape == shape and v.shape == shape
            and slots.get_device() == k.get_device() == v.get_device() == index
            and slots.is_contiguous() and k.is_contiguous() and v.is_contiguous()):
        raise ValueError(f"k and v must be contiguous float32 tensors {shape} and slots a "
                         f"contiguous int32 tensor [{n_tok}] on {cache.device}")
    fn = lib().bh_kv_store_paged
    _call(lambda ref, s: fn(ref, k.data_ptr(), v.data_ptr(), slots.data_ptr(), n_tok, s), cache,
          stream)


def make_attention_paged_args(cache: PagedCache, q, q_start, kv_len, block_table, out=None,
                              max_new: int = 0, bad_page=None,
                              workspace=None) -> AttentionPagedArgs:
    """Queries q [n_tok, n_head, hd] f32 of the requests whose tokens begin at
    q_start int32 [n_req + 1], over kv_len int32 [n_req] positions in the pages
    block_table int32 [n_req, width].  The result is args.out_tensor (if out is
    None, zeros made on the current stream); rows of no request are left as they
    were.  workspace: a uint8 tensor
    of attention_paged_workspace(args) bytes for calls that may overlap; None:
    the library's scratch."""
    import torch
    i32, dev = (torch.int32,), cache.device
    if q.dim() != 3 or q.shape[2] != cache.hd:
        raise ValueError(f"q must be [n_tok, n_head, {cache.hd}], got {tuple(q.shape)}")
    if block_table.dim() != 2:
        raise ValueError("block_table must be [n_req, width]")
    n_req = kv_len.numel()
    _dev_tensor(q, "q", (torch.float32,), dev)
    out = torch.zeros_like(q) if out is None else out
    _dev_tensor(out, "out", (torch.float32,), dev, q.shape)
    _dev_tensor(q_start, "q_start", i32, dev, (n_req + 1,))
    _dev_tensor(kv_len, "kv_len", i32, dev, (n_req,))
    _dev_tensor(block_table, "block_table", i32, dev, (n_req, block_table.shape[1]))
    if bad_page is not None:
        _dev_tensor(bad_page, "bad_page", i32, dev)
    args = AttentionPagedArgs(cache, _ptr(q), _ptr(out), _ptr(q_start), _ptr(kv_len),
                              _ptr(block_table), _ptr(bad_page), q.shape[0], n_req, q.shape[1],
                              block_table.shape[1], max_new, None, 0)
    if workspace is not None:
        _dev_tensor(workspace, "workspace", (torch.uint8,), dev)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.numel()
    args.out_tensor = out
    return _hold(args, dev, cache.tensors, q, out, q_start, kv_len, block_table, bad_page,
                 workspace)


def attention_paged_workspace(args: AttentionPagedArgs) -> int:
    """Bytes of workspace of attention_paged(args) on the args' device."""
    import torch
    with torch.cuda.device(args.device):
        return int(lib().bh_attention_paged_workspace(ctypes.byref(args)))


def attention_paged(args: AttentionPagedArgs, stream=None):
    """attention for many requests at once over a paged cache; returns the
    output tensor of the arguments."""
    _call(lib().bh_attention_paged, args, stream)
    return args.out_tensor


def make_token_logprobs_args(x, tokens=None, n_top: int = 0, inv_temp: float = 1.0, *,
                             logprob=None, entropy=None, top_ids=None, top_logprobs=None,
                             bad_id=None, workspace=None) -> TokenLogprobsArgs:
    """Logits x [n_rows, vocab] f32 (rows any stride apart), tokens int32 or
    uint32 [n_rows].  Outputs that are None are made (logprob with tokens,
    top_ids / top_logprobs with n_top); args.results holds (logprob, entropy,
    top_ids, top_logprobs)."""
    import torch
    dev, f32, ids = x.device, (torch.float32,), _ids_dtypes()
    if x.dim() != 2 or x.dtype != torch.float32 or not x.is_cuda:
        raise ValueError("x must be a float32 CUDA tensor [n_rows, vocab]")
    n_rows, vocab = x.shape
    if vocab > 1 and x.stride(1) != 1:
        raise ValueError("a row's logits must lie side by side")
    if n_rows > 1 and x.stride(0) < vocab:
        raise ValueError("rows of x must not overlap")
    if tokens is not None:
        _dev_tensor(tokens, "tokens", ids, dev, (n_rows,))
        logprob = torch.empty(n_rows, dtype=torch.float32, device=dev) if logprob is None \
            else _dev_tensor(logprob, "logprob", f32, dev, (n_rows,))
    elif logprob is not None:
        raise ValueError("logprob needs tokens")
    entropy = torch.empty(n_rows, dtype=torch.float32, device=dev) if entropy is None \
        else _dev_tensor(entropy, "entropy", f32, dev, (n_rows,))
    if n_top:
        shape = (n_rows, n_top)
        top_ids = torch.empty(shape, dtype=torch.int32, device=dev) if top_ids is None \
            else _dev_tensor(top_ids, "top_ids", ids, dev, shape)
        top_logprobs = torch.empty(shape, dtype=torch.float32, device=dev) \
            if top_logprobs is None else _dev_tensor(top_logprobs, "top_logprobs", f32, dev, shape)
    else:
        top_ids = top_logprobs = None
    if bad_id is not None:
        _dev_tensor(bad_id, "bad_id", ids, dev)
    args = TokenLogprobsArgs(_ptr(x), _ptr(tokens), _ptr(logprob), _ptr(entropy), _ptr(top_ids),
                             _ptr(top_logprobs), _ptr(bad_id), n_rows, vocab,
                             x.stride(0) if n_rows > 1 else vocab, n_top, inv_temp, None, 0)
    if workspace is not None:
        _dev_tensor(workspace, "workspace", (torch.uint8,), dev)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.numel()
    args.results = (logprob, entropy, top_ids, top_logprobs)
    return _hold(args, dev, x, tokens, logprob, entropy, top_ids, top_logprobs, bad_id, workspace)


def token_logprobs_workspace(args: TokenLogprobsArgs) -> int:
    """Bytes of workspace of token_logprobs(args) on the args' device."""
    import torch
    with torch.cuda.device(args.device):
        return int(lib().bh_token_logprobs_workspace(ctypes.byref(args)))


def token_logprobs(args: TokenLogprobsArgs, stream=None):
    """(logprob, entropy, top_ids, top_logprobs) of each row of logits."""
    _call(lib().bh_token_logprobs, args, stream)
    return args.results


# ---------------------------------------------------------------------------
# recurrent layers of many requests, and beam search (include/bonsai_hip_batch.h)
# ---------------------------------------------------------------------------

BH_MAX_BEAMS = 32


def _rows_of(t, name: str, device, shape):
    """t, checked: float32 rows of whole `shape[1:]` blocks, any stride apart; the stride."""
    import torch
    if t.dtype != torch.float32 or not t.is_cuda or t.get_device() != device.index:
        raise ValueError(f"{name} must be a float32 tensor on {device}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    inner = 1
    for n, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        if n > 1 and stride != inner:
            raise ValueError(f"what lies within a row of {name} must be contiguous")
        inner *= n
    if t.shape[0] > 1 and t.stride(0) < inner:
        raise ValueError(f"rows of {name} must not overlap")
    return t.stride(0) if t.shape[0] > 1 else inner


def _step_of(q_start, src_slot, dst_slot, bad_slot, dev):
    """Checks what names a ragged step's requests; their number."""
    i32 = (_ids_dtypes()[0],)
    n_req = src_slot.numel()
    _dev_tensor(q_start, "q_start", i32, dev, (n_req + 1,))
    _dev_tensor(src_slot, "src_slot", i32, dev, (n_req,))
    _dev_tensor(dst_slot, "dst_slot", i32, dev, (n_req,))
    if bad_slot is not None:
        _dev_tensor(bad_slot, "bad_slot", i32, dev)
    return n_req


def make_conv_ragged_args(x, w, state, q_start, src_slot, dst_slot, out=None, l2_dim: int = 0,
                          head_dim: int = 0, eps: float = EPS, max_new: int = 0,
                          bad_slot=None) -> ConvRaggedArgs:
    """Inputs x [n_tok, ch] f32 (rows any stride apart) of the requests whose tokens
    begin at q_start int32 [n_req + 1], taps w [ch, k], the pool state
    [n_slots, ch, k - 1] (slots any stride apart), slots int32 [n_req].  The result
    is args.out_tensor (if out is None, zeros made on the current stream)."""
    import torch
    dev, f32 = x.device, (torch.float32,)
    if x.dim() != 2 or w.dim() != 2:
        raise ValueError("x must be [n_tok, ch] and w [ch, k]")
    n_tok, ch = x.shape
    k = w.shape[1]
    x_stride = _rows_of(x, "x", dev, x.shape)
    _dev_tensor(w, "w", f32, dev, (ch, k))
    if state is None and k > 1:
        raise ValueError("state must be [n_slots, ch, k - 1]")
    n_slots = 0 if state is None else state.shape[0]
    slot_stride = 0 if state is None else _rows_of(state, "state", dev, (n_slots, ch, k - 1))
    n_req = _step_of(q_start, src_slot, dst_slot, bad_slot, dev)
    out = torch.zeros((n_tok, ch), dtype=torch.float32, device=dev) if out is None else out
    _dev_tensor(out, "out", f32, dev, (n_tok, ch))
    args = ConvRaggedArgs(_ptr(x), _ptr(w), _ptr(state), _ptr(out), _ptr(q_start), _ptr(src_slot),
                          _ptr(dst_slot), _ptr(bad_slot), n_tok, n_req, ch, k, l2_dim, head_dim,
                          n_slots, x_stride, slot_stride, max_new, eps)
    args.out_tensor = out
    return _hold(args, dev, x, w, state, out, q_start, src_slot, dst_slot, bad_slot)


def conv1d_silu_ragged(args: ConvRaggedArgs, stream=None):
    """conv1d_silu (and L2 norms) of many requests at once, states in slots; returns
    the output tensor of the arguments."""
    _call(lib().bh_conv1d_silu_ragged, args, stream)
    return args.out_tensor


def make_gdn_ragged_args(q, k, v, gate, beta, state, q_start, src_slot, dst_slot, attn=None,
                         max_new: int = 0, bad_slot=None, workspace=None) -> GdnRaggedArgs:
    """q, k [n_tok, h_k, s], v [n_tok, h_v, s] f32 (tokens any stride apart, so that
    they may be parts of one row), gate, beta [n_tok, h_v], the pool state
    [n_slots, h_v, s, s] (slots any stride apart), int32 q_start [n_req + 1] and slots
    [n_req].  The result is args.attn_tensor (if attn is None, zeros made on the
    current stream)."""
    import torch
    dev, f32 = q.device, (torch.float32,)
    if q.dim() != 3 or v.dim() != 3 or state.dim() != 4:
        raise ValueError("q, k, v must be [n_tok, heads, s] and state [n_slots, h_v, s, s]")
    n_tok, h_k, s = q.shape
    h_v, n_slots = v.shape[1], state.shape[0]
    strides = [_rows_of(q, "q", dev, (n_tok, h_k, s)), _rows_of(k, "k", dev, (n_tok, h_k, s)),
               _rows_of(v, "v", dev, (n_tok, h_v, s)),
               _rows_of(state, "state", dev, (n_slots, h_v, s, s))]
    _dev_tensor(gate, "gate", f32, dev, (n_tok, h_v))
    _dev_tensor(beta, "beta", f32, dev, (n_tok, h_v))
    n_req = _step_of(q_start, src_slot, dst_slot, bad_slot, dev)
    attn = torch.zeros((n_tok, h_v, s), dtype=torch.float32, device=dev) if attn is None else attn
    _dev_tensor(attn, "attn", f32, dev, (n_tok, h_v, s))
    args = GdnRaggedArgs(_ptr(q), _ptr(k), _ptr(v), _ptr(gate), _ptr(beta), _ptr(state),
                         _ptr(attn), _ptr(q_start), _ptr(src_slot), _ptr(dst_slot),
                         _ptr(bad_slot), n_tok, n_req, h_k, h_v, s, n_slots, *strides, max_new,
                         None, 0)
    if workspace is not None:
        _dev_tensor(workspace, "workspace", (torch.uint8,), dev)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.numel()
    args.attn_tensor = attn
    return _hold(args, dev, q, k, v, gate, beta, state, attn, q_start, src_slot, dst_slot,
                 bad_slot, workspace)


def gdn_ragged_workspace(args: GdnRaggedArgs) -> int:
    """Bytes of workspace of gdn_ragged(args) on the args' device."""
    import torch
    with torch.cuda.device(args.device):
        return int(lib().bh_gdn_ragged_workspace(ctypes.byref(args)))


def gdn_ragged(args: GdnRaggedArgs, stream=None):
    """gdn_step of many requests at once, states in slots; returns the attn tensor of
    the arguments."""
    _call(lib().bh_gdn_ragged, args, stream)
    return args.attn_tensor


def make_attention_shared_args(cache: PagedCache, q, q_start, kv_len, block_table, group,
                               group_start, shared_len, out=None, max_new: int = 0,
                               max_group_new: int = 0, bad_page=None,
                               workspace=None) -> AttentionSharedArgs:
    """make_attention_paged_args, and the groups that share a prefix: group int32
    [n_req], group_start int32 [n_group + 1], shared_len int32 [n_group]."""
    paged = make_attention_paged_args(cache, q, q_start, kv_len, block_table, out, max_new,
                                      bad_page, workspace)
    i32, dev, n_group = (_ids_dtypes()[0],), paged.device, shared_len.numel()
    _dev_tensor(group, "group", i32, dev, (paged.n_req,))
    _dev_tensor(group_start, "group_start", i32, dev, (n_group + 1,))
    _dev_tensor(shared_len, "shared_len", i32, dev, (n_group,))
    args = AttentionSharedArgs(paged, _ptr(group), _ptr(group_start), _ptr(shared_len), n_group,
                               max_group_new)
    args.out_tensor = paged.out_tensor
    return _hold(args, dev, paged.tensors, group, group_start, shared_len)


def attention_shared_workspace(args: AttentionSharedArgs) -> int:
    """Bytes of workspace of attention_shared(args) on the args' device."""
    import torch
    with torch.cuda.device(args.device):
        return int(lib().bh_attention_shared_workspace(ctypes.byref(args)))


def attention_shared(args: AttentionSharedArgs, stream=None):
    """attention_paged of requests that share a prefix, which is read once a tile of
    rows of a group; returns the output tensor of the arguments."""
    _call(lib().bh_attention_shared, args, stream)
    return args.out_tensor


def make_beam_select_args(x, score, width: int, n_best: int, inv_temp: float = 1.0, *,
                          parent=None, token=None, score_out=None,
                          workspace=None) -> BeamSelectArgs:
    """Logits x [n_group * width, vocab] f32 (rows any stride apart) and the beams'
    scores f32 [n_group * width].  Outputs that are None are made; args.results holds
    (parent, token, score_out), [n_group, n_best] each."""
    import torch
    dev, f32, ids = x.device, (torch.float32,), _ids_dtypes()
    if x.dim() != 2 or width < 1 or x.shape[0] % width != 0:
        raise ValueError("x must be [n_group * width, vocab]")
    stride = _rows_of(x, "x", dev, x.shape)
    _dev_tensor(score, "score", f32, dev, (x.shape[0],))
    shape = (x.shape[0] // width, n_best)
    parent = torch.empty(shape, dtype=torch.int32, device=dev) if parent is None \
        else _dev_tensor(parent, "parent", ids[:1], dev, shape)
    token = torch.empty(shape, dtype=torch.int32, device=dev) if token is None \
        else _dev_tensor(token, "token", ids, dev, shape)
    if score_out is None:
        score_out = torch.empty(shape, dtype=torch.float32, device=dev)
    elif score_out.data_ptr() != score.data_ptr():
        _dev_tensor(score_out, "score_out", f32, dev, shape)
    else:  # the scores in place, of any shape (a vector)
        _dev_tensor(score_out, "score_out", f32, dev)
        if score_out.numel() != shape[0] * n_best:
            raise ValueError("score_out may be score only where n_best is width")
    args = BeamSelectArgs(_ptr(x), _ptr(score), _ptr(parent), _ptr(token), _ptr(score_out),
                          shape[0], width, x.shape[1], stride, n_best, inv_temp, None, 0)
    if workspace is not None:
        _dev_tensor(workspace, "workspace", (torch.uint8,), dev)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.numel()
    args.results = (parent, token, score_out)
    return _hold(args, dev, x, score, parent, token, score_out, workspace)


def beam_select_workspace(args: BeamSelectArgs) -> int:
    """Bytes of workspace of beam_select(args) on the args' device."""
    import torch
    with torch.cuda.device(args.device):
        return int(lib().bh_beam_select_workspace(ctypes.byref(args)))


def beam_select(args: BeamSelectArgs, stream=None):
    """(parent, token, score) of each group's best continuations."""
    _call(lib().bh_beam_select, args, stream)
    return args.results


def make_beam_reorder_args(parent, block_table, *, copy_from, src_slot=None, dst_slot=None,
                           spare_slot=None) -> BeamReorderArgs:
    """int32 tensors: parent [n_group, width] (rows any stride apart, as a slice of
    beam_select's), block_table [n_group * width, table_width] and copy_from, src_slot,
    dst_slot, spare_slot [n_group * width]."""
    i32, dev = (_ids_dtypes()[0],), parent.device
    if parent.dim() != 2 or block_table.dim() != 2:
        raise ValueError("parent must be [n_group, width] and block_table a matrix")
    n_group, width = parent.shape
    stride = parent.stride(0) if n_group > 1 else width
    if parent.dtype != i32[0] or not parent.is_cuda or (width > 1 and parent.stride(1) != 1) \
            or stride < width:
        raise ValueError("parent must be an int32 CUDA tensor of contiguous rows")
    _dev_tensor(block_table, "block_table", i32, dev, (n_group * width, block_table.shape[1]))
    for name, t in (("copy_from", copy_from), ("src_slot", src_slot), ("dst_slot", dst_slot),
                    ("spare_slot", spare_slot)):
        if t is not None:
            _dev_tensor(t, name, i32, dev, (n_group * width,))
    return _hold(BeamReorderArgs(_ptr(parent), _ptr(block_table), _ptr(copy_from),
                                 _ptr(src_slot), _ptr(dst_slot), _ptr(spare_slot), n_group, width,
                                 stride, block_table.shape[1]),
                 dev, parent, block_table, copy_from, src_slot, dst_slot, spare_slot)


def beam_reorder(args: BeamReorderArgs, stream=None) -> None:
    """The beams' page tables and state slots in the order of the beams selected."""
    _call(lib().bh_beam_reorder, args, stream)


def make_kv_copy_args(cache: PagedCache, block_table, copy_from, begin, end) -> KvCopyArgs:
    """int32 tensors: block_table [n_req, table_width], copy_from, begin (or None), end
    [n_req]."""
    i32, dev, n_req = (_ids_dtypes()[0],), cache.device, copy_from.numel()
    if block_table.dim() != 2:
        raise ValueError("block_table must be [n_req, table_width]")
    _dev_tensor(block_table, "block_table", i32, dev, (n_req, block_table.shape[1]))
    _dev_tensor(copy_from, "copy_from", i32, dev)
    _dev_tensor(end, "end", i32, dev, (n_req,))
    if begin is not None:
        _dev_tensor(begin, "begin", i32, dev, (n_req,))
    return _hold(KvCopyArgs(cache, _ptr(block_table), _ptr(copy_from), _ptr(begin), _ptr(end),
                            n_req, block_table.shape[1]),
                 dev, cache.tensors, block_table, copy_from, begin, end)


def kv_copy_paged(args: KvCopyArgs, stream=None) -> None:
    """The pages of one layer's cache of requests that go on from another's."""
    _call(lib().bh_kv_copy_paged, args, stream)


def env_info() -> dict:
    return {"lib": str(LIB_PATH), "version": lib().bh_version().decode(),
            "pid": os.getpid()}
