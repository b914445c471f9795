"""ikv — Python bindings for the MI355X KV-cache hot path.

Thin ctypes layer over the C-ABI declared in ``include/ikv.h`` and built into
``infer-llm_amd/lib/libikv.so``. PyTorch is used only as plumbing: device
buffers and the current HIP stream. Every call goes to the HIP kernels; there
is no CPU fallback, and loading fails loudly when the library is missing.

Return codes follow ikv.h: 0 ok, negative errno for rejected arguments,
positive hipError_t for a failed launch. Non-zero codes raise ``IkvError``.
"""
from __future__ import annotations

import ctypes
import errno
import os
import pathlib
import re
from typing import Optional

PKG_ROOT = pathlib.Path(__file__).resolve().parents[1]  # infer-llm_amd/
REPO_ROOT = PKG_ROOT.parent
LIB_PATH = PKG_ROOT / "lib" / "libikv.so"
HEADER_DIR = REPO_ROOT / "include"

_c_void_p = ctypes.c_void_p
_c_size_t = ctypes.c_size_t
_c_int = ctypes.c_int
_c_int64 = ctypes.c_int64
_c_float = ctypes.c_float


class KvPages(ctypes.Structure):
    """ikv_kv_pages (include/ikv.h): a paged KV pool's block table."""
    _fields_ = [("block_table", ctypes.c_void_p), ("block_tokens", ctypes.c_int64),
                ("n_pool_blocks", ctypes.c_int64), ("status", ctypes.c_void_p)]


_c_pages = ctypes.POINTER(KvPages)


class KvBatch(ctypes.Structure):
    """ikv_kv_batch (include/ikv_batch.h): the block tables of several sequences."""
    _fields_ = [("block_tables", ctypes.c_void_p), ("table_stride", ctypes.c_int64),
                ("block_tokens", ctypes.c_int64), ("n_pool_blocks", ctypes.c_int64),
                ("n_seq", ctypes.c_int64), ("status", ctypes.c_void_p)]


_c_batch = ctypes.POINTER(KvBatch)


class KvQ8(ctypes.Structure):
    """ikv_kv_q8 (include/ikv_batch.h): a paged cache of 8 bits an element."""
    _fields_ = [("k_codes", ctypes.c_void_p), ("k_scales", ctypes.c_void_p),
                ("v_codes", ctypes.c_void_p), ("v_scales", ctypes.c_void_p),
                ("n_head_kv", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("format", ctypes.c_int32)]


_c_q8 = ctypes.POINTER(KvQ8)


class LogitRules(ctypes.Structure):
    """ikv_logit_rules (include/ikv_model.h)."""
    _fields_ = [("history", ctypes.c_void_p), ("history_stride", ctypes.c_int64),
                ("n_history", ctypes.c_void_p), ("n_prompt", ctypes.c_void_p),
                ("repetition", ctypes.c_void_p), ("presence", ctypes.c_void_p),
                ("frequency", ctypes.c_void_p), ("bias_tokens", ctypes.c_void_p),
                ("bias_values", ctypes.c_void_p), ("bias_stride", ctypes.c_int64),
                ("n_bias", ctypes.c_void_p), ("masks", ctypes.c_void_p), ("n_masks", ctypes.c_int64),
                ("mask_of", ctypes.c_void_p)]

# name -> (restype, argtypes); include/ikv.h, ikv_batch.h, then ikv_model.h
SIGNATURES = {
    "ikv_version": (ctypes.c_char_p, []),
    "ikv_append_f32": (_c_int, [_c_void_p, _c_void_p, _c_size_t, _c_size_t, _c_void_p]),
    "ikv_attn_decode_workspace_bytes": (_c_size_t, [_c_int, _c_int, _c_int, _c_int64]),
    "ikv_attn_decode_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p,
         _c_int, _c_int, _c_int, _c_int64, _c_float, _c_void_p, _c_size_t, _c_void_p],
    ),
    "ikv_attn_decode_noalloc_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p,
         _c_int, _c_int, _c_int, _c_int64, _c_float, _c_void_p],
    ),
    "ikv_attn_decode_rope_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_int, _c_int, _c_int,
         _c_int64, _c_float, _c_void_p, _c_void_p, _c_float, _c_void_p, _c_void_p, _c_void_p,
         _c_int64, _c_void_p, _c_void_p, _c_size_t, _c_void_p],
    ),
    "ikv_qkv_attn_decode_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_float, _c_void_p, _c_void_p,
         _c_void_p, _c_int64, _c_void_p, _c_void_p, _c_void_p, _c_int, _c_int, _c_int, _c_int64,
         _c_float, _c_void_p, _c_void_p, _c_float, _c_void_p, _c_void_p, _c_void_p, _c_int64,
         _c_void_p, _c_void_p, _c_size_t, _c_void_p],
    ),
    "ikv_qkv_attn_decode_replay_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_float, _c_void_p, _c_void_p,
         _c_void_p, _c_int64, _c_void_p, _c_void_p, _c_void_p, _c_int, _c_int, _c_int, _c_int64,
         _c_float, _c_void_p, _c_void_p, _c_float, _c_void_p, _c_void_p, _c_void_p, _c_int64,
         _c_void_p, _c_void_p, _c_size_t, _c_void_p],
    ),
    "ikv_attn_decode_rope_replay_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_int, _c_int, _c_int,
         _c_int64, _c_float, _c_void_p, _c_void_p, _c_float, _c_void_p, _c_void_p, _c_void_p,
         _c_int64, _c_void_p, _c_void_p, _c_size_t, _c_void_p],
    ),
    "ikv_attn_decode_replay_limit": (_c_int64, [_c_int, _c_int, _c_int, _c_int64, _c_int64]),
    "ikv_attn_prefill_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_int, _c_int, _c_int,
         _c_int64, _c_int64, _c_int64, _c_float, _c_void_p],
    ),
    "ikv_append_paged_f32": (
        _c_int, [_c_void_p, _c_void_p, _c_pages, _c_int64, _c_size_t, _c_size_t, _c_void_p]),
    "ikv_attn_decode_paged_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_pages, _c_void_p, _c_void_p, _c_void_p,
         _c_int, _c_int, _c_int, _c_int64, _c_float, _c_void_p, _c_size_t, _c_void_p],
    ),
    "ikv_attn_decode_rope_paged_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_pages, _c_void_p, _c_int,
         _c_int, _c_int, _c_int64, _c_float, _c_void_p, _c_void_p, _c_float, _c_void_p,
         _c_void_p, _c_void_p, _c_int64, _c_void_p, _c_void_p, _c_size_t, _c_void_p],
    ),
    "ikv_attn_decode_rope_paged_replay_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_pages, _c_void_p, _c_int,
         _c_int, _c_int, _c_int64, _c_float, _c_void_p, _c_void_p, _c_float, _c_void_p,
         _c_void_p, _c_void_p, _c_int64, _c_void_p, _c_void_p, _c_size_t, _c_void_p],
    ),
    "ikv_attn_prefill_paged_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_pages, _c_void_p, _c_int, _c_int, _c_int,
         _c_int64, _c_int64, _c_int64, _c_float, _c_void_p],
    ),
    "ikv_rms_norm_f32": (
        _c_int, [_c_void_p, _c_void_p, _c_void_p, _c_int64, _c_int64, _c_float, _c_void_p]),
    "ikv_rope_theta_table_f32": (_c_int, [_c_float, _c_int, _c_int64, _c_void_p]),
    "ikv_rope_sincos_table_f32": (_c_int, [_c_void_p, _c_size_t, _c_void_p, _c_void_p]),
    "ikv_rope_neox_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_int64, _c_int, _c_int, _c_void_p, _c_void_p,
         _c_int64, _c_void_p, _c_void_p],
    ),
    "ikv_qk_norm_rope_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_int64, _c_int, _c_int, _c_float,
         _c_void_p, _c_void_p, _c_int64, _c_void_p, _c_void_p],
    ),
    # include/ikv_batch.h
    "ikv_append_packed_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_batch, _c_void_p, _c_void_p, _c_int64,
         _c_size_t, _c_void_p],
    ),
    "ikv_attn_prefill_packed_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_int64, _c_int64, _c_void_p, _c_int, _c_int,
         _c_int, _c_float, _c_void_p, _c_void_p],
    ),
    "ikv_attn_prefill_packed_paged_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_batch, _c_void_p, _c_void_p, _c_int64, _c_void_p,
         _c_int, _c_int, _c_int, _c_float, _c_void_p, _c_size_t, _c_void_p],
    ),
    "ikv_attn_prefill_packed_paged_workspace_bytes": (
        _c_size_t, [_c_int64, _c_int64, _c_int64, _c_int, _c_int, _c_int]),
    "ikv_attn_decode_batch_workspace_bytes": (_c_size_t, [_c_int, _c_int, _c_int]),
    "ikv_attn_decode_batch_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_batch, _c_void_p, _c_void_p, _c_void_p, _c_void_p,
         _c_int, _c_int, _c_int, _c_float, _c_void_p, _c_size_t, _c_void_p],
    ),
    "ikv_append_packed_q8": (
        _c_int,
        [_c_q8, _c_void_p, _c_void_p, _c_batch, _c_void_p, _c_void_p, _c_int64, _c_void_p],
    ),
    "ikv_read_packed_q8": (
        _c_int,
        [_c_q8, _c_void_p, _c_void_p, _c_batch, _c_void_p, _c_void_p, _c_void_p, _c_int64, _c_void_p],
    ),
    "ikv_attn_decode_batch_q8_workspace_bytes": (_c_size_t, [_c_int, _c_int, _c_int]),
    "ikv_attn_decode_batch_q8": (
        _c_int,
        [_c_void_p, _c_q8, _c_batch, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_int, _c_float,
         _c_void_p, _c_size_t, _c_void_p],
    ),
    "ikv_attn_decode_shared_workspace_bytes": (
        _c_size_t, [_c_int64, _c_int64, _c_int, _c_int, _c_int]),
    "ikv_attn_decode_shared_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_batch, _c_void_p, _c_void_p, _c_int64, _c_void_p,
         _c_void_p, _c_void_p, _c_void_p, _c_int, _c_int, _c_int, _c_float, _c_void_p, _c_size_t,
         _c_void_p],
    ),
    # include/ikv_model.h
    "ikv_mul_mat_f32": (
        _c_int, [_c_void_p, _c_void_p, _c_void_p, _c_int64, _c_int64, _c_int64, _c_void_p, _c_void_p]),
    "ikv_gemm_nt_f32": (
        _c_int, [_c_void_p, _c_void_p, _c_void_p, _c_int64, _c_int64, _c_int64, _c_void_p, _c_void_p]),
    "ikv_gemv3_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p,
         _c_int64, _c_int64, _c_int64, _c_int64, _c_void_p, _c_float, _c_void_p],
    ),
    "ikv_gemv_swiglu_f32": (
        _c_int, [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_int64, _c_int64, _c_void_p, _c_float,
                 _c_void_p]),
    "ikv_get_rows_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_int64, _c_int64, _c_int64, _c_void_p, _c_void_p]),
    "ikv_add_f32": (_c_int, [_c_void_p, _c_void_p, _c_void_p, _c_int64, _c_void_p]),
    "ikv_mul_f32": (_c_int, [_c_void_p, _c_void_p, _c_void_p, _c_int64, _c_void_p]),
    "ikv_silu_f32": (_c_int, [_c_void_p, _c_void_p, _c_int64, _c_void_p]),
    "ikv_silu_mul_f32": (_c_int, [_c_void_p, _c_void_p, _c_void_p, _c_int64, _c_void_p]),
    "ikv_argmax_f32": (_c_int, [_c_void_p, _c_int64, _c_void_p, _c_void_p, _c_void_p]),
    "ikv_argmax_workspace_bytes": (_c_size_t, []),
    "ikv_argmax_ws_f32": (
        _c_int, [_c_void_p, _c_int64, _c_void_p, _c_void_p, _c_void_p, _c_size_t, _c_void_p]),
    "ikv_adjust_logits_f32": (
        _c_int,
        [_c_void_p, _c_void_p, ctypes.POINTER(LogitRules), _c_int64, _c_int64, _c_void_p, _c_void_p]),
    "ikv_sample_workspace_bytes": (_c_size_t, [_c_int64, _c_int64]),
    "ikv_sample_f32": (
        _c_int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_int64, _c_int64,
         _c_void_p, _c_void_p, _c_void_p, _c_size_t, _c_void_p],
    ),
    "ikv_synth_normal_f32": (
        _c_int, [ctypes.c_uint64, ctypes.c_uint64, _c_size_t, ctypes.c_double, _c_void_p, _c_int]),
}

# libikv_bench.so, the measurement library (infer-llm_amd/bench/ikv_bench.h):
# its own entry points; its decode build also has include/ikv.h's decode ones
BENCH_LIB_PATH = PKG_ROOT / "lib" / "libikv_bench.so"
BENCH_HEADER = PKG_ROOT / "bench" / "ikv_bench.h"
BENCH_SIGNATURES = {
    "ikv_probe_read": (_c_int, [_c_void_p, _c_size_t, _c_void_p, _c_int, _c_int, _c_void_p]),
    "ikv_probe_empty": (_c_int, [_c_int, _c_void_p]),
    "ikv_bench_timeline_read": (_c_int, [_c_void_p, _c_size_t]),
    "ikv_bench_timeline_clear": (_c_int, []),
    "ikv_bench_gemm_nt_tile_f32": (
        _c_int, [_c_void_p, _c_void_p, _c_void_p, _c_int64, _c_int64, _c_int64, _c_void_p, _c_int,
                 _c_int, _c_void_p, _c_size_t, _c_void_p]),
    "ikv_bench_gemm_plan": (_c_int, [_c_int64, _c_int64, _c_int64, _c_void_p, _c_void_p]),
    "ikv_bench_gemm_choice": (_c_int, [_c_int64, _c_int64, _c_int64, _c_void_p, _c_void_p]),
}


class IkvError(RuntimeError):
    """A C-ABI entry point returned a non-zero code."""

    def __init__(self, fn: str, rc: int):
        self.fn, self.rc = fn, rc
        if rc < 0:
            what = errno.errorcode.get(-rc, str(-rc))
            super().__init__(f"{fn} rejected its arguments: -{what}")
        else:
            super().__init__(f"{fn} launch failed: hipError_t {rc}")


_lib: Optional[ctypes.CDLL] = None
_bench_lib: Optional[ctypes.CDLL] = None


def header_functions() -> list[str]:
    """Names of the entry points declared in include/*.h."""
    names = set()
    for h in sorted(HEADER_DIR.glob("*.h")):
        text = re.sub(r"/\*.*?\*/", "", h.read_text(), flags=re.S)
        names |= set(re.findall(r"\b(ikv_[a-z0-9_]+)\s*\(", text))
    return sorted(names)


def load_bench() -> ctypes.CDLL:
    """Load libikv_bench.so (once): the probes, the timeline reader, and the
    stamped decode build's entry points (with include/ikv.h's signatures).
    Its own symbols stay local to its handle, apart from libikv.so's."""
    global _bench_lib
    if _bench_lib is not None:
        return _bench_lib
    if not BENCH_LIB_PATH.exists():
        raise FileNotFoundError(f"{BENCH_LIB_PATH} is not built")
    lib = ctypes.CDLL(str(BENCH_LIB_PATH))
    for name, (res, args) in BENCH_SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    for name in ("ikv_attn_decode_f32", "ikv_attn_decode_workspace_bytes"):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = SIGNATURES[name]
    _bench_lib = lib
    return lib


def load() -> ctypes.CDLL:
    """Load libikv.so (once). Raises if the library has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise FileNotFoundError(
            f"{LIB_PATH} is not built; run `python -c 'import __graft_entry__ as g; g.build()'`")
    lib = ctypes.CDLL(str(LIB_PATH))
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


def _check(fn: str, rc: int) -> None:
    if rc != 0:
        raise IkvError(fn, rc)


# ----------------------------------------------------------------------------
# torch plumbing
# ----------------------------------------------------------------------------

def _torch():
    import torch  # imported lazily so CPU-only users of the ABI need no torch
    return torch


def _ptr(t) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _stream(stream=None) -> int:
    if stream is not None:
        return stream.cuda_stream
    torch = _torch()
    if torch.cuda.is_initialized():
        # the current stream's handle without a Stream object around it: 0.3 us
        # against 2.9, of a call's 7.4 (a one-row norm)
        return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())
    return torch.cuda.current_stream().cuda_stream


def _need_f32_dev(name: str, t) -> None:
    torch = _torch()
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


# ----------------------------------------------------------------------------
# entry points
# ----------------------------------------------------------------------------

def version() -> str:
    return load().ikv_version().decode()


def append(dst_rows, src_rows, stream=None) -> None:
    """KV append: copy src_rows into dst_rows (both contiguous device tensors of
    equal byte size; dst_rows is the writable cache view)."""
    _need_f32_dev("dst_rows", dst_rows)
    _need_f32_dev("src_rows", src_rows)
    if dst_rows.numel() != src_rows.numel():
        raise ValueError("append: size mismatch")
    n_rows = src_rows.shape[0] if src_rows.dim() > 0 else 1
    row_bytes = src_rows.numel() * 4 // max(n_rows, 1)
    _check("ikv_append_f32",
           load().ikv_append_f32(_ptr(dst_rows), _ptr(src_rows), n_rows, row_bytes, _stream(stream)))


def decode_replay_limit(n_head: int, n_head_kv: int, head_dim: int, n_kv: int, width: int) -> int:
    return int(load().ikv_attn_decode_replay_limit(n_head, n_head_kv, head_dim, n_kv, width))


def decode_workspace_bytes(n_head: int, n_head_kv: int, head_dim: int, n_kv: int) -> int:
    return int(load().ikv_attn_decode_workspace_bytes(n_head, n_head_kv, head_dim, n_kv))


def decode_workspace(n_head: int, n_head_kv: int, head_dim: int, n_kv: int, device="cuda"):
    """Zero-filled workspace for attn_decode at every context up to n_kv
    (reusable across ordered launches). The split count is not monotone in
    the context (it peaks where a split's tile count steps down), so every
    context is asked."""
    torch = _torch()
    nbytes = 256
    for n in range(1, n_kv + 1):
        nbytes = max(nbytes, decode_workspace_bytes(n_head, n_head_kv, head_dim, n))
    return torch.zeros((nbytes + 3) // 4, dtype=torch.float32, device=device)


def attn_decode(q, k_cache, v_cache, n_kv: int, *, k_new=None, v_new=None, out=None,
                scale: float = 0.0, workspace=None, stream=None):
    """Decode attention for one query token over cache rows [0, n_kv).

    q: [n_head, D]; k_cache/v_cache: [capacity, n_head_kv, D]; when k_new/v_new
    ([n_head_kv, D]) are given, row n_kv-1 is taken from them and appended."""
    torch = _torch()
    for name, t in (("q", q), ("k_cache", k_cache), ("v_cache", v_cache)):
        _need_f32_dev(name, t)
    n_head, D = q.shape[-2], q.shape[-1]
    n_head_kv = k_cache.shape[-2]
    if k_cache.shape[0] < n_kv or v_cache.shape[0] < n_kv:
        raise ValueError("cache shorter than n_kv")
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new go together")
    if k_new is not None:
        _need_f32_dev("k_new", k_new)
        _need_f32_dev("v_new", v_new)
        if k_new.numel() != n_head_kv * D or v_new.numel() != n_head_kv * D:
            raise ValueError("k_new/v_new must hold one token row")
    if out is None:
        out = torch.empty((n_head, D), dtype=torch.float32, device=q.device)
    _need_f32_dev("out", out)
    if workspace is None:
        workspace = decode_workspace(n_head, n_head_kv, D, n_kv, device=q.device)
    rc = load().ikv_attn_decode_f32(
        _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(k_new), _ptr(v_new), _ptr(out),
        n_head, n_head_kv, D, n_kv, scale, _ptr(workspace), workspace.numel() * 4, _stream(stream))
    _check("ikv_attn_decode_f32", rc)
    return out


# IKV_STATUS_* bits (include/ikv.h) a kernel raises in a device status word
STATUS_POSITION, STATUS_BLOCK, STATUS_TOKEN = 1, 2, 4

# IKV_DECODE_NOALLOC_SCRATCH_BYTES (include/ikv.h): the device array that
# attn_decode_noalloc keeps its split partials and counters in
NOALLOC_SCRATCH_BYTES = 2 << 20


def attn_decode_noalloc(q, k_cache, v_cache, n_kv: int, *, out, k_new=None, v_new=None,
                        scale: float = 0.0, stream=None):
    """attn_decode without a workspace: nothing is allocated (out is the
    caller's). The library's per-device scratch array holds the split
    partials, so calls on one device must be ordered on one stream."""
    for name, t in (("q", q), ("k_cache", k_cache), ("v_cache", v_cache), ("out", out)):
        _need_f32_dev(name, t)
    n_head, D = q.shape[-2], q.shape[-1]
    n_head_kv = k_cache.shape[-2]
    if k_cache.shape[0] < n_kv or v_cache.shape[0] < n_kv:
        raise ValueError("cache shorter than n_kv")
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new go together")
    if k_new is not None:
        _need_f32_dev("k_new", k_new)
        _need_f32_dev("v_new", v_new)
        if k_new.numel() != n_head_kv * D or v_new.numel() != n_head_kv * D:
            raise ValueError("k_new/v_new must hold one token row")
    if out.numel() != n_head * D:
        raise ValueError("out must hold n_head rows")
    rc = load().ikv_attn_decode_noalloc_f32(
        _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(k_new), _ptr(v_new), _ptr(out),
        n_head, n_head_kv, D, n_kv, scale, _stream(stream))
    _check("ikv_attn_decode_noalloc_f32", rc)
    return out


def qkv_attn_decode(w_q, w_k, w_v, x, k_cache, v_cache, n_kv: int, q_norm_w, k_norm_w,
                    eps: float, pos, sin_tab, cos_tab, *, attn_norm_w=None, attn_eps: float = 0.0,
                    q_out=None, k_out=None, v_out=None, out=None, scale: float = 0.0, status=None,
                    workspace=None, replay=False, stream=None):
    """One token's q/k/v projections (attn_norm folded in when attn_norm_w is
    given) and its decode (qk-norm + RoPE + append + attention) in one launch,
    for contexts of one decode split. Returns (out, q_out, k_out, v_out).
    replay=True: the replay form, n_kv is then the planned maximum and the
    context is pos[0] + 1, read on the device."""
    torch = _torch()
    n_embd = x.numel()
    D = k_cache.shape[-1]
    n_head_kv = k_cache.shape[-2]
    n_head = w_q.shape[0] // D
    dev = x.device
    if q_out is None:
        q_out = torch.empty((n_head, D), dtype=torch.float32, device=dev)
    if k_out is None:
        k_out = torch.empty((n_head_kv, D), dtype=torch.float32, device=dev)
    if v_out is None:
        v_out = torch.empty((n_head_kv, D), dtype=torch.float32, device=dev)
    if out is None:
        out = torch.empty((n_head, D), dtype=torch.float32, device=dev)
    if workspace is None:
        workspace = decode_workspace(n_head, n_head_kv, D, n_kv, device=dev)
    fn = "ikv_qkv_attn_decode_replay_f32" if replay else "ikv_qkv_attn_decode_f32"
    rc = getattr(load(), fn)(
        _ptr(w_q), _ptr(w_k), _ptr(w_v), _ptr(x), _ptr(attn_norm_w), attn_eps, _ptr(q_out),
        _ptr(k_out), _ptr(v_out), n_embd, _ptr(k_cache), _ptr(v_cache), _ptr(out), n_head,
        n_head_kv, D, n_kv, scale, _ptr(q_norm_w), _ptr(k_norm_w), eps, _ptr(pos), _ptr(sin_tab),
        _ptr(cos_tab), sin_tab.shape[0], _ptr(status), _ptr(workspace), workspace.numel() * 4,
        _stream(stream))
    _check(fn, rc)
    return out, q_out, k_out, v_out


def attn_decode_rope(q_raw, k_raw, v_new, k_cache, v_cache, n_kv: int, q_norm_w, k_norm_w,
                     eps: float, pos, sin_tab, cos_tab, *, out=None, scale: float = 0.0,
                     status=None, workspace=None, replay=False, stream=None):
    """Decode with qk-RMSNorm + RoPE folded in: q/k rotated at position pos[0],
    k (rotated) and v_new appended at row n_kv-1, attention over [0, n_kv).
    replay=True: the replay form, n_kv is then the planned maximum and the
    context is pos[0] + 1, read on the device."""
    torch = _torch()
    n_head, D = q_raw.shape[-2], q_raw.shape[-1]
    n_head_kv = k_cache.shape[-2]
    if out is None:
        out = torch.empty((n_head, D), dtype=torch.float32, device=q_raw.device)
    if workspace is None:
        workspace = decode_workspace(n_head, n_head_kv, D, n_kv, device=q_raw.device)
    fn = "ikv_attn_decode_rope_replay_f32" if replay else "ikv_attn_decode_rope_f32"
    rc = getattr(load(), fn)(
        _ptr(q_raw), _ptr(k_raw), _ptr(v_new), _ptr(k_cache), _ptr(v_cache), _ptr(out), n_head,
        n_head_kv, D, n_kv, scale, _ptr(q_norm_w), _ptr(k_norm_w), eps, _ptr(pos), _ptr(sin_tab),
        _ptr(cos_tab), sin_tab.shape[0], _ptr(status), _ptr(workspace), workspace.numel() * 4,
        _stream(stream))
    _check(fn, rc)
    return out


def attn_prefill(q, k, v, n_past: int = 0, *, n_kv: Optional[int] = None, out=None,
                 scale: float = 0.0, stream=None):
    """Causal attention for q [n_q, n_head, D] over k, v [>= n_kv, n_head_kv, D]."""
    torch = _torch()
    for name, t in (("q", q), ("k", k), ("v", v)):
        _need_f32_dev(name, t)
    n_q, n_head, D = q.shape
    n_head_kv = k.shape[1]
    if n_kv is None:
        n_kv = n_past + n_q
    if out is None:
        out = torch.empty_like(q)
    _need_f32_dev("out", out)
    rc = load().ikv_attn_prefill_f32(_ptr(q), _ptr(k), _ptr(v), _ptr(out), n_head, n_head_kv, D,
                                     n_q, n_kv, n_past, scale, _stream(stream))
    _check("ikv_attn_prefill_f32", rc)
    return out


# ----------------------------------------------------------------------------
# paged KV pool: [n_blocks * block_tokens, n_head_kv, D] per K and V; logical
# token t in pool row table[t // block_tokens] * block_tokens + t % block_tokens
# ----------------------------------------------------------------------------

def kv_pages(table, block_tokens: int, pool, status=None) -> KvPages:
    """The ikv_kv_pages descriptor of a device int32 block table over `pool`."""
    torch = _torch()
    if table.dtype != torch.int32 or not table.is_cuda or not table.is_contiguous():
        raise ValueError("block table must be a contiguous device int32 tensor")
    if pool.shape[0] % block_tokens:
        raise ValueError("pool rows must be whole blocks")
    return KvPages(table.data_ptr(), block_tokens, pool.shape[0] // block_tokens, _ptr(status))


def append_paged(pool, src_rows, table, block_tokens: int, first_token: int, status=None,
                 stream=None) -> None:
    """Writes src_rows [n, n_head_kv, D] to logical tokens first_token.. of the pool."""
    _need_f32_dev("pool", pool)
    _need_f32_dev("src_rows", src_rows)
    n_rows = src_rows.shape[0]
    row_bytes = src_rows[0].numel() * 4 if n_rows else 0
    pg = kv_pages(table, block_tokens, pool, status)
    _check("ikv_append_paged_f32",
           load().ikv_append_paged_f32(_ptr(pool), _ptr(src_rows), ctypes.byref(pg), first_token,
                                       n_rows, row_bytes, _stream(stream)))


def attn_decode_paged(q, k_pool, v_pool, table, block_tokens: int, n_kv: int, *, k_new=None,
                      v_new=None, out=None, scale: float = 0.0, status=None, workspace=None,
                      stream=None):
    """attn_decode over a paged pool (logical rows [0, n_kv) through `table`)."""
    torch = _torch()
    for name, t in (("q", q), ("k_pool", k_pool), ("v_pool", v_pool)):
        _need_f32_dev(name, t)
    n_head, D = q.shape[-2], q.shape[-1]
    n_head_kv = k_pool.shape[-2]
    if out is None:
        out = torch.empty((n_head, D), dtype=torch.float32, device=q.device)
    if workspace is None:
        workspace = decode_workspace(n_head, n_head_kv, D, n_kv, device=q.device)
    pg = kv_pages(table, block_tokens, k_pool, status)
    rc = load().ikv_attn_decode_paged_f32(
        _ptr(q), _ptr(k_pool), _ptr(v_pool), ctypes.byref(pg), _ptr(k_new), _ptr(v_new),
        _ptr(out), n_head, n_head_kv, D, n_kv, scale, _ptr(workspace), workspace.numel() * 4,
        _stream(stream))
    _check("ikv_attn_decode_paged_f32", rc)
    return out


def attn_decode_rope_paged(q_raw, k_raw, v_new, k_pool, v_pool, table, block_tokens: int,
                           n_kv: int, q_norm_w, k_norm_w, eps: float, pos, sin_tab, cos_tab, *,
                           out=None, scale: float = 0.0, status=None, page_status=None,
                           workspace=None, replay=False, stream=None):
    """attn_decode_rope over a paged pool (replay=True: the replay form, n_kv
    the planned maximum, the context pos[0] + 1 read on the device)."""
    torch = _torch()
    n_head, D = q_raw.shape[-2], q_raw.shape[-1]
    n_head_kv = k_pool.shape[-2]
    if out is None:
        out = torch.empty((n_head, D), dtype=torch.float32, device=q_raw.device)
    if workspace is None:
        workspace = decode_workspace(n_head, n_head_kv, D, n_kv, device=q_raw.device)
    pg = kv_pages(table, block_tokens, k_pool, page_status)
    fn = "ikv_attn_decode_rope_paged_replay_f32" if replay else "ikv_attn_decode_rope_paged_f32"
    rc = getattr(load(), fn)(
        _ptr(q_raw), _ptr(k_raw), _ptr(v_new), _ptr(k_pool), _ptr(v_pool), ctypes.byref(pg),
        _ptr(out), n_head, n_head_kv, D, n_kv, scale, _ptr(q_norm_w), _ptr(k_norm_w), eps,
        _ptr(pos), _ptr(sin_tab), _ptr(cos_tab), sin_tab.shape[0], _ptr(status), _ptr(workspace),
        workspace.numel() * 4, _stream(stream))
    _check(fn, rc)
    return out


def attn_prefill_paged(q, k_pool, v_pool, table, block_tokens: int, n_past: int = 0, *,
                       n_kv: Optional[int] = None, out=None, scale: float = 0.0, status=None,
                       stream=None):
    """attn_prefill over a paged pool."""
    torch = _torch()
    for name, t in (("q", q), ("k_pool", k_pool), ("v_pool", v_pool)):
        _need_f32_dev(name, t)
    n_q, n_head, D = q.shape
    n_head_kv = k_pool.shape[1]
    if n_kv is None:
        n_kv = n_past + n_q
    if out is None:
        out = torch.empty_like(q)
    pg = kv_pages(table, block_tokens, k_pool, status)
    rc = load().ikv_attn_prefill_paged_f32(_ptr(q), _ptr(k_pool), _ptr(v_pool), ctypes.byref(pg),
                                           _ptr(out), n_head, n_head_kv, D, n_q, n_kv, n_past,
                                           scale, _stream(stream))
    _check("ikv_attn_prefill_paged_f32", rc)
    return out


# ----------------------------------------------------------------------------
# a step over several sequences (include/ikv_batch.h): the pools as above, a
# block table per sequence ([n_seq, blocks] int32), and the sequences' sizes as
# device int32 tensors, which a captured call reads anew at every replay
# ----------------------------------------------------------------------------

def _operands(device, floats, float_names, ints, int_names):
    """Contiguous float32 and int32 tensors on `device`, a device; None is left out."""
    torch = _torch()
    index = device.index if device.type == "cuda" else None
    for want, tensors, names in ((torch.float32, floats, float_names), (torch.int32, ints, int_names)):
        for t in tensors:
            # (get_device: below 0 off the GPUs; 0.04 us where comparing devices took 0.14)
            if t is None or (t.dtype is want and t.get_device() == index and t.is_contiguous()):
                continue
            name = names.split()[next(i for i, x in enumerate(tensors) if x is t)]
            if t.dtype is not want:
                raise TypeError(f"{name} must be {want}, got {t.dtype}")
            if t.device != device or not t.is_cuda:
                raise ValueError(f"{name} must be on the device of the others")
            raise ValueError(f"{name} must be contiguous")


class _Here:
    """The current device and stream as they are."""

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_here = _Here()


def _raw_stream(device) -> int:
    """The handle of the current stream of `device`, on which there are tensors."""
    return _torch()._C._cuda_getCurrentRawStream(device.index)


def _on(device, stream):
    """The context of a launch on `device`, on which there are tensors: its current
    stream, or `stream`. What is allocated in it belongs to that stream."""
    torch = _torch()
    if stream is None:
        if torch._C._cuda_getDevice() == device.index:
            return _here
        return torch.cuda.stream(torch.cuda.current_stream(device))
    if stream.device != device:
        raise ValueError("stream and tensors must be on one device")
    return torch.cuda.stream(stream)


def kv_batch(tables, block_tokens: int, pool, status=None) -> KvBatch:
    """The ikv_kv_batch descriptor of device int32 block tables [n_seq, blocks]
    over `pool` (and the V pool of its shape)."""
    if tables.dim() != 2:
        raise ValueError("tables must be [n_seq, blocks]")
    if block_tokens <= 0 or pool.shape[0] % block_tokens:
        raise ValueError("pool rows must be whole blocks")
    n_seq, width = tables.shape
    return KvBatch(tables.data_ptr(), width, block_tokens, pool.shape[0] // block_tokens, n_seq,
                   _ptr(status))


def _need_pools(k_pool, v_pool, n_head_kv: int, head_dim: int) -> None:
    if k_pool.dim() != 3 or k_pool.shape != v_pool.shape:
        raise ValueError("k_pool and v_pool must be of one shape [rows, n_head_kv, head_dim]")
    if k_pool.shape[1] != n_head_kv or k_pool.shape[2] != head_dim:
        raise ValueError("the pools' heads differ from the rows'")


def append_packed(k_pool, v_pool, k_rows, v_rows, tables, block_tokens: int, row_start,
                  first_token=None, *, status=None, stream=None) -> None:
    """Rows [row_start[s], row_start[s + 1]) of k_rows and v_rows [n, n_head_kv, D]
    become sequence s's tokens first_token[s].. (0.. without it) in the pools."""
    dev = k_pool.device
    _operands(dev, (k_pool, v_pool, k_rows, v_rows), "k_pool v_pool k_rows v_rows",
              (tables, row_start, first_token, status), "tables row_start first_token status")
    if k_rows.dim() != 3 or k_rows.shape != v_rows.shape:
        raise ValueError("k_rows and v_rows must be of one shape [rows, n_head_kv, head_dim]")
    n_rows, n_head_kv, D = k_rows.shape
    _need_pools(k_pool, v_pool, n_head_kv, D)
    bt = kv_batch(tables, block_tokens, k_pool, status)
    if row_start.numel() != bt.n_seq + 1:
        raise ValueError("row_start must hold n_seq + 1 rows")
    if first_token is not None and first_token.numel() != bt.n_seq:
        raise ValueError("first_token must hold a token per sequence")
    with _on(dev, stream):
        _check("ikv_append_packed_f32",
               load().ikv_append_packed_f32(_ptr(k_pool), _ptr(v_pool), _ptr(k_rows), _ptr(v_rows),
                                            ctypes.byref(bt), _ptr(row_start), _ptr(first_token),
                                            n_rows, n_head_kv * D * 4, _raw_stream(dev)))


def attn_prefill_packed(q, k, v, row_start, *, out=None, scale: float = 0.0, status=None,
                        stream=None):
    """Causal attention of several prompts packed one behind the other: rows
    [row_start[s], row_start[s + 1]) of q [n, n_head, D] and of k, v
    [n, n_head_kv, D]. Rows of no sequence are left as `out` has them (an `out`
    that is allocated here: undefined)."""
    torch = _torch()
    dev = q.device
    _operands(dev, (q, k, v, out), "q k v out", (row_start, status), "row_start status")
    n_rows, n_head, D = q.shape
    if k.dim() != 3 or k.shape != v.shape or k.shape[0] != n_rows or k.shape[2] != D:
        raise ValueError("k and v must be [rows of q, n_head_kv, head_dim]")
    if row_start.numel() < 1:
        raise ValueError("row_start must hold n_seq + 1 rows")
    if out is not None and out.shape != q.shape:
        raise ValueError("out must be of q's shape")
    with _on(dev, stream):
        if out is None:
            out = torch.empty_like(q)
        _check("ikv_attn_prefill_packed_f32",
               load().ikv_attn_prefill_packed_f32(_ptr(q), _ptr(k), _ptr(v), _ptr(row_start),
                                                  row_start.numel() - 1, n_rows, _ptr(out), n_head,
                                                  k.shape[1], D, scale, _ptr(status), _raw_stream(dev)))
    return out


def prefill_packed_workspace(n_seq: int, n_rows: int, max_tokens: int, n_head: int, n_head_kv: int,
                             head_dim: int, device="cuda"):
    """Workspace of attn_prefill_packed_paged for these sizes (max_tokens: what a
    table covers), or None where it uses none."""
    torch = _torch()
    nbytes = int(load().ikv_attn_prefill_packed_paged_workspace_bytes(n_seq, n_rows, max_tokens, n_head,
                                                                      n_head_kv, head_dim))
    return torch.empty((nbytes + 3) // 4, dtype=torch.float32, device=device) if nbytes else None


def attn_prefill_packed_paged(q, k_pool, v_pool, tables, block_tokens: int, row_start, n_past=None,
                              *, out=None, scale: float = 0.0, status=None, workspace=None, stream=None):
    """attn_prefill_packed over paged pools that hold the new rows already, each
    sequence's queries behind n_past[s] cached tokens (none without it). Without
    `workspace` (prefill_packed_workspace) one is allocated where it is used."""
    torch = _torch()
    dev = q.device
    _operands(dev, (q, k_pool, v_pool, out, workspace), "q k_pool v_pool out workspace",
              (tables, row_start, n_past, status), "tables row_start n_past status")
    n_rows, n_head, D = q.shape
    n_head_kv = k_pool.shape[-2]
    _need_pools(k_pool, v_pool, n_head_kv, D)
    bt = kv_batch(tables, block_tokens, k_pool, status)
    if row_start.numel() != bt.n_seq + 1:
        raise ValueError("row_start must hold n_seq + 1 rows")
    if n_past is not None and n_past.numel() != bt.n_seq:
        raise ValueError("n_past must hold a count per sequence")
    if out is not None and out.shape != q.shape:
        raise ValueError("out must be of q's shape")
    with _on(dev, stream):
        if out is None:
            out = torch.empty_like(q)
        if workspace is None and n_past is not None:
            workspace = prefill_packed_workspace(bt.n_seq, n_rows, bt.table_stride * block_tokens, n_head,
                                                 n_head_kv, D, device=dev)
        _check("ikv_attn_prefill_packed_paged_f32",
               load().ikv_attn_prefill_packed_paged_f32(
                   _ptr(q), _ptr(k_pool), _ptr(v_pool), ctypes.byref(bt), _ptr(row_start),
                   _ptr(n_past), n_rows, _ptr(out), n_head, n_head_kv, D, scale, _ptr(workspace),
                   0 if workspace is None else workspace.numel() * 4, _raw_stream(dev)))
    return out


def decode_batch_workspace(n_head: int, n_head_kv: int, head_dim: int, device="cuda"):
    """Zero-filled workspace of attn_decode_batch for these heads: any number of
    sequences, any lengths (reusable across ordered launches)."""
    torch = _torch()
    nbytes = int(load().ikv_attn_decode_batch_workspace_bytes(n_head, n_head_kv, head_dim))
    return torch.zeros((nbytes + 3) // 4, dtype=torch.float32, device=device)


def attn_decode_batch(q, k_pool, v_pool, tables, block_tokens: int, n_kv, *, k_new=None, v_new=None,
                      out=None, scale: float = 0.0, status=None, workspace=None, stream=None):
    """Decode attention of one new token per sequence: q [n_seq, n_head, D] over
    the n_kv[s] keys of each sequence (0: an idle slot, a zero row); with k_new
    and v_new [n_seq, n_head_kv, D] the last of them is taken from there and
    appended."""
    torch = _torch()
    dev = q.device
    _operands(dev, (q, k_pool, v_pool, k_new, v_new, out, workspace),
              "q k_pool v_pool k_new v_new out workspace", (tables, n_kv, status), "tables n_kv status")
    n_seq, n_head, D = q.shape
    n_head_kv = k_pool.shape[-2]
    _need_pools(k_pool, v_pool, n_head_kv, D)
    bt = kv_batch(tables, block_tokens, k_pool, status)
    if bt.n_seq != n_seq or n_kv.numel() != n_seq:
        raise ValueError("tables and n_kv must hold an entry per row of q")
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new go together")
    if k_new is not None and (k_new.shape != (n_seq, n_head_kv, D) or v_new.shape != k_new.shape):
        raise ValueError("k_new and v_new must hold one token row per sequence")
    if out is not None and out.shape != q.shape:
        raise ValueError("out must be of q's shape")
    with _on(dev, stream):
        if out is None:
            out = torch.empty_like(q)
        if workspace is None:
            workspace = decode_batch_workspace(n_head, n_head_kv, D, device=dev)
        _check("ikv_attn_decode_batch_f32",
               load().ikv_attn_decode_batch_f32(
                   _ptr(q), _ptr(k_pool), _ptr(v_pool), ctypes.byref(bt), _ptr(n_kv), _ptr(k_new),
                   _ptr(v_new), _ptr(out), n_head, n_head_kv, D, scale, _ptr(workspace),
                   workspace.numel() * 4, _raw_stream(dev)))
    return out


def decode_shared_workspace(n_seq: int, n_groups: int, n_head: int, n_head_kv: int, head_dim: int,
                            device="cuda"):
    """Zero-filled workspace of attn_decode_shared for up to so many sequences and
    groups, of any lengths (reusable across ordered launches)."""
    torch = _torch()
    nbytes = int(load().ikv_attn_decode_shared_workspace_bytes(n_seq, n_groups, n_head, n_head_kv,
                                                               head_dim))
    return torch.zeros((nbytes + 3) // 4, dtype=torch.float32, device=device)


def attn_decode_shared(q, k_pool, v_pool, tables, block_tokens: int, group_start, shared_blocks, n_kv,
                       *, k_new=None, v_new=None, out=None, scale: float = 0.0, status=None,
                       workspace=None, stream=None):
    """attn_decode_batch where the sequences [group_start[g], group_start[g + 1]) of
    each group have the first shared_blocks[g] blocks of their tables in common:
    these are read once for all of them. The tables of idle slots are not read."""
    torch = _torch()
    dev = q.device
    _operands(dev, (q, k_pool, v_pool, k_new, v_new, out, workspace),
              "q k_pool v_pool k_new v_new out workspace",
              (tables, group_start, shared_blocks, n_kv, status),
              "tables group_start shared_blocks n_kv status")
    n_seq, n_head, D = q.shape
    n_head_kv = k_pool.shape[-2]
    _need_pools(k_pool, v_pool, n_head_kv, D)
    bt = kv_batch(tables, block_tokens, k_pool, status)
    if bt.n_seq != n_seq or n_kv.numel() != n_seq:
        raise ValueError("tables and n_kv must hold an entry per row of q")
    n_groups = shared_blocks.numel()
    if group_start.numel() != n_groups + 1:
        raise ValueError("group_start must hold n_groups + 1 sequences")
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new go together")
    if k_new is not None and (k_new.shape != (n_seq, n_head_kv, D) or v_new.shape != k_new.shape):
        raise ValueError("k_new and v_new must hold one token row per sequence")
    if out is not None and out.shape != q.shape:
        raise ValueError("out must be of q's shape")
    with _on(dev, stream):
        if out is None:
            out = torch.empty_like(q)
        if workspace is None:
            workspace = decode_shared_workspace(n_seq, n_groups, n_head, n_head_kv, D, device=dev)
        _check("ikv_attn_decode_shared_f32",
               load().ikv_attn_decode_shared_f32(
                   _ptr(q), _ptr(k_pool), _ptr(v_pool), ctypes.byref(bt), _ptr(group_start),
                   _ptr(shared_blocks), n_groups, _ptr(n_kv), _ptr(k_new), _ptr(v_new), _ptr(out),
                   n_head, n_head_kv, D, scale, _ptr(workspace), workspace.numel() * 4,
                   _raw_stream(dev)))
    return out


# ----------------------------------------------------------------------------
# a cache of 8 bits an element: (k_codes, k_scales, v_codes, v_scales), codes int8 or
# float8_e4m3fn [blocks, n_head_kv, block_tokens, D], scales float32 [blocks, n_head_kv,
# block_tokens]
# ----------------------------------------------------------------------------

def cache_q8(n_blocks: int, block_tokens: int, n_head_kv: int, head_dim: int, dtype=None,
             device="cuda"):
    """A paged cache of 8 bits an element, of int8 codes or of `dtype`
    torch.float8_e4m3fn."""
    torch = _torch()
    if dtype is None:
        dtype = torch.int8
    if dtype not in (torch.int8, torch.float8_e4m3fn):
        raise TypeError(f"dtype must be int8 or float8_e4m3fn, got {dtype}")
    shape = (n_blocks, n_head_kv, block_tokens, head_dim)
    codes = [torch.zeros(shape, dtype=torch.int8, device=device).view(dtype) for _ in range(2)]
    scales = [torch.zeros(shape[:-1], dtype=torch.float32, device=device) for _ in range(2)]
    return codes[0], scales[0], codes[1], scales[1]


def _cache_q8(cache, tables, status):
    """The descriptors of a cache and of block tables over it, and its shape."""
    torch = _torch()
    k, k_scales, v, v_scales = cache
    shape = k.shape
    if k.dtype is torch.int8:
        fmt = 0
    elif k.dtype is torch.float8_e4m3fn:
        fmt = 1
    else:
        raise TypeError(f"codes must be int8 or float8_e4m3fn, got {k.dtype}")
    if v.dtype is not k.dtype:
        raise TypeError(f"k and v codes must be of one type, got {k.dtype} and {v.dtype}")
    if k.device != v.device or not k.is_cuda:
        raise ValueError("codes must be on one GPU")
    if len(shape) != 4 or v.shape != shape or k_scales.shape != shape[:3] or v_scales.shape != shape[:3]:
        raise ValueError("codes must be [blocks, n_head_kv, block_tokens, head_dim], scales one less")
    if not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("codes must be contiguous")
    if tables.dim() != 2:
        raise ValueError("tables must be [n_seq, blocks]")
    n_seq, width = tables.shape
    return (KvQ8(k.data_ptr(), k_scales.data_ptr(), v.data_ptr(), v_scales.data_ptr(), shape[1], shape[3], fmt),
            KvBatch(tables.data_ptr(), width, shape[2], shape[0], n_seq, _ptr(status)), shape)


def append_packed_q8(cache, k_rows, v_rows, tables, row_start, first_token=None, *, status=None,
                     stream=None) -> None:
    """append_packed into a cache of 8 bits an element (cache_q8)."""
    dev = k_rows.device
    _operands(dev, (k_rows, v_rows, cache[1], cache[3]), "k_rows v_rows k_scales v_scales",
              (tables, row_start, first_token, status), "tables row_start first_token status")
    q8, bt, shape = _cache_q8(cache, tables, status)
    if cache[0].get_device() != dev.index:
        raise ValueError("codes must be on the device of the others")
    if k_rows.dim() != 3 or k_rows.shape != v_rows.shape or k_rows.shape[1:] != (shape[1], shape[3]):
        raise ValueError("k_rows and v_rows must be [rows, n_head_kv, head_dim] of the cache's heads")
    if row_start.numel() != bt.n_seq + 1:
        raise ValueError("row_start must hold n_seq + 1 rows")
    if first_token is not None and first_token.numel() != bt.n_seq:
        raise ValueError("first_token must hold a token per sequence")
    with _on(dev, stream):
        _check("ikv_append_packed_q8",
               load().ikv_append_packed_q8(ctypes.byref(q8), _ptr(k_rows), _ptr(v_rows),
                                           ctypes.byref(bt), _ptr(row_start), _ptr(first_token),
                                           k_rows.shape[0], _raw_stream(dev)))


def read_packed_q8(cache, tables, row_start, n_rows: int, first_token=None, n_kv=None, *, k_rows=None,
                   v_rows=None, status=None, stream=None):
    """Rows [row_start[s], row_start[s + 1]) of (k_rows, v_rows) [n_rows, n_head_kv, D]
    become the values of sequence s's tokens first_token[s].. (0.. without it), but
    for those from n_kv[s] on. Rows of no token are left as k_rows and v_rows have
    them (where they are allocated here: undefined)."""
    torch = _torch()
    dev = cache[1].device
    _operands(dev, (cache[1], cache[3], k_rows, v_rows), "k_scales v_scales k_rows v_rows",
              (tables, row_start, first_token, n_kv, status), "tables row_start first_token n_kv status")
    q8, bt, shape = _cache_q8(cache, tables, status)
    if cache[0].get_device() != dev.index:
        raise ValueError("codes must be on the device of the others")
    if row_start.numel() != bt.n_seq + 1:
        raise ValueError("row_start must hold n_seq + 1 rows")
    for t in (first_token, n_kv):
        if t is not None and t.numel() != bt.n_seq:
            raise ValueError("first_token and n_kv must hold a token per sequence")
    rows = (n_rows, shape[1], shape[3])
    for t in (k_rows, v_rows):
        if t is not None and t.shape != rows:
            raise ValueError("k_rows and v_rows must be [n_rows, n_head_kv, head_dim]")
    with _on(dev, stream):
        if k_rows is None:
            k_rows = torch.empty(rows, dtype=torch.float32, device=dev)
        if v_rows is None:
            v_rows = torch.empty(rows, dtype=torch.float32, device=dev)
        _check("ikv_read_packed_q8",
               load().ikv_read_packed_q8(ctypes.byref(q8), _ptr(k_rows), _ptr(v_rows),
                                         ctypes.byref(bt), _ptr(row_start), _ptr(first_token),
                                         _ptr(n_kv), n_rows, _raw_stream(dev)))
    return k_rows, v_rows


def decode_batch_q8_workspace(n_head: int, n_head_kv: int, head_dim: int, device="cuda"):
    """decode_batch_workspace of attn_decode_batch_q8."""
    torch = _torch()
    nbytes = int(load().ikv_attn_decode_batch_q8_workspace_bytes(n_head, n_head_kv, head_dim))
    return torch.zeros((nbytes + 3) // 4, dtype=torch.float32, device=device)


def attn_decode_batch_q8(q, cache, tables, n_kv, *, k_new=None, v_new=None, out=None,
                         scale: float = 0.0, status=None, workspace=None, stream=None):
    """attn_decode_batch over a cache of 8 bits an element (cache_q8): the new rows
    are quantised, appended and attended to as they are held."""
    torch = _torch()
    dev = q.device
    _operands(dev, (q, cache[1], cache[3], k_new, v_new, out, workspace),
              "q k_scales v_scales k_new v_new out workspace", (tables, n_kv, status),
              "tables n_kv status")
    q8, bt, shape = _cache_q8(cache, tables, status)
    n_seq, n_head, D = q.shape
    if cache[0].get_device() != dev.index:
        raise ValueError("codes must be on the device of the others")
    if shape[3] != D:
        raise ValueError("the cache's heads differ from q's")
    if bt.n_seq != n_seq or n_kv.numel() != n_seq:
        raise ValueError("tables and n_kv must hold an entry per row of q")
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new go together")
    if k_new is not None and (k_new.shape != (n_seq, shape[1], D) or v_new.shape != k_new.shape):
        raise ValueError("k_new and v_new must hold one token row per sequence")
    if out is not None and out.shape != q.shape:
        raise ValueError("out must be of q's shape")
    with _on(dev, stream):
        if out is None:
            out = torch.empty_like(q)
        if workspace is None:
            workspace = decode_batch_q8_workspace(n_head, shape[1], D, device=dev)
        _check("ikv_attn_decode_batch_q8",
               load().ikv_attn_decode_batch_q8(
                   _ptr(q), ctypes.byref(q8), ctypes.byref(bt), _ptr(n_kv), _ptr(k_new), _ptr(v_new),
                   _ptr(out), n_head, scale, _ptr(workspace), workspace.numel() * 4,
                   _raw_stream(dev)))
    return out


def rms_norm(x, w, eps: float, out=None, stream=None):
    torch = _torch()
    _need_f32_dev("x", x)
    _need_f32_dev("w", w)
    dim = x.shape[-1]
    if w.numel() != dim:
        raise ValueError("weight length must equal the last dim")
    if out is None:
        out = torch.empty_like(x)
    rows = x.numel() // dim
    _check("ikv_rms_norm_f32",
           load().ikv_rms_norm_f32(_ptr(x), _ptr(w), _ptr(out), rows, dim, eps, _stream(stream)))
    return out


def rope_theta_table(theta_base: float, head_dim: int, n_ctx: int):
    """Host RoPE angle table [n_ctx][head_dim/2] (numpy float32), the
    engine's own (GraphContext::get_rope_theta_table)."""
    import numpy as np
    out = np.empty((n_ctx, head_dim // 2), dtype=np.float32)
    _check("ikv_rope_theta_table_f32",
           load().ikv_rope_theta_table_f32(theta_base, head_dim, n_ctx, out.ctypes.data))
    return out


def rope_sincos_table(theta):
    """Host sin/cos tables (numpy float32) from a host angle table."""
    import numpy as np
    theta = np.ascontiguousarray(theta, dtype=np.float32)
    s = np.empty_like(theta)
    c = np.empty_like(theta)
    _check("ikv_rope_sincos_table_f32",
           load().ikv_rope_sincos_table_f32(theta.ctypes.data, theta.size, s.ctypes.data,
                                            c.ctypes.data))
    return s, c


def rope_neox(x, pos, sin_tab, cos_tab, out=None, status=None, stream=None):
    """x: [n_tokens, n_heads, D]; pos: int32 [n_tokens]; tables [n_ctx, D/2]."""
    torch = _torch()
    _need_f32_dev("x", x)
    n_tokens, n_heads, D = x.shape
    if out is None:
        out = torch.empty_like(x)
    rc = load().ikv_rope_neox_f32(_ptr(x), _ptr(out), _ptr(pos), n_tokens, n_heads, D,
                                  _ptr(sin_tab), _ptr(cos_tab), sin_tab.shape[0], _ptr(status),
                                  _stream(stream))
    _check("ikv_rope_neox_f32", rc)
    return out


def qk_norm_rope(x, w, pos, eps: float, sin_tab, cos_tab, out=None, status=None, stream=None):
    torch = _torch()
    _need_f32_dev("x", x)
    n_tokens, n_heads, D = x.shape
    if out is None:
        out = torch.empty_like(x)
    rc = load().ikv_qk_norm_rope_f32(_ptr(x), _ptr(w), _ptr(out), _ptr(pos), n_tokens, n_heads, D,
                                     eps, _ptr(sin_tab), _ptr(cos_tab), sin_tab.shape[0],
                                     _ptr(status), _stream(stream))
    _check("ikv_qk_norm_rope_f32", rc)
    return out


# ----------------------------------------------------------------------------
# ops around the path (include/ikv_model.h)
# ----------------------------------------------------------------------------

def mul_mat(w, x, out=None, residual=None, stream=None):
    """out[m, n] = x[m, :] . w[n, :] (+ residual); w [n_out, k], x [m, k] or [k]."""
    torch = _torch()
    _need_f32_dev("w", w)
    _need_f32_dev("x", x)
    n_out, k = w.shape
    m = x.numel() // k
    if x.numel() != m * k:
        raise ValueError("x length must be a multiple of k")
    if out is None:
        out = torch.empty((m, n_out) if x.dim() > 1 else (n_out,), device=x.device)
    _check("ikv_mul_mat_f32", load().ikv_mul_mat_f32(_ptr(w), _ptr(x), _ptr(out), n_out, k, m,
                                                      _ptr(residual), _stream(stream)))
    return out


def gemm_nt(w, x, out=None, residual=None, stream=None):
    """The MFMA GEMM of mul_mat for any number of tokens: out[m, n] =
    x[m, :] . w[n, :] (+ residual); n_out % 64 == 0 and k % 64 == 0."""
    torch = _torch()
    _need_f32_dev("w", w)
    _need_f32_dev("x", x)
    n_out, k = w.shape
    m = x.numel() // k
    if x.numel() != m * k:
        raise ValueError("x length must be a multiple of k")
    if out is None:
        out = torch.empty((m, n_out), device=x.device)
    _check("ikv_gemm_nt_f32", load().ikv_gemm_nt_f32(_ptr(w), _ptr(x), _ptr(out), n_out, k, m,
                                                      _ptr(residual), _stream(stream)))
    return out


def gemv3(w0, w1, w2, x, norm_w=None, eps: float = 1e-6, stream=None):
    """[w_i . x'] for i = 0, 1, 2; x' = rms_norm(x, norm_w, eps) when norm_w is given."""
    torch = _torch()
    k = x.numel()
    outs = [torch.empty(w.shape[0], device=x.device) for w in (w0, w1, w2)]
    _check("ikv_gemv3_f32", load().ikv_gemv3_f32(
        _ptr(w0), _ptr(w1), _ptr(w2), _ptr(x), _ptr(outs[0]), _ptr(outs[1]), _ptr(outs[2]),
        w0.shape[0], w1.shape[0], w2.shape[0], k, _ptr(norm_w), eps, _stream(stream)))
    return outs


def gemv_swiglu(w_gate, w_up, x, out=None, norm_w=None, eps: float = 1e-6, stream=None):
    torch = _torch()
    n_out, k = w_gate.shape
    if out is None:
        out = torch.empty(n_out, device=x.device)
    _check("ikv_gemv_swiglu_f32", load().ikv_gemv_swiglu_f32(
        _ptr(w_gate), _ptr(w_up), _ptr(x), _ptr(out), n_out, k, _ptr(norm_w), eps,
        _stream(stream)))
    return out


def get_rows(table, ids, out=None, status=None, stream=None):
    torch = _torch()
    n_rows, row_len = table.shape
    if out is None:
        out = torch.empty((ids.numel(), row_len), device=table.device)
    _check("ikv_get_rows_f32", load().ikv_get_rows_f32(
        _ptr(table), _ptr(ids), _ptr(out), ids.numel(), row_len, n_rows, _ptr(status),
        _stream(stream)))
    return out


def elementwise(op: str, a, b=None, out=None, stream=None):
    torch = _torch()
    if out is None:
        out = torch.empty_like(a)
    lib = load()
    if op == "silu":
        rc = lib.ikv_silu_f32(_ptr(a), _ptr(out), a.numel(), _stream(stream))
    else:
        rc = getattr(lib, f"ikv_{op}_f32")(_ptr(a), _ptr(b), _ptr(out), a.numel(), _stream(stream))
    _check(f"ikv_{op}_f32", rc)
    return out


def argmax(logits, token=None, mirror=None, workspace=None, stream=None):
    """Device int32 [1]: greedy token of logits (ties -> lowest id; -1 on NaN/+inf);
    `mirror` (e.g. a pinned host tensor) receives a copy. With `workspace`
    (argmax_workspace()), the multi-workgroup form runs."""
    torch = _torch()
    if token is None:
        token = torch.empty(1, dtype=torch.int32, device=logits.device)
    if workspace is None:
        _check("ikv_argmax_f32", load().ikv_argmax_f32(_ptr(logits), logits.numel(), _ptr(token),
                                                        _ptr(mirror), _stream(stream)))
    else:
        _check("ikv_argmax_ws_f32",
               load().ikv_argmax_ws_f32(_ptr(logits), logits.numel(), _ptr(token), _ptr(mirror),
                                        _ptr(workspace), workspace.numel() * workspace.element_size(),
                                        _stream(stream)))
    return token


def argmax_workspace(device=None):
    """Zeroed device workspace of the multi-workgroup greedy sampler."""
    torch = _torch()
    n = int(load().ikv_argmax_workspace_bytes())
    return torch.zeros(n, dtype=torch.uint8, device=device or "cuda")


def adjust_logits(logits, *, history=None, n_history=None, n_prompt=None, repetition=None,
                  presence=None, frequency=None, bias_tokens=None, bias_values=None, n_bias=None,
                  masks=None, mask_of=None, out=None, status=None, stream=None):
    """The rows of logits [n_rows, n_vocab] with penalties for the first n_history[r]
    tokens of history [n_rows, .] (repetition for all, presence and frequency for those
    behind the first n_prompt[r]), with the first n_bias[r] of bias_values added at
    bias_tokens [n_rows, .], and -inf where the bits of masks [n_masks, words] (int32
    words of 32 tokens; row mask_of[r], none where that is negative) are 0. `out` may
    be logits."""
    torch = _torch()
    dev = logits.device
    _operands(dev, (logits, out, repetition, presence, frequency, bias_values),
              "logits out repetition presence frequency bias_values",
              (history, n_history, n_prompt, bias_tokens, n_bias, masks, mask_of, status),
              "history n_history n_prompt bias_tokens n_bias masks mask_of status")
    if logits.dim() != 2:
        raise ValueError("logits must be [n_rows, n_vocab]")
    n_rows, n_vocab = logits.shape
    for t in (n_history, n_prompt, repetition, presence, frequency, n_bias, mask_of):
        if t is not None and t.numel() != n_rows:
            raise ValueError("lengths, penalties and mask_of must hold a value per row")
    for t in (history, bias_tokens):
        if t is not None and (t.dim() != 2 or t.shape[0] != n_rows):
            raise ValueError("history and bias_tokens must be [n_rows, tokens]")
    if (bias_tokens is None) != (bias_values is None):
        raise ValueError("bias_tokens and bias_values go together")
    if bias_tokens is not None and bias_tokens.shape != bias_values.shape:
        raise ValueError("bias_tokens and bias_values must be of one shape")
    if masks is None:
        if mask_of is not None:
            raise ValueError("mask_of goes with masks")
    elif masks.dim() != 2 or masks.shape[0] == 0 or masks.shape[1] != (n_vocab + 31) // 32:
        raise ValueError("masks must be [n_masks, (n_vocab + 31) // 32], one at least")
    if out is not None and out.shape != logits.shape:
        raise ValueError("out must be of logits' shape")
    with _on(dev, stream):
        if out is None:
            out = torch.empty_like(logits)
        # (an empty list has no address, but its lengths are looked at)
        at = [None if t is None else t.data_ptr() or logits.data_ptr()
              for t in (history, bias_tokens, bias_values)]
        rules = LogitRules(at[0], 0 if history is None else history.shape[1], _ptr(n_history),
                           _ptr(n_prompt), _ptr(repetition), _ptr(presence), _ptr(frequency),
                           at[1], at[2],
                           0 if bias_tokens is None else bias_tokens.shape[1], _ptr(n_bias),
                           _ptr(masks), 0 if masks is None else masks.shape[0], _ptr(mask_of))
        _check("ikv_adjust_logits_f32",
               load().ikv_adjust_logits_f32(_ptr(logits), _ptr(out), ctypes.byref(rules), n_rows, n_vocab,
                                            _ptr(status), _raw_stream(dev)))
    return out


def sample_workspace(n_rows: int, n_vocab: int, device="cuda"):
    """Workspace of sample() for up to n_rows rows (reusable across ordered launches)."""
    torch = _torch()
    nbytes = int(load().ikv_sample_workspace_bytes(n_rows, n_vocab))
    return torch.empty((nbytes + 3) // 4, dtype=torch.float32, device=device)


def sample(logits, u, *, temperature=None, top_k=None, top_p=None, min_p=None, token=None,
           logprob=None, workspace=None, stream=None):
    """The next token of each row of logits [n_rows, n_vocab] from uniform numbers
    u [n_rows], with each row's temperature (<= 0: greedy), top_k (<= 0: all),
    top_p and min_p (device tensors [n_rows], or None). Returns (token, logprob),
    int32 and float32 [n_rows]."""
    torch = _torch()
    dev = logits.device
    _operands(dev, (logits, u, temperature, top_p, min_p, logprob, workspace),
              "logits u temperature top_p min_p logprob workspace", (top_k, token), "top_k token")
    if logits.dim() != 2:
        raise ValueError("logits must be [n_rows, n_vocab]")
    n_rows, n_vocab = logits.shape
    for t in (u, temperature, top_k, top_p, min_p, token, logprob):
        if t is not None and t.numel() != n_rows:
            raise ValueError("u, the parameters and the results must hold a value per row")
    with _on(dev, stream):
        if token is None:
            token = torch.empty(n_rows, dtype=torch.int32, device=dev)
        if logprob is None:
            logprob = torch.empty(n_rows, dtype=torch.float32, device=dev)
        if workspace is None:
            workspace = sample_workspace(n_rows, n_vocab, device=dev)
        _check("ikv_sample_f32",
               load().ikv_sample_f32(_ptr(logits), _ptr(u), _ptr(temperature), _ptr(top_k), _ptr(top_p),
                                     _ptr(min_p), n_rows, n_vocab, _ptr(token), _ptr(logprob),
                                     _ptr(workspace), workspace.numel() * 4, _raw_stream(dev)))
    return token, logprob


def synth_normal(seed: int, shape, std: float = 1.0, offset: int = 0, threads: int = 8):
    """Host float32 N(0, std^2) array from the product's synthetic initialiser."""
    import numpy as np
    out = np.empty(shape, dtype=np.float32)
    _check("ikv_synth_normal_f32", load().ikv_synth_normal_f32(
        seed & 0xFFFFFFFFFFFFFFFF, offset, out.size, std, out.ctypes.data, threads))
    return out
