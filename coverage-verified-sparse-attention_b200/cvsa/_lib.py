"""ctypes binding of libcvsa_b200.so (include/cvsa_b200.h).

The library is the product: every CVSA op in this package is a call into it on
the current CUDA stream. There is no CPU or Triton fallback -- if the library
cannot be loaded, or a tensor is not on a CUDA device, the call raises.

Status codes map to the exception types the reference raises for the same
conditions: CVSA_ERR_INVALID -> ValueError (cvsa/backend.py:150-178),
CVSA_ERR_POOL -> AssertionError (cvsa/runtime/kv_cache.py:55-56), the rest
-> RuntimeError.
"""

from __future__ import annotations

import ctypes
import os
import struct
import threading
from typing import Optional

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libcvsa_b200.so")

DTYPE_F32, DTYPE_F16, DTYPE_BF16, DTYPE_E4M3 = 0, 1, 2, 3
OK, ERR_INVALID, ERR_UNSUPPORTED, ERR_WORKSPACE, ERR_CUDA, ERR_POOL = 0, -1, -2, -3, -4, -5
MODE_SCORE, MODE_LAZY, MODE_REUSE, MODE_DENSE = 0, 1, 2, 3
RECOVERY_EXACT, RECOVERY_NONE, RECOVERY_APPROX = 0, 1, 2
(CTR_PAGES_ATTENDED, CTR_PAGES_MAX, CTR_HEAD_ACCEPT, CTR_HEAD_TOTAL, CTR_ACCEPT_STEPS,
 CTR_REJECT_STEPS, CTR_SCORING_STEPS, CTR_COVERAGE_CHECKS) = range(8)
NUM_COUNTERS = 8
EV_SCORE_BEGIN, EV_SCORE_END, EV_SELECT_BEGIN, EV_SELECT_END, EV_ATTEND_BEGIN, EV_ATTEND_END = (
    range(6))
NUM_EVENTS = 6
(DEV_ERR_BLOCK_RANGE, DEV_ERR_PAGE_RANGE, DEV_ERR_POOL, DEV_ERR_TABLE_FULL, DEV_ERR_TIMEOUT,
 DEV_ERR_RAGGED) = (1, 2, 4, 8, 16, 32)

_TORCH_TO_DT = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}


class KvDesc(ctypes.Structure):
    _fields_ = [
        ("k_cache", ctypes.c_void_p), ("v_cache", ctypes.c_void_p),
        ("dtype", ctypes.c_int32), ("num_blocks", ctypes.c_int32),
        ("block_size", ctypes.c_int32), ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32), ("reserved0", ctypes.c_int32),
        ("stride_block", ctypes.c_int64), ("stride_token", ctypes.c_int64),
        ("stride_head", ctypes.c_int64),
    ]


class QueryDesc(ctypes.Structure):
    _fields_ = [
        ("q", ctypes.c_void_p), ("dtype", ctypes.c_int32), ("batch", ctypes.c_int32),
        ("num_q_heads", ctypes.c_int32), ("max_pages", ctypes.c_int32),
        ("block_tables", ctypes.c_void_p), ("context_lens", ctypes.c_void_p),
    ]


class StepConfig(ctypes.Structure):
    _fields_ = [
        ("mode", ctypes.c_int32), ("budget", ctypes.c_int32),
        ("sink_pages", ctypes.c_int32), ("local_pages", ctypes.c_int32),
        ("tau", ctypes.c_float), ("recovery", ctypes.c_int32),
        ("has_cache", ctypes.c_int32), ("lazy_stats", ctypes.c_int32),
        ("approx_budget", ctypes.c_int32),
    ]


class StepIO(ctypes.Structure):
    _fields_ = [
        ("cached_indices", ctypes.c_void_p), ("cached_n", ctypes.c_void_p),
        ("max_sel", ctypes.c_int32), ("phase", ctypes.c_int32),
        ("out", ctypes.c_void_p), ("page_scores", ctypes.c_void_p),
        ("accept", ctypes.c_void_p), ("coverage", ctypes.c_void_p),
        ("counters", ctypes.c_void_p), ("step_flags", ctypes.c_void_p),
        ("dev_error", ctypes.c_void_p), ("timing_events", ctypes.c_void_p),
    ]


class SplitDesc(ctypes.Structure):
    _fields_ = [
        ("world", ctypes.c_int32), ("rank", ctypes.c_int32), ("batch", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32), ("max_pages", ctypes.c_int32),
        ("block_size", ctypes.c_int32), ("budget", ctypes.c_int32), ("max_sel", ctypes.c_int32),
        ("sink_pages", ctypes.c_int32), ("local_pages", ctypes.c_int32), ("tau", ctypes.c_float),
    ]


class PeerDesc(ctypes.Structure):
    _fields_ = [
        ("bases", ctypes.c_void_p), ("world", ctypes.c_int32), ("rank", ctypes.c_int32),
        ("row_cap", ctypes.c_int64), ("dev_error", ctypes.c_void_p),
    ]


class RaggedDesc(ctypes.Structure):
    _fields_ = [
        ("cu_tokens", ctypes.c_void_p), ("seq_ids", ctypes.c_void_p),
        ("start_positions", ctypes.c_void_p), ("block_tables", ctypes.c_void_p),
        ("context_lens", ctypes.c_void_p), ("batch", ctypes.c_int32),
        ("num_tokens", ctypes.c_int32), ("num_seqs", ctypes.c_int32),
        ("max_pages", ctypes.c_int32),
    ]


class RopeAppend(ctypes.Structure):
    _fields_ = [
        ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
        ("q_out", ctypes.c_void_p), ("dtype", ctypes.c_int32), ("num_q_heads", ctypes.c_int32),
        ("q_stride_token", ctypes.c_int64), ("q_stride_head", ctypes.c_int64),
        ("k_stride_token", ctypes.c_int64), ("k_stride_head", ctypes.c_int64),
        ("v_stride_token", ctypes.c_int64), ("v_stride_head", ctypes.c_int64),
        ("q_out_stride_token", ctypes.c_int64), ("q_out_stride_head", ctypes.c_int64),
        ("cos_sin", ctypes.c_void_p), ("max_positions", ctypes.c_int32),
        ("rot_dim", ctypes.c_int32), ("interleaved", ctypes.c_int32),
        ("norm_dtype", ctypes.c_int32), ("q_norm", ctypes.c_void_p),
        ("k_norm", ctypes.c_void_p), ("eps", ctypes.c_float),
    ]


class ChunkAttend(ctypes.Structure):
    _fields_ = [
        ("q", ctypes.c_void_p), ("out", ctypes.c_void_p), ("lse", ctypes.c_void_p),
        ("dtype", ctypes.c_int32), ("num_q_heads", ctypes.c_int32),
        ("q_stride_token", ctypes.c_int64), ("q_stride_head", ctypes.c_int64),
        ("out_stride_token", ctypes.c_int64), ("out_stride_head", ctypes.c_int64),
        ("scale", ctypes.c_float), ("causal", ctypes.c_int32), ("window", ctypes.c_int32),
    ]


class KeyWeights(ctypes.Structure):
    _fields_ = [
        ("q", ctypes.c_void_p), ("lse", ctypes.c_void_p), ("dtype", ctypes.c_int32),
        ("num_q_heads", ctypes.c_int32), ("q_stride_token", ctypes.c_int64),
        ("q_stride_head", ctypes.c_int64), ("scale", ctypes.c_float), ("decay", ctypes.c_float),
        ("causal", ctypes.c_int32), ("window", ctypes.c_int32), ("prior", ctypes.c_void_p),
        ("out", ctypes.c_void_p), ("weights_stride", ctypes.c_int64),
    ]


class Evict(ctypes.Structure):
    _fields_ = [
        ("weights", ctypes.c_void_p), ("weights_stride", ctypes.c_int64),
        ("out_weights", ctypes.c_void_p), ("out_stride", ctypes.c_int64),
        ("new_tables", ctypes.c_void_p), ("new_pages", ctypes.c_int32),
        ("kept", ctypes.c_void_p), ("keep", ctypes.c_int32), ("sink", ctypes.c_int32),
        ("recent", ctypes.c_int32),
    ]


class EvictPages(ctypes.Structure):
    _fields_ = [
        ("block_tables", ctypes.c_void_p), ("context_lens", ctypes.c_void_p),
        ("pages_allocated", ctypes.c_void_p), ("evicted", ctypes.c_void_p),
        ("free_list", ctypes.c_void_p), ("free_head", ctypes.c_void_p),
        ("new_tables", ctypes.c_void_p), ("plan_lens", ctypes.c_void_p),
        ("num_seqs", ctypes.c_int32), ("max_pages", ctypes.c_int32),
        ("block_size", ctypes.c_int32), ("keep", ctypes.c_int32),
        ("free_list_len", ctypes.c_int32),
    ]


_P = ctypes.c_void_p
_I = ctypes.c_int32
_SIGS = {
    "cvsa_abi_version": ([], ctypes.c_int),
    "cvsa_status_string": ([ctypes.c_int], ctypes.c_char_p),
    "cvsa_last_error": ([], ctypes.c_char_p),
    "cvsa_score_pages": ([ctypes.POINTER(QueryDesc), ctypes.POINTER(KvDesc), _P, _P], ctypes.c_int),
    "cvsa_quest_scores": ([ctypes.POINTER(QueryDesc), ctypes.POINTER(KvDesc), _P, _P, _P],
                          ctypes.c_int),
    "cvsa_select_pages": ([_P, _I, _I, _I, _P, _I, _I, _I, _I, _P, _I, _P, _P], ctypes.c_int),
    "cvsa_check_coverage": ([_P, _I, _I, _I, _P, _I, _P, ctypes.c_float, _P, _P, _P], ctypes.c_int),
    "cvsa_compute_complement": ([_P, _I, _P, _P, _I, _I, _I, _P, _P, _I, _P, _P], ctypes.c_int),
    "cvsa_decode_workspace_size": ([ctypes.POINTER(QueryDesc), ctypes.POINTER(KvDesc), _I],
                                   ctypes.c_size_t),
    "cvsa_sparse_decode": ([ctypes.POINTER(QueryDesc), ctypes.POINTER(KvDesc), _P, _I, _P, _P, _P,
                            _P, _P, _I, _P, ctypes.c_size_t, _P], ctypes.c_int),
    "cvsa_lse_merge": ([_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P, _I, _P], ctypes.c_int),
    "cvsa_page_lse": ([_P, _I, _I, _P, _I, _P, _P, _P, _P], ctypes.c_int),
    "cvsa_rank_accept": ([_P, _I, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, _I,
                          ctypes.c_float, _P, _P], ctypes.c_int),
    "cvsa_split_row_floats": ([ctypes.POINTER(SplitDesc)], ctypes.c_int64),
    "cvsa_split_propose": ([ctypes.POINTER(SplitDesc), _P, _P, _P, _P, _P, _P, _P], ctypes.c_int),
    "cvsa_split_gate": ([ctypes.POINTER(SplitDesc), _P, ctypes.c_int64, _P, _P, _I, _I, _P, _P,
                         _P, _P, _P, _P, _P, _P], ctypes.c_int),
    "cvsa_split_attend": ([ctypes.POINTER(QueryDesc), ctypes.POINTER(KvDesc), _P, _P, _P, _P, _I,
                           _P, _P, _P, _P, _P, _P, _P, _P, ctypes.c_size_t, _P], ctypes.c_int),
    "cvsa_peer_buffer_bytes": ([_I, ctypes.c_int64], ctypes.c_size_t),
    "cvsa_peer_alloc": ([ctypes.c_size_t, ctypes.POINTER(ctypes.c_void_p), _P], ctypes.c_int),
    "cvsa_peer_open": ([_P, ctypes.POINTER(ctypes.c_void_p)], ctypes.c_int),
    "cvsa_peer_close": ([_P], ctypes.c_int),
    "cvsa_peer_free": ([_P], ctypes.c_int),
    "cvsa_peer_allgather": ([ctypes.POINTER(PeerDesc), _P, ctypes.c_int64, _P, _P], ctypes.c_int),
    "cvsa_peer_min_i32": ([ctypes.POINTER(PeerDesc), _P, ctypes.c_int64, _P, _P], ctypes.c_int),
    "cvsa_peer_merge": ([ctypes.POINTER(PeerDesc), _P, _I, _I, _I, _I, _P, _P, _I, _P],
                        ctypes.c_int),
    "cvsa_rank_merge": ([_P, _I, ctypes.c_int64, _I, _I, _I, _I, _P, _P, _I, _P], ctypes.c_int),
    "cvsa_recover_merge": ([ctypes.POINTER(QueryDesc), ctypes.POINTER(KvDesc), _P, _I, _P, _P, _P,
                            _P, _P, _P, _I, _P, ctypes.c_size_t, _P], ctypes.c_int),
    "cvsa_step_workspace_size": ([ctypes.POINTER(QueryDesc), ctypes.POINTER(KvDesc),
                                  ctypes.POINTER(StepConfig), _I], ctypes.c_size_t),
    "cvsa_decode_step": ([ctypes.POINTER(QueryDesc), ctypes.POINTER(KvDesc),
                          ctypes.POINTER(StepConfig), ctypes.POINTER(StepIO), _P, ctypes.c_size_t,
                          _P], ctypes.c_int),
    "cvsa_set_wait_limit": ([ctypes.c_uint32], ctypes.c_int),
    "cvsa_workspace_reset": ([_P, ctypes.c_size_t, _P], ctypes.c_int),
    "cvsa_step_decision_word": ([_P, ctypes.POINTER(ctypes.c_void_p)], ctypes.c_int),
    "cvsa_paged_append": ([ctypes.POINTER(KvDesc), _P, _P, _I, _P, _P, _I, _P, _P, _P, _I, _P, _P,
                           _P], ctypes.c_int),
    "cvsa_paged_gather": ([ctypes.POINTER(KvDesc), _P, _I, _P, _P, _P, _P], ctypes.c_int),
    "cvsa_paged_reserve": ([_I, _P, _P, _I, _I, _P, _I, _P, _P, _P, _I, _P, _P, _P, _P],
                           ctypes.c_int),
    "cvsa_rope_append": ([ctypes.POINTER(KvDesc), ctypes.POINTER(RaggedDesc),
                          ctypes.POINTER(RopeAppend), _P, _P], ctypes.c_int),
    "cvsa_rope_append_check": ([ctypes.POINTER(KvDesc), ctypes.POINTER(RaggedDesc),
                                ctypes.POINTER(RopeAppend)], ctypes.c_int),
    "cvsa_chunk_attend_check": ([ctypes.POINTER(KvDesc), ctypes.POINTER(RaggedDesc),
                                 ctypes.POINTER(ChunkAttend)], ctypes.c_int),
    "cvsa_chunk_attend_workspace_size": ([ctypes.POINTER(KvDesc), ctypes.POINTER(RaggedDesc),
                                          ctypes.POINTER(ChunkAttend)], ctypes.c_size_t),
    "cvsa_chunk_attend": ([ctypes.POINTER(KvDesc), ctypes.POINTER(RaggedDesc),
                           ctypes.POINTER(ChunkAttend), _P, _P, ctypes.c_size_t, _P],
                          ctypes.c_int),
    "cvsa_rope_append_to": ([ctypes.POINTER(KvDesc), _P, _P, ctypes.POINTER(RaggedDesc),
                             ctypes.POINTER(RopeAppend), _P, _P, _P], ctypes.c_int),
    "cvsa_rope_append_to_check": ([ctypes.POINTER(KvDesc), _P, _P, ctypes.POINTER(RaggedDesc),
                                   ctypes.POINTER(RopeAppend), _P], ctypes.c_int),
    "cvsa_chunk_attend_q8_check": ([ctypes.POINTER(KvDesc), _P, _P, ctypes.POINTER(RaggedDesc),
                                    ctypes.POINTER(ChunkAttend)], ctypes.c_int),
    "cvsa_chunk_attend_q8_workspace_size": (
        [ctypes.POINTER(KvDesc), _P, _P, ctypes.POINTER(RaggedDesc),
         ctypes.POINTER(ChunkAttend)], ctypes.c_size_t),
    "cvsa_chunk_attend_q8": ([ctypes.POINTER(KvDesc), _P, _P, ctypes.POINTER(RaggedDesc),
                              ctypes.POINTER(ChunkAttend), _P, _P, ctypes.c_size_t, _P],
                             ctypes.c_int),
    "cvsa_key_weights": ([ctypes.POINTER(KvDesc), _P, ctypes.POINTER(RaggedDesc),
                          ctypes.POINTER(KeyWeights), _P, _P], ctypes.c_int),
    "cvsa_key_weights_check": ([ctypes.POINTER(KvDesc), _P, ctypes.POINTER(RaggedDesc),
                                ctypes.POINTER(KeyWeights)], ctypes.c_int),
    "cvsa_evict": ([ctypes.POINTER(KvDesc), _P, _P, _P, _P, _I, _I, ctypes.POINTER(Evict), _P,
                    _P], ctypes.c_int),
    "cvsa_evict_reserve": ([ctypes.POINTER(EvictPages), _P, _P], ctypes.c_int),
    "cvsa_evict_commit": ([ctypes.POINTER(EvictPages), _P, _P], ctypes.c_int),
    "cvsa_sparse_decode_noalloc": ([ctypes.POINTER(QueryDesc), ctypes.POINTER(KvDesc), _P, _I, _P,
                                    _P, _P, _P, _P, _I, _P], ctypes.c_int),
}
NOALLOC_SCRATCH_BYTES = 8 << 20
ABI_VERSION = 2
# cvsa_decode_step phases (include/cvsa_b200.h CVSA_PHASE_*)
PHASE_ALL, PHASE_SELECT, PHASE_ATTEND = 0, 1, 2

_lib = None
_lock = threading.Lock()


def exported_symbols():
    """Names of every entry point this binding expects the library to export."""
    return sorted(_SIGS)


def load(path: Optional[str] = None) -> ctypes.CDLL:
    """Load libcvsa_b200.so once (raises if it is missing: no fallback)."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    with _lock:
        if _lib is not None and path is None:
            return _lib
        p = path or LIB_PATH
        if not os.path.exists(p):
            raise RuntimeError(
                f"libcvsa_b200.so not found at {p}; build it with "
                "`python coverage-verified-sparse-attention_b200/build_lib.py` "
                "(the CVSA ops have no CPU fallback)")
        lib = ctypes.CDLL(p)
        for name, (args, res) in _SIGS.items():
            fn = getattr(lib, name)
            fn.argtypes = args
            fn.restype = res
        if lib.cvsa_abi_version() != ABI_VERSION:
            raise RuntimeError("libcvsa_b200.so ABI version mismatch")
        if path is None:
            _lib = lib
        return lib


def check(status: int, what: str = "") -> None:
    if status == OK:
        return
    msg = (load().cvsa_last_error() or b"").decode()
    text = f"{what}: {msg}" if what else msg
    if status == ERR_INVALID:
        raise ValueError(text)
    if status == ERR_POOL:
        raise AssertionError(text)
    raise RuntimeError(f"{text} (status {status})")


def dtype_code(dt: torch.dtype) -> int:
    try:
        return _TORCH_TO_DT[dt]
    except KeyError:
        raise ValueError(f"unsupported dtype {dt}")


def ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def require_cuda(*tensors: Optional[torch.Tensor]) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("CVSA ops run on CUDA tensors only (no CPU fallback); "
                               f"got a tensor on {t.device}")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} and {t.device}")
    return dev


def stream_ptr(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def raw_stream(index: int) -> int:
    """The current stream's handle by device index (no stream object is built)."""
    return torch._C._cuda_getCurrentRawStream(index)


def same_device(first: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """Device index shared by all tensors; the errors are require_cuda's."""
    dev = first.get_device()
    ok = dev >= 0
    for t in others:
        if t is not None and t.get_device() != dev:
            ok = False
    if not ok:
        require_cuda(first, *others)
    return dev


def kv_desc(k_cache: torch.Tensor, v_cache: torch.Tensor) -> KvDesc:
    """[num_blocks, block_size, num_kv_heads, head_dim] pools (kv_cache.py:38-43)."""
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError("k_cache/v_cache must both be [num_blocks, block_size, H_kv, D]")
    if k_cache.dtype != v_cache.dtype:
        raise ValueError("k_cache and v_cache dtypes differ")
    if k_cache.stride() != v_cache.stride() or k_cache.stride(3) != 1:
        raise ValueError("k_cache/v_cache must share strides with a contiguous head_dim")
    nb, bs, h, d = k_cache.shape
    return KvDesc(k_cache.data_ptr(), v_cache.data_ptr(), dtype_code(k_cache.dtype), nb, bs, h, d,
                  0, k_cache.stride(0), k_cache.stride(1), k_cache.stride(2))


def query_desc(q: Optional[torch.Tensor], block_tables: torch.Tensor,
               context_lens: torch.Tensor, num_q_heads: Optional[int] = None) -> QueryDesc:
    if block_tables.dtype != torch.int32 or context_lens.dtype != torch.int32:
        raise ValueError("block_tables and context_lens must be int32")
    if not block_tables.is_contiguous() or not context_lens.is_contiguous():
        raise ValueError("block_tables/context_lens must be contiguous")
    B, W = block_tables.shape
    if q is not None:
        if q.dim() != 3 or not q.is_contiguous():
            raise ValueError("q must be a contiguous [B, H_q, D] tensor")
        return QueryDesc(q.data_ptr(), dtype_code(q.dtype), B, q.shape[1], W,
                         block_tables.data_ptr(), context_lens.data_ptr())
    return QueryDesc(None, DTYPE_BF16, B, num_q_heads or 1, W, block_tables.data_ptr(),
                     context_lens.data_ptr())


def ragged_desc(**kw) -> RaggedDesc:
    """RaggedDesc of ragged_fields' arguments."""
    return RaggedDesc(*ragged_fields(**kw))


def ragged_fields(num_tokens: int, cu_tokens: torch.Tensor, block_tables: torch.Tensor,
                  context_lens: torch.Tensor, seq_ids: Optional[torch.Tensor],
                  start_positions: Optional[torch.Tensor]) -> tuple:
    """The packed new tokens of a batch and the tables of the sequences they belong to."""
    i32 = torch.int32
    for t in (cu_tokens, block_tables, context_lens, seq_ids, start_positions):
        if t is not None and not (t.dtype is i32 and t.is_contiguous()):
            raise ValueError("cu_tokens, block_tables, context_lens, seq_ids and "
                             "start_positions must be contiguous int32")
    B = cu_tokens.numel() - 1
    if block_tables.dim() != 2 or cu_tokens.dim() != 1 or B < 0:
        raise ValueError("block_tables must be [num_seqs, max_pages], cu_tokens [batch + 1]")
    S, W = block_tables.shape
    if context_lens.dim() != 1 or context_lens.numel() != S:
        raise ValueError("context_lens must be [num_seqs]")
    for t in (seq_ids, start_positions):
        if t is not None and (t.dim() != 1 or t.numel() != B):
            raise ValueError("seq_ids and start_positions must be [batch]")
    return (cu_tokens.data_ptr(), 0 if seq_ids is None else seq_ids.data_ptr(),
            0 if start_positions is None else start_positions.data_ptr(),
            block_tables.data_ptr(), context_lens.data_ptr(), B, num_tokens, S, W)


class _ArgMemory(threading.local):
    """Per-thread argument structs of the ragged-batch calls over one buffer, which one
    pack fills (constructing the three structs field by field costs 5 us a call)."""

    _KV, _RG = "QQiiiiiiqqq", "QQQQQiiii"

    def __init__(self):
        self.buf = ctypes.create_string_buffer(64 + 56 + 152)
        self.kv = KvDesc.from_buffer(self.buf, 0)
        self.rg = RaggedDesc.from_buffer(self.buf, 64)
        self.chunk = ChunkAttend.from_buffer(self.buf, 120)
        self.rope = RopeAppend.from_buffer(self.buf, 120)
        self.weights = KeyWeights.from_buffer(self.buf, 120)
        self.evict = Evict.from_buffer(self.buf, 64)
        self.pack_chunk = struct.Struct("<" + self._KV + self._RG + "QQQiiqqqqfii").pack_into
        self.pack_rope = struct.Struct("<" + self._KV + self._RG
                                       + "QQQQiiqqqqqqqqQiiiiQQf").pack_into
        self.pack_weights = struct.Struct("<" + self._KV + self._RG
                                          + "QQiiqqffiiQQq").pack_into
        self.pack_evict = struct.Struct("<" + self._KV + "QqQqQi4xQiii4x").pack_into


ARGS = _ArgMemory()


def kv_fields(k_cache: torch.Tensor, v_cache: torch.Tensor, scaled: bool = False) -> tuple:
    """KvDesc's fields (kv_desc's checks); scaled: the call has scales, for 8-bit pools."""
    shape, stride, dt = k_cache.shape, k_cache.stride(), k_cache.dtype
    if (len(shape) != 4 or v_cache.shape != shape or v_cache.dtype != dt
            or v_cache.stride() != stride or stride[3] != 1):
        kv_desc(k_cache, v_cache)  # raises
    if scaled != (dt is torch.float8_e4m3fn):
        raise ValueError("an 8-bit cache (float8_e4m3fn) needs its scales, another has none")
    return (k_cache.data_ptr(), v_cache.data_ptr(), DTYPE_E4M3 if scaled else dtype_code(dt),
            *shape, 0, *stride[:3])


def scale_ptr(scale: Optional[torch.Tensor], cache: torch.Tensor, name: str) -> Optional[int]:
    """Address of an 8-bit cache's scales (None without)."""
    if scale is None:
        return None
    if (cache.dim() != 4 or scale.dtype is not torch.float32 or not scale.is_contiguous()
            or scale.shape != (cache.shape[0], cache.shape[2])):
        raise ValueError(f"{name} must be a contiguous float32 [num_blocks, H_kv]")
    return scale.data_ptr()


# A selection names pages by their place in a sequence's table. An eviction puts other keys
# there, so the tables' memory (views of it too) carries how often that happened, for who
# keeps selections.
def renumbered(tables: torch.Tensor) -> int:
    """How often so far; -1 where a replayed graph may have done it unseen."""
    memory = tables.untyped_storage()
    if getattr(memory, "cvsa_replays", False) and not torch.cuda.is_current_stream_capturing():
        return -1
    return getattr(memory, "cvsa_renumbered", 0)


def renumber(tables: torch.Tensor):
    memory = tables.untyped_storage()
    memory.cvsa_renumbered = getattr(memory, "cvsa_renumbered", 0) + 1
    if torch.cuda.is_current_stream_capturing():
        memory.cvsa_replays = True


def token_rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """A [num_tokens, heads, head_dim] view the kernels can read: 16-byte rows (copied if not)."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be [num_tokens, heads, head_dim]")
    st, sh, sd = t.stride()
    if t.numel() and (sd != 1 or t.data_ptr() % 16 or (st | sh) * t.element_size() % 16):
        return t.clone(memory_format=torch.contiguous_format)
    return t


class Workspace:
    """Per-device, per-stream cache of zeroed workspace buffers, grown on demand.

    Kernels that use a ticket counter leave it at zero, so a buffer is zeroed
    once, when it is created.
    """

    def __init__(self):
        self._bufs = {}
        self.lock = threading.Lock()

    def get(self, nbytes: int, device: torch.device, tag: str = "") -> torch.Tensor:
        key = (device, torch.cuda.current_stream(device).cuda_stream, tag)
        buf = self._bufs.get(key)
        if buf is None or buf.numel() < nbytes:
            buf = torch.zeros(max(nbytes, 256) + 256, dtype=torch.uint8, device=device)
            self._bufs[key] = buf
        off = (-buf.data_ptr()) % 256
        return buf[off:]

    def address(self, nbytes: int, device: torch.device, stream: int, tag: str) -> int:
        """Aligned address of nbytes, for calls that pass no tensor on; a buffer for each size,
        kept. Under `lock`, until the call has enqueued all its kernels: threads share a stream
        (the default one), and what one call's kernels leave for one another is lost if another
        call's come between. Not for a call that is captured: every graph would hold the same
        buffer, and graphs may run at the same time."""
        key = (device.index, stream, tag, nbytes)
        got = self._bufs.get(key)
        if got is None:
            buf = torch.zeros(nbytes + 256, dtype=torch.uint8, device=device)
            got = (buf, buf.data_ptr() + (-buf.data_ptr()) % 256)
            self._bufs[key] = got
        return got[1]


WORKSPACE = Workspace()
