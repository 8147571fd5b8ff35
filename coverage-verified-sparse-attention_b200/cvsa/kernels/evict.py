"""Eviction from the paged cache by accumulated attention weight.

`evict` keeps, for each KV head of a sequence that is too long, the first keys,
the last ones and those of largest weight between, and moves them to new pages
(csrc/evict.cu). `SequenceKVManager.evict` calls it with the pages of its cache.
The reference has no counterpart: it keeps every page and reads few of them.
"""

import struct
from typing import Optional

import torch

from cvsa import _lib


def evict(k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
          context_lens: torch.Tensor, weights: torch.Tensor, new_tables: torch.Tensor, keep: int,
          sink: int = 0, recent: int = 0, out_weights: Optional[torch.Tensor] = None,
          kept: Optional[torch.Tensor] = None, dev_error: Optional[torch.Tensor] = None, *,
          k_scale: Optional[torch.Tensor] = None,
          v_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Kept keys [num_seqs, H_kv, keep] int32 of the sequences longer than keep (-1: shorter).

    The first `sink` keys, the last `recent` and the keep - sink - recent of
    largest weight between (equal weights: the earlier; NaN below everything),
    in their order. Their keys and values go to the pages of new_tables
    [num_seqs, ceil(keep / block_size)], which no sequence may be using, their
    weights to out_weights [num_seqs, H_kv, >= keep] (None: to the front of
    weights, float32 [num_seqs, H_kv, >= max_pages * block_size], where those behind
    become 0 up to the old length). Tables and lengths stay as they are.
    k_scale, v_scale: of an 8-bit cache, whose new pages get the largest scale of
    their rows.
    """
    dev = _lib.same_device(k_cache, v_cache, block_tables, context_lens, weights, new_tables,
                           out_weights, kept, dev_error, k_scale, v_scale)
    if dev != torch.cuda.current_device():  # a launch goes to the current device
        with torch.cuda.device(dev):
            return evict(k_cache, v_cache, block_tables, context_lens, weights, new_tables, keep,
                         sink, recent, out_weights, kept, dev_error, k_scale=k_scale,
                         v_scale=v_scale)
    scaled = k_scale is not None
    if scaled != (v_scale is not None):
        raise ValueError("k_scale and v_scale go together")
    i32, f32, mem = torch.int32, torch.float32, _lib.ARGS
    kv = _lib.kv_fields(k_cache, v_cache, scaled)
    page, H = kv[4], kv[5]
    for t in (block_tables, context_lens, new_tables):
        if t.dtype is not i32 or not t.is_contiguous():
            raise ValueError("block_tables, context_lens and new_tables must be contiguous int32")
    if block_tables.dim() != 2 or context_lens.shape != block_tables.shape[:1]:
        raise ValueError("block_tables must be [num_seqs, max_pages], context_lens [num_seqs]")
    if not 0 < keep < 2 ** 31 or not 0 <= sink <= keep or not 0 <= recent <= keep - sink:
        raise ValueError("keep must be positive, sink and recent >= 0 and together at most keep")
    S, W = block_tables.shape
    if new_tables.shape != (S, -(-keep // page)):
        raise ValueError("new_tables must be [num_seqs, ceil(keep / block_size)]")
    if out_weights is None:
        out_weights = weights
    for t in (weights, out_weights):
        if t.dim() != 3 or t.dtype is not f32 or not t.is_contiguous() or t.shape[:2] != (S, H):
            raise ValueError("weights and out_weights must be contiguous float32 "
                             "[num_seqs, H_kv, keys]")
    w, o = weights.data_ptr(), out_weights.data_ptr()
    if out_weights is not weights and _overlap(weights, out_weights) and (
            w != o or weights.shape != out_weights.shape):
        raise ValueError("out_weights must be weights itself or memory of its own")
    if kept is None:
        kept = torch.empty((S, H, keep), dtype=i32, device=weights.device)
    elif kept.shape != (S, H, keep) or kept.dtype is not i32 or not kept.is_contiguous():
        raise ValueError("kept must be a contiguous int32 [num_seqs, H_kv, keep]")
    try:
        mem.pack_evict(mem.buf, 0, *kv, w, weights.shape[2], o, out_weights.shape[2],
                       new_tables.data_ptr(), new_tables.shape[1], kept.data_ptr(), keep, sink,
                       recent)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"evict: an argument is out of range ({e})") from None
    st = _lib.load().cvsa_evict(
        mem.kv, _lib.scale_ptr(k_scale, k_cache, "k_scale"),
        _lib.scale_ptr(v_scale, k_cache, "v_scale"), block_tables.data_ptr(),
        context_lens.data_ptr(), S, W, mem.evict, _lib.ptr(dev_error), _lib.raw_stream(dev))
    if st:
        _lib.check(st, "cvsa_evict")
    return kept


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two contiguous tensors share memory."""
    return (a.data_ptr() < b.data_ptr() + b.numel() * b.element_size()
            and b.data_ptr() < a.data_ptr() + a.numel() * a.element_size())
