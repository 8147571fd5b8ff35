"""Attention weight that cached keys got from new tokens.

`key_weights` goes with `chunk_attention`: given its queries and the
log-sum-exp that it returned, it adds up for every cached key and KV head the
softmax weights of the rows that see it (csrc/key_weights.cu). What a key
gathered over time says which keys a sequence can do without
(`cvsa.kernels.evict`). The reference has no counterpart.
"""

import struct
from typing import Optional

import torch

from cvsa import _lib
from cvsa.kernels.evict import _overlap

_ALL = 2 ** 31 - 1  # keys: more than a sequence can hold


def key_weights(q: torch.Tensor, lse: torch.Tensor, k_cache: torch.Tensor,
                block_tables: torch.Tensor, context_lens: torch.Tensor,
                cu_tokens: torch.Tensor, weights: torch.Tensor,
                out: Optional[torch.Tensor] = None, decay: float = 1.0, causal: bool = True,
                window: int = 0, scale: Optional[float] = None,
                seq_ids: Optional[torch.Tensor] = None,
                start_positions: Optional[torch.Tensor] = None,
                dev_error: Optional[torch.Tensor] = None, *,
                k_scale: Optional[torch.Tensor] = None,
                check_only: bool = False) -> torch.Tensor:
    """decay * weights + what the batch's tokens gave each key, [num_seqs, H_kv, capacity].

    q [T, H_q, D] and lse [T, H_q] float32 as given to and filled by
    `chunk_attention`, with its causal, window and scale; weights float32,
    capacity at least max_pages * block_size. The new tokens' own keys start
    from 0. `out` may be another tensor than weights (None: in place); keys past
    a context and sequences outside the batch are not written. k_scale
    [num_blocks, H_kv]: of an 8-bit cache. check_only raises what the call would be
    refused with, without a launch.
    """
    dev = _lib.same_device(q, lse, k_cache, block_tables, context_lens, cu_tokens, weights, out,
                           seq_ids, start_positions, dev_error, k_scale)
    if dev != torch.cuda.current_device():  # a launch goes to the current device
        with torch.cuda.device(dev):
            return key_weights(q, lse, k_cache, block_tables, context_lens, cu_tokens, weights,
                               out, decay, causal, window, scale, seq_ids, start_positions,
                               dev_error, k_scale=k_scale, check_only=check_only)
    q = _lib.token_rows(q, "q")
    T, Hq, D = q.shape
    if k_cache.dim() != 4 or k_cache.shape[3] != D:
        raise ValueError("q's head_dim does not match the cache")
    if lse.shape != (T, Hq) or lse.dtype is not torch.float32 or not lse.is_contiguous():
        raise ValueError("lse must be a contiguous float32 [T, H_q]")
    if out is None:
        out = weights
    for t in (weights, out):
        if (t.dim() != 3 or t.dtype is not torch.float32 or not t.is_contiguous()
                or t.shape[:2] != (block_tables.shape[0], k_cache.shape[2])
                or t.shape != weights.shape):
            raise ValueError("weights and out must be contiguous float32 "
                             "[num_seqs, H_kv, capacity]")
    if out is not weights and out.data_ptr() != weights.data_ptr() and _overlap(weights, out):
        raise ValueError("out must be weights itself or memory of its own")
    qs, mem = q.stride(), _lib.ARGS
    try:
        mem.pack_weights(mem.buf, 0, *_lib.kv_fields(k_cache, k_cache, k_scale is not None),
                         *_lib.ragged_fields(T, cu_tokens, block_tables, context_lens, seq_ids,
                                             start_positions),
                         q.data_ptr(), lse.data_ptr(), _lib.dtype_code(q.dtype), Hq, qs[0], qs[1],
                         D ** -0.5 if scale is None else scale, decay, causal,
                         window if window < _ALL else _ALL, weights.data_ptr(), out.data_ptr(),
                         weights.shape[2])
    except (struct.error, OverflowError) as e:
        raise ValueError(f"key_weights: an argument is out of range ({e})") from None
    lib, ks = _lib.load(), _lib.scale_ptr(k_scale, k_cache, "k_scale")
    if check_only:
        st = lib.cvsa_key_weights_check(mem.kv, ks, mem.rg, mem.weights)
    else:
        st = lib.cvsa_key_weights(mem.kv, ks, mem.rg, mem.weights, _lib.ptr(dev_error),
                                  _lib.raw_stream(dev))
    if st:
        _lib.check(st, "cvsa_key_weights")
    return out
