"""Attention of new tokens on the paged cache: prompts, chunks, drafts, single tokens.

The step before (or beside) the sparse decode: one layer's projections of a
ragged batch of new tokens are appended to the cache of the decode step and
attend to everything their sequences hold. The reference runs prompts in the
model library and copies the keys into its cache afterwards
(eval/latency_benchmark.py:376-420, cvsa/runtime/kv_cache.py:102-131).
"""

from typing import Optional

import torch

from cvsa.kernels.chunk_attend import chunk_attention
from cvsa.kernels.rope_append import rope_append


class ChunkedAttention:
    """reserve -> rope_append -> chunk_attention for one layer's cache.

    cos_sin is a `rope_table` (None: the projections are already rotated);
    q_norm / k_norm are the layer's per-head RMS-norm weights [D] or None;
    window limits how many keys a token sees (0: all)."""

    def __init__(self, cos_sin: Optional[torch.Tensor] = None,
                 q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
                 eps: float = 1e-6, interleaved: bool = False, window: int = 0,
                 scale: Optional[float] = None):
        self.cos_sin = cos_sin
        self.q_norm = q_norm
        self.k_norm = k_norm
        self.eps = eps
        self.interleaved = interleaved
        self.window = window
        self.scale = scale

    def append(self, manager, q, k, v, cu_tokens, seq_ids=None, out=None):
        """Reserve pages, write the keys and values, return (rotated queries, start positions).

        For a decode step: the queries go to the sparse backend. A call that is
        refused (ValueError, RuntimeError) has reserved nothing."""
        c = manager.cache
        cu, ids = _int32(cu_tokens), _int32(seq_ids)
        starts = torch.empty((max(cu.numel() - 1, 0),), dtype=torch.int32, device=cu.device)
        q = rope_append(q, k, v, c.k_cache, c.v_cache, manager.block_tables,
                        manager.context_lens, cu, cos_sin=self.cos_sin,
                        q_norm=self.q_norm, k_norm=self.k_norm, eps=self.eps,
                        interleaved=self.interleaved, seq_ids=ids, start_positions=starts,
                        out=out, dev_error=c.dev_error,
                        _reserve=lambda: manager._reserve(cu, ids, starts))
        return q, starts

    def __call__(self, manager, q, k, v, cu_tokens, seq_ids=None):
        """q [T, H_q, D], k and v [T, H_kv, D] of the packed new tokens -> [T, H_q, D].

        manager is the layer's `SequenceKVManager`; sequence seq_ids[b] (default
        b) owns tokens cu_tokens[b]..cu_tokens[b + 1] (on the device). Nothing
        synchronises: a sequence that does not fit yields zeros and
        `manager.cache.check()` raises. A call that is refused (ValueError,
        RuntimeError) has appended nothing."""
        c = manager.cache
        cu, ids = _int32(cu_tokens), _int32(seq_ids)
        rotated = q.new_empty(q.shape)
        form = dict(window=self.window, scale=self.scale, seq_ids=ids, dev_error=c.dev_error)
        out = chunk_attention(rotated, c.k_cache, c.v_cache, manager.block_tables,
                              manager.context_lens, cu, check_only=True, **form)
        _, starts = self.append(manager, q, k, v, cu, ids, out=rotated)
        return chunk_attention(rotated, c.k_cache, c.v_cache, manager.block_tables,
                               manager.context_lens, cu, start_positions=starts, out=out, **form)


def _int32(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.to(torch.int32).contiguous()
