"""Eviction of a layer's cached keys by the attention weight they gathered.

The sparse decode step reads few pages of a cache that holds every key; where the
pool itself is short, this drops the keys that the tokens so far hardly looked at.
The reference has no counterpart.
"""

from typing import Optional

import torch

from cvsa.kernels.key_weights import key_weights


class WeightedEviction:
    """The weights of one layer's cached keys, and the cut to `keep` of them.

        eviction = WeightedEviction(manager, keep=4096, sink=4, recent=256)
        out = layer(manager, q, k, v, cu_tokens, eviction=eviction)   # every step
        eviction.evict()                                              # now and then

    manager is the layer's `SequenceKVManager`. A key's weight is the sum of the
    softmax weights of all query heads of its KV head's group, `decay` times
    what it was a step before; a key that came in a call without the counting begins
    at 0 with the next one that counts. The first `sink` and the last `recent` keys of a
    sequence are kept whatever their weight. A sliding window counts the keys that
    are left, not positions."""

    def __init__(self, manager, keep: int, sink: int = 0, recent: int = 0, decay: float = 1.0):
        if keep <= 0 or sink < 0 or recent < 0 or sink + recent > keep:
            raise ValueError("keep must be positive, sink and recent >= 0 and together at most "
                             "keep")
        self.manager = manager
        self.keep = keep
        self.sink = sink
        self.recent = recent
        self.decay = decay
        c = manager.cache
        manager.track_evictions()
        self.weights = torch.zeros(
            manager.batch_size, c.num_kv_heads, manager.max_pages * manager.block_size,
            device=c.k_cache.device)
        manager._counting.add(self)  # prefill_kv clears a slot that it fills anew

    def observe(self, q: torch.Tensor, lse: torch.Tensor, cu_tokens: torch.Tensor,
                seq_ids: Optional[torch.Tensor] = None,
                start_positions: Optional[torch.Tensor] = None, window: int = 0,
                scale: Optional[float] = None, check_only: bool = False):
        """Add what the tokens of a batch gave each key; arguments as in `chunk_attention`."""
        m = self.manager
        c = m.cache
        key_weights(q, lse, c.k_cache, m.block_tables, m.context_lens, cu_tokens, self.weights,
                    decay=self.decay, window=window, scale=scale, seq_ids=seq_ids,
                    start_positions=start_positions, dev_error=c.dev_error, k_scale=c.k_scale,
                    check_only=check_only)

    def evict(self) -> torch.Tensor:
        """`SequenceKVManager.evict` with these weights; the kept keys."""
        return self.manager.evict(self.weights, self.keep, self.sink, self.recent)
