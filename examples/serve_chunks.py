"""Serve a few prompts: chunked prompts, then sparse decode, on one set of paged caches.

Every layer norms and rotates its projections, appends them to its paged cache
and attends: prompts in chunks of several sequences at a time
(`ChunkedAttention`), then one token a sequence and step through the
coverage-verified sparse backend. The model around the attention is synthetic
(random projections), the attention path is the real one.

    python examples/serve_chunks.py
"""

import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "coverage-verified-sparse-attention_b200"))
from cvsa.backend import CVSABackend  # noqa: E402
from cvsa.kernels.rope_append import rope_table  # noqa: E402
from cvsa.runtime.chunked import ChunkedAttention  # noqa: E402
from cvsa.runtime.kv_cache import PagedKVCache, SequenceKVManager  # noqa: E402


class Layer:
    """One attention layer: a fused projection, its cache and its attention."""

    def __init__(self, hidden, hq, hkv, d, page, batch, max_ctx, table, gen, dtype, device):
        self.shape = (hq, hkv, d)
        w = torch.randn((hidden, (hq + 2 * hkv) * d), generator=gen, device=device)
        self.w_qkv = (w * hidden ** -0.5).to(dtype)
        self.w_out = (torch.randn((hq * d, hidden), generator=gen, device=device)
                      * (hq * d) ** -0.5).to(dtype)
        pages = batch * ((max_ctx + page - 1) // page + 1)
        self.manager = SequenceKVManager(
            PagedKVCache(pages, page, hkv, d, dtype=dtype, device=device), batch, max_ctx)
        norm = torch.ones(d, dtype=dtype, device=device)
        self.attention = ChunkedAttention(cos_sin=table, q_norm=norm, k_norm=norm)

    def project(self, x):
        hq, hkv, d = self.shape
        qkv = x @ self.w_qkv                      # q, k and v stay views of one tensor
        T = x.shape[0]
        return (qkv[:, :hq * d].view(T, hq, d), qkv[:, hq * d:(hq + hkv) * d].view(T, hkv, d),
                qkv[:, (hq + hkv) * d:].view(T, hkv, d))


def serve(prompts, steps, chunk=256, layers=2, hidden=512, hq=8, hkv=2, d=128, page=16,
          dtype=torch.bfloat16, device="cuda", seed=0):
    """Hidden states of every new token of prompts and steps, and the layers."""
    gen = torch.Generator(device=device).manual_seed(seed)
    B, max_ctx = len(prompts), max(prompts) + steps
    table = rope_table(max_ctx, d, device=device)
    net = [Layer(hidden, hq, hkv, d, page, B, max_ctx, table, gen, dtype, device)
           for _ in range(layers)]
    decode = CVSABackend(hkv, hq, d, page, num_layers=layers, budget_pct=0.25,
                         coverage_threshold=0.9, sink_pages=1, local_pages=2, lazy=True,
                         check_interval=4)
    embed = [torch.randn((n + steps, hidden), generator=gen, device=device).to(dtype)
             for n in prompts]
    hidden_out = [[] for _ in prompts]
    # prompts: a chunk of every sequence that has one left, in one ragged batch
    done = [0] * B
    while any(done[b] < prompts[b] for b in range(B)):
        ids = [b for b in range(B) if done[b] < prompts[b]]
        new = [min(chunk, prompts[b] - done[b]) for b in ids]
        cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32,
                          device=device)
        seq = torch.tensor(ids, dtype=torch.int32, device=device)
        x = torch.cat([embed[b][done[b]:done[b] + n] for b, n in zip(ids, new)])
        for layer in net:
            o = layer.attention(layer.manager, *layer.project(x), cu, seq)
            x = x + o.flatten(1) @ layer.w_out
        for i, (b, n) in enumerate(zip(ids, new)):
            hidden_out[b].append(x[int(sum(new[:i])):int(sum(new[:i + 1]))])
            done[b] += n
    # decode: one token a sequence, attention by the sparse backend
    cu = torch.arange(B + 1, dtype=torch.int32, device=device)
    decode.reset()
    for step in range(steps):
        x = torch.stack([embed[b][prompts[b] + step] for b in range(B)])
        for i, layer in enumerate(net):
            m = layer.manager
            q, _ = layer.attention.append(m, *layer.project(x), cu)
            o = decode(q, m.cache.k_cache, m.cache.v_cache, m.block_tables, m.context_lens, i)
            decode.step_done(i, layers)
            x = x + o.flatten(1) @ layer.w_out
        for b in range(B):
            hidden_out[b].append(x[b:b + 1])
    for layer in net:
        layer.manager.cache.check()
    return [torch.cat(h) for h in hidden_out], net, embed, decode


if __name__ == "__main__":
    prompts, steps = [1900, 333, 1024, 57], 12
    out, net, _, decode = serve(prompts, steps)
    torch.cuda.synchronize()
    print("tokens served:", [h.shape[0] for h in out])
    print("cached tokens:", net[0].manager.context_lens.tolist())
    stats = decode.get_stats()
    print("decode steps:", stats["total_decode_steps"],
          "effective budget: %.1f%%" % stats["effective_budget_pct"])
