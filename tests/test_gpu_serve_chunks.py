"""The new tokens' path end to end: the example's chunked prompts and sparse
decode against dense attention in 64 bits, layer by layer.

Each layer's reference starts from the layer input the run itself had (the
residual stream is recomputed in the run's types), so errors do not pile up
and the bar is one layer's: projections and residuals round to bf16 (2^-8), the
attention output passes one random projection of unit gain."""

import importlib.util
import os

import pytest
import torch

from conftest import ROOT

_spec = importlib.util.spec_from_file_location("serve_chunks",
                                               os.path.join(ROOT, "examples", "serve_chunks.py"))
S = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(S)

pytestmark = pytest.mark.gpu


def dense_layer(layer, x):
    """One sequence's layer over all its tokens at once, 64-bit attention."""
    hq, hkv, d = layer.shape
    q, k, v = (t.double() for t in layer.project(x))
    q, k = (t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) for t in (q, k))
    n = x.shape[0]
    tab = layer.attention.cos_sin[:n].double()[:, None]
    cos, sin = tab[..., :d // 2], tab[..., d // 2:]
    q, k = (torch.cat([t[..., :d // 2] * cos - t[..., d // 2:] * sin,
                       t[..., d // 2:] * cos + t[..., :d // 2] * sin], -1) for t in (q, k))
    k, v = (t.repeat_interleave(hq // hkv, 1) for t in (k, v))
    s = torch.einsum("qhd,khd->hqk", q, k) * d ** -0.5
    s.masked_fill_(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), float("-inf"))
    o = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v)
    return x + o.to(x.dtype).flatten(1) @ layer.w_out


@pytest.mark.parametrize("chunk", [64, 256, 4096])
def test_chunked_prompts_match_dense(cuda, chunk):
    prompts = [700, 33, 257, 1]
    out, net, embed, _ = S.serve(prompts, 0, chunk=chunk, layers=1, seed=3)
    for b, n in enumerate(prompts):
        want = dense_layer(net[0], embed[b][:n])
        err = (out[b].float() - want.float()).abs().max()
        assert out[b].shape == want.shape and float(err) < 4e-2, (b, float(err))
    assert net[0].manager.context_lens.tolist() == prompts


def test_prompts_then_sparse_decode(cuda):
    """The decode steps read what the chunks wrote: with every head verified at
    every step (no reuse; threshold above 1: every page recovered) the outputs
    are dense attention's."""
    prompts, steps = [300, 65, 129], 5
    real = S.CVSABackend

    def exact(*a, **kw):
        kw.update(coverage_threshold=1.5, check_interval=1)
        return real(*a, **kw)

    S.CVSABackend = exact
    try:
        out, net, embed, _ = S.serve(prompts, steps, layers=1, seed=4)
    finally:
        S.CVSABackend = real
    for b, n in enumerate(prompts):
        want = dense_layer(net[0], embed[b][:n + steps])
        assert float((out[b].float() - want.float()).abs().max()) < 4e-2
    assert net[0].manager.context_lens.tolist() == [n + steps for n in prompts]


def test_chunk_size_does_not_matter(cuda):
    """Two layers: the same tokens in chunks of 50 and of 400 give the same
    cached keys up to the rounding of what the first layer passes on."""
    a, na, _, _ = S.serve([390, 77], 0, chunk=50, seed=5)
    b, nb, _, _ = S.serve([390, 77], 0, chunk=400, seed=5)
    for x, y in zip(a, b):
        assert float((x.float() - y.float()).abs().max()) < 6e-2
