"""The page-sparse decode step between evictions: a selection of pages names them by their
place in a sequence's table, and an eviction renumbers them."""

import pytest
import torch

from conftest import sel_sets
from cvsa.backend import CVSABackend
from cvsa.runtime.chunked import ChunkedAttention
from cvsa.runtime.eviction import WeightedEviction
from cvsa.runtime.kv_cache import PagedKVCache, SequenceKVManager
from ragged_ref import cu_of

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
HQ, H, D, PAGE = 8, 2, 128, 16


def grown(cuda, lens=(1500, 700), seed=0):
    """A manager with sequences, and their eviction with weights of one call."""
    m = SequenceKVManager(PagedKVCache(400, PAGE, H, D), len(lens), 2048)
    ev = WeightedEviction(m, keep=400, sink=4, recent=50)
    g = torch.Generator(device=cuda).manual_seed(seed)
    q, k, v = (torch.randn((sum(lens), h, D), generator=g, device=cuda).to(BF16)
               for h in (HQ, H, H))
    ChunkedAttention()(m, q, k, v, cu_of(list(lens), cuda), eviction=ev)
    return m, ev, [torch.randn((len(lens), HQ, D), generator=g, device=cuda).to(BF16)
                   for _ in range(8)]


def step(be, m, q, layer=0, rows=None):
    c = m.cache
    out = be(q[:rows], c.k_cache, c.v_cache, m.block_tables[:rows], m.context_lens[:rows], layer)
    be.step_done(layer, be.num_layers)
    return out


FORMS = [dict(reuse_interval=16), dict(lazy=True, check_interval=8),
         dict(lazy=True, check_interval=8, coverage_interval=1),
         dict(lazy=True, check_interval=8, selector="quest"),
         dict(lazy=True, check_interval=8, coverage_interval=1, top_p=0.8),
         dict(reuse_interval=16, adaptive_selection=True),
         dict(lazy=True, check_interval=4, sink_pages=1, local_pages=2)]


def backend(kw):
    return CVSABackend(H, HQ, D, PAGE, num_layers=1, budget_pct=0.1, coverage_threshold=0.5, **kw)


@pytest.mark.parametrize("kw", FORMS)
@pytest.mark.parametrize("rows", [None, 1])
def test_a_selection_does_not_outlive_an_eviction(cuda, kw, rows):
    """The step behind an eviction selects anew: it gives what a backend gives that never saw
    the longer sequences, and so do the steps that reuse its selection."""
    m, ev, q = grown(cuda)
    be, fresh = backend(kw), backend(kw)
    step(be, m, q[0], rows=rows)
    ev.evict()
    m.cache.check()
    assert m.context_lens.tolist() == [400, 400]
    for x in q[1:4]:
        got, want = step(be, m, x, rows=rows), step(fresh, m, x, rows=rows)
        assert torch.equal(got, want)
    assert be.device_errors() == 0
    a, b = ([x.cpu() for x in who.cached_selection(0)] for who in (be, fresh))
    assert sel_sets(*a) == sel_sets(*b)


@pytest.mark.parametrize("kw", FORMS[:2])
def test_evictions_of_other_tables_drop_nothing(cuda, kw):
    """Layers and managers are apart: a backend selects anew for the evicted tables alone."""
    (m, ev, q), (other, _, _) = grown(cuda), grown(cuda, seed=1)
    be = CVSABackend(H, HQ, D, PAGE, num_layers=2, budget_pct=0.1, coverage_threshold=0.5, **kw)
    for i in range(3):
        step(be, m, q[i], 0)
        step(be, other, q[i], 1)
    assert be.get_stats()["total_scoring_steps"] == 2
    ev.evict()
    for i in range(3, 6):
        step(be, m, q[i], 0)
        step(be, other, q[i], 1)
    assert be.get_stats()["total_scoring_steps"] == 3


@pytest.mark.parametrize("kw", FORMS)
def test_forget_selections(cuda, kw):
    """For tables that are copies of a manager's: the selections of a layer, or of all, are
    dropped by hand; steps and statistics go on."""
    m, ev, q = grown(cuda)
    be, fresh = backend(kw), backend(kw)

    def go(be, x):
        c = m.cache
        out = be(x, c.k_cache, c.v_cache, m.block_tables.clone(), m.context_lens, 0)
        be.step_done(0, 1)
        return out

    go(be, q[0])
    ev.evict()
    be.forget_selections(0)
    assert be.cached_selection(0) is None
    for x in q[1:4]:
        assert torch.equal(go(be, x), go(fresh, x))
    be.forget_selections()
    assert be.cached_selection(0) is None and be.get_stats()["total_decode_steps"] == 4


@pytest.mark.parametrize("kw", FORMS[:4])
def test_a_replayed_eviction(cuda, kw):
    """The host does not see a graph that evicts being replayed: steps beside it select anew
    every time. Steps in the graph reuse what the graph's own first step selected."""
    m, ev, q = grown(cuda)
    be, fresh = backend(kw), backend(kw)
    graph, g = torch.cuda.CUDAGraph(), torch.Generator(device=cuda).manual_seed(9)
    with torch.cuda.graph(graph):
        ev.evict()
    for i in range(2):
        step(be, m, q[3 * i])
        graph.replay()
        m.cache.check()
        assert m.context_lens.tolist() == [400, 400]
        for x in q[3 * i + 1:3 * i + 3]:
            assert torch.equal(step(be, m, x), step(fresh, m, x))
        k, v = (torch.randn((900, H, D), generator=g, device=cuda).to(BF16) for _ in range(2))
        zero = torch.zeros((900, HQ, D), dtype=BF16, device=cuda)
        ChunkedAttention()(m, zero, k, v, cu_of([600, 300], cuda), eviction=ev)


def test_an_eviction_and_its_steps_in_a_graph(cuda):
    m, ev, q = grown(cuda)
    be, fresh = backend(FORMS[0]), backend(FORMS[0])
    step(be, m, q[0])
    state = [t.clone() for t in (m.block_tables, m.context_lens, m.pages_allocated,
                                 m.cache.free_list, m.cache.free_head, ev.weights)]
    step(fresh, m, q[0])  # workspaces of both exist before the capture
    fresh.forget_selections()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ev.evict()
        out = [step(be, m, x) for x in q[1:4]]
    for t, was in zip((m.block_tables, m.context_lens, m.pages_allocated, m.cache.free_list,
                       m.cache.free_head, ev.weights), state):
        assert torch.equal(t, was)  # a capture runs nothing
    graph.replay()
    m.cache.check()
    assert m.context_lens.tolist() == [400, 400]
    got = [x.clone() for x in out]
    fresh.reset()
    c = m.cache
    bt = m.block_tables.clone()  # not known to be evicted from
    for x, y in zip(q[1:4], got):
        want = fresh(x, c.k_cache, c.v_cache, bt, m.context_lens, 0)
        fresh.step_done(0, 1)
        assert torch.equal(y, want)
