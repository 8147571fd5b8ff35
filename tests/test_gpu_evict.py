"""Key weights and eviction against 64-bit references, and the layer that uses both."""

import pytest
import torch

from cache8_ref import F8, Problem8, exponent, kept64, near8, values, weights64
from cvsa import _lib
from cvsa.kernels.chunk_attend import chunk_attention
from cvsa.kernels.evict import evict
from cvsa.kernels.key_weights import key_weights
from cvsa.kernels.rope_append import rope_append, rope_table
from cvsa.runtime.chunked import ChunkedAttention
from cvsa.runtime.eviction import WeightedEviction
from cvsa.runtime.kv_cache import PagedKVCache, SequenceKVManager
from ragged_ref import Problem, assert_within, attend64, cu_of, rope64

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
I32 = dict(dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------
# key weights
# ---------------------------------------------------------------------------
def problem(new, ctx, hq, hkv, d, cache8=False, **kw):
    P = (Problem8 if cache8 else Problem)(new, ctx, hq, hkv, d, **kw)
    P.more = dict(k_scale=P.k_scale) if cache8 else {}
    return P


def lse_of(P, **kw):
    """The rows' log-sum-exps from the definition, as the attention would return them."""
    return attend64(P, **kw)[1].float()


def check_weights(P, decay=1.0, in_place=False, starts=None, lse=None, **kw):
    lse = lse_of(P, starts=starts, **kw) if lse is None else lse
    g = torch.Generator(device="cuda").manual_seed(5)
    S, cap = P.lens.numel(), P.tables.shape[1] * P.page + 3
    prior = torch.rand((S, P.hkv, cap), generator=g, device="cuda")
    # what the new tokens' own slots and those past a context hold does not count
    for b, (n, c) in enumerate(zip(P.new, P.ctx)):
        prior[P.rows[b], :, max(0, c - n if starts is None else starts[b]):] = 9.0
    given = prior.clone() if in_place else torch.full_like(prior, 7.0)
    st = None if starts is None else torch.tensor(starts, **I32)
    got = key_weights(P.q, lse, P.k_cache, P.tables, P.lens, P.cu,
                      given if in_place else prior, out=None if in_place else given, decay=decay,
                      seq_ids=P.seq_ids, start_positions=st, dev_error=P.dev_error, **P.more, **kw)
    torch.cuda.synchronize()
    assert got is given and int(P.dev_error.item()) == 0
    want, tol = weights64(P, P.q, lse, prior, decay, starts=starts, **kw)
    if not in_place:  # not written: past a context, rows of no sequence, refused sequences
        live = torch.zeros(want.shape, dtype=torch.bool, device="cuda")
        for b, c in enumerate(P.ctx):
            if starts is None or starts[b] >= 0:
                live[P.rows[b], :, :c] = True
        want = torch.where(live, want, 7.0)
    assert_within(got, want, tol, "weights")
    return got


@pytest.mark.parametrize("dtype,cache8", [(BF16, False), (F16, False), (F32, False), (BF16, True),
                                          (F16, True), (F32, True)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (7, 1)])
def test_weights_ragged_batch(cuda, dtype, cache8, d, hq, hkv):
    check_weights(problem([1, 0, 33, 5, 130, 1, 2, 1], [1, 40, 33, 127, 259, 128, 129, 1000], hq,
                          hkv, d, cache8, dtype=dtype, seed=3))


@pytest.mark.parametrize("cache8", [False, True])
@pytest.mark.parametrize("new", [[1, 1, 1], [300, 1, 64]])
@pytest.mark.parametrize("kw", [
    dict(decay=0.5), dict(decay=0.0), dict(in_place=True), dict(in_place=True, decay=0.25),
    dict(causal=False), dict(window=1), dict(window=17), dict(window=200), dict(scale=0.3),
    dict(window=2 ** 31 - 1)])
def test_weights_forms(cuda, cache8, new, kw):
    check_weights(problem(new, [400, 333, 65], 8, 2, 128, cache8, seed=4), **kw)


@pytest.mark.parametrize("cache8", [False, True])
@pytest.mark.parametrize("G", [1, 2, 3, 5, 8, 16, 17, 33, 64])
@pytest.mark.parametrize("new", [[1, 1], [70, 1]])
def test_weights_group_sizes(cuda, cache8, G, new):
    check_weights(problem(new, [200, 150], 2 * G, 2, 64, cache8, seed=G))


@pytest.mark.parametrize("cache8", [False, True])
@pytest.mark.parametrize("page", [1, 2, 16, 24, 64, 256])
@pytest.mark.parametrize("new", [[1, 2], [150, 3]])
def test_weights_pages(cuda, cache8, page, new):
    check_weights(problem(new, [301, 77], 8, 4, 128, cache8, page=page, seed=page))


@pytest.mark.parametrize("cache8", [False, True])
def test_weights_long(cuda, cache8):
    check_weights(problem([1, 40], [20011, 5000], 4, 1, 128, cache8, seed=9))
    n = 300
    check_weights(problem([1 + i % 3 for i in range(n)], [3 + (i * 7) % 50 for i in range(n)], 2,
                          1, 64, cache8, seed=4))
    check_weights(problem([700], [900], 16, 2, 128, cache8, seed=6))


@pytest.mark.parametrize("q_dtype,kv_dtype", [(BF16, F32), (F32, BF16), (F16, BF16)])
def test_weights_mixed_types(cuda, q_dtype, kv_dtype):
    check_weights(problem([30, 1], [100, 300], 8, 2, 128, dtype=q_dtype, kv_dtype=kv_dtype, seed=6))


@pytest.mark.parametrize("cache8", [False, True])
def test_weights_rows_and_sequences(cuda, cache8):
    """Table rows in another order, padding, start positions, refused sequences, contexts
    shorter than the chunk."""
    check_weights(problem([2, 33, 1], [20, 33, 260], 8, 2, 64, cache8, seq_ids=[3, 0, 5],
                          pad_tokens=9))
    check_weights(problem([2, 33, 1], [60, 90, 260], 8, 2, 64, cache8), starts=[58, -1, 259])
    check_weights(problem([2, 33, 1], [60, 90, 260], 8, 2, 64, cache8), starts=[10, 57, 100])
    check_weights(problem([10, 3, 4], [4, 0, 300], 8, 2, 128, cache8, seed=2))


@pytest.mark.parametrize("cache8", [False, True])
@pytest.mark.parametrize("n", [1, 100])
def test_weights_without_a_number(cuda, cache8, n):
    """Rows whose log-sum-exp is -inf add nothing, a NaN key is a NaN weight where a row
    sees it and reaches no other."""
    P = problem([n], [333], 4, 2, 128, cache8, seed=7)
    lse = lse_of(P)
    lse[0] = float("-inf")
    check_weights(P, lse=lse)
    P.put(0, 300, k=float("nan"))
    lse = lse_of(problem([n], [333], 4, 2, 128, cache8, seed=7))
    got = check_weights(P, lse=lse)
    assert bool(torch.isnan(got[0, :, 300]).all()) and int(torch.isnan(got).sum()) == 2


@pytest.mark.parametrize("cache8", [False, True])
@pytest.mark.parametrize("n", [1, 100])
def test_weights_bad_pages(cuda, cache8, n):
    P = problem([n], [333], 4, 2, 128, cache8, seed=7)
    lse = lse_of(P)
    prior = torch.rand((1, 2, P.tables.shape[1] * 16), device=cuda)
    good = key_weights(P.q, lse, P.k_cache, P.tables, P.lens, P.cu, prior,
                       out=torch.zeros_like(prior), **P.more)
    P.tables[0, 3], P.tables[0, 7] = P.k_cache.shape[0], -2
    got = key_weights(P.q, lse, P.k_cache, P.tables, P.lens, P.cu, prior,
                      out=torch.zeros_like(prior), dev_error=P.dev_error, **P.more)
    assert int(P.dev_error.item()) == _lib.DEV_ERR_BLOCK_RANGE
    for p in (3, 7):  # what the keys had before
        good[:, :, 16 * p:16 * p + 16] = prior[:, :, 16 * p:16 * p + 16]
    assert torch.equal(got, good)


def test_weights_sum_to_the_rows(cuda):
    """With the attention's own log-sum-exps every row gives 1 in all."""
    P = problem([200, 1, 9], [700, 400, 1000], 16, 4, 128, seed=8)
    lse = torch.empty((P.T, 16), device=cuda)
    chunk_attention(P.q, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, lse=lse)
    w = torch.zeros((3, 4, P.tables.shape[1] * 16), device=cuda)
    key_weights(P.q, lse, P.k_cache, P.tables, P.lens, P.cu, w)
    # a score errs by about 1e-5, a weight relatively by as much
    assert torch.allclose(w.double().sum(-1), torch.tensor([800.0, 4.0, 36.0], device=cuda)
                          .double()[:, None].expand(3, 4), rtol=5e-5)


def test_weights_other_stream_and_graph(cuda):
    P = problem([1, 30], [500, 700], 8, 2, 128, seed=16)
    lse = lse_of(P)
    w = torch.rand((2, 2, P.tables.shape[1] * 16), device=cuda)
    want = key_weights(P.q, lse, P.k_cache, P.tables, P.lens, P.cu, w, out=torch.zeros_like(w))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = key_weights(P.q, lse, P.k_cache, P.tables, P.lens, P.cu, w, out=torch.zeros_like(w))
    s.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        key_weights(P.q, lse, P.k_cache, P.tables, P.lens, P.cu, w, out=out)
    graph.replay()
    assert torch.equal(out, want)
    P.lens[1] = 600  # as many new tokens of a shorter sequence
    want = key_weights(P.q, lse, P.k_cache, P.tables, P.lens, P.cu, w, out=torch.zeros_like(w))
    out.zero_()
    graph.replay()
    assert torch.equal(out, want)


# ---------------------------------------------------------------------------
# evict
# ---------------------------------------------------------------------------
class Cut:
    """Caches of sequences with weights, and what eviction should make of them."""

    def __init__(self, lens, keep, sink=0, recent=0, hkv=2, d=64, page=16, dtype=BF16, seed=0,
                 ties=0, extra=3):
        g = torch.Generator().manual_seed(seed)
        self.lens_, self.keep, self.sink, self.recent = lens, keep, sink, recent
        S, self.page, self.hkv = len(lens), page, hkv
        W = max(1, max(-(-n // page) for n in lens))
        n_new = -(-keep // page)
        blocks = sum(-(-n // page) for n in lens) + S * n_new + 1
        order = torch.randperm(blocks, generator=g).to(torch.int32)
        self.tables = torch.full((S, W), -9, dtype=torch.int32)  # past a context: never read
        at = 0
        for s, n in enumerate(lens):
            p = -(-n // page)
            self.tables[s, :p] = order[at:at + p]
            at += p
        self.new = order[at:at + S * n_new].view(S, n_new).clone().cuda()
        self.tables, self.lens = self.tables.cuda(), torch.tensor(lens, **I32)
        if dtype is F8:
            self.pools = [torch.randint(0, 255, (blocks, page, hkv, d), generator=g,
                                        dtype=torch.uint8).cuda().view(F8) for _ in range(2)]
            self.scales = [(2.0 ** torch.randint(-15, 8, (blocks, hkv), generator=g)).float()
                           .cuda() for _ in range(2)]
        else:
            self.pools = [torch.randn((blocks, page, hkv, d), generator=g).to(dtype).cuda()
                          for _ in range(2)]
            self.scales = []
        w = torch.rand((S, hkv, W * page + extra), generator=g) ** 4
        if ties:
            w = torch.round(w * ties) / ties
        self.w = w.cuda()
        self.err = torch.zeros(1, **I32)

    def run(self, out=None, **kw):
        more = dict(zip(("k_scale", "v_scale"), self.scales))
        got = evict(*self.pools, self.tables, self.lens, self.w, self.new, self.keep,
                    sink=self.sink, recent=self.recent, out_weights=out, dev_error=self.err,
                    **more, **kw)
        torch.cuda.synchronize()
        return got

    def check(self, in_place=True):
        pools0 = [p.clone() for p in self.pools]
        scales0 = [s.clone() for s in self.scales]
        w0 = self.w.clone()
        out = None if in_place else torch.full((len(self.lens_), self.hkv, self.keep), 5.0,
                                               device="cuda")
        kept = self.run(out).cpu()
        assert int(self.err.item()) == 0
        got_w = self.w if in_place else out
        want = [p.clone() for p in pools0]
        want_s = [s.clone() for s in scales0]
        for s, n in enumerate(self.lens_):
            if n <= self.keep:
                assert bool((kept[s] == -1).all())
                assert torch.equal(got_w[s], w0[s] if in_place else out[s])
                if not in_place:
                    assert bool((out[s] == 5).all())
                continue
            for h in range(self.hkv):
                idx = kept64(w0[s, h].tolist(), n, self.keep, self.sink, self.recent)
                assert kept[s, h].tolist() == idx, (s, h)
                idx = torch.tensor(idx, device="cuda")
                ww = w0[s, h][idx]
                assert torch.equal(torch.nan_to_num(got_w[s, h, :self.keep], 77.0),
                                   torch.nan_to_num(ww, 77.0))
                i = torch.arange(self.keep, device="cuda")
                src = self.tables[s].long()[idx // self.page]
                dst = self.new[s].long()[i // self.page]
                for j in range(2):
                    raw0 = pools0[j].view(torch.uint8) if self.scales else pools0[j]
                    raw = want[j].view(torch.uint8) if self.scales else want[j]
                    rows = raw0[src, idx % self.page, h]
                    if self.scales:
                        mine = scales0[j][src, h]
                        for p in range(self.new.shape[1]):
                            here = i // self.page == p
                            top = mine[here].max()
                            want_s[j][self.new[s, p].long(), h] = top
                            old = rows[here].view(F8).double() * mine[here].double()[:, None]
                            rows[here] = near8(old / top.double()).float().to(F8).view(torch.uint8)
                    raw[dst, i % self.page, h] = rows
        for a, b in zip(self.pools, want):
            if self.scales:  # NaN has two codes, the sign aside: compare the values
                a, b = a.double(), b.double()
            assert torch.equal(torch.nan_to_num(a.double(), 1e9), torch.nan_to_num(b.double(), 1e9))
        for a, b in zip(self.scales, want_s):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F16, F32, F8])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_evict_types(cuda, dtype, d):
    Cut([100, 33, 30, 0, 500], 32, 3, 7, d=d, dtype=dtype, seed=d).check()


@pytest.mark.parametrize("dtype", [BF16, F8])
@pytest.mark.parametrize("keep,sink,recent", [
    (1, 0, 0), (1, 1, 0), (1, 0, 1), (16, 16, 0), (16, 0, 16), (17, 4, 13), (31, 0, 0),
    (64, 1, 62), (200, 10, 20)])
def test_evict_shares(cuda, dtype, keep, sink, recent):
    Cut([201, 350, keep, keep + 1], keep, sink, recent, dtype=dtype, seed=keep).check(False)


@pytest.mark.parametrize("dtype", [F16, F8])
@pytest.mark.parametrize("page", [1, 2, 16, 24, 33, 64, 256])
def test_evict_pages(cuda, dtype, page):
    Cut([301, 77, 500], 70, 2, 9, page=page, dtype=dtype, seed=page).check()


@pytest.mark.parametrize("ties", [1, 3, 50])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_ties(cuda, ties, in_place):
    """Few different weights (with ties=1, mostly zeros): the earlier key goes first."""
    Cut([3000, 129], 100, 4, 20, ties=ties, seed=ties).check(in_place)
    c = Cut([3000, 129], 100, 4, 20, seed=ties)
    c.w.fill_(0.25)
    c.check(in_place)


@pytest.mark.parametrize("n,keep", [(8192, 8191), (8193, 100), (20000, 5000), (60001, 1000),
                                    (131072, 4096)])
def test_evict_long(cuda, n, keep):
    """Rows past one round of the block, and past what shared memory holds."""
    Cut([n, n // 2 + 1], keep, 5, keep // 10, hkv=1, seed=n).check()
    Cut([n], keep, 0, 0, hkv=2, seed=n, ties=1000).check(False)


def test_evict_weights_without_a_number(cuda):
    """Infinities and NaN in the weights: NaN goes last, -0 and 0 are one."""
    c = Cut([400], 50, 2, 3, hkv=1, seed=3)
    c.w[0, 0, 10:200] = float("nan")
    c.w[0, 0, 200:210] = float("inf")
    c.w[0, 0, 210:260] = float("-inf")
    c.w[0, 0, 260:300] = -0.0
    c.w[0, 0, 300:330] = 0.0
    c.check()
    c = Cut([400], 350, 2, 3, hkv=1, seed=3)  # some NaN have to stay
    c.w[0, 0, 10:200] = float("nan")
    c.check(False)


def test_evict_out_of_range(cuda):
    c = Cut([100, 90], 32, 1, 1)
    pools = [p.clone() for p in c.pools]
    c.new.fill_(c.pools[0].shape[0])
    c.run()
    assert int(c.err.item()) == _lib.DEV_ERR_BLOCK_RANGE
    assert all(torch.equal(a, b) for a, b in zip(pools, c.pools))
    c = Cut([100, 90], 32, 1, 1)
    c.tables.fill_(-1)
    pools = [p.clone() for p in c.pools]
    c.run()
    assert int(c.err.item()) == _lib.DEV_ERR_BLOCK_RANGE
    assert all(torch.equal(a, b) for a, b in zip(pools, c.pools))
    c = Cut([100, 90], 32, 1, 1)
    c.lens[0], c.lens[1] = -4, 1 << 30
    assert bool((c.run() == -1).all())
    assert int(c.err.item()) == _lib.DEV_ERR_RAGGED


def test_evict_other_stream_and_graph(cuda):
    c = Cut([1000, 700], 200, 4, 30, dtype=F8, seed=5)
    out = torch.zeros((2, 2, 200), device=cuda)
    want = c.run(out).clone()
    w, pools = out.clone(), [p.clone().view(torch.uint8) for p in c.pools]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.run(out)
    s.synchronize()
    assert torch.equal(got, want)
    kept = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    more = dict(zip(("k_scale", "v_scale"), c.scales))
    with torch.cuda.graph(graph):
        evict(*c.pools, c.tables, c.lens, c.w, c.new, 200, 4, 30, out_weights=out, kept=kept,
              **more)
    out.zero_()
    graph.replay()
    assert torch.equal(kept, want) and torch.equal(out, w)
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(pools, c.pools))


# ---------------------------------------------------------------------------
# the manager and the layer
# ---------------------------------------------------------------------------
def pages_of(m):
    """Every page of the pool once: in a table or free."""
    c = m.cache
    used = [p for s in range(m.batch_size)
            for p in m.block_tables[s, :int(m.pages_allocated[s])].tolist()]
    free = c.free_list[int(c.free_head):].tolist()
    assert sorted(used + free) == list(range(c.k_cache.shape[0]))
    return len(free)


@pytest.mark.parametrize("dtype", [BF16, F8])
def test_manager_gives_pages_back(cuda, dtype):
    H, d, page = 2, 64, 16
    order = torch.randperm(80, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    m = SequenceKVManager(PagedKVCache(80, page, H, d, dtype=dtype, free_list=order), 4, 512)
    lens = [300, 40, 200, 33]
    T = sum(lens)
    g = torch.Generator(device=cuda).manual_seed(2)
    k, v = (torch.randn((T, H, d), generator=g, device=cuda).to(BF16) for _ in range(2))
    starts = m.reserve(cu_of(lens, cuda))
    c = m.cache
    more = dict(k_scale=c.k_scale, v_scale=c.v_scale)
    rope_append(None, k, v, c.k_cache, c.v_cache, m.block_tables, m.context_lens, cu_of(lens, cuda),
                start_positions=starts, **more)
    before = pages_of(m)
    w = torch.rand((4, H, 512), generator=g, device=cuda)
    w0, t0 = w.clone(), m.block_tables.clone()
    whole = [values(x, s) if dtype is F8 else x.double() for x, s in
             ((c.k_cache, c.k_scale), (c.v_cache, c.v_scale))]
    kept = m.evict(w, 50, 2, 10)
    c.check()
    assert m.context_lens.tolist() == [50, 40, 50, 33]
    assert m.pages_allocated.tolist() == [4, 3, 4, 3] and m.evicted.tolist() == [250, 0, 150, 0]
    assert pages_of(m) == before + 19 - 4 + 13 - 4
    now = [values(x, s) if dtype is F8 else x.double() for x, s in
           ((c.k_cache, c.k_scale), (c.v_cache, c.v_scale))]
    for s, n in enumerate(lens):
        if n <= 50:
            assert bool((kept[s] == -1).all()) and torch.equal(m.block_tables[s], t0[s])
            continue
        for h in range(H):
            idx = torch.tensor(kept64(w0[s, h].tolist(), n, 50, 2, 10), device=cuda)
            assert torch.equal(kept[s, h].long(), idx)
            assert torch.equal(w[s, h, :50], w0[s, h][idx])
            i = torch.arange(50, device=cuda)
            for a, b, sc in zip(now, whole, (c.k_scale, c.v_scale)):
                x = a[m.block_tables[s].long()[i // page], i % page, h]
                y = b[t0[s].long()[idx // page], idx % page, h]
                # an 8-bit row may have moved to a larger scale: subnormal there
                assert torch.equal(x, y) if dtype is BF16 else \
                    bool(((x - y).abs() <= 2.0 ** -10 * sc.max()).all())
    # the pages that came back are handed out again
    starts = m.reserve(cu_of([200, 0, 300, 0], cuda))
    c.check()
    assert starts.tolist() == [50, 40, 50, 33]
    pages_of(m)


def test_manager_without_room(cuda):
    """A sequence that the pool has no pages for stays as it is; the others are cut."""
    m = SequenceKVManager(PagedKVCache(32, 16, 1, 64), 3, 256)
    m.reserve(cu_of([160, 160, 160], cuda))  # 30 of 32 pages
    tables = m.block_tables.clone()
    w = torch.rand((3, 1, 256), device=cuda)
    kept = m.evict(w, 32)
    assert m.context_lens.tolist() == [32, 160, 160] and m.evicted.tolist() == [128, 0, 0]
    assert torch.equal(m.block_tables[1:], tables[1:]) and bool((kept[1:] == -1).all())
    with pytest.raises(AssertionError):
        m.cache.check()
    m.cache.dev_error.zero_()
    assert pages_of(m) == 10
    m.evict(w, 32)
    m.cache.check()
    assert m.context_lens.tolist() == [32, 32, 32] and pages_of(m) == 26
    m.evict(w, 32)  # nothing to do
    m.cache.check()
    assert m.context_lens.tolist() == [32, 32, 32] and pages_of(m) == 26


def test_manager_does_not_take_foreign_pages(cuda):
    """Tables that the pool did not hand out are not given to it: nothing is evicted."""
    m = SequenceKVManager(PagedKVCache(40, 16, 1, 64), 1, 512)
    m.block_tables[0, :20] = torch.arange(20, 40)
    m.context_lens[0], m.pages_allocated[0] = 320, 20
    m.evict(torch.rand((1, 1, 512), device=cuda), 16)
    assert m.context_lens.tolist() == [320] and int(m.cache.free_head) == 0
    with pytest.raises(AssertionError):
        m.cache.check()


def test_many_sequences_of_a_manager(cuda):
    """More sequences than the bookkeeping block has threads."""
    n = 1500
    m = SequenceKVManager(PagedKVCache(2 * n + n // 2, 1, 1, 64), n, 4)
    m.reserve(cu_of([1 + i % 2 for i in range(n)], cuda))
    m.cache.check()
    m.evict(torch.rand((n, 1, 4), device=cuda), 1)
    m.cache.check()
    assert m.context_lens.tolist() == [1] * n and pages_of(m) == n + n // 2
    assert m.evicted.tolist() == [i % 2 for i in range(n)]


@pytest.mark.parametrize("dtype", [BF16, F8])
@pytest.mark.parametrize("hq", [2, 8])
def test_layer_with_eviction(cuda, dtype, hq):
    """Chunks, single tokens and evictions in turn: every call's output is the 64-bit
    attention over what its heads still hold, new tokens are rotated by their true
    position, and the weights are those of the definition."""
    H, d, page, B = 2, 64, 16, 2
    m = SequenceKVManager(PagedKVCache(100, page, H, d, dtype=dtype), B, 320)
    tab = rope_table(2000, d, device=cuda)
    layer = ChunkedAttention(cos_sin=tab)
    ev = WeightedEviction(m, keep=100, sink=4, recent=20, decay=0.9)
    g = torch.Generator(device=cuda).manual_seed(hq)
    seen = [0, 0]
    model = torch.zeros((B, H, 320), dtype=torch.float64, device=cuda)
    c = m.cache
    for step in range(24):
        new = [int(torch.randint(0, 60, (1,), generator=g, device=cuda)), 1] if step % 3 else [1, 1]
        T = sum(new)
        q, k, v = (torch.randn((T, h, d), generator=g, device=cuda).to(BF16) for h in (hq, H, H))
        out = layer(m, q, k, v, cu_of(new, cuda), eviction=ev)
        kv, vv = ((values(x, s) if dtype is F8 else x.double()) for x, s in
                  ((c.k_cache, c.k_scale), (c.v_cache, c.v_scale)))
        t, lens = 0, m.context_lens.tolist()
        for b, n in enumerate(new):
            L = lens[b]
            pos = torch.arange(L, device=cuda)
            blk = m.block_tables[b].long()[pos // page]
            kk, vvv = kv[blk, pos % page], vv[blk, pos % page]
            at = torch.arange(seen[b], seen[b] + n, device=cuda)
            seen[b] += n
            qq = rope64(q[t:t + n], at, tab, d, False, None, 0)[0].view(n, H, hq // H, d)
            mine = rope64(k[t:t + n], at, tab, d, False, None, 0)[0]
            u = 2.0 ** -4 if dtype is F8 else 2.0 ** -8
            if n:  # its own keys, turned by the positions in the text
                top = mine.abs().max()
                assert bool(((kk[L - n:] - mine).abs()
                             <= u * mine.abs() + 2.0 ** -9 * 2.0 ** exponent(4 * top)).all())
            s = torch.einsum("nhgd,lhd->hgnl", qq, kk) * d ** -0.5
            mag = torch.einsum("nhgd,lhd->hgnl", qq.abs(), kk.abs()) * d ** -0.5
            hide = pos[None] > torch.arange(L - n, L, device=cuda)[:, None]
            s.masked_fill_(hide, float("-inf"))
            p = torch.softmax(s, -1)
            want = torch.einsum("hgnl,lhd->nhgd", p, vvv).reshape(n, hq, d)
            A = torch.einsum("hgnl,lhd->nhgd", p, vvv.abs()).reshape(n, hq, d)
            ds = 2.0 ** -8 * (mag * ~hide).amax(-1) if n else mag.sum(-1)
            rel = (1.05 * (2 * ds + 2.0 ** -8)).permute(2, 0, 1).reshape(n, hq, 1)
            assert_within(out[t:t + n], want, 1.01 * rel * A + 2.0 ** -8 * want.abs(), (step, b))
            # weights: rows' scores err by ds (the queries' rounding)
            model[b, :, :L] = torch.where(pos < L - n, 0.9 * model[b, :, :L], 0.0) \
                + p.sum((1, 2))
            bar = (2 * ds.amax() if n else 0.0) + 1e-4
            gap = (ev.weights[b, :, :L].double() - model[b, :, :L]).abs()
            assert bool((gap <= 1.1 * bar * model[b, :, :L] + 1e-6).all()), (step, b)
            model[b, :, :L] = ev.weights[b, :, :L].double()  # errors do not pile up here
            t += n
        if step % 4 == 3:
            before = model.clone()
            kept = ev.evict()
            c.check()
            for b in range(B):
                if lens[b] > 100:
                    for h in range(H):
                        idx = kept64(before[b, h].tolist(), lens[b], 100, 4, 20)
                        assert kept[b, h].tolist() == idx
                        model[b, h, :100] = before[b, h][torch.tensor(idx, device=cuda)]
            assert [n + e for n, e in zip(m.context_lens.tolist(), m.evicted.tolist())] == seen
            pages_of(m)
    assert max(m.evicted.tolist()) > 200


def test_eviction_of_another_manager(cuda):
    a, b = (SequenceKVManager(PagedKVCache(8, 16, 2, 64), 1, 64) for _ in range(2))
    layer = ChunkedAttention()
    x = torch.zeros((1, 2, 64), dtype=BF16, device=cuda)
    with pytest.raises(ValueError, match="another manager"):
        layer(a, x, x, x, cu_of([1], cuda), eviction=WeightedEviction(b, 16))
    assert a.context_lens.tolist() == [0]


@pytest.mark.parametrize("cache8", [False, True])
def test_weights_without_tokens_and_odd_queries(cuda, cache8):
    """A batch of no tokens decays what was there; queries whose heads share memory (no
    tensor copy takes them) give what copies of them give."""
    P = problem([0, 0], [300, 40], 8, 2, 128, cache8)
    check_weights(P, decay=0.5)
    P = problem([100, 60], [300, 400], 8, 2, 128, cache8)
    lse = lse_of(P)
    P.q = P.q[:, :1].expand(-1, 8, -1)
    w = torch.rand((2, 2, P.tables.shape[1] * 16), device=cuda)
    got, want = (key_weights(q, lse, P.k_cache, P.tables, P.lens, P.cu, w,
                             out=torch.zeros_like(w), **P.more) for q in (P.q, P.q.contiguous()))
    assert torch.allclose(got, want, rtol=2e-5, atol=1e-6)  # two kernels' sums in 32 bits


def test_weights_wait_that_runs_out(cuda):
    """One poll of a wait lasts about 4 us. Each of the 4 * 157 items of 256 keys takes 32
    steps of more than 0.3 us (its products alone), and a CTA has four: its third waits for
    the first one's keys to be done with, which is longer than that."""
    P = problem([1024], [39000], 8, 4, 128)
    lse, w = lse_of(P), torch.rand((1, 4, P.tables.shape[1] * 16), device=cuda)
    args = (P.q, lse, P.k_cache, P.tables, P.lens, P.cu, w)
    want = key_weights(*args, out=torch.zeros_like(w))
    lib = _lib.load()
    try:
        lib.cvsa_set_wait_limit(1)
        key_weights(*args, out=torch.zeros_like(w), dev_error=P.dev_error)
        torch.cuda.synchronize()
    finally:
        lib.cvsa_set_wait_limit(0)
    assert int(P.dev_error.item()) == _lib.DEV_ERR_TIMEOUT
    assert torch.equal(key_weights(*args, out=torch.zeros_like(w)), want)


@pytest.mark.parametrize("cache8", [False, True])
def test_weights_many_short_items(cuda, cache8):
    """Items of one to nine steps in all orders: the groups of warps that share a CTA fall
    behind and catch up with one another."""
    new = [33, 300, 64, 1, 130, 500, 40, 65, 90, 200]
    for reps in (1, 3):
        check_weights(problem(new * reps, [n + 7 * i for i, n in enumerate(new * reps)], 16, 4, 64,
                              cache8, seed=reps))


def test_evict_in_a_graph(cuda):
    """A captured eviction, replayed as the sequences grow; one captured before the counting
    began is refused."""
    m = SequenceKVManager(PagedKVCache(60, 16, 2, 64), 2, 256)
    w = torch.rand((2, 2, 256), device=cuda)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            m.evict(w, 50, 2, 10)
    m.track_evictions()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = m.evict(w, 50, 2, 10)
    assert not m._evict_plan  # the graph's own memory is not kept for other calls
    for step in range(3):
        m.reserve(cu_of([100, 40], cuda))
        lens, w0 = m.context_lens.tolist(), w.clone()
        graph.replay()
        m.cache.check()
        for b in range(2):
            for h in range(2):
                idx = kept64(w0[b, h].tolist(), lens[b], 50, 2, 10) if lens[b] > 50 else [-1] * 50
                assert kept[b, h].tolist() == idx
        pages_of(m)
    assert m.evicted.tolist() == [250, 70]


# ---------------------------------------------------------------------------
# weights of keys that no counted call appended
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n,keep", [(33, 32), (500, 60), (20000, 4096), (131072, 100),
                                    (400000, 30000)])
def test_evict_clears_what_stood_behind(cuda, n, keep):
    """In place, the slots between the kept weights and the old length belong to no key any
    more and are 0; what lies past the length, shorter sequences and other memory stay. Rows
    of one block and of several, and one that shared memory does not hold."""
    c = Cut([n, n // 2 + 1, keep], keep, 2, keep // 10, hkv=1, seed=keep)
    w0 = c.w.clone()
    c.check()
    for s, m in enumerate(c.lens_):
        if m > keep:
            assert not bool(c.w[s, :, keep:m].any())
            assert torch.equal(c.w[s, :, m:], w0[s, :, m:])
        else:
            assert torch.equal(c.w[s], w0[s])
    c = Cut([n, n // 2 + 1, keep], keep, 2, keep // 10, hkv=1, seed=keep)
    out = torch.full((3, 1, keep + 40), 5.0, device=cuda)
    c.run(out)
    assert torch.equal(c.w, w0) and bool((out[..., keep:] == 5).all())


def uniform(layer, m, ev, n, hq, cuda):
    """n tokens whose queries are 0: a token gives each key it sees the same weight."""
    H, d = m.cache.num_kv_heads, m.cache.head_dim
    z = torch.zeros((n, hq, d), dtype=BF16, device=cuda)
    layer(m, z, z[:, :H], z[:, :H], cu_of([n], cuda), eviction=ev)


@pytest.mark.parametrize("how", ["layer", "append", "batch", "token"])
def test_keys_that_were_not_counted_begin_at_zero(cuda, how):
    """After an eviction, keys that come without the counting have no weight: not what the
    keys that had their slots before it left there."""
    H, hq, d, keep = 2, 4, 64, 50
    m = SequenceKVManager(PagedKVCache(40, 16, H, d), 1, 400)
    layer, ev = ChunkedAttention(), WeightedEviction(m, keep, 2, 5)
    g = torch.Generator(device=cuda).manual_seed(3)
    q, k, v = (torch.randn((200, h, d), generator=g, device=cuda).to(BF16) for h in (hq, H, H))
    layer(m, q, k, v, cu_of([200], cuda), eviction=ev)
    assert float(ev.weights[0, :, keep:200].min()) > 0
    ev.evict()
    if how == "layer":
        layer(m, q[:60], k[:60], v[:60], cu_of([60], cuda))
    elif how == "append":
        layer.append(m, q[:60], k[:60], v[:60], cu_of([60], cuda))
    else:
        for i in range(60):
            if how == "batch":
                m.append_batch(k[i:i + 1], v[i:i + 1])
            else:
                m.append_token_kv(0, k[i], v[i])
    assert m.context_lens.tolist() == [110]
    assert not bool(ev.weights[0, :, keep:].any())
    before = ev.weights.double()
    uniform(layer, m, ev, 1, hq, cuda)
    m.cache.check()
    want = before + 0.0
    want[0, :, :111] += (hq // H) / 111.0
    # scores are 0, so a weight errs as the log of a sum of 111 terms does ((111 + 16) 2^-24 and
    # 4 * 4.8 * 2^-24, and 2^-21 for each of two exponentials: below 2^-16), the sum by 2^-23
    tol = 2.0 ** -16 * (hq // H) / 111.0 + 2.0 ** -22 * want
    assert bool(((ev.weights.double() - want).abs() <= tol).all())
    w0, kept = ev.weights[0].cpu(), ev.evict()
    for h in range(H):
        assert kept[0, h].tolist() == kept64(w0[h].tolist(), 111, keep, 2, 5)


@pytest.mark.parametrize("registered", [1, 2])
def test_a_slot_that_is_filled_anew_has_no_weights(cuda, registered):
    """prefill_kv puts another sequence where one gathered weights: its keys begin at 0, the
    other sequences' stay."""
    H, hq, d, keep = 2, 4, 64, 50
    m = SequenceKVManager(PagedKVCache(80, 16, H, d), 3, 200)
    layer, evs = ChunkedAttention(), [WeightedEviction(m, keep) for _ in range(registered)]
    g = torch.Generator(device=cuda).manual_seed(4)
    q, k, v = (torch.randn((270, h, d), generator=g, device=cuda).to(BF16) for h in (hq, H, H))
    for ev in evs:
        layer(m, q, k, v, cu_of([90, 90, 90], cuda), eviction=ev)
    was = [ev.weights.clone() for ev in evs]
    m.prefill_kv(1, k[:120], v[:120])
    for ev, w in zip(evs, was):
        assert not bool(ev.weights[1].any())
        for s in (0, 2):
            assert torch.equal(ev.weights[s], w[s]) and bool(w[s].any())
    ev = evs[0]
    z = torch.zeros((1, hq, d), dtype=BF16, device=cuda)
    layer(m, z, z[:, :H], z[:, :H], cu_of([1], cuda),
          torch.ones(1, dtype=torch.int32, device=cuda), eviction=ev)
    m.cache.check()
    want = torch.zeros_like(ev.weights[1]).double()
    want[:, :121] = (hq // H) / 121.0
    assert bool(((ev.weights[1].double() - want).abs() <= 2.0 ** -16 * want).all())
    evs.clear()
    del ev
    m.prefill_kv(2, k[:10], v[:10])  # nobody counts any more


# ---------------------------------------------------------------------------
# keys that no row sees
# ---------------------------------------------------------------------------
def hidden_pages(P, window, starts=None, causal=True):
    """(table row, page) of the pages that hold keys of a context but none that a row sees."""
    out = []
    for b, (n, c) in enumerate(zip(P.new, P.ctx)):
        first = c - n if starts is None else starts[b]
        lo = max(0, first - window + 1) if window else 0
        hi = (min(c, first + n) if causal else c) if n else 0
        for p in range(-(-c // P.page)):
            if min(c, (p + 1) * P.page) <= lo or p * P.page >= hi:
                out.append((P.rows[b], p))
    return out


@pytest.mark.parametrize("dtype,cache8,d,page", [
    (BF16, False, 128, 16), (BF16, True, 128, 16), (F16, True, 64, 64), (F16, False, 64, 32),
    (F32, False, 128, 16), (BF16, True, 256, 16), (BF16, False, 64, 24)])
@pytest.mark.parametrize("new,kw", [
    ([1, 1, 0], dict(window=16)), ([1, 3, 2], dict(window=40)), ([100, 64, 1], dict(window=33)),
    ([150, 20, 0], dict(window=1)), ([1, 2, 0], dict()), ([4, 0, 90], dict())])
@pytest.mark.parametrize("early", [False, True])
def test_weights_of_pages_nobody_sees(cuda, dtype, cache8, d, page, new, kw, early):
    """Pages behind a window, past the last row's position or of a sequence without new
    tokens are not looked up, as in the attention: table entries out of range there are no
    error, and their keys keep decay times what they had."""
    P = problem(new, [901, 640, 333], 8, 2, d, cache8, dtype=dtype, page=page, seed=d)
    starts = [c - n - 150 for n, c in zip(new, P.ctx)] if early else None
    lse = lse_of(P, starts=starts, **kw)
    hidden = hidden_pages(P, kw.get("window", 0), starts)
    assert hidden
    prior = torch.rand((3, 2, P.tables.shape[1] * page), device=cuda)
    st = None if starts is None else torch.tensor(starts, **I32)
    args = (P.q, lse, P.k_cache, P.tables, P.lens, P.cu, prior)
    form = dict(decay=0.5, start_positions=st, dev_error=P.dev_error, **P.more, **kw)
    want = key_weights(*args, out=torch.full_like(prior, 7.0), **form)
    for i, (r, p) in enumerate(hidden):
        P.tables[r, p] = -1 - i if i % 2 else P.k_cache.shape[0] + i
    got = key_weights(*args, out=torch.full_like(prior, 7.0), **form)
    scales = dict(k_scale=P.k_scale, v_scale=P.v_scale) if cache8 else {}
    chunk_attention(P.q, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, start_positions=st,
                    dev_error=P.dev_error, **scales, **kw)
    torch.cuda.synchronize()
    assert int(P.dev_error.item()) == 0
    assert torch.equal(got, want)
