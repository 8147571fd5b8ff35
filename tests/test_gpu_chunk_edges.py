"""chunk_attention and its layer where a call can go wrong without being refused:
weights far below the largest, rows of refused sequences, calls that are refused
after a reservation, captured and concurrent calls."""

import threading

import pytest
import torch

from cvsa import _lib
from cvsa.kernels.chunk_attend import chunk_attention
from cvsa.kernels.rope_append import rope_table
from cvsa.runtime.chunked import ChunkedAttention
from cvsa.runtime.kv_cache import PagedKVCache, SequenceKVManager
from ragged_ref import E32, U, Problem

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


# ---------------------------------------------------------------------------
# weights far below the largest
# ---------------------------------------------------------------------------

def sink_call(cuda, dtype, n, gap, new=1, d=64, sink=0, steps=None, seqs=1):
    """`new` tokens over n keys of page 16 whose scores are 0, but `gap` bits (log2 of the
    weight) at key `sink`, or as `steps` [n] says. Values: 0 at the sink, else 0.75 to 1.25.
    All is exact in 16 bits up to the gap's own rounding. `seqs` sequences hold the same
    pages. Returns (out, lse, want, want_lse) of the last one, which all others have to equal,
    the definition in 64 bits, and the largest score."""
    bits = torch.zeros(n, dtype=torch.float64)
    bits[sink] = gap
    if steps is not None:
        bits = steps.double()
    q = torch.zeros((seqs * new, 1, d), dtype=dtype, device=cuda)
    q[:, 0, 0] = 1.0
    k = torch.zeros((n, 1, d), dtype=dtype)
    k[:, 0, 0] = bits.to(dtype)               # score = k0 * scale, scale = ln 2
    scale = 0.6931471805599453
    v = 1.0 + (((torch.arange(n)[:, None] * 7 + torch.arange(d) * 3) % 33) - 16) / 64.0
    if steps is None:
        v[sink] = 0.0
    v = v.to(dtype)
    page, blocks = 16, -(-n // 16)
    kc = torch.zeros((blocks * page, 1, d), dtype=dtype)
    vc = torch.zeros((blocks * page, 1, d), dtype=dtype)
    kc[:n], vc[:n, 0] = k, v
    table = torch.arange(blocks, dtype=torch.int32, device=cuda).repeat(seqs, 1)
    lens = torch.full((seqs,), n, dtype=torch.int32, device=cuda)
    cu = torch.arange(seqs + 1, dtype=torch.int32, device=cuda) * new
    lse = torch.empty((seqs * new, 1), device=cuda)
    out = chunk_attention(q, kc.view(blocks, page, 1, d).to(cuda),
                          vc.view(blocks, page, 1, d).to(cuda), table, lens, cu, scale=scale,
                          lse=lse)
    out, lse = out[:, 0].double().view(seqs, new, d), lse[:, 0].double().view(seqs, new)
    s = (k[:, 0, 0].double() * scale).to(cuda)
    v64 = v.double().to(cuda)
    want = torch.stack([torch.softmax(s[:n - new + i + 1], 0) @ v64[:n - new + i + 1]
                        for i in range(new)])
    wl = torch.stack([torch.logsumexp(s[:n - new + i + 1], 0) for i in range(new)])
    return out, lse, want, wl, float(s.abs().max())


def bounds(dtype, want, wl, n, smax, vmax=1.25):
    """A weight is rounded to the 16-bit type: u relative, and in f16, where the row's largest
    weight is held at 2^11 or more and the smallest step is 2^-24, at most 2^-36 of the
    largest a key. The rest as in ragged_ref.attend64 (scores here are one exact product,
    so the exponential's 2^-21 (1 + |s|) and the sums' (n + 16) 2^-24 are left)."""
    u = U[dtype]
    rel = 2 * 2.0 ** -21 * (1 + smax) + (n + 16) * E32 + (u if dtype != F32 else 0.0)
    low = n * 2.0 ** -36 * vmax if dtype == F16 else 0.0
    otol = 1.01 * (rel * want.abs() + low) + u * want.abs() * (1 + rel) + 6e-8
    ltol = 2.0 ** -21 * (1 + smax) + (n + 16) * E32 + 4 * E32 * wl.abs()
    return otol, ltol


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("gap", [17.5, 24.0, 25.125, 27.0])
@pytest.mark.parametrize("n,new,seqs", [(131072, 1, 1), (70001, 150, 1), (65536, 1, 300),
                                        (65536, 150, 150)])
def test_sink_over_a_long_context(cuda, dtype, gap, n, new, seqs):
    """One early key takes nearly all of the weight and has value 0: what is left of the
    output is the many keys whose weights are 2^-gap of the largest. With one sequence the
    keys are shared by many CTAs, with more than there are CTAs one walks them all."""
    if dtype == F32 and seqs > 1:
        n = 8192
    out, lse, want, wl, smax = sink_call(cuda, dtype, n, gap, new=new, seqs=seqs)
    otol, ltol = bounds(dtype, want, wl, n, smax)
    assert bool(((out - want).abs() <= otol).all()), float(((out - want).abs() / otol).max())
    assert bool(((lse - wl).abs() <= ltol).all()), float(((lse - wl).abs() / ltol).max())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d,new", [(64, 1), (128, 40), (128, 150)])
@pytest.mark.parametrize("rise", [0.5, 2.0, 3.75, 4.0, 4.25, 7.75, 8.0, 8.25, 11.0, 20.0])
def test_maximum_rises_by_steps(cuda, dtype, d, new, rise):
    """Every 128 keys the scores rise by `rise` bits: the largest weight before the reference
    maximum follows stays finite in f16, and the earlier keys keep their share."""
    n = 1500
    steps = torch.arange(n) // 128 * rise
    out, lse, want, wl, smax = sink_call(cuda, dtype, n, 0.0, new=new, d=d, steps=steps)
    otol, ltol = bounds(dtype, want, wl, n, smax)
    assert bool(torch.isfinite(out).all())
    assert bool(((out - want).abs() <= otol).all()), float(((out - want).abs() / otol).max())
    assert bool(((lse - wl).abs() <= ltol).all()), float(((lse - wl).abs() / ltol).max())


# ---------------------------------------------------------------------------
# captured and concurrent calls
# ---------------------------------------------------------------------------

def split_problems(n):
    """Calls of different batches whose items are all split over CTAs and merged."""
    return [Problem([1 + 5 * i, 40], [9000 + 700 * i, 3000], 8, 2, 128, seed=40 + i)
            for i in range(n)]


def attend(P, **kw):
    return chunk_attention(P.q, P.k_cache, P.v_cache, P.tables, P.lens, P.cu,
                           dev_error=P.dev_error, **kw)


def test_graphs_of_one_capture_stream_run_at_the_same_time(cuda):
    """torch captures every graph on one stream if told of none: their workspaces differ."""
    problems = split_problems(2)
    want = [attend(P) for P in problems]
    outs = [torch.empty_like(P.q) for P in problems]
    graphs = [torch.cuda.CUDAGraph() for _ in problems]
    for g, P, out in zip(graphs, problems, outs):
        with torch.cuda.graph(g):
            attend(P, out=out)
    streams = [torch.cuda.Stream() for _ in problems]
    torch.cuda.synchronize()
    for _ in range(20):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(5):
                    g.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out, w)
    assert all(int(P.dev_error.item()) == 0 for P in problems)


def test_threads_on_the_default_stream(cuda):
    problems = split_problems(3)
    want = [attend(P) for P in problems]
    wrong, errors = [], []

    def work(P, w):
        try:
            got = [attend(P) for _ in range(40)]
            wrong.extend(not torch.equal(x, w) for x in got)
        except Exception as e:  # noqa: BLE001 - shown by the assertion below
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(problems, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and len(wrong) == 120 and not any(wrong)


# ---------------------------------------------------------------------------
# refused sequences
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F16, 128), (BF16, 256), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("bad", [-1, 5, 1 << 30])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_of_a_bad_table_row_are_zero(cuda, dtype, d, bad, causal):
    """The rows of a sequence whose table row is out of range belong to the caller's output:
    0 and -inf, not what the memory held. The other sequences are as if alone."""
    P = Problem([4, 150, 5, 1], [60, 190, 33, 700], 4, 2, d, dtype=dtype, seed=19)
    good = attend(P, causal=causal)
    for b in range(4):
        ids = torch.arange(4, dtype=torch.int32, device=cuda)
        ids[b] = bad
        out = torch.full_like(P.q, float("nan"))
        lse = torch.full((P.T, P.hq), float("nan"), device=cuda)
        attend(P, causal=causal, seq_ids=ids, out=out, lse=lse)
        lo, hi = P.cu[b].item(), P.cu[b + 1].item()
        assert bool((out[lo:hi] == 0).all()) and bool((lse[lo:hi] == float("-inf")).all())
        rest = torch.cat([torch.arange(lo), torch.arange(hi, P.T)]).to(cuda)
        # a refused sequence moves the cut of the work: equal up to the order of the sums
        far = 2 * U[dtype] if dtype != F32 else 1e-5
        assert float((out[rest].float() - good[rest].float()).abs().max()) <= far * float(
            good.float().abs().max())
        assert bool(torch.isfinite(lse[rest]).all())
        assert int(P.dev_error.item()) == _lib.DEV_ERR_RAGGED
        P.dev_error.zero_()


# ---------------------------------------------------------------------------
# refused calls of a layer
# ---------------------------------------------------------------------------

def layer_state(manager):
    c = manager.cache
    return [t.clone() for t in (manager.context_lens, manager.pages_allocated,
                                manager.block_tables, c.free_head, c.k_cache, c.v_cache)]


def layer_call(cuda, T=21, hq=8, hkv=2, d=128, dtype=BF16):
    q = torch.randn((T, hq, d), device=cuda).to(dtype)
    k, v = (torch.randn((T, hkv, d), device=cuda).to(dtype) for _ in range(2))
    return q, k, v


REFUSED = {  # what is wrong: (layer's settings, changes of the call)
    "dtype of k": ({}, dict(k=lambda q, k, v: k.float())),
    "no such dtype": ({}, dict(q=lambda q, k, v: q.double(), k=lambda q, k, v: k.double(),
                               v=lambda q, k, v: v.double())),
    "tokens of q": ({}, dict(q=lambda q, k, v: q[:-1])),
    "heads of k": ({}, dict(k=lambda q, k, v: k[:, :1], v=lambda q, k, v: v[:, :1])),
    "shape of v": ({}, dict(v=lambda q, k, v: v[:, :, :64])),
    "dimensions": ({}, dict(q=lambda q, k, v: q.flatten(1))),
    "offsets' shape": ({}, dict(cu=lambda cu: cu[None])),
    "table rows' shape": ({}, dict(ids=[0])),
    "more sequences than rows": ({}, dict(cu=lambda cu: torch.cat([cu, cu[-1:].expand(3)]))),
    "norm's width": (dict(q_norm=64, k_norm=64), {}),
    "norm's dtype": (dict(k_norm=F16), {}),
    "eps": (dict(k_norm=BF16, eps=-1.0), {}),
    "rotated width": (dict(table=48), {}),
    "table's dtype": (dict(table=F16), {}),
}
REFUSED_ATTENTION = {  # by the attention that follows the append
    "scale": (dict(scale=-1.0), {}),
    "window": (dict(window=-3), {}),
    "query heads": ({}, dict(q=lambda q, k, v: q[:, :7])),
    "query heads a KV head": ({}, dict(q=lambda q, k, v: q.repeat(1, 17, 1))),
}


@pytest.mark.parametrize("what", list(REFUSED) + list(REFUSED_ATTENTION))
def test_a_refused_layer_call_reserves_nothing(cuda, what):
    """Lengths, tables, pool and cache are as before, so the call can be made again."""
    settings, change = {**REFUSED, **REFUSED_ATTENTION}[what]
    settings = dict(settings)
    table = settings.pop("table", None)
    if table is not None:
        table = rope_table(64, 48, device=cuda) if table == 48 else \
            rope_table(64, 128, device=cuda).to(table)
    for name in ("q_norm", "k_norm"):
        if name in settings:
            w = settings[name]
            settings[name] = torch.ones(64, dtype=BF16, device=cuda) if w == 64 else \
                torch.ones(128, dtype=w, device=cuda)
    layer = ChunkedAttention(cos_sin=table, **settings)
    manager = SequenceKVManager(PagedKVCache(16, 16, 2, 128, device="cuda"), 2, 64)
    q, k, v = layer_call(cuda)
    cu = torch.tensor([0, 18, 21], dtype=torch.int32, device=cuda)
    new = {name: change[name](q, k, v) if name in change else x
           for name, x in (("q", q), ("k", k), ("v", v))}
    cu_bad = change["cu"](cu) if "cu" in change else cu
    ids = torch.tensor(change["ids"], dtype=torch.int32, device=cuda) if "ids" in change else None
    ChunkedAttention()(manager, q, k, v, cu)          # the sequences hold something
    before = layer_state(manager)
    calls = [layer] if what in REFUSED_ATTENTION else [layer, layer.append]
    for call in calls:
        with pytest.raises((ValueError, RuntimeError)):
            call(manager, new["q"], new["k"], new["v"], cu_bad, ids)
        torch.cuda.synchronize()
        for a, b in zip(before, layer_state(manager)):
            assert torch.equal(a, b)
    manager.cache.check()


def test_a_layer_takes_64_bit_offsets_and_rows(cuda):
    """torch's default integers: converted once, for the reservation and for the calls."""
    q, k, v = layer_call(cuda)
    outs, states = [], []
    for dtype in (torch.int32, torch.int64):
        manager = SequenceKVManager(PagedKVCache(16, 16, 2, 128, device="cuda"), 3, 64)
        cu = torch.tensor([0, 18, 21], dtype=dtype, device=cuda)
        ids = torch.tensor([2, 0], dtype=dtype, device=cuda)
        layer = ChunkedAttention(cos_sin=rope_table(64, 128, device=cuda))
        outs.append(layer(manager, q, k, v, cu, ids))
        rotated, starts = layer.append(manager, q, k, v, cu, ids)
        outs.append(rotated)
        assert starts.tolist() == [18, 3]
        states.append(layer_state(manager))
        manager.cache.check()
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
    assert all(torch.equal(a, b) for a, b in zip(*states))


@pytest.mark.parametrize("dtype,pairs", [(BF16, 550), (BF16, 1100), (F32, 600)])
def test_offsets_that_name_all_tokens_again_and_again(cuda, dtype, pairs):
    """Offsets 0, T, 0, T, ...: every second sequence is out of order, the others own all
    tokens, and the work of all of them does not fit the plan's 31 bits. Flagged, nothing
    written; the next call is as ever."""
    T, ctx, hkv, d, page = 8192, 131072, 2, 64, 16
    pool = torch.zeros((ctx // page, page, hkv, d), dtype=dtype, device=cuda)
    q = torch.zeros((1, 64 * hkv, d), dtype=dtype, device=cuda).expand(T, -1, -1)
    tables = torch.arange(ctx // page, dtype=torch.int32, device=cuda)[None]
    lens = torch.tensor([ctx], dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, T] * pairs + [0], dtype=torch.int32, device=cuda)
    ids = torch.zeros(2 * pairs, dtype=torch.int32, device=cuda)
    out = torch.full(q.shape, 3.0, dtype=dtype, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    chunk_attention(q, pool, pool, tables, lens, cu, causal=False, seq_ids=ids, out=out,
                    dev_error=err)
    assert int(err.item()) == _lib.DEV_ERR_RAGGED
    assert bool((out == 3).all())
    P = Problem([3, 140], [700, 300], 8, 2, d, dtype=dtype, seed=50)
    got = attend(P)
    assert int(P.dev_error.item()) == 0 and bool(torch.isfinite(got).all())


def test_reservations_that_ask_for_more_than_31_bits_of_pages(cuda):
    """Offsets 0, n, 0, n, ... over one row: 512 times 2^22 pages, the sum of which passes 31
    bits. Every one is refused; the pool and the row keep their state."""
    cache = PagedKVCache(64, 1, 1, 64, device="cuda")
    manager = SequenceKVManager(cache, 1, 1 << 22)
    cu = torch.tensor([0, 1 << 22] * 512 + [0], dtype=torch.int32, device=cuda)
    ids = torch.zeros(1024, dtype=torch.int32, device=cuda)
    starts = manager.reserve(cu, ids)
    assert starts.tolist() == [-1] * 1024
    assert int(cache.dev_error.item()) == _lib.DEV_ERR_RAGGED | _lib.DEV_ERR_POOL
    assert cache._next_free == 0 and manager.context_lens.tolist() == [0]
    assert manager.pages_allocated.tolist() == [0] and int(manager.block_tables.abs().max()) == 0
