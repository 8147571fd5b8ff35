"""rope_append and reserve against 64-bit references.

rope_append computes in 32 bits and rounds once, so an element's error is at
most u |y| + 8 * 2^-24 * (sum of the magnitudes of its terms), u the output
type's unit roundoff; with a norm, another (D + 8) * 2^-24 relative."""

import pytest
import torch

from cvsa import _lib
from cvsa.kernels.rope_append import rope_append, rope_table
from cvsa.runtime.kv_cache import PagedKVCache, SequenceKVManager
from ragged_ref import E32, U, Problem, assert_within, cu_of, rope64

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def tol_of(y, mag, dtype, D, norm):
    rel = (8 + (D + 8 if norm else 0)) * E32
    tiny = {F16: 2.0 ** -25, BF16: 1e-38, F32: 1e-38}[dtype]
    return U[dtype] * (y.abs() + rel * mag) + rel * mag + tiny


def check(new, ctx, hq, hkv, d, dtype, kv_dtype=None, rot=None, interleaved=False, norm=None,
          page=16, seq_ids=None, pad=0, inplace=False, fused=True, table=True, with_q=True, seed=0):
    P = Problem(new, ctx, hq, hkv, d, page=page, dtype=dtype, kv_dtype=kv_dtype, seed=seed,
                seq_ids=seq_ids, pad_tokens=pad)
    dev, T = P.q.device, P.T
    g = torch.Generator(device=dev).manual_seed(seed)
    if fused:
        qkv = torch.randn((T, (hq + 2 * hkv) * d), generator=g, device=dev).to(dtype)
        q = qkv[:, :hq * d].view(T, hq, d)
        k = qkv[:, hq * d:(hq + hkv) * d].view(T, hkv, d)
        v = qkv[:, (hq + hkv) * d:].view(T, hkv, d)
    else:
        q, k, v = (torch.randn((T, h, d), generator=g, device=dev).to(dtype)
                   for h in (hq, hkv, hkv))
    rot = d if rot is None else rot
    tab = rope_table(max(ctx) + 1, rot, device=dev) if table else None
    wq = wk = None
    if norm is not None:
        wq, wk = (torch.empty(d, device=dev).uniform_(0.5, 1.5, generator=g).to(norm)
                  for _ in range(2))
    kc0, vc0 = P.k_cache.clone(), P.v_cache.clone()
    q0 = q.clone()
    out = rope_append(q if with_q else None, k, v, P.k_cache, P.v_cache, P.tables, P.lens, P.cu,
                      cos_sin=tab, q_norm=wq if with_q else None, k_norm=wk, eps=1e-5,
                      interleaved=interleaved, seq_ids=P.seq_ids, out=q if inplace else None,
                      dev_error=P.dev_error)
    torch.cuda.synchronize()
    assert int(P.dev_error.item()) == 0
    kvt = kv_dtype or dtype
    kc, vc = kc0.double(), vc0.double()
    ktol = torch.zeros_like(kc)
    t = 0
    for b, (n, c) in enumerate(zip(new, ctx)):
        if n == 0:
            continue
        pos = torch.arange(c - n, c, device=dev)
        sl = slice(t, t + n)
        if with_q:
            y, mag = rope64(q0[sl], pos, tab, rot, interleaved, wq, 1e-5)
            assert_within(out[sl], y, tol_of(y, mag, dtype, d, norm is not None), f"q of {b}")
        y, mag = rope64(k[sl], pos, tab, rot, interleaved, wk, 1e-5)
        blk = P.tables[P.rows[b]].long()[pos // page]
        kc[blk, pos % page] = y
        ktol[blk, pos % page] = tol_of(y, mag, kvt, d, norm is not None)
        vc[blk, pos % page] = v[sl].double()
        t += n
    assert_within(P.k_cache, kc, ktol, "keys")                # NaN where nothing was written
    assert_within(P.v_cache, vc, U[kvt] * vc.abs().nan_to_num() + 2.0 ** -25, "values")
    if not with_q:
        assert out is None


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("interleaved", [False, True])
def test_types_and_layouts(cuda, dtype, d, interleaved):
    check([1, 0, 17, 3, 100], [1, 9, 17, 64, 333], 8, 2, d, dtype, interleaved=interleaved)


@pytest.mark.parametrize("dtype,norm", [(BF16, BF16), (BF16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("d,rot", [(128, 128), (128, 32), (64, 32), (256, 96)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norms_and_partial_rotation(cuda, dtype, norm, d, rot, interleaved):
    check([5, 40, 1], [5, 60, 900], 10, 2, d, dtype, rot=rot, norm=norm, interleaved=interleaved)


@pytest.mark.parametrize("kw", [
    dict(hq=1, hkv=1), dict(hq=7, hkv=1), dict(hq=64, hkv=8), dict(hq=8, hkv=2, page=1),
    dict(hq=8, hkv=2, page=24), dict(hq=8, hkv=2, page=256), dict(hq=8, hkv=2, inplace=True),
    dict(hq=8, hkv=2, inplace=True, fused=False), dict(hq=8, hkv=2, table=False),
    dict(hq=8, hkv=2, table=False, norm=BF16), dict(hq=8, hkv=2, with_q=False),
    dict(hq=8, hkv=2, seq_ids=[3, 0, 5, 1], pad=9), dict(hq=8, hkv=2, kv_dtype=F32),
    dict(hq=8, hkv=2, kv_dtype=F16)])
def test_forms(cuda, kw):
    kw = dict(kw)
    hq, hkv = kw.pop("hq"), kw.pop("hkv")
    check([2, 33, 1, 4], [20, 33, 260, 4], hq, hkv, 128, BF16, **kw)


@pytest.mark.parametrize("n", [1, 31, 32, 33, 1000, 1025])
def test_many_sequences(cuda, n):
    """The token's sequence is found by 32-way probes: batches around their powers."""
    check([(i * 5) % 3 for i in range(n - 1)] + [2], [3 + i % 40 for i in range(n)], 2, 1, 64, BF16)


def test_long_positions(cuda):
    """Position 131071: the table's angles are formed in 64 bits."""
    tab = rope_table(131072, 128, device=cuda)
    ang = 131071.0 * 10000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    want = torch.cat([ang.cos(), ang.sin()])
    assert (tab[131071].double().cpu() - want).abs().max() < 1e-7
    check([3], [131072], 4, 1, 128, BF16)


def test_skipped_tokens(cuda):
    """Refused sequences, positions past the table of cosines or before 0:
    query rows 0, nothing written, padded tokens untouched."""
    P = Problem([4, 5, 6], [30, 20, 40], 4, 2, 64, seed=1, pad_tokens=2)
    q = torch.randn((17, 4, 64), device=cuda).to(BF16)
    k = torch.randn((17, 2, 64), device=cuda).to(BF16)
    before = P.k_cache.clone()
    starts = torch.tensor([26, -1, 34], dtype=torch.int32, device=cuda)
    out = torch.full_like(q, 5.0)
    tab = rope_table(38, 64, device=cuda)                       # positions 38, 39 are past it
    rope_append(q, k, k, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, cos_sin=tab,
                start_positions=starts, out=out, dev_error=P.dev_error)
    assert int(P.dev_error.item()) == _lib.DEV_ERR_RAGGED
    assert bool((out[4:9] == 0).all()) and bool((out[13:15] == 0).all())
    assert bool((out[15:] == 5).all())
    assert bool((out[:4] != 5).any()) and bool((out[9:13] != 0).any())
    for b, pos in ((1, 15), (1, 19), (2, 38), (2, 39)):
        blk, off = P.slot(b, pos)
        assert torch.equal(P.k_cache[blk, off], before[blk, off])
    P.dev_error.zero_()
    P.tables[0, 1] = 1 << 20
    rope_append(q, k, k, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, dev_error=P.dev_error)
    assert int(P.dev_error.item()) == _lib.DEV_ERR_BLOCK_RANGE
    assert torch.equal(rope_append(q[:0], k[:0], k[:0], P.k_cache, P.v_cache, P.tables, P.lens,
                                   P.cu[:1]), q[:0])


# ---------------------------------------------------------------------------
# reserve
# ---------------------------------------------------------------------------

def reserve_ref(tables, lens, pages, free, head, cu, ids, bs):
    """Sequential restatement on host lists; returns starts and the new head."""
    W, starts, refused_pool = tables.shape[1], [], False
    for b in range(len(cu) - 1):
        n, s = cu[b + 1] - cu[b], ids[b]
        end = lens[s] + n
        if end > W * bs:
            starts.append(-1)
            continue
        first = max(pages[s], -(-lens[s] // bs))
        need = max(0, -(-end // bs) - first)
        if need and (refused_pool or head + need > len(free)):
            refused_pool = True
            starts.append(-1)
            continue
        for i in range(need):
            tables[s, first + i] = free[head + i]
        head += need
        if need:
            pages[s] = first + need
        starts.append(int(lens[s]))
        lens[s] = end
    return starts, head


@pytest.mark.parametrize("n,bs,pool", [(5, 16, 400), (5, 16, 20), (40, 4, 3000), (1500, 16, 9000),
                                       (1500, 16, 2500)])
def test_reserve_matches_sequential(cuda, n, bs, pool):
    g = torch.Generator().manual_seed(n + pool)
    free = torch.randperm(pool, generator=g).to(torch.int32)
    cache = PagedKVCache(pool, bs, 1, 64, device="cuda", free_list=free)
    mgr = SequenceKVManager(cache, n + 3, 40 * bs)
    tables, lens = mgr.block_tables.cpu().clone(), [0] * (n + 3)
    pages, head, errors = [0] * (n + 3), 0, False
    for step in range(4):
        counts = torch.randint(0, (3 if step else 7) * bs, (n,), generator=g).tolist()
        ids = torch.randperm(n + 3, generator=g)[:n].to(torch.int32)
        cu = cu_of(counts, "cpu")
        starts = mgr.reserve(cu.to(cuda), ids.to(cuda))
        want, head = reserve_ref(tables, lens, pages, free.tolist(), head, cu.tolist(),
                                 ids.tolist(), bs)
        errors = errors or -1 in want
        assert starts.tolist() == want
        assert mgr.context_lens.tolist() == lens and mgr.pages_allocated.tolist() == pages
        assert cache._next_free == head
        assert torch.equal(mgr.block_tables.cpu(), tables)
    assert (int(cache.dev_error.item()) != 0) == errors
    if errors:
        with pytest.raises((AssertionError, ValueError)):
            cache.check()


def test_reserve_table_full_and_bad_rows(cuda):
    cache = PagedKVCache(32, 16, 1, 64, device="cuda")
    mgr = SequenceKVManager(cache, 3, 64)
    starts = mgr.reserve(cu_of([65, 64, 0], cuda))
    assert starts.tolist() == [-1, 0, 0] and mgr.context_lens.tolist() == [0, 64, 0]
    assert int(cache.dev_error.item()) == _lib.DEV_ERR_TABLE_FULL
    cache.dev_error.zero_()
    ids = torch.tensor([0, 3], dtype=torch.int32, device=cuda)
    assert mgr.reserve(cu_of([1, 1], cuda), ids).tolist() == [0, -1]
    assert int(cache.dev_error.item()) == _lib.DEV_ERR_RAGGED


def test_reserve_then_append_batch(cuda):
    """The batched reservation and the single-token append share one state."""
    cache = PagedKVCache(64, 16, 2, 64, device="cuda")
    mgr = SequenceKVManager(cache, 2, 256)
    cu = cu_of([15, 33], cuda)
    x = torch.randn((48, 2, 64), device=cuda).to(BF16)
    starts = mgr.reserve(cu)
    rope_append(None, x, x, cache.k_cache, cache.v_cache, mgr.block_tables, mgr.context_lens, cu,
                start_positions=starts, dev_error=cache.dev_error)
    y = torch.randn((3, 2, 2, 64), device=cuda).to(BF16)
    for i in range(3):
        mgr.append_batch(y[i], y[i])
    cache.check()
    assert mgr.context_lens.tolist() == [18, 36] and mgr._pages_allocated == [2, 3]
    for b, (lo, hi) in enumerate(((0, 15), (15, 48))):
        k, v = cache.gather_pages(mgr.block_tables[b, :3 if b else 2])
        n = hi - lo
        assert torch.equal(k[:n], x[lo:hi]) and torch.equal(v[n:n + 3], y[:, b])
