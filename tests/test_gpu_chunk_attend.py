"""chunk_attention against a 64-bit reference, element by element.

Unused cache slots hold NaN in every problem, so a key that reaches a row it
should not shows. Tolerances are derived in ragged_ref.attend64 from the
kernels' arithmetic (32-bit accumulation; weights rounded to the 16-bit type
where the pool is 16-bit)."""

import pytest
import torch

from cvsa import _lib
from cvsa.kernels.chunk_attend import chunk_attention
from ragged_ref import U, Problem, assert_within, attend64

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def run(P, **kw):
    lse = torch.empty((P.T, P.hq), device=P.q.device)
    out = chunk_attention(P.q, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, seq_ids=P.seq_ids,
                          lse=lse, dev_error=P.dev_error, **kw)
    torch.cuda.synchronize()
    return out, lse


def check(P, **kw):
    out, lse = run(P, **kw)
    u = U[P.k_cache.dtype] if P.k_cache.dtype != F32 else 0.0
    want, wl, otol, ltol = attend64(P, weight_u=u, **kw)
    n = sum(P.new)
    assert_within(out[:n], want[:n], otol[:n], "out")
    assert_within(lse[:n], wl[:n], ltol[:n], "lse")
    assert int(P.dev_error.item()) == 0


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (7, 1)])
def test_ragged_batch(cuda, dtype, d, hq, hkv):
    """Lengths around the tile sizes, one-token and empty sequences together."""
    check(Problem([1, 0, 33, 5, 130, 1, 2, 1], [1, 40, 33, 127, 259, 128, 129, 1000], hq, hkv, d,
                  dtype=dtype, seed=3))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("G", [1, 2, 5, 16, 33, 64])
def test_group_sizes(cuda, dtype, G):
    check(Problem([70, 1], [200, 150], 2 * G, 2, 128, dtype=dtype, seed=G))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page", [1, 16, 24, 64, 256])
def test_page_sizes(cuda, dtype, page):
    check(Problem([40, 3], [301, 77], 8, 4, 64, page=page, dtype=dtype, seed=page))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("window", [1, 2, 17, 128, 130, 5000, 2 ** 31 - 1])
def test_window(cuda, dtype, window):
    check(Problem([150, 1, 20], [700, 400, 20], 8, 2, 128, dtype=dtype, seed=window),
          window=window)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_not_causal(cuda, dtype):
    check(Problem([9, 140, 1], [300, 140, 257], 4, 2, 64, dtype=dtype, seed=1), causal=False)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_without_keys(cuda, dtype):
    """Contexts shorter than the chunk put the first rows before position 0;
    a context of 0 leaves every row empty: 0 and -inf."""
    P = Problem([10, 3, 4], [4, 0, 300], 8, 2, 128, dtype=dtype, seed=2)
    check(P)
    out, lse = run(P)
    assert bool((out[:6] == 0).all()) and bool((lse[:6] == float("-inf")).all())
    assert bool((out[10:13] == 0).all())
    check(P, causal=False)


@pytest.mark.parametrize("dtype,new,ctx,hq,hkv,d", [
    (BF16, [1], [20011], 4, 1, 128), (BF16, [3], [30001], 8, 2, 64), (F16, [40], [9000], 8, 1, 128),
    (F32, [2], [9001], 4, 1, 64), (BF16, [300], [300], 32, 8, 128), (BF16, [1] * 40, [
        17 + 61 * i for i in range(40)], 8, 4, 128)])
def test_split_over_ctas(cuda, dtype, new, ctx, hq, hkv, d):
    """Few items over a long cache: every item is shared by many CTAs and merged."""
    check(Problem(new, ctx, hq, hkv, d, dtype=dtype, seed=9))


def test_many_sequences(cuda):
    """More sequences and groups than the planning round's threads."""
    n = 700
    check(Problem([1 + i % 3 for i in range(n)], [3 + (i * 7) % 50 for i in range(n)], 2, 1, 64,
                  seed=4))
    check(Problem([1 + i % 3 for i in range(n)], [3 + (i * 7) % 50 for i in range(n)], 2, 1, 64,
                  dtype=F32, seed=4))


@pytest.mark.parametrize("q_dtype,kv_dtype", [(BF16, F32), (F32, BF16), (F16, BF16), (BF16, F16)])
def test_mixed_types(cuda, q_dtype, kv_dtype):
    P = Problem([30, 1], [100, 300], 8, 2, 128, dtype=q_dtype, kv_dtype=kv_dtype, seed=6)
    check(P)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_a_row_does_not_see(cuda, dtype, bad):
    """A non-finite value of a late token reaches only the rows at or behind
    it; one that left the window reaches no row; a non-finite key row that no
    row sees reaches none."""
    P = Problem([150], [333], 4, 2, 128, dtype=dtype, seed=7)
    P.put(0, 300, v=bad)
    out, _ = run(P)
    u = U[dtype] if dtype != F32 else 0.0
    want, _, otol, _ = attend64(P, weight_u=u)
    before = 300 - (333 - 150)
    assert_within(out[:before], want[:before], otol[:before], "rows before the value")
    assert not bool(torch.isfinite(out[before:].float()).any())
    P = Problem([150], [333], 4, 2, 128, dtype=dtype, seed=8)
    P.put(0, 100, k=bad, v=bad)
    check(P, window=83)          # the first row, at 183, sees 101 onwards
    P = Problem([20], [333], 4, 2, 128, dtype=dtype, seed=8)
    P.put(0, 332, k=float("nan"))
    out, _ = run(P)
    want, _, otol, _ = attend64(P, weight_u=u)
    assert_within(out[:19], want[:19], otol[:19], "rows before the key")
    assert bool(torch.isnan(out[19].float()).all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_extreme_scores(cuda, dtype):
    """Scores of +-1e4 and more: one key takes all, nothing overflows; equal
    scores of the type's lowest magnitude weigh alike."""
    P = Problem([17, 130], [400, 130], 4, 2, 128, dtype=dtype, seed=11, heat=300.0)
    out, lse = run(P)
    u = U[dtype] if dtype != F32 else 0.0
    want, wl, otol, ltol = attend64(P, weight_u=u)
    assert_within(out, want, otol, "out")
    assert_within(lse, wl, ltol, "lse")
    P = Problem([17], [400], 4, 2, 128, dtype=dtype, seed=12, heat=0.0)
    check(P)
    P = Problem([40, 2], [400, 700], 4, 2, 128, dtype=dtype, seed=13)
    check(P, scale=1e-6)
    check(P, scale=3.0)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rising_maximum(cuda, dtype):
    """Keys that grow along the sequence raise the running maximum every tile."""
    P = Problem([20, 1], [1500, 1500], 4, 1, 64, dtype=dtype, seed=14)
    for b in range(2):
        for pos in range(0, 1500, 37):
            row = P.q[0 if b == 0 else 20, 0].float().cpu()
            row = (row / row.norm() * (pos / 60.0)).to(dtype).float()
            blk, off = P.slot(b, pos)
            P.k_cache[blk, off, 0] = row.to(P.k_cache.dtype).to(P.q.device)
            P.k64[b][pos, 0] = row
    check(P)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides_padding_and_table_rows(cuda, dtype):
    """q as a column range of a projection's output, table rows picked by
    seq_ids, padded tokens left alone, strided pools and output."""
    P = Problem([5, 60, 1], [50, 200, 900], 8, 2, 128, dtype=dtype, seed=15, seq_ids=[4, 0, 2],
                pad_tokens=6)
    wide = torch.zeros((P.T, 13 * 128), dtype=dtype, device=cuda)
    wide[:, 128:9 * 128] = P.q.reshape(P.T, -1)
    P.q = wide[:, 128:9 * 128].view(P.T, 8, 128)
    both = torch.stack([P.k_cache, P.v_cache], 1)    # K and V of a block side by side
    P.k_cache, P.v_cache = both[:, 0], both[:, 1]
    buf = torch.full((P.T, 8, 256), 3.0, dtype=dtype, device=cuda)
    out = buf[:, :, :128]
    chunk_attention(P.q, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, seq_ids=P.seq_ids, out=out,
                    dev_error=P.dev_error)
    torch.cuda.synchronize()
    u = U[dtype] if dtype != F32 else 0.0
    want, _, otol, _ = attend64(P, weight_u=u)
    assert_within(out[:66], want[:66], otol[:66], "out")
    assert bool((buf[66:] == 3).all()) and bool((buf[:, :, 128:] == 3).all())
    assert int(P.dev_error.item()) == 0
    # rows that are not 16-byte aligned are copied
    odd = torch.zeros((P.T, 8, 129), dtype=dtype, device=cuda)
    odd[:, :, 1:] = P.q
    again = chunk_attention(odd[:, :, 1:], P.k_cache, P.v_cache, P.tables, P.lens, P.cu,
                            seq_ids=P.seq_ids)
    assert torch.equal(again[:66], out[:66])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_start_positions(cuda, dtype):
    """start_positions place the tokens; a refused sequence (-1) yields zeros."""
    P = Problem([4, 7, 3], [90, 200, 50], 4, 2, 64, dtype=dtype, seed=16)
    starts = [20, -1, 47]
    out = chunk_attention(P.q, P.k_cache, P.v_cache, P.tables, P.lens, P.cu,
                          start_positions=torch.tensor(starts, dtype=torch.int32, device=cuda))
    u = U[dtype] if dtype != F32 else 0.0
    want, _, otol, _ = attend64(P, weight_u=u, starts=starts)
    assert_within(out, want, otol, "out")
    assert bool((out[4:11] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_deterministic_graph_and_streams(cuda, dtype):
    """Equal bits on every run, in a CUDA graph whose lengths change between
    replays, and on another stream."""
    P = Problem([1, 200, 9], [900, 333, 5000], 8, 2, 128, dtype=dtype, seed=17)
    first, _ = run(P)
    for _ in range(3):
        assert torch.equal(run(P)[0], first)
    s = torch.cuda.Stream()
    out = torch.empty_like(P.q)
    with torch.cuda.stream(s):
        chunk_attention(P.q, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, out=out)
        s.synchronize()
        assert torch.equal(out, first)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            chunk_attention(P.q, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, out=out)
        out.zero_()
        g.replay()
        s.synchronize()
        assert torch.equal(out, first)
        cu2, ctx2 = [0, 30, 31, 210], [500, 20, 4000]
        P.cu.copy_(torch.tensor(cu2, dtype=torch.int32))
        P.lens[:3] = torch.tensor(ctx2, dtype=torch.int32, device=cuda)
        g.replay()
        s.synchronize()
    P.new, P.ctx = [30, 1, 179], ctx2
    P.k64 = [k[:c] if k.shape[0] >= c else k for k, c in zip(P.k64, ctx2)]
    P.v64 = [v[:c] if v.shape[0] >= c else v for v, c in zip(P.v64, ctx2)]
    u = U[dtype] if dtype != F32 else 0.0
    want, _, otol, _ = attend64(P, weight_u=u)
    assert_within(out, want, otol, "replay on other lengths")


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_bad_blocks_are_skipped(cuda, dtype):
    """Table entries past the pool the kernel is told of (allocated memory
    behind a view): their keys are left out and the error word says so."""
    P = Problem([20, 1], [300, 410], 4, 2, 64, dtype=dtype, seed=18)
    nb = P.k_cache.shape[0]
    k = torch.cat([P.k_cache, torch.zeros_like(P.k_cache[:2])])[:nb]
    v = torch.cat([P.v_cache, torch.zeros_like(P.v_cache[:2])])[:nb]
    P.k_cache, P.v_cache = k, v
    P.tables[0, 3], P.tables[1, 11] = nb + 1, -2
    out, _ = run(P)
    assert int(P.dev_error.item()) == _lib.DEV_ERR_BLOCK_RANGE
    # the definition over the remaining keys
    keep = [[p for p in range(300) if p // 16 != 3], [p for p in range(410) if p // 16 != 11]]
    Q = Problem([20, 1], [300 - 16, 410 - 16], 4, 2, 64, dtype=dtype, seed=18)
    Q.q, Q.dev_error = P.q, P.dev_error
    Q.k64 = [P.k64[b][keep[b]] for b in range(2)]
    Q.v64 = [P.v64[b][keep[b]] for b in range(2)]
    u = U[dtype] if dtype != F32 else 0.0
    want, _, otol, _ = attend64(Q, weight_u=u)
    assert_within(out, want, otol, "out")


def test_bad_ragged_arrays_set_the_error_word(cuda):
    """Offsets past the tokens, a table row past the table, a length past the
    table's pages: flagged, the other sequences as if alone."""
    P = Problem([4, 6, 5], [60, 90, 33], 4, 2, 64, seed=19)
    good, _ = run(P)
    ids = torch.tensor([0, 3, 2], dtype=torch.int32, device=cuda)      # 3 rows: row 3 is past
    out = torch.full_like(P.q, 2.0)
    chunk_attention(P.q, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, seq_ids=ids, out=out,
                    dev_error=P.dev_error)
    assert int(P.dev_error.item()) == _lib.DEV_ERR_RAGGED
    assert torch.equal(out[:4], good[:4]) and torch.equal(out[10:], good[10:])
    P.dev_error.zero_()
    cu = P.cu.clone()
    cu[3] = 16                                                          # 15 tokens
    chunk_attention(P.q, P.k_cache, P.v_cache, P.tables, P.lens, cu, out=out,
                    dev_error=P.dev_error)
    assert int(P.dev_error.item()) == _lib.DEV_ERR_RAGGED
    assert torch.equal(out[:10], good[:10])
    P.dev_error.zero_()
    P.tables.clamp_(min=0)                      # whatever the long length reads is a block
    P.lens[1] = 5000
    run(P)
    assert int(P.dev_error.item()) & _lib.DEV_ERR_RAGGED


def test_empty_calls(cuda):
    P = Problem([3], [20], 4, 2, 64, seed=20)
    z = P.q[:0]
    assert chunk_attention(z, P.k_cache, P.v_cache, P.tables, P.lens,
                           torch.zeros(2, dtype=torch.int32, device=cuda)).shape == (0, 4, 64)
    assert chunk_attention(z, P.k_cache, P.v_cache, P.tables, P.lens,
                           torch.zeros(1, dtype=torch.int32, device=cuda)).shape == (0, 4, 64)


def test_long_pool_offsets(cuda):
    """Blocks whose element offset passes 32 bits."""
    page, hkv, d = 256, 8, 128
    nb = (1 << 32) // (page * hkv * d) + 4           # 2^32 elements and more
    k = torch.empty((nb, page, hkv, d), dtype=BF16, device=cuda)
    P = Problem([3, 50], [600, 100], 16, hkv, d, page=page, seed=21)
    n = P.k_cache.shape[0]
    k[nb - n:] = P.k_cache
    # V shares the pool tensor's strides; its blocks are K's blocks here
    k64 = [x.clone() for x in P.k64]
    P.v64 = k64
    P.tables = torch.where(P.tables >= 0, P.tables + (nb - n), P.tables)
    P.k_cache = P.v_cache = k
    check(P)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64)])
def test_mixed_items_in_one_cta(cuda, dtype, d):
    """Items of two, one and small single query tiles, with and without keys,
    follow one another in every CTA's range: far more items than CTAs."""
    new = [(37 * i * i + 11) % 97 for i in range(60)] + [130, 1, 300, 0, 2, 64, 65]
    ctx = [n + (53 * i) % 400 for i, n in enumerate(new)]
    P = Problem(new, ctx, 28, 4, d, dtype=dtype, seed=22)
    check(P)
    check(P, window=100)


@pytest.mark.parametrize("d", [64, 128])
def test_wait_limit_runs_out_and_recovers(cuda, d):
    """One poll a wait (about 4 us): the call ends with CVSA_DEV_ERR_TIMEOUT
    instead of waiting, and the next call with the default limit is as before.
    With thousands of sequences every CTA's plan takes several times a poll, and
    the other warps wait for its first item."""
    P = Problem([1] * 4000, [3 + i % 20 for i in range(4000)], 2, 1, d, seed=23)
    first, _ = run(P)
    assert int(P.dev_error.item()) == 0
    lib = _lib.load()
    lib.cvsa_set_wait_limit(1)
    try:
        run(P)
    finally:
        lib.cvsa_set_wait_limit(0)
    assert int(P.dev_error.item()) == _lib.DEV_ERR_TIMEOUT
    P.dev_error.zero_()
    again, _ = run(P)
    assert torch.equal(again, first) and int(P.dev_error.item()) == 0


def test_graph_survives_a_larger_call(cuda):
    """A captured call's workspace stays its own when a later call on the same
    stream needs a larger one."""
    P = Problem([40, 1], [900, 7000], 8, 2, 64, seed=24)
    Q = Problem([40, 1], [900, 7000], 8, 2, 128, seed=25)
    s, out = torch.cuda.Stream(), torch.empty_like(P.q)
    with torch.cuda.stream(s):
        chunk_attention(P.q, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, out=out)
        s.synchronize()
        want = out.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            chunk_attention(P.q, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, out=out)
        big, _ = run(Q)
        junk = [torch.full((1 << 22,), float("nan"), device=cuda) for _ in range(16)]
        out.zero_()
        g.replay()
        s.synchronize()
        assert torch.equal(out, want)
        assert all(bool(torch.isnan(j).all()) for j in junk)
        assert torch.equal(run(Q)[0], big)
