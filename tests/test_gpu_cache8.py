"""The 8-bit cache: the append against 64-bit references, code by code, and the attention
over it, element by element. Slots that nothing uses hold NaN."""

import pytest
import torch

from cache8_ref import F8, NAN8, Problem8, exponent, near8, values
from cvsa import _lib
from cvsa.kernels.chunk_attend import chunk_attention
from cvsa.kernels.rope_append import rope_append, rope_table
from cvsa.runtime.chunked import ChunkedAttention
from cvsa.runtime.kv_cache import PagedKVCache, SequenceKVManager
from ragged_ref import E32, Problem, U, assert_within, attend64, cu_of, rope64

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def check_append(new, ctx, hq=8, hkv=2, d=128, dtype=BF16, page=16, rot=None, interleaved=False,
                 norm=None, seq_ids=None, pad=0, shift=None, size=1.0, seed=0, with_q=True):
    P = Problem8(new, ctx, hq, hkv, d, page=page, dtype=dtype, seed=seed, seq_ids=seq_ids,
                 pad_tokens=pad)
    dev, T = P.q.device, P.T
    g = torch.Generator(device=dev).manual_seed(seed)
    qkv = torch.randn((T, (hq + 2 * hkv) * d), generator=g, device=dev)
    # tokens differ in size, so pages grow their scales
    qkv = (qkv * size * torch.empty((T, 1), device=dev).uniform_(0.3, 4.0, generator=g)).to(dtype)
    q = qkv[:, :hq * d].view(T, hq, d)
    k = qkv[:, hq * d:(hq + hkv) * d].view(T, hkv, d)
    v = qkv[:, (hq + hkv) * d:].view(T, hkv, d)
    rot = d if rot is None else rot
    tab = rope_table(max(ctx) + 50, rot, device=dev)
    wq = wk = None
    if norm is not None:
        wq, wk = (torch.empty(d, device=dev).uniform_(0.5, 1.5, generator=g).to(norm)
                  for _ in range(2))
    S = P.lens.numel()
    turn = None if shift is None else torch.tensor([shift] * S, dtype=torch.int32, device=dev)
    before = {n: getattr(P, n).clone() for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    out = rope_append(q if with_q else None, k, v, P.k_cache, P.v_cache, P.tables, P.lens, P.cu,
                      cos_sin=tab, q_norm=wq if with_q else None, k_norm=wk, eps=1e-5,
                      interleaved=interleaved, seq_ids=P.seq_ids, dev_error=P.dev_error,
                      position_shift=turn, **P.scales)
    torch.cuda.synchronize()
    assert int(P.dev_error.item()) == 0
    # what is expected of each pool: values, tolerances, scales
    rel = (8 + (d + 8 if norm is not None else 0)) * E32
    want = {n: values(before[n + "_cache"], before[n + "_scale"]) for n in "kv"}
    tol = {n: torch.zeros_like(want[n]) for n in "kv"}
    scales = {n: before[n + "_scale"].double().clone() for n in "kv"}
    t = 0
    for b, (n, c) in enumerate(zip(new, ctx)):
        if n == 0:
            continue
        pos = torch.arange(c - n, c, device=dev)
        sl = slice(t, t + n)
        t += n
        at = pos + (shift or 0)
        if with_q:
            y, mag = rope64(q[sl], at, tab, rot, interleaved, wq, 1e-5)
            assert_within(out[sl], y, U[dtype] * (y.abs() + rel * mag) + rel * mag + 2.0 ** -25,
                          f"q of {b}")
        blk = P.tables[P.rows[b]].long()[pos // page]
        for name, (y, mag) in (("k", rope64(k[sl], at, tab, rot, interleaved, wk, 1e-5)),
                               ("v", (v[sl].double(), None))):
            err = torch.zeros_like(y) if mag is None else rel * mag
            got = getattr(P, name + "_scale")
            for p in torch.unique(pos // page).tolist():
                here = pos // page == p
                bk = int(P.tables[P.rows[b], p])
                top = y[here].abs().amax((0, 2))
                slack = err[here].amax((0, 2))
                lo, hi = exponent(top - slack), exponent(top + slack)
                begun = (c - n) - p * page
                if begun > 0:
                    had = exponent(448.0 * before[name + "_scale"][bk])
                    lo, hi = torch.maximum(lo, had), torch.maximum(hi, had)
                e = torch.frexp(got[bk].double())[1] - 1
                assert bool(((e >= lo) & (e <= hi)).all()), (name, b, p)
                scales[name][bk] = got[bk].double()
                if begun > 0:  # the codes in use moved to the new scale
                    old = want[name][bk, :begun]
                    want[name][bk, :begun] = near8(old / got[bk].double()[:, None]) \
                        * got[bk].double()[:, None]
            sc = got[blk].double()[..., None]
            want[name][blk, pos % page] = near8(y / sc) * sc
            # a code is off only where the 32-bit value lies across a border: by a step then
            r = (y / sc).abs()
            near = near8(((y + err) / sc)) != near8((y - err) / sc)
            step = torch.ldexp(torch.ones_like(r), torch.frexp(r)[1].clamp(min=-5) - 4) * sc
            tol[name][blk, pos % page] = torch.where(near, 2.0 * step, 0.0)
    for name in "kv":
        got = values(getattr(P, name + "_cache"), getattr(P, name + "_scale"))
        assert torch.equal(getattr(P, name + "_scale").double(), scales[name])
        assert_within(got, want[name], tol[name], name)
    assert float((tol["v"] != 0).sum()) == 0  # values are exact to the code
    return P


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_types_and_layouts(cuda, dtype, d, interleaved):
    check_append([1, 0, 17, 3, 100], [1, 9, 17, 64, 333], d=d, dtype=dtype,
                 interleaved=interleaved)


@pytest.mark.parametrize("page", [1, 2, 16, 24, 64, 256])
@pytest.mark.parametrize("d", [64, 256])
def test_append_pages(cuda, page, d):
    check_append([40, 1, 33], [301, 77, 65], page=page, d=d, seed=page)


@pytest.mark.parametrize("kw", [
    dict(hq=1, hkv=1), dict(hq=7, hkv=1), dict(hq=40, hkv=8), dict(with_q=False),
    dict(seq_ids=[3, 0, 5, 1], pad=9), dict(norm=BF16), dict(norm=F32, rot=32, interleaved=True),
    dict(shift=37), dict(size=1e-6), dict(size=4e4, dtype=F32), dict(size=1e-3, dtype=F16)])
def test_append_forms(cuda, kw):
    check_append([2, 33, 1, 4], [20, 33, 260, 4], **kw)


@pytest.mark.parametrize("n", [31, 33, 700])
def test_append_many_sequences(cuda, n):
    check_append([(i * 5) % 3 for i in range(n - 1)] + [2], [3 + i % 40 for i in range(n)], hq=2,
                 hkv=1, d=64)


def test_append_token_by_token(cuda):
    """Ten tokens, each twice the one before: the page's scale follows, and every token
    keeps three bits of what it was appended with, a rounding for each time it moved into
    the subnormal numbers."""
    H, d = 2, 64
    c = PagedKVCache(4, 16, H, d, dtype=F8)
    m = SequenceKVManager(c, 1, 32)
    g = torch.Generator(device=cuda).manual_seed(1)
    toks = [torch.randn((1, H, d), generator=g, device=cuda) * 2.0 ** i for i in range(10)]
    for x in toks:
        m.append_batch(x, -x)
    c.check()
    got = values(c.k_cache, c.k_scale)[int(m.block_tables[0, 0]), :10]
    want = torch.cat(toks).double()
    top = c.k_scale[int(m.block_tables[0, 0])].double()
    err = (got - want).abs()
    # the first rounding, and half a subnormal step at each later scale: twice the last's
    bar = want.abs() * 2.0 ** -4 + 3 * 2.0 ** -10 * top[None, :, None]
    assert bool((err <= bar).all())
    assert torch.equal(2.0 ** exponent(want.abs().amax((0, 2))).double(), top)
    v = values(c.v_cache, c.v_scale)[int(m.block_tables[0, 0]), :10]
    assert torch.equal(v, -got)


def test_append_values_without_a_code(cuda):
    """NaN stays NaN, infinities and what passes the largest scale saturate, neither moves
    the scale; zeros get the smallest."""
    P = Problem8([4], [4], 2, 2, 64, dtype=F32)
    k = torch.zeros((4, 2, 64), device=cuda)
    k[0, 0, 0], k[1, 0, 1], k[2, 0, 2], k[3, 0, 3] = float("nan"), float("inf"), -1e30, 3.0
    k[0, 1, 5] = float("-inf")
    v = torch.zeros_like(k)
    rope_append(None, k, v, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, **P.scales)
    blk = int(P.tables[0, 0])
    assert P.k_scale[blk].tolist() == [2.0 ** 7, 2.0 ** -15]
    assert P.v_scale[blk].tolist() == [2.0 ** -15] * 2
    got = values(P.k_cache, P.k_scale)[blk, :4]
    assert got[0, 0, 0] != got[0, 0, 0] and got[1, 0, 1] == 57344 and got[2, 0, 2] == -57344
    assert got[3, 0, 3] == 3.0 and got[0, 1, 5] == -448 * 2.0 ** -15
    got[0, 0, 0] = got[1, 0, 1] = got[2, 0, 2] = got[3, 0, 3] = got[0, 1, 5] = 0
    assert not bool(got.any())


def test_append_skips_what_is_out_of_range(cuda):
    P = Problem8([3, 2, 2], [20, 18, 40], 2, 2, 64)
    before = [t.clone().view(torch.uint8) for t in (P.k_cache, P.v_cache)] + [
        P.k_scale.clone(), P.v_scale.clone()]

    def call(**kw):
        args = dict(tables=P.tables, lens=P.lens, cu=P.cu, ids=None, starts=None, tab=None)
        args.update(kw)
        x = torch.ones((P.T, 2, 64), dtype=BF16, device=cuda)
        q = torch.full((P.T, 2, 64), 7.0, dtype=BF16, device=cuda)
        P.dev_error.zero_()
        out = rope_append(q, x, x, P.k_cache, P.v_cache, args["tables"], args["lens"], args["cu"],
                          cos_sin=args["tab"], seq_ids=args["ids"],
                          start_positions=args["starts"], dev_error=P.dev_error, **P.scales)
        return out, int(P.dev_error.item())

    def unchanged():
        now = [t.view(torch.uint8) for t in (P.k_cache, P.v_cache)] + [P.k_scale, P.v_scale]
        return all(torch.equal(a, b) for a, b in zip(before, now))

    i32 = dict(dtype=torch.int32, device=cuda)
    refused = torch.tensor([-1, -1, -1], **i32)
    out, err = call(starts=refused)
    assert err == 0 and unchanged() and not bool(out.any())
    for ids in ([-1, 50, 3], [3, 3, 1 << 30]):
        out, err = call(ids=torch.tensor(ids, **i32))
        assert err == _lib.DEV_ERR_RAGGED and unchanged() and not bool(out.any())
    for lens in ([1 << 30] * 3, [-5] * 3):
        out, err = call(lens=torch.tensor(lens, **i32))
        assert err == _lib.DEV_ERR_RAGGED and unchanged() and not bool(out.any())
    _, err = call(tables=torch.full_like(P.tables, P.k_cache.shape[0]))
    assert err == _lib.DEV_ERR_BLOCK_RANGE and unchanged()
    _, err = call(tables=torch.full_like(P.tables, -1))
    assert err == _lib.DEV_ERR_BLOCK_RANGE and unchanged()
    _, err = call(tab=rope_table(10, 64, device=cuda))  # no angles for these positions
    assert err == _lib.DEV_ERR_RAGGED and unchanged()
    _, err = call(cu=torch.tensor([0, 3, 1, 1 << 30], **i32))
    assert err & _lib.DEV_ERR_RAGGED


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def run(P, **kw):
    lse = torch.full((P.T, P.hq), 7.0, device=P.q.device)
    out = torch.full_like(P.q, 7.0)
    got = chunk_attention(P.q, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, seq_ids=P.seq_ids,
                          out=out, lse=lse, dev_error=P.dev_error, **P.scales, **kw)
    assert got is out
    torch.cuda.synchronize()
    return out, lse


def check(P, **kw):
    out, lse = run(P, **kw)
    u = U[P.q.dtype] if P.q.dtype != F32 else 0.0  # the weights' rounding
    want, wl, otol, ltol = attend64(P, weight_u=u, **kw)
    n = sum(P.new)
    assert_within(out[:n], want[:n], otol[:n], "out")
    assert_within(lse[:n], wl[:n], ltol[:n], "lse")
    assert bool((out[n:] == 7).all()) and bool((lse[n:] == 7).all())
    assert int(P.dev_error.item()) == 0
    again = run(P, **kw)
    assert torch.equal(again[0].view(torch.uint8), out.view(torch.uint8))  # a fixed order


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (7, 1)])
def test_ragged_batch(cuda, dtype, d, hq, hkv):
    check(Problem8([1, 0, 33, 5, 130, 1, 2, 1], [1, 40, 33, 127, 259, 128, 129, 1000], hq, hkv, d,
                   dtype=dtype, seed=3))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("G", [1, 3, 4, 8, 16, 17])
def test_single_tokens(cuda, dtype, d, G):
    ctx = [1, 2, 15, 16, 17, 31, 33, 64, 100, 129, 555, 2049]
    check(Problem8([1] * len(ctx), ctx, 2 * G, 2, d, dtype=dtype, seed=G))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("G", [1, 2, 5, 16, 33, 64])
@pytest.mark.parametrize("new", [[70, 1], [3, 1], [1, 1]])
def test_group_sizes(cuda, dtype, G, new):
    check(Problem8(new, [200, 150], 2 * G, 2, 128, dtype=dtype, seed=G))


@pytest.mark.parametrize("new", [[40, 3], [1, 2]])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [1, 2, 8, 16, 24, 40, 64, 256])
def test_page_sizes(cuda, page, d, new):
    check(Problem8(new, [301, 77], 8, 4, d, page=page, seed=page))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("window", [1, 2, 17, 128, 130, 5000, 2 ** 31 - 1])
@pytest.mark.parametrize("new", [[150, 1, 20], [1, 2, 1]])
def test_window(cuda, dtype, window, new):
    check(Problem8(new, [700, 400, 20], 8, 2, 128, dtype=dtype, seed=window), window=window)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("new", [[9, 140, 1], [1, 2, 3]])
def test_not_causal(cuda, dtype, new):
    check(Problem8(new, [300, 140, 257], 4, 2, 64, dtype=dtype, seed=1), causal=False)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("new,ctx", [([10, 3, 4], [4, 0, 300]), ([2, 1, 1], [1, 0, 300])])
def test_rows_without_keys(cuda, dtype, new, ctx):
    P = Problem8(new, ctx, 8, 2, 128, dtype=dtype, seed=2)
    check(P)
    out, lse = run(P)
    short = new[0] - ctx[0]
    assert bool((out[:short] == 0).all()) and bool((lse[:short] == float("-inf")).all())
    assert bool((out[new[0]:new[0] + new[1]] == 0).all())
    check(P, causal=False)


@pytest.mark.parametrize("dtype,new,ctx,hq,hkv,d", [
    (BF16, [1], [20011], 4, 1, 128), (BF16, [3], [30001], 8, 2, 64), (F16, [40], [9000], 8, 1, 128),
    (F32, [2], [9001], 4, 1, 64), (BF16, [300], [300], 32, 8, 128), (F16, [1], [131072], 8, 1, 64),
    (BF16, [1] * 40, [17 + 61 * i for i in range(40)], 8, 4, 128)])
def test_split_over_ctas(cuda, dtype, new, ctx, hq, hkv, d):
    check(Problem8(new, ctx, hq, hkv, d, dtype=dtype, seed=9))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_sequences(cuda, dtype):
    n = 700
    check(Problem8([1 + i % 3 for i in range(n)], [3 + (i * 7) % 50 for i in range(n)], 2, 1, 64,
                   dtype=dtype, seed=4))
    check(Problem8([1] * n, [3 + (i * 7) % 50 for i in range(n)], 2, 1, 64, dtype=dtype, seed=5,
                   seq_ids=list(range(n))[::-1], pad_tokens=3))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [150, 2])
def test_values_a_row_does_not_see(cuda, dtype, n):
    nan = float("nan")
    P = Problem8([n], [333], 4, 2, 128, dtype=dtype, seed=7)
    at = 333 - n // 2
    P.put(0, at, v=nan)
    out, _ = run(P)
    want, _, otol, _ = attend64(P, weight_u=U[dtype] if dtype != F32 else 0.0)
    before = at - (333 - n)
    assert_within(out[:before], want[:before], otol[:before], "rows before the value")
    assert bool(torch.isnan(out[before:].float()).all())
    P = Problem8([n], [333], 4, 2, 128, dtype=dtype, seed=8)
    P.put(0, 100, k=nan, v=nan)
    check(P, window=333 - n - 100)  # the first row sees 101 onwards
    P = Problem8([n], [333], 4, 2, 128, dtype=dtype, seed=8)
    P.put(0, 332, k=nan)
    out, _ = run(P)
    want, _, otol, _ = attend64(P, weight_u=U[dtype] if dtype != F32 else 0.0)
    assert_within(out[:n - 1], want[:n - 1], otol[:n - 1], "rows before the key")
    assert bool(torch.isnan(out[n - 1].float()).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("e", [-15, 7])
@pytest.mark.parametrize("new", [[1, 1], [90, 20]])
def test_ends_of_the_scales(cuda, dtype, e, new):
    """Pages of the smallest and the largest scale, with codes from the smallest subnormal
    to 448; queries that bring the scores into range."""
    P = Problem8(new, [100, 333], 8, 2, 128, dtype=dtype, seed=11)
    g = torch.Generator().manual_seed(e)
    for name in ("k", "v"):
        pool = getattr(P, name + "_cache")
        codes = torch.randint(0, 0x7f, pool.shape, generator=g, dtype=torch.uint8)
        codes |= torch.randint(0, 2, pool.shape, generator=g, dtype=torch.uint8) * 0x80
        pool.view(torch.uint8).copy_(codes)
        getattr(P, name + "_scale").fill_(2.0 ** e)
        val = values(pool, getattr(P, name + "_scale")).cpu()
        for b, (r, c) in enumerate(zip(P.rows, P.ctx)):
            pos = torch.arange(c)
            getattr(P, name + "64")[b] = val[P.tables[r].cpu().long()[pos // P.page],
                                             pos % P.page]
    if dtype is F16 and e == -15:
        check(P, scale=2.0 ** 10)
    else:
        P.q = (P.q.float() * 2.0 ** (-e - 6)).to(dtype)
        check(P)


@pytest.mark.parametrize("new", [[1], [2], [100]])
def test_long_tails_of_small_weights(cuda, new):
    """One key takes nearly all the weight and has value 0; thousands of others at 2^-20 of
    it each are the output."""
    P = Problem8(new, [6000], 4, 1, 64, dtype=F16, seed=12)
    P.q.fill_(1.0)
    for b, pos, k, v in [(0, 5, 3.5, 0.0)]:
        blk = P.tables[0].long()[torch.arange(6000) // 16]
        P.k_cache.view(torch.uint8)[blk, torch.arange(6000) % 16] = 0
        P.k64[0].zero_()
        P.put(b, pos, k=k, v=v)
    check(P, scale=14.0 / 3.5 / 64)


def test_other_layouts(cuda):
    """Strided pools (heads outermost in a page), strided queries and outputs."""
    P = Problem8([1, 20, 1], [70, 90, 333], 8, 2, 128, seed=13)
    want, _ = run(P)
    kc, vc = (t.view(torch.uint8).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3).view(F8)
              for t in (P.k_cache, P.v_cache))
    wide = torch.randn((P.T, 12, 160), device=cuda).to(BF16)
    q = wide[:, 2:10, 16:144]
    q.copy_(P.q)
    out = torch.zeros((P.T, 16, 128), dtype=BF16, device=cuda)[:, ::2]
    got = chunk_attention(q, kc, vc, P.tables, P.lens, P.cu, out=out, **P.scales)
    assert torch.equal(got, want)


def test_matches_the_wide_cache(cuda):
    """Over a 16-bit cache that holds the same values, rows and log-sum-exps agree to the
    kernels' own tolerances, and for whole chunks bit by bit."""
    for dtype in (BF16, F16):
        P = Problem8([200, 64], [900, 333], 8, 2, 128, dtype=dtype, seed=14)
        kc, vc = (values(c, s).to(dtype) for c, s in ((P.k_cache, P.k_scale),
                                                      (P.v_cache, P.v_scale)))
        out, lse = run(P)
        l16 = torch.empty_like(lse)
        o16 = chunk_attention(P.q, kc, vc, P.tables, P.lens, P.cu, lse=l16)
        _, _, otol, ltol = attend64(P, weight_u=U[dtype])
        assert_within(out, o16.double(), 2 * otol, "out")
        assert_within(lse, l16.double(), 2 * ltol, "lse")


def test_bad_pages(cuda):
    """Table entries out of range are skipped: their keys count as unseen."""
    for new in ([1], [40]):
        P = Problem8(new, [100], 4, 2, 128, seed=15)
        P.tables[0, 2] = P.k_cache.shape[0]
        P.tables[0, 4] = -1
        out, _ = run(P)
        assert int(P.dev_error.item()) == _lib.DEV_ERR_BLOCK_RANGE
        assert bool(torch.isfinite(out.float()).all())
        k, v = P.k64[0], P.v64[0]
        seen = torch.ones(100, dtype=torch.bool)
        seen[32:48] = seen[64:80] = False
        q = P.q[-1].double().cpu().view(2, 2, 128)
        s = torch.einsum("hgd,lhd->hgl", q, k[seen].double()) * 128 ** -0.5
        want = torch.einsum("hgl,lhd->hgd", torch.softmax(s, -1), v[seen].double()).view(4, 128)
        assert float((out[-1].double().cpu() - want).abs().max()) < 2e-2


def test_graph_replay_with_other_lengths(cuda):
    """A captured layer step on the 8-bit cache, replayed as the sequences grow."""
    H, hq, d = 2, 8, 128
    layer = ChunkedAttention(cos_sin=rope_table(512, d, device=cuda))
    made = []
    for _ in range(2):
        made.append(SequenceKVManager(PagedKVCache(64, 16, H, d, dtype=F8), 3, 256))
    a, b = made
    cu = cu_of([1, 1, 1], cuda)
    g = torch.Generator(device=cuda).manual_seed(3)

    def tokens():
        return tuple(torch.randn((3, h, d), generator=g, device=cuda).to(BF16) for h in (hq, H, H))

    first = tokens()
    for m in made:
        layer(m, *first, cu)
    held = [t.clone() for t in first]
    graph = torch.cuda.CUDAGraph()
    state = [t.clone() for t in (b.block_tables, b.context_lens, b.pages_allocated,
                                 b.cache.free_head)]
    with torch.cuda.graph(graph):
        out = layer(b, *held, cu)
    for t, was in zip((b.block_tables, b.context_lens, b.pages_allocated, b.cache.free_head),
                      state):
        t.copy_(was)
    for _ in range(20):
        now = tokens()
        want = layer(a, *now, cu)
        for t, x in zip(held, now):
            t.copy_(x)
        graph.replay()
        assert torch.equal(out, want)
    assert torch.equal(a.cache.k_scale, b.cache.k_scale)
    assert torch.equal(a.cache.k_cache.view(torch.uint8), b.cache.k_cache.view(torch.uint8))


def test_other_stream(cuda):
    P = Problem8([1, 30], [500, 700], 8, 2, 128, seed=16)
    want, _ = run(P)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [chunk_attention(P.q, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, **P.scales)
               for _ in range(3)]
    s.synchronize()
    assert all(torch.equal(x, want) for x in got)


@pytest.mark.parametrize("chunk", [7, 64, 300])
def test_chunked_layer(cuda, chunk):
    """Prompts in chunks, then single tokens, through ChunkedAttention on an 8-bit cache,
    against 64-bit attention over the values the cache holds at each call."""
    hq, H, d, lens = 8, 2, 64, [300, 45]
    m = SequenceKVManager(PagedKVCache(60, 16, H, d, dtype=F8), 2, 400)
    layer = ChunkedAttention(cos_sin=rope_table(400, d, device=cuda))
    g = torch.Generator(device=cuda).manual_seed(chunk)
    done = [0, 0]
    for step in range(1000):
        new = [min(chunk, n - x) if x < n else int(x < n + 3) for n, x in zip(lens, done)]
        if not any(new):
            break
        T = sum(new)
        q, k, v = (torch.randn((T, h, d), generator=g, device=cuda).to(BF16) for h in (hq, H, H))
        out = layer(m, q, k, v, cu_of(new, cuda))
        done = [a + b for a, b in zip(done, new)]
        assert m.context_lens.tolist() == done
        kv, vv = values(m.cache.k_cache, m.cache.k_scale), values(m.cache.v_cache, m.cache.v_scale)
        tab, t = rope_table(400, d, device=cuda), 0
        for b, (n, c) in enumerate(zip(new, done)):
            pos = torch.arange(c, device=cuda)
            blk = m.block_tables[b].long()[pos // 16]
            kk, vvv = kv[blk, pos % 16], vv[blk, pos % 16]
            qq, _ = rope64(q[t:t + n], torch.arange(c - n, c, device=cuda), tab, d, False, None, 0)
            s = torch.einsum("nhgd,lhd->hgnl", qq.view(n, H, hq // H, d), kk) * d ** -0.5
            mag = torch.einsum("nhgd,lhd->hgnl", qq.view(n, H, hq // H, d).abs(), kk.abs())
            s.masked_fill_(pos[None] > torch.arange(c - n, c, device=cuda)[:, None], float("-inf"))
            w = torch.softmax(s, -1)
            want = torch.einsum("hgnl,lhd->nhgd", w, vvv).reshape(n, hq, d)
            A = torch.einsum("hgnl,lhd->nhgd", w, vvv.abs()).reshape(n, hq, d)
            # queries, weights and outputs are rounded to bf16 (2^-8): scores err by ds
            ds = 2.0 ** -8 * d ** -0.5 * (mag * torch.isfinite(s)).amax(-1)
            rel = (1.05 * (2 * ds + 2.0 ** -8)).permute(2, 0, 1).reshape(n, hq, 1)
            assert_within(out[t:t + n], want, rel * A * 1.01 + 2.0 ** -8 * want.abs(), step)
            t += n
    m.cache.check()


def test_eight_bit_cache_refusals(cuda):
    c = PagedKVCache(4, 16, 2, 64, dtype=F8)
    m = SequenceKVManager(c, 1, 64)
    x = torch.zeros((3, 2, 64), device=cuda)
    with pytest.raises(ValueError, match="8-bit"):
        m.prefill_kv(0, x, x)
    with pytest.raises(ValueError, match="8-bit"):
        c.write_kv(0, 0, x[0], x[0])
    with pytest.raises(ValueError, match="8-bit"):
        c.write_kv_block(0, x, x, 3)
    with pytest.raises(ValueError):
        c.gather_pages(torch.zeros(1, dtype=torch.int32, device=cuda))


@pytest.mark.parametrize("new", [[1, 1], [90, 40]])
def test_graphs_with_pools_of_their_own(cuda, new):
    """Two captured calls replayed at the same time on two streams."""
    problems = [Problem8(new, [9000, 5000], 8, 2, 128, seed=s) for s in (21, 22)]
    want = [run(P)[0] for P in problems]
    graphs, outs = [], []
    for P in problems:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(chunk_attention(P.q, P.k_cache, P.v_cache, P.tables, P.lens, P.cu,
                                        **P.scales))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_wait_that_runs_out(cuda):
    """A wait limit of one poll makes the tensor-core kernel give up: the timeout bit, and the
    next call with the default limit is as before."""
    P = Problem8([200, 64], [900, 333], 8, 2, 128, seed=23)
    want, _ = run(P)
    lib = _lib.load()
    try:
        lib.cvsa_set_wait_limit(1)
        chunk_attention(P.q, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, dev_error=P.dev_error,
                        **P.scales)
        torch.cuda.synchronize()
    finally:
        lib.cvsa_set_wait_limit(0)
    assert int(P.dev_error.item()) == _lib.DEV_ERR_TIMEOUT
    P.dev_error.zero_()
    assert torch.equal(run(P)[0], want) and int(P.dev_error.item()) == 0


def test_mean_of_rows_that_misleads(cuda):
    """The kernel goes by the batch's mean of rows: sequences far from it, and padding that
    no sequence owns, come out the same."""
    check(Problem8([1, 60, 0, 0, 1, 0, 1, 2], [500, 700, 9, 40, 333, 0, 17, 2000], 8, 2, 128,
                   seed=24))
    check(Problem8([1, 2], [500, 700], 8, 2, 128, seed=25, pad_tokens=500))
    check(Problem8([0, 0, 1], [500, 700, 300], 8, 2, 64, seed=26))


@pytest.mark.parametrize("page", [16, 64, 256])
def test_append_in_the_middle(cuda, page):
    """Tokens written over some in the middle of a sequence: those before and behind them on
    their pages keep their values, moved to the pages' new scales."""
    n, c, start = 37, 300, 101
    P = Problem8([n], [c], 4, 2, 64, page=page, seed=30)
    P.k_scale.fill_(2.0 ** -6), P.v_scale.fill_(2.0 ** -6)
    old = {x: values(getattr(P, x + "_cache"), getattr(P, x + "_scale")) for x in "kv"}
    g = torch.Generator(device="cuda").manual_seed(31)
    k, v = (torch.randn((n, 2, 64), generator=g, device="cuda") * 100 for _ in range(2))
    rope_append(None, k, v, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, dev_error=P.dev_error,
                start_positions=torch.tensor([start], dtype=torch.int32, device="cuda"),
                **P.scales)
    assert int(P.dev_error.item()) == 0
    for x, new in (("k", k), ("v", v)):
        pool, scale = getattr(P, x + "_cache"), getattr(P, x + "_scale").double()
        got = values(pool, getattr(P, x + "_scale"))
        for pos in range(c):
            blk, off = P.slot(0, pos)
            sc = scale[blk][:, None]
            if start <= pos < start + n:
                want = new[pos - start].double()
                assert bool((sc > 2.0 ** -6).all())
            else:
                want = old[x][blk, off]
            assert torch.equal(got[blk, off], near8(want / sc) * sc), (x, pos)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_shift_of_a_wider_cache(cuda, dtype):
    """position_shift with pools of the tokens' own type: each sequence turns by its own."""
    new, ctx, shift, d = [3, 1, 20], [50, 9, 20], [7, 0, 1000], 64
    P = Problem(new, ctx, 4, 2, d, dtype=dtype, seed=33)
    g = torch.Generator(device="cuda").manual_seed(34)
    q, k, v = (torch.randn((P.T, h, d), generator=g, device="cuda").to(dtype) for h in (4, 2, 2))
    tab = rope_table(1100, d, device="cuda")
    out = rope_append(q, k, v, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, cos_sin=tab,
                      dev_error=P.dev_error, position_shift=torch.tensor(
                          shift, dtype=torch.int32, device="cuda")[:P.lens.numel()])
    assert int(P.dev_error.item()) == 0
    t = 0
    for b, (n, c, s) in enumerate(zip(new, ctx, shift)):
        at = torch.arange(c - n, c, device="cuda") + s
        for got, x in ((out[t:t + n], q), (None, k)):
            y, mag = rope64(x[t:t + n], at, tab, d, False, None, 1e-5)
            if got is None:
                got = torch.stack([P.k_cache[P.slot(b, p)] for p in range(c - n, c)])
            assert_within(got, y, U[dtype] * (y.abs() + 8 * E32 * mag) + 8 * E32 * mag + 2.0 ** -25,
                          f"{b}")
        assert all(torch.equal(P.v_cache[P.slot(b, c - n + i)], v[t + i]) for i in range(n))
        t += n
    P.dev_error.zero_()  # past the table of turns: the token is skipped
    rope_append(q, k, v, P.k_cache, P.v_cache, P.tables, P.lens, P.cu, cos_sin=tab,
                dev_error=P.dev_error, out=out, position_shift=torch.full_like(P.lens, 2 ** 31 - 1))
    assert int(P.dev_error.item()) == _lib.DEV_ERR_RAGGED and float(out.abs().max()) == 0.0


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (8, 2, 64), (2, 2, 128), (40, 8, 64)])
def test_items_with_and_without_a_second_tile(cuda, hq, hkv, d):
    """Items of one tile of query rows before items of two: the warps of the second tile
    have nothing to do in the former and must not run ahead of the latter's queries."""
    G = hq // hkv
    new = [max(1, n // G) for n in [70, 100, 222, 90, 250, 120, 256, 66, 80, 70, 240] * 6]
    P = Problem8(new, [n + 300 + 37 * (i % 9) for i, n in enumerate(new)], hq, hkv, d, seed=41)
    first, _ = run(P)
    check(P)
    for _ in range(20):
        assert torch.equal(run(P)[0], first)
