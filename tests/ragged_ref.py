"""64-bit references and problem builders for the ragged-batch operators
(rope_append, chunk_attention, reserve), shared by their tests."""

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
E32 = 2.0 ** -24


def cu_of(new, device):
    return torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32,
                        device=device)


class Problem:
    """A paged cache whose unused slots hold NaN, with ragged new tokens."""

    def __init__(self, new, ctx, hq, hkv, d, page=16, dtype=torch.bfloat16, kv_dtype=None, seed=0,
                 seq_ids=None, pad_tokens=0, heat=2.0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.new, self.ctx, self.hq, self.hkv, self.d, self.page = new, ctx, hq, hkv, d, page
        kv_dtype = kv_dtype or dtype
        S = len(new) if seq_ids is None else max(seq_ids) + 2
        rows = list(range(len(new))) if seq_ids is None else seq_ids
        self.rows = rows
        W = max(1, max(-(-c // page) for c in ctx)) + 1
        NB = sum(-(-c // page) for c in ctx) + 3
        order = torch.randperm(NB, generator=g)
        tables = torch.full((S, W), -7, dtype=torch.int32)   # never read past a context
        lens = torch.full((S,), 1 << 20, dtype=torch.int32)  # rows no sequence names
        k = torch.full((NB, page, hkv, d), float("nan"))
        v = torch.full((NB, page, hkv, d), float("nan"))
        self.k64, self.v64 = [], []
        at = 0
        for b, (r, c) in enumerate(zip(rows, ctx)):
            n = -(-c // page)
            tables[r, :n] = order[at:at + n].to(torch.int32)
            lens[r] = c
            kk = torch.randn((c, hkv, d), generator=g).to(kv_dtype).float()
            vv = torch.randn((c, hkv, d), generator=g).to(kv_dtype).float()
            for p in range(n):
                m = min(page, c - p * page)
                k[order[at + p], :m] = kk[p * page:p * page + m]
                v[order[at + p], :m] = vv[p * page:p * page + m]
            at += n
            self.k64.append(kk)
            self.v64.append(vv)
        T = sum(new) + pad_tokens
        self.T = T
        self.q = (torch.randn((T, hq, d), generator=g) * heat).to(dtype).to(device)
        self.k_cache, self.v_cache = k.to(kv_dtype).to(device), v.to(kv_dtype).to(device)
        self.tables, self.lens = tables.to(device), lens.to(device)
        self.cu = cu_of(new, device)
        self.seq_ids = None if seq_ids is None else torch.tensor(seq_ids, dtype=torch.int32,
                                                                 device=device)
        self.dev_error = torch.zeros(1, dtype=torch.int32, device=device)

    def slot(self, b, pos):
        return (int(self.tables[self.rows[b], pos // self.page]), pos % self.page)

    def put(self, b, pos, k=None, v=None):
        """Overwrite the key / value row of one position (every head) with a constant."""
        blk, off = self.slot(b, pos)
        if k is not None:
            self.k_cache[blk, off] = k
            self.k64[b][pos] = k
        if v is not None:
            self.v_cache[blk, off] = v
            self.v64[b][pos] = v


def attend64(P, causal=True, window=0, scale=None, weight_u=0.0, starts=None):
    """(out, lse, out_tol, lse_tol), 64 bits, from the definition row by row.

    Tolerances, per element, with A = sum_j p_j |v_j| (the weights' absolute
    moment): a score is a sum of D products accumulated in 32 bits, so its
    error is at most (D + 4) 2^-24 scale sum |q||k| =: ds, plus 2^-21 relative
    for the scaled exponential; weights then err by 2 ds relative, sums of n
    terms by (n + 16) 2^-24; weights rounded to a 16-bit type add weight_u; the
    output is rounded once to its type."""
    scale = P.d ** -0.5 if scale is None else scale
    G = P.hq // P.hkv
    out = torch.zeros((P.T, P.hq, P.d), dtype=torch.float64, device=P.q.device)
    lse = torch.full((P.T, P.hq), float("-inf"), dtype=torch.float64, device=P.q.device)
    otol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    t = 0
    for b, (n, c) in enumerate(zip(P.new, P.ctx)):
        k = P.k64[b].double().to(P.q.device)
        v = P.v64[b].double().to(P.q.device)
        first = c - n if starts is None else starts[b]
        for i in range(n):
            p = first + i
            hi = min(c, p + 1) if causal else c
            lo = max(0, p - window + 1) if window else 0
            if starts is not None and first < 0:
                hi = 0
            if hi <= lo:
                t += 1
                continue
            q = P.q[t].double().view(P.hkv, G, P.d)
            ks, vs = k[lo:hi].permute(1, 0, 2), v[lo:hi].permute(1, 0, 2)
            s = torch.einsum("hgd,hld->hgl", q, ks) * scale
            mag = torch.einsum("hgd,hld->hgl", q.abs(), ks.abs()) * scale
            w = torch.softmax(s, -1)
            o = torch.einsum("hgl,hld->hgd", w, vs)
            A = torch.einsum("hgl,hld->hgd", w, vs.abs())
            ds = ((P.d + 4) * E32 * mag.amax(-1) + 2.0 ** -21 * (1 + s.abs().amax(-1)))
            rel = (2 * ds + (hi - lo + 16) * E32 + weight_u)[..., None]
            out[t] = o.reshape(P.hq, P.d)
            lse[t] = torch.logsumexp(s, -1).reshape(P.hq)
            u = U[P.q.dtype]
            otol[t] = (1.01 * rel * A + u * (o.abs() + rel * A) + 1e-30
                       + (6e-8 if P.q.dtype == torch.float16 else 0.0)).reshape(P.hq, P.d)
            ltol[t] = (ds + (hi - lo + 16) * E32 + 4 * E32 * lse[t].reshape(P.hkv, G).abs()
                       ).reshape(P.hq)
            t += 1
    return out, lse, otol, ltol


def assert_within(got, want, tol, what=""):
    got = got.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN positions differ"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    d = (got[fin] - want[fin]).abs()
    bad = d > tol[fin]
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond tolerance, "
                                 f"worst {float((d / tol[fin].clamp(min=1e-300)).max()):.2f}x")


def rope64(x, pos, table, rot, interleaved, w, eps):
    """Norm and rotation of rows [n, H, D] at positions [n], 64 bits, and the
    magnitude sum |terms| of every element (for tolerances)."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    if table is None:
        return x, x.abs()
    h = rot // 2
    c, s = table[pos, :h].double()[:, None], table[pos, h:].double()[:, None]
    y, mag = x.clone(), x.abs()
    for i in range(h):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + h)
        xa, xb, ci, si = x[..., a], x[..., b], c[..., i], s[..., i]
        y[..., a], y[..., b] = xa * ci - xb * si, xb * ci + xa * si
        mag[..., a] = (xa * ci).abs() + (xb * si).abs()
        mag[..., b] = (xb * ci).abs() + (xa * si).abs()
    return y, mag
