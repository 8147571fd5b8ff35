"""64-bit references and problems of the 8-bit cache, the key weights and the eviction."""

import torch

from ragged_ref import E32, Problem

F8 = torch.float8_e4m3fn
NAN8 = 0x7f


def exponent(amax):
    """The least e in [-15, 7] with amax <= 448 * 2^e (7 beyond)."""
    e = torch.full(amax.shape, -15, dtype=torch.int64, device=amax.device)
    for i in range(-15, 7):
        e = torch.where(amax.double() > 448.0 * 2.0 ** i, i + 1, e)
    return e


def near8(x):
    """x rounded to e4m3, halves to even, saturating; NaN stays."""
    x = x.double()
    e = torch.frexp(x)[1].clamp(min=-5) - 1
    step = torch.ldexp(torch.ones_like(x), e - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def values(cache, scale):
    """What an 8-bit cache holds, in 64 bits."""
    return cache.double() * scale.double()[:, None, :, None]


class Problem8(Problem):
    """A Problem whose cache is of 8 bits: k64 / v64 hold the values it stands for.
    Scales differ from page to page; slots that no sequence uses are NaN."""

    def __init__(self, *a, spread=2.0, **kw):
        super().__init__(*a, **kw)
        g = torch.Generator().manual_seed(kw.get("seed", 0) + 1)
        for name in ("k", "v"):
            x = getattr(self, name + "_cache").float().cpu()
            x = x * (torch.rand((x.shape[0], 1, self.hkv, 1), generator=g) * spread + 0.2)
            e = exponent(torch.nan_to_num(x).abs().amax((1, 3)))
            e = (e + torch.randint(0, 3, e.shape, generator=g)).clamp(max=7)
            scale = 2.0 ** e.double()
            code = near8(x.double() / scale[:, None, :, None])
            val = code * scale[:, None, :, None]
            code8 = code.float().to(F8)
            setattr(self, name + "_cache", code8.to(self.q.device))
            setattr(self, name + "_scale", scale.float().to(self.q.device))
            rows = getattr(self, name + "64")
            for b, (r, c) in enumerate(zip(self.rows, self.ctx)):
                blk = self.tables[r].cpu().long()
                pos = torch.arange(c)
                rows[b] = val[blk[pos // self.page], pos % self.page]

    @property
    def scales(self):
        return dict(k_scale=self.k_scale, v_scale=self.v_scale)

    def put(self, b, pos, k=None, v=None):
        """As Problem.put; the constant is NaN or a value the page's scale holds."""
        blk, off = self.slot(b, pos)
        for name, x in (("k", k), ("v", v)):
            if x is not None:
                scale = getattr(self, name + "_scale")[blk].double().cpu()
                code = near8(torch.full((self.hkv,), float(x), dtype=torch.float64) / scale)
                pool = getattr(self, name + "_cache").view(torch.uint8)
                pool[blk, off] = code.float().to(F8).view(torch.uint8)[:, None].to(pool.device)
                getattr(self, name + "64")[b][pos] = (code * scale)[:, None]


def weights64(P, q, lse, prior, decay=1.0, causal=True, window=0, scale=None, starts=None):
    """(weights, tolerance) [num_seqs, H_kv, capacity] of key_weights, row by row.

    A weight is e^(s - lse); s, a sum of D products in 32 bits, errs by at most
    (D + 4) 2^-24 scale sum |q||k|, the difference by 2^-24 of itself, the
    exponential by 2^-21; the sum of n weights by (n + 8) 2^-24 of itself."""
    scale = P.d ** -0.5 if scale is None else scale
    G = P.hq // P.hkv
    out, tol = prior.double().clone(), torch.zeros(prior.shape, dtype=torch.float64,
                                                   device=prior.device)
    t = 0
    for b, (n, c) in enumerate(zip(P.new, P.ctx)):
        first = c - n if starts is None else starts[b]
        row, k = P.rows[b], P.k64[b].double().to(q.device)
        if starts is not None and first < 0:
            t += n
            continue
        got = torch.zeros((P.hkv, c), dtype=torch.float64, device=q.device)
        err, terms = torch.zeros_like(got), 0
        for i in range(n):
            p = first + i
            hi = min(c, p + 1) if causal else c
            lo = max(0, p - window + 1) if window else 0
            if hi > lo:
                qq = q[t].double().view(P.hkv, G, P.d)
                s = torch.einsum("hgd,lhd->hgl", qq, k[lo:hi]) * scale
                mag = torch.einsum("hgd,lhd->hgl", qq.abs(), k[lo:hi].abs()) * scale
                l = lse[t].double().view(P.hkv, G, 1)
                w = torch.exp(s - l)
                w = torch.where(l == float("-inf"), 0.0, w)
                ds = (P.d + 4) * E32 * mag + 4 * E32 * (s - l).abs() + 2.0 ** -21
                got[:, lo:hi] += w.sum(1)
                err[:, lo:hi] += (w * torch.where(torch.isfinite(ds), ds, 0.0)).sum(1)
                terms += G
            t += 1
        j = torch.arange(c, device=q.device)
        had = torch.where(j < first, decay * prior[row, :, :c].double(), 0.0)
        out[row, :, :c] = had + got
        tol[row, :, :c] = 1.01 * err + (terms + 8) * E32 * (had.abs() + got) + 1e-37
    return out, tol


def kept64(w, n, keep, sink, recent):
    """Kept keys of one head, from its weights' first n."""
    mid = list(range(sink, n - recent))
    rank = {j: (float("-inf") if w[j] != w[j] else float(w[j]), w[j] == w[j]) for j in mid}
    mid.sort(key=lambda j: (-rank[j][0], not rank[j][1], j))
    return sorted(list(range(sink)) + mid[:keep - sink - recent] + list(range(n - recent, n)))
