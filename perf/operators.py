"""Performance cases of the operators that bring new tokens into the paged cache.

Two operators over one ragged batch of new tokens (sequence b owns rows
cu[b]..cu[b+1] of the packed token arrays, its keys live in the pages its block
table lists):

- `append`: the norm of every query and key row (optional), the rotation by
  the token's position, the rotated queries out, the keys and values into
  their pages (`cvsa.kernels.rope_append`);
- `attend`: attention of the new tokens over everything their sequences have
  cached, causal, optionally over a sliding window (`cvsa.kernels.chunk_attend`).

`run` computes them in plain torch operations in 32 bits, or, with `own` set,
through the package. Lengths come from the case alone (its `mix` seeds
them), values and the pages' order from the seed.
"""

import math
import os
import random
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_PKG = "coverage-verified-sparse-attention_b200"


def _case(name, op, dtype, hq, hkv, d, page, seqs, new, ctx, **more):
    c = dict(name=name, op=op, dtype=dtype, hq=hq, hkv=hkv, d=d, page=page, seqs=seqs,
             new_lo=new[0], new_hi=new[1], ctx_lo=ctx[0], ctx_hi=ctx[1], mix=1, window=0,
             norm=False, interleaved=False, rot=d)
    c.update(more)
    return c


def listed():
    return [
        # attention: a short follow-up question in a short chat; a call of this size is all latency
        _case("attend 17 new at 300", "attend", "bf16", 32, 8, 128, 16, 1, (17, 17), (300, 300)),
        # one token for each sequence of a batch, ragged contexts up to 8K: the serving form
        _case("attend 32x1 ragged 8K", "attend", "bf16", 32, 8, 128, 16, 32, (1, 1), (1024, 8192)),
        # a few drafted tokens verified per sequence (8 to 40 query rows a KV head)
        _case("attend 8x(2-8) at 8K-16K", "attend", "bf16", 32, 8, 128, 16, 8, (2, 8),
              (8192, 16384)),
        # a whole prompt from nothing, one sequence
        _case("attend prompt 4096", "attend", "bf16", 32, 8, 128, 16, 1, (4096, 4096),
              (4096, 4096)),
        # a prompt's chunk far into a long document, 64 query heads
        _case("attend 1024 at 32K, 64 heads", "attend", "bf16", 64, 8, 128, 16, 1, (1024, 1024),
              (32768, 32768)),
        # the last chunk of a 128K document
        _case("attend 509 at 128K", "attend", "bf16", 32, 8, 128, 16, 1, (509, 509),
              (131072, 131072)),
        # chunks of several prompts in one call, odd lengths, 7 query heads a KV head
        _case("attend 6 odd chunks f16 G7", "attend", "f16", 28, 4, 128, 16, 6, (1, 700),
              (701, 5001), mix=3),
        # sliding window, 64-wide heads, pages of 64
        _case("attend window 1000, D 64", "attend", "f16", 16, 4, 64, 64, 3, (300, 1100),
              (1100, 9000), window=1000, mix=2),
        # 32-bit cache (the accuracy configuration)
        _case("attend 250 at 4096 f32", "attend", "f32", 8, 2, 64, 16, 1, (250, 250), (4096, 4096)),
        # one token of 32 sequences into the cache, once a layer and step
        _case("append 32x1", "append", "bf16", 32, 8, 128, 16, 32, (1, 1), (100, 2048)),
        # a whole prompt's keys and values into the cache
        _case("append prompt 8192", "append", "bf16", 32, 8, 128, 16, 1, (8192, 8192),
              (8192, 8192)),
        # ragged chunks with query and key norms, half of each head rotated in neighbouring pairs
        _case("append 9 odd chunks, norms", "append", "f16", 40, 8, 128, 16, 9, (1, 900),
              (900, 1900), norm=True, interleaved=True, rot=64, mix=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"]) if op == "append" else \
        rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"])
    d = rng.choice([64, 128, 128])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 4, 5, 7, 8])
    page = rng.choice([16, 16, 16, 64])
    while True:
        seqs = _log(rng, 1, 64)
        new_hi = _log(rng, 1, 8192)
        new_lo = new_hi if rng.random() < 0.3 else rng.randint(1, new_hi)
        if op == "append":
            ctx_lo = new_hi
            ctx_hi = new_hi + _log(rng, 1, 1024)
            if seqs * new_hi * (hq + 2 * hkv) * d <= 8192 * 48 * 128:
                break
        else:
            ctx_lo = max(new_hi, _log(rng, 16, 131072))
            ctx_hi = min(131072, ctx_lo * rng.choice([1, 2, 4]))
            rows = seqs * hq * new_hi * ctx_hi
            cap = 2 ** 31 if dtype != "f32" else 2 ** 29
            if rows <= cap and rows * d * 4 <= 1.0e12 and seqs * ctx_hi * hkv * d <= 2 ** 29:
                break
    window = _log(rng, 16, 4096) if op == "attend" and rng.random() < 0.25 else 0
    c = _case("", op, dtype, hq, hkv, d, page, seqs, (new_lo, new_hi), (ctx_lo, ctx_hi),
              mix=rng.randrange(1 << 20), window=window, norm=op == "append" and rng.random() < 0.5,
              interleaved=rng.random() < 0.5, rot=rng.choice([d, d, d // 2]))
    del c["name"]
    return c


def _lengths(c):
    """(new tokens, context length with them) of each sequence."""
    r = random.Random(c["mix"])
    new = [r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["seqs"])]
    ctx = [max(n, r.randint(c["ctx_lo"], c["ctx_hi"])) for n in new]
    return new, ctx


def prepare(case, seed):
    c = case
    dev, dt = torch.device("cuda"), _DT[c["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    new, ctx = _lengths(c)
    page, width = c["page"], max(-(-x // c["page"]) for x in ctx)
    blocks = sum(-(-x // page) for x in ctx)
    T, hq, hkv, d = sum(new), c["hq"], c["hkv"], c["d"]
    order = torch.randperm(blocks, generator=g, device=dev).to(torch.int32)
    tables = torch.zeros((c["seqs"], width), dtype=torch.int32, device=dev)
    at = 0
    for b, x in enumerate(ctx):
        n = -(-x // page)
        tables[b, :n] = order[at:at + n]
        at += n
    shape = (blocks, page, hkv, d)
    k_cache = torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dt)
    v_cache = torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dt)
    lens = torch.tensor(ctx, dtype=torch.int32, device=dev)
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=dev)
    s = dict(case=c, k_cache=k_cache, v_cache=v_cache, tables=tables, lens=lens, cu=cu,
             max_new=max(new), max_ctx=max(ctx))
    if c["op"] == "attend":
        # slots past a context hold whatever was there: NaN here
        for b, x in enumerate(ctx):
            if x % page:
                k_cache[tables[b, x // page].long(), x % page:] = float("nan")
                v_cache[tables[b, x // page].long(), x % page:] = float("nan")
        # logits spread like trained heads': some rows look at a few keys, some at many
        heat = torch.empty((1, hq, 1), device=dev).uniform_(0.5, 2.5, generator=g)
        s["q"] = (torch.randn((T, hq, d), generator=g, device=dev) * heat).to(dt)
    else:
        # one projection's output: q, k and v are its column ranges
        qkv = torch.randn((T, (hq + 2 * hkv) * d), generator=g, device=dev).to(dt)
        s["q"] = qkv[:, :hq * d].view(T, hq, d)
        s["k"] = qkv[:, hq * d:(hq + hkv) * d].view(T, hkv, d)
        s["v"] = qkv[:, (hq + hkv) * d:].view(T, hkv, d)
        rot = c["rot"]
        freq = 10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
        ang = torch.arange(max(ctx), device=dev, dtype=torch.float64)[:, None] * freq
        s["cos_sin"] = torch.cat([ang.cos(), ang.sin()], 1).float().contiguous()
        if c["norm"]:
            s["q_norm"] = torch.empty(d, device=dev).uniform_(0.5, 1.5, generator=g).to(dt)
            s["k_norm"] = torch.empty(d, device=dev).uniform_(0.5, 1.5, generator=g).to(dt)
    return s


_mod = {}


def _package():
    if not _mod:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), _PKG)
        if root not in sys.path:
            sys.path.insert(0, root)
        from cvsa.kernels.chunk_attend import chunk_attention
        from cvsa.kernels.rope_append import rope_append
        _mod["attend"], _mod["append"] = chunk_attention, rope_append
    return _mod


def run(state):
    s, c = state, state["case"]
    if own:
        if c["op"] == "attend":
            return {"out": _package()["attend"](s["q"], s["k_cache"], s["v_cache"], s["tables"],
                                                s["lens"], s["cu"], window=c["window"])}
        q = _package()["append"](s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["tables"],
                                 s["lens"], s["cu"], cos_sin=s["cos_sin"],
                                 q_norm=s.get("q_norm"), k_norm=s.get("k_norm"), eps=1e-6,
                                 interleaved=c["interleaved"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    return _plain_attend(s, c) if c["op"] == "attend" else _plain_append(s, c)


def _tokens(s):
    """Sequence and position of every new token."""
    cu, lens = s["cu"].long(), s["lens"].long()
    t = torch.arange(s["q"].shape[0], device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    return b, lens[b] - (cu[b + 1] - t)


def _plain_attend(s, c):
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    G, B, N, L = hq // hkv, c["seqs"], s["max_new"], s["max_ctx"]
    b, pos = _tokens(s)
    cu, lens = s["cu"].long(), s["lens"].long()
    i = torch.arange(s["q"].shape[0], device=b.device) - cu[b]
    # pages in table order, padded to the longest sequence; what no sequence holds is zero
    key = torch.arange(L, device=b.device)
    slot = s["tables"].long()[:, key // page] * page + key % page
    held = (key[None] < lens[:, None])[..., None, None]
    k = torch.where(held, s["k_cache"].view(-1, hkv, d)[slot].float(), 0.0).permute(0, 2, 3, 1)
    v = torch.where(held, s["v_cache"].view(-1, hkv, d)[slot].float(), 0.0).permute(0, 2, 1, 3)
    q = torch.zeros((B, N, hq, d), device=b.device)
    q[b, i] = s["q"].float()
    q = q.view(B, N, hkv, G, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * N, d)
    x = torch.matmul(q, k).mul_(d ** -0.5).view(B, hkv, G, N, L)
    p = torch.full((B, N), -1, device=b.device)
    p[b, i] = pos
    hidden = key[None, None] > p[..., None]
    if c["window"]:
        hidden |= key[None, None] <= p[..., None] - c["window"]
    x.masked_fill_(hidden[:, None, None], float("-inf"))
    x.sub_(x.amax(-1, keepdim=True).clamp_(min=-3.0e38)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, hkv, G * N, L), v).view(B, hkv, G, N, d) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, N, hq, d)
    return {"out": o[b, i].to(s["q"].dtype)}


def _plain_append(s, c):
    rot, half, d = c["rot"], c["rot"] // 2, c["d"]
    b, pos = _tokens(s)
    cs = s["cos_sin"][pos][:, None]
    cos, sin = cs[..., :half], cs[..., half:]

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
        head = x[..., :rot]
        if c["interleaved"]:
            x0, x1 = head[..., 0::2], head[..., 1::2]
            y = torch.stack([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1).flatten(-2)
        else:
            x0, x1 = head[..., :half], head[..., half:]
            y = torch.cat([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1)
        return torch.cat([y, x[..., rot:]], -1) if rot < d else y

    page = c["page"]
    slot = s["tables"].long()[b, pos // page] * page + pos % page
    dt = s["k_cache"].dtype
    s["k_cache"].view(-1, c["hkv"], d)[slot] = turned(s["k"], s.get("k_norm")).to(dt)
    s["v_cache"].view(-1, c["hkv"], d)[slot] = s["v"]
    q = turned(s["q"], s.get("q_norm")).to(s["q"].dtype)
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _bytes(c):
    return {"bf16": 2, "f16": 2, "f32": 4}[c["dtype"]]


def work(case):
    c = case
    new, ctx = _lengths(c)
    T, eb, d = sum(new), _bytes(c), c["d"]
    if c["op"] == "append":
        rows = T * (c["hq"] + 2 * c["hkv"])
        return {"bytes": 2 * rows * d * eb + T * (c["rot"] + 1) * 4 + len(new) * 8,
                "flops": T * (c["hq"] + c["hkv"]) * (3 * c["rot"] + (4 * d if c["norm"] else 0))}
    pairs = keys = 0
    for n, x in zip(new, ctx):
        if not c["window"]:
            pairs += n * x - n * (n - 1) // 2
            keys += x
            continue
        w = c["window"]
        keys += x - max(0, x - n - w + 1)  # from the first row's window to the last row
        whole = min(n, max(0, x - w + 1))  # rows whose window the start does not cut
        cut = n - whole
        pairs += whole * w + cut * (x - n + 1) + cut * (cut - 1) // 2
    return {"bytes": 2 * keys * c["hkv"] * d * eb + 2 * T * c["hq"] * d * eb,
            "flops": 4 * d * c["hq"] * pairs}


def exact(case, seed):
    """The definition in 64 bits, one sequence and KV head at a time."""
    s, c = prepare(case, seed), case
    new, ctx = _lengths(c)
    hkv, G, d, page = c["hkv"], c["hq"] // c["hkv"], c["d"], c["page"]
    t0 = 0
    if c["op"] == "append":
        q64 = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        rot = c["rot"]

        def spin(x, w, cos, sin):  # as a complex product over the pairs
            x = x.double()
            if w is not None:
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + 1e-6) * w.double()
            a = x[..., :rot]
            z = torch.view_as_complex(
                (a.unflatten(-1, (rot // 2, 2)) if c["interleaved"]
                 else a.unflatten(-1, (2, rot // 2)).transpose(-1, -2)).contiguous())
            z = torch.view_as_real(z * torch.complex(cos, sin)[:, None])
            z = z if c["interleaved"] else z.transpose(-1, -2)
            return torch.cat([z.flatten(-2), x[..., rot:]], -1)

        for b, (n, x) in enumerate(zip(new, ctx)):
            p = torch.arange(x - n, x, device="cuda")
            cs = s["cos_sin"][p].double()
            cos, sin = cs[:, :rot // 2], cs[:, rot // 2:]
            sl = slice(t0, t0 + n)
            q64[sl] = spin(s["q"][sl], s.get("q_norm"), cos, sin)
            blk, off = s["tables"][b, p // page].long(), p % page
            kc[blk, off] = spin(s["k"][sl], s.get("k_norm"), cos, sin)
            vc[blk, off] = s["v"][sl].double()
            t0 += n
        return {"q": q64, "k_cache": kc, "v_cache": vc}
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (n, x) in enumerate(zip(new, ctx)):
        blk = s["tables"][b, :-(-x // page)].long()
        j = torch.arange(x, device="cuda")[None, None]
        for h in range(hkv):
            k = s["k_cache"][blk, :, h].reshape(-1, d)[:x].double()
            v = s["v_cache"][blk, :, h].reshape(-1, d)[:x].double()
            q = s["q"][t0:t0 + n, h * G:(h + 1) * G].double()
            for i in range(0, n, 256):
                z = torch.einsum("ngd,ld->ngl", q[i:i + 256], k) / math.sqrt(d)
                p = torch.arange(x - n + i, x - n + min(n, i + 256), device="cuda")[:, None, None]
                seen = (j <= p) & (j > p - c["window"]) if c["window"] else j <= p
                z = torch.softmax(z.masked_fill(~seen, float("-inf")), -1)
                out[t0 + i:t0 + min(n, i + 256), h * G:(h + 1) * G] = torch.einsum(
                    "ngl,ld->ngd", z, v)
        t0 += n
    return {"out": out}
