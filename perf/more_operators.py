"""Performance cases of the operators that make the paged cache smaller.

Four operators over the paged cache and a ragged batch (sequence b owns rows
cu[b]..cu[b + 1] of the packed token arrays and the pages of row b of the tables):

- `append8`: the rotating append into a cache of 8-bit floats (e4m3) with a
  power-of-two scale for each page and KV head, keys and values apart
  (`cvsa.kernels.rope_append`);
- `attend8`: attention of the new tokens over such a cache
  (`cvsa.kernels.chunk_attend`);
- `weights`: the attention weight that each cached key got from the new tokens,
  added to what it had (`cvsa.kernels.key_weights`);
- `evict`: the keys of largest weight of each KV head, the first and the last
  ones of a sequence among them, moved to new pages (`cvsa.kernels.evict`).

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
_F8 = torch.float8_e4m3fn
_PKG = "coverage-verified-sparse-attention_b200"
_LO, _HI = -15, 7  # exponents of a page's scale: every value is an f16 and a bf16 number


def _case(name, op, dtype, hq, hkv, d, page, seqs, new, ctx, **more):
    c = dict(name=name, op=op, dtype=dtype, hq=hq, hkv=hkv, d=d, page=page, seqs=seqs,
             new_lo=new[0], new_hi=new[1], ctx_lo=ctx[0], ctx_hi=ctx[1], mix=1, window=0,
             norm=False, interleaved=False, rot=d, cache8=op in ("append8", "attend8"),
             keep=0, sink=0, recent=0, decay=1.0)
    c.update(more)
    return c


def listed():
    return [
        # one token of 32 sequences into the 8-bit cache, once a layer and step; most go to
        # a page that holds others already
        _case("append8 32x1", "append8", "bf16", 32, 8, 128, 16, 32, (1, 1), (100, 2048)),
        # a whole prompt's keys and values into the 8-bit cache
        _case("append8 prompt 8192", "append8", "bf16", 32, 8, 128, 16, 1, (8192, 8192),
              (8192, 8192)),
        # ragged chunks with query and key norms, half of each head rotated in neighbouring pairs
        _case("append8 9 odd chunks, norms", "append8", "f16", 40, 8, 128, 16, 9, (1, 900),
              (900, 1900), norm=True, interleaved=True, rot=64, mix=4),
        # a short question in a short chat on the 8-bit cache: a call of this size is latency
        _case("attend8 1 at 300", "attend8", "bf16", 32, 8, 128, 16, 1, (1, 1), (300, 300)),
        # one token for each sequence of a batch, ragged contexts up to 8K: the serving form
        _case("attend8 32x1 ragged 8K", "attend8", "bf16", 32, 8, 128, 16, 32, (1, 1),
              (1024, 8192)),
        # a few drafted tokens verified per sequence, 64-wide heads, pages of 64
        _case("attend8 8x(2-8) D 64", "attend8", "f16", 32, 8, 64, 64, 8, (2, 8), (8192, 16384)),
        # a prompt's chunk far into a long document
        _case("attend8 1024 at 32K", "attend8", "bf16", 32, 8, 128, 16, 1, (1024, 1024),
              (32768, 32768)),
        # chunks of several prompts in one call, odd lengths, 7 query heads a KV head
        _case("attend8 6 odd chunks f16 G7", "attend8", "f16", 28, 4, 128, 16, 6, (1, 700),
              (701, 5001), mix=3),
        # weights of a decode step's keys over the 16-bit cache
        _case("weights 32x1 ragged 8K", "weights", "bf16", 32, 8, 128, 16, 32, (1, 1),
              (1024, 8192)),
        # weights that the last tokens of a long prompt give its keys, 8-bit cache
        _case("weights 256 at 32K, 8 bits", "weights", "bf16", 32, 8, 128, 16, 1, (256, 256),
              (32768, 32768), cache8=True),
        # a long prompt cut to an eighth before decoding
        _case("evict 32K to 4096", "evict", "bf16", 32, 8, 128, 16, 1, (1, 1), (32768, 32768),
              keep=4096, sink=4, recent=256),
        # a batch that outgrew its share of the 8-bit cache
        _case("evict 16 ragged to 1000, 8 bits", "evict", "bf16", 32, 8, 128, 16, 16, (1, 1),
              (1001, 3000), keep=1000, sink=16, recent=100, cache8=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append8", "attend8", "attend8", "weights", "evict"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    d = rng.choice([64, 128, 128])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 4, 5, 7, 8])
    page = rng.choice([16, 16, 16, 64])
    more = dict(mix=rng.randrange(1 << 20))
    cache8 = op in ("append8", "attend8") or rng.random() < 0.5
    while True:
        seqs = _log(rng, 1, 64)
        new_hi = 1 if op == "evict" or rng.random() < 0.3 else _log(rng, 1, 8192)
        new_lo = new_hi if rng.random() < 0.3 else rng.randint(1, new_hi)
        if op == "append8":
            ctx_lo = new_hi
            ctx_hi = new_hi + _log(rng, 1, 1024)
            if seqs * new_hi * (hq + 2 * hkv) * d <= 8192 * 48 * 128:
                break
            continue
        ctx_lo = max(new_hi, _log(rng, 16, 131072))
        ctx_hi = min(131072, ctx_lo * rng.choice([1, 2, 4]))
        if seqs * ctx_hi * hkv * d > 2 ** 28:
            continue
        if op == "evict":
            if ctx_lo < 32 or seqs * ctx_hi * hkv > 2 ** 21:
                continue
            keep = min(ctx_lo, _log(rng, 16, 8192))
            if seqs * keep * hkv * d > 2 ** 25:
                continue
            sink = rng.choice([0, 0, rng.randint(0, min(keep, 64))])
            more.update(keep=keep, sink=sink, recent=rng.randint(0, keep - sink))
            break
        rows = seqs * hq * new_hi * ctx_hi
        if rows <= (2 ** 30 if dtype != "f32" else 2 ** 28) and rows * d <= 2 ** 37:
            break
    if op in ("attend8", "weights") and rng.random() < 0.25:
        more["window"] = _log(rng, 16, 4096)
    if op == "append8":
        more.update(norm=rng.random() < 0.5, interleaved=rng.random() < 0.5,
                    rot=rng.choice([d, d, d // 2]))
    if op == "weights":
        more["decay"] = rng.choice([1.0, 1.0, 0.875])
    c = _case("", op, dtype, hq, hkv, d, page, seqs, (new_lo, new_hi), (ctx_lo, ctx_hi),
              cache8=cache8, **more)
    del c["name"]
    return c


def _lengths(c):
    """(new tokens, context length with them) of each sequence."""
    r = random.Random(c["mix"])
    new = [r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["seqs"])]
    ctx = [max(n, r.randint(c["ctx_lo"], c["ctx_hi"])) for n in new]
    return new, ctx


def _exponent(amax):
    """The least e with amax <= 448 * 2^e, in the range of a page's scale."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, e, _LO).clamp(_LO, _HI)


def prepare(case, seed):
    c = case
    dev, dt = torch.device("cuda"), _DT[c["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    new, ctx = _lengths(c)
    page, width = c["page"], max(-(-x // c["page"]) for x in ctx)
    T, hq, hkv, d = sum(new), c["hq"], c["hkv"], c["d"]
    kept = -(-c["keep"] // page)  # new pages of a sequence
    held = sum(-(-x // page) for x in ctx)
    blocks = held + c["seqs"] * kept
    order = torch.randperm(blocks, generator=g, device=dev).to(torch.int32)
    tables = torch.zeros((c["seqs"], width), dtype=torch.int32, device=dev)
    at = 0
    for b, x in enumerate(ctx):
        n = -(-x // page)
        tables[b, :n] = order[at:at + n]
        at += n
    shape = (blocks, page, hkv, d)
    lens = torch.tensor(ctx, dtype=torch.int32, device=dev)
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=dev)
    s = dict(case=c, tables=tables, lens=lens, cu=cu, max_new=max(new), max_ctx=max(ctx))
    for name in ("k", "v"):
        x = torch.randn(shape, generator=g, device=dev)
        # pages differ in size, as the tokens of a text do
        x *= torch.empty((blocks, 1, hkv, 1), device=dev).uniform_(0.5, 2.0, generator=g)
        if c["cache8"]:
            e = _exponent(x.abs().amax((1, 3)))
            s[name + "_scale"] = torch.ldexp(torch.ones(e.shape, device=dev), e)
            s[name + "_cache"] = (x / s[name + "_scale"][:, None, :, None]).to(_F8)
        else:
            s[name + "_cache"] = x.to(dt)
        del x
    if c["op"] == "append8":
        # one projection's output: q, k and v are its column ranges
        qkv = torch.randn((T, (hq + 2 * hkv) * d), generator=g, device=dev)
        qkv *= torch.empty((T, 1), device=dev).uniform_(0.5, 3.0, generator=g)
        qkv = qkv.to(dt)
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
    if c["op"] == "evict":
        # most of a head's weight lies on few keys
        w = torch.empty((c["seqs"], hkv, width * page), device=dev).uniform_(generator=g)
        s["weights"] = w.pow_(8).mul_(100.0)
        s["out_weights"] = torch.zeros((c["seqs"], hkv, c["keep"]), device=dev)
        s["new_tables"] = order[held:].view(c["seqs"], kept)
        return s
    # slots past a context hold whatever was there: NaN here
    for b, x in enumerate(ctx):
        if x % page:
            for name in ("k_cache", "v_cache"):
                pool = s[name].view(torch.uint8) if c["cache8"] else s[name]
                pool[tables[b, x // page].long(), x % page:] = 0x7f if c["cache8"] \
                    else float("nan")
    # logits spread like trained heads': some rows look at a few keys, some at many
    heat = torch.empty((1, hq, 1), device=dev).uniform_(0.5, 2.5, generator=g)
    s["q"] = (torch.randn((T, hq, d), generator=g, device=dev) * heat).to(dt)
    if c["op"] == "weights":
        # what a key had is of the size of what it gets
        s["weights"] = torch.empty((c["seqs"], hkv, width * page), device=dev).uniform_(
            generator=g).mul_(hq // hkv * T / sum(ctx))
        s["out"] = torch.zeros_like(s["weights"])
        x, seen = _scores(s, c)
        s["lse"] = _packed(torch.logsumexp(x.masked_fill_(~seen, float("-inf")), -1), s, c)
        s["lse"] = s["lse"].contiguous()
    return s


_mod = {}


def _package():
    if not _mod:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), _PKG)
        if root not in sys.path:
            sys.path.insert(0, root)
        from cvsa.kernels.chunk_attend import chunk_attention
        from cvsa.kernels.evict import evict
        from cvsa.kernels.key_weights import key_weights
        from cvsa.kernels.rope_append import rope_append
        _mod.update(attend8=chunk_attention, append8=rope_append, weights=key_weights,
                    evict=evict)
    return _mod


def run(state):
    s, c = state, state["case"]
    if own:
        f = _package()[c["op"]]
        ks, vs = s.get("k_scale"), s.get("v_scale")
        if c["op"] == "attend8":
            return {"out": f(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["cu"],
                             window=c["window"], k_scale=ks, v_scale=vs)}
        if c["op"] == "weights":
            return {"out": f(s["q"], s["lse"], s["k_cache"], s["tables"], s["lens"], s["cu"],
                             s["weights"], out=s["out"], decay=c["decay"], window=c["window"],
                             k_scale=ks)}
        if c["op"] == "evict":
            s["kept"] = f(s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["weights"],
                          s["new_tables"], c["keep"], sink=c["sink"], recent=c["recent"],
                          out_weights=s["out_weights"], k_scale=ks, v_scale=vs)
            return _evicted(s)
        q = f(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["cu"],
              cos_sin=s["cos_sin"], q_norm=s.get("q_norm"), k_norm=s.get("k_norm"), eps=1e-6,
              interleaved=c["interleaved"], k_scale=ks, v_scale=vs)
        return dict(_pools(s), q=q)
    if c["op"] == "attend8":
        return _plain_attend(s, c)
    if c["op"] == "weights":
        return _plain_weights(s, c)
    return _plain_evict(s, c) if c["op"] == "evict" else _plain_append(s, c)


def _pools(s):
    return {k: s[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale") if k in s}


def _evicted(s):
    return dict(_pools(s), kept=s["kept"], weights=s["out_weights"])


def _tokens(s):
    """Sequence, position, and index in its sequence of every new token."""
    cu, lens = s["cu"].long(), s["lens"].long()
    t = torch.arange(s["q"].shape[0], device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    return b, lens[b] - (cu[b + 1] - t), t - cu[b]


def _dense(s, name):
    """[seqs, hkv, max_ctx, d] in 32 bits: pages in table order, zeros past a context."""
    c = s["case"]
    key = torch.arange(s["max_ctx"], device=s["lens"].device)
    blk = s["tables"].long()[:, key // c["page"]]
    pool = s[name + "_cache"]
    x = (pool.view(torch.uint8) if c["cache8"] else pool)[blk, key % c["page"]]
    x = (x.view(_F8) if c["cache8"] else x).float()
    if c["cache8"]:
        x *= s[name + "_scale"][blk][..., None]
    held = (key[None] < s["lens"].long()[:, None])[..., None, None]
    return torch.where(held, x, 0.0).permute(0, 2, 1, 3)


def _scores(s, c):
    """Scaled scores [seqs, hkv, G, max_new, max_ctx] in 32 bits, and which are seen."""
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    G, B, N, L = hq // hkv, c["seqs"], s["max_new"], s["max_ctx"]
    b, pos, i = _tokens(s)
    q = torch.zeros((B, N, hq, d), device=b.device)
    q[b, i] = s["q"].float()
    q = q.view(B, N, hkv, G, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * N, d)
    x = torch.matmul(q, _dense(s, "k").transpose(-1, -2)).mul_(d ** -0.5)
    key = torch.arange(L, device=b.device)
    p = torch.full((B, N), -1, device=b.device)
    p[b, i] = pos
    seen = key[None, None] <= p[..., None]
    if c["window"]:
        seen &= key[None, None] > p[..., None] - c["window"]
    return x.view(B, hkv, G, N, L), seen[:, None, None]


def _packed(x, s, c):
    """[seqs, hkv, G, max_new, ...] to the packed tokens' [T, hq, ...]."""
    b, _, i = _tokens(s)
    return x.movedim(3, 1).flatten(2, 3)[b, i]


def _plain_attend(s, c):
    x, seen = _scores(s, c)
    x.masked_fill_(~seen, float("-inf"))
    x.sub_(x.amax(-1, keepdim=True).clamp_(min=-3.0e38)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.flatten(2, 3), _dense(s, "v")).view(*x.shape[:4], c["d"])
    return {"out": _packed(o / total.clamp(min=1e-30), s, c).to(s["q"].dtype)}


def _plain_weights(s, c):
    x, seen = _scores(s, c)
    b, _, i = _tokens(s)
    hkv, G = c["hkv"], c["hq"] // c["hkv"]
    lse = torch.zeros((c["seqs"], s["max_new"], hkv, G), device=x.device)
    lse[b, i] = s["lse"].view(-1, hkv, G)
    x.sub_(lse.permute(0, 2, 3, 1)[..., None]).exp_().masked_fill_(~seen, 0.0)
    key, lens = torch.arange(s["max_ctx"], device=x.device), s["lens"].long()[:, None]
    start = lens - (s["cu"][1:] - s["cu"][:-1]).long()[:, None]
    out, L = s["out"], s["max_ctx"]
    # the new tokens' own keys had no weight before
    prior = torch.where((key < start)[:, None], s["weights"][..., :L], 0.0) * c["decay"]
    total = prior + x.sum((2, 3))
    out[..., :L] = torch.where((key < lens)[:, None], total, out[..., :L])
    return {"out": out}


def _put(pool, where, x):
    """pool[where] = x, also for 8-bit floats."""
    if pool.dtype == _F8:
        pool.view(torch.uint8)[where] = x.to(_F8).view(torch.uint8)
    else:
        pool[where] = x.to(pool.dtype)


def _plain_evict(s, c):
    page, keep, lens = c["page"], c["keep"], s["lens"].long()[:, None, None]
    w = s["weights"]
    key = torch.arange(w.shape[2], device=w.device)
    must = (key < c["sink"]) | (key >= lens - c["recent"])
    rank = torch.where(must, float("inf"), w).masked_fill(key >= lens, float("-inf"))
    kept = torch.sort(rank, dim=-1, descending=True, stable=True)[1][..., :keep]
    kept = torch.sort(kept, dim=-1)[0]
    moved = lens > keep
    b = torch.arange(c["seqs"], device=w.device)[:, None, None]
    h = torch.arange(c["hkv"], device=w.device)[None, :, None]
    i = torch.arange(keep, device=w.device)
    src = (s["tables"].long()[b, kept // page], kept % page, h)
    dst = (s["new_tables"].long()[b, i // page], i % page, h)
    some = moved.expand(kept.shape)
    src, dst = tuple(t.expand(kept.shape)[some] for t in src), \
        tuple(t.expand(kept.shape)[some] for t in dst)
    for name in ("k", "v"):
        pool = s[name + "_cache"]
        if not c["cache8"]:
            pool[dst] = pool[src]
            continue
        scale = s[name + "_scale"]
        x = pool.view(torch.uint8)[src].view(_F8).float()
        x, mine = x * scale[src[0], src[2]][:, None], scale[src[0], src[2]]
        scale[dst[0], dst[2]] = 0.0
        scale.view(-1).scatter_reduce_(0, dst[0] * c["hkv"] + dst[2], mine, "amax")
        _put(pool, dst, x / scale[dst[0], dst[2]][:, None])
    s["kept"] = torch.where(moved, kept, -1).to(torch.int32)
    s["out_weights"].copy_(torch.where(moved, w.gather(2, kept), s["out_weights"]))
    return _evicted(s)


def _plain_append(s, c):
    rot, half, d, hkv, page = c["rot"], c["rot"] // 2, c["d"], c["hkv"], c["page"]
    b, pos, _ = _tokens(s)
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

    tables, lens = s["tables"].long(), s["lens"].long()
    start = lens - (s["cu"][1:] - s["cu"][:-1]).long()
    blk = tables[b, pos // page]
    # the page that each sequence had begun, and its slots in use
    begun = tables[torch.arange(c["seqs"], device=b.device), start // page]
    used = torch.arange(page, device=b.device) < (start % page)[:, None]
    begun, used = begun[:, None].expand(used.shape)[used], used.nonzero()[:, 1]
    for name, x in (("k", turned(s["k"], s.get("k_norm"))), ("v", s["v"].float())):
        pool, scale = s[name + "_cache"], s[name + "_scale"]
        amax = torch.zeros(scale.shape, device=b.device)
        amax.scatter_reduce_(0, blk[:, None].expand(-1, hkv), x.abs().amax(-1), "amax")
        fresh = torch.ldexp(torch.ones_like(amax), _exponent(amax))
        had = scale[begun].clone()
        old = pool.view(torch.uint8)[begun, used].view(_F8).float() * had[..., None]
        scale[blk] = fresh[blk]
        scale[begun] = torch.maximum(had, fresh[begun])
        _put(pool, (begun, used), old / scale[begun][..., None])
        _put(pool, (blk, pos % page), (x / scale[blk][..., None]).clamp(-448.0, 448.0))
    q = turned(s["q"], s.get("q_norm")).to(s["q"].dtype)
    return dict(_pools(s), q=q)


def _bytes(c):
    return {"bf16": 2, "f16": 2, "f32": 4}[c["dtype"]]


def work(case):
    c = case
    new, ctx = _lengths(c)
    T, eb, d, hkv = sum(new), _bytes(c), c["d"], c["hkv"]
    cb = 1 if c["cache8"] else eb
    if c["op"] == "append8":
        rows = T * (c["hq"] + 2 * hkv)
        old = sum((x - n) % c["page"] for n, x in zip(new, ctx))
        pages = sum((x - 1) // c["page"] - (x - n) // c["page"] + 1 for n, x in zip(new, ctx))
        # the slots in use of a begun page are read and written only where its scale grows
        return {"bytes": rows * d * eb + T * c["hq"] * d * eb + 2 * T * hkv * d +
                T * (c["rot"] + 1) * 4 + pages * hkv * 8 + len(new) * 8,
                "flops": T * (c["hq"] + hkv) * (3 * c["rot"] + (4 * d if c["norm"] else 0)) +
                2 * (T + old) * hkv * d * 2}
    if c["op"] == "evict":
        moved = [x for x in ctx if x > c["keep"]]
        n = len(moved) * hkv * c["keep"]
        return {"bytes": 2 * 2 * n * d * cb + sum(moved) * hkv * 4 + n * 8,
                "flops": sum(moved) * hkv}
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
    scales = -(-keys // c["page"]) * hkv * 4 if c["cache8"] else 0
    if c["op"] == "weights":
        return {"bytes": keys * hkv * d * cb + scales + T * c["hq"] * (d * eb + 4) +
                2 * sum(ctx) * hkv * 4, "flops": 2 * d * c["hq"] * pairs}
    return {"bytes": 2 * keys * hkv * d * cb + 2 * scales + 2 * T * c["hq"] * d * eb,
            "flops": 4 * d * c["hq"] * pairs}


def _near(x):
    """x rounded to the nearest e4m3 number, halves to even, in 64 bits."""
    e = torch.frexp(x)[1].clamp(min=-5) - 1  # x = f 2^e, 1 <= f < 2, or below the normal numbers
    step = torch.ldexp(torch.ones_like(x), e - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _scale64(amax):
    """The page's scale from its largest absolute value, in 64 bits."""
    e = torch.full_like(amax, _LO)
    for i in range(_LO, _HI):
        e = torch.where(amax > 448.0 * 2.0 ** i, float(i + 1), e)
    return 2.0 ** e


def _exact_append(s, c):
    new, ctx = _lengths(c)
    d, page, rot, t0 = c["d"], c["page"], c["rot"], 0
    out = {"q": torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")}
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        out[name] = s[name].double()

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
        out["q"][sl] = spin(s["q"][sl], s.get("q_norm"), cos, sin)
        for name, rows in (("k", spin(s["k"][sl], s.get("k_norm"), cos, sin)),
                           ("v", s["v"][sl].double())):
            pool, scale = out[name + "_cache"], out[name + "_scale"]
            # whole pages from the one that the first token falls into, zeros around the tokens
            first, pages = (x - n) // page, (x - 1) // page - (x - n) // page + 1
            lead = (x - n) % page
            grid = torch.zeros((pages * page,) + rows.shape[1:], dtype=torch.float64,
                               device="cuda")
            grid[lead:lead + n] = rows
            grid = grid.unflatten(0, (pages, page))
            blk = s["tables"][b, first:first + pages].long()
            sc = _scale64(grid.abs().amax((1, 3)))
            if lead:
                had = scale[blk[0]].clone()
                sc[0] = torch.maximum(sc[0], had)
                old = pool[blk[0], :lead] * had[None, :, None]
                pool[blk[0], :lead] = _near(old / sc[0][None, :, None])
            scale[blk] = sc
            code = _near(grid / sc[:, None, :, None]).flatten(0, 1)[lead:lead + n]
            pool[blk[(p // page) - first], p % page] = code
        t0 += n
    return out


def _exact_evict(s, c):
    _, ctx = _lengths(c)
    page, keep, hkv = c["page"], c["keep"], c["hkv"]
    out = {k: v.double() for k, v in _pools(s).items()}
    out["kept"] = torch.full((c["seqs"], hkv, keep), -1, dtype=torch.int32, device="cuda")
    out["weights"] = s["out_weights"].double()
    at = torch.arange(keep, device="cuda")
    for b, x in enumerate(ctx):
        if x <= keep:
            continue
        lo, hi, n = c["sink"], x - c["recent"], keep - c["sink"] - c["recent"]
        mid = s["weights"][b, :, lo:hi].double()
        # the n largest: those above the n-th, and the first of those equal to it
        if n > 0:
            cut = mid.topk(n, dim=-1)[0][:, -1:]
            above, same = mid > cut, mid == cut
            room = n - above.sum(-1, keepdim=True)
            take = above | (same & (same.cumsum(-1) <= room))
        else:
            take = torch.zeros_like(mid, dtype=torch.bool)
        all_ = torch.ones((hkv, x), dtype=torch.bool, device="cuda")
        all_[:, lo:hi] = take
        idx = all_.nonzero()[:, 1].view(hkv, keep)
        out["kept"][b] = idx.to(torch.int32)
        out["weights"][b] = s["weights"][b].gather(1, idx).double()
        to = s["new_tables"][b].long()[at // page]
        for h in range(hkv):
            frm = s["tables"][b].long()[idx[h] // page]
            for name in ("k", "v"):
                rows = s[name + "_cache"][frm, idx[h] % page, h] if not c["cache8"] else \
                    s[name + "_cache"].view(torch.uint8)[frm, idx[h] % page, h].view(_F8)
                rows = rows.double()
                if c["cache8"]:
                    mine = s[name + "_scale"][frm, h].double()
                    pages = -(-keep // page)
                    full = torch.zeros(pages * page, dtype=torch.float64, device="cuda")
                    full[:keep] = mine
                    top = full.view(pages, page).amax(1)
                    out[name + "_scale"][s["new_tables"][b].long(), h] = top
                    rows = _near(rows * (mine / top[at // page])[:, None])
                out[name + "_cache"][to, at % page, h] = rows
    return out


def exact(case, seed):
    """The definitions in 64 bits, one sequence and KV head at a time."""
    s, c = prepare(case, seed), case
    if c["op"] == "append8":
        return _exact_append(s, c)
    if c["op"] == "evict":
        return _exact_evict(s, c)
    new, ctx = _lengths(c)
    hkv, G, d = c["hkv"], c["hq"] // c["hkv"], c["d"]

    def rows(name, b, h, x):
        blk = s["tables"][b, :-(-x // c["page"])].long()
        if not c["cache8"]:
            return s[name + "_cache"][blk, :, h].reshape(-1, d)[:x].double()
        code = s[name + "_cache"].view(torch.uint8)[blk, :, h].view(_F8).double()
        return (code * s[name + "_scale"][blk, h].double()[:, None, None]).reshape(-1, d)[:x]

    t0 = 0
    if c["op"] == "weights":
        out = s["out"].double()
    else:
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (n, x) in enumerate(zip(new, ctx)):
        j = torch.arange(x, device="cuda")[None, None]
        for h in range(hkv):
            k, q = rows("k", b, h, x), s["q"][t0:t0 + n, h * G:(h + 1) * G].double()
            got = torch.zeros(x, dtype=torch.float64, device="cuda")
            for i in range(0, n, 256):
                z = torch.einsum("ngd,ld->ngl", q[i:i + 256], k) / math.sqrt(d)
                p = torch.arange(x - n + i, x - n + min(n, i + 256), device="cuda")[:, None, None]
                seen = (j <= p) & (j > p - c["window"]) if c["window"] else j <= p
                z = z.masked_fill(~seen, float("-inf"))
                if c["op"] == "weights":
                    lse = s["lse"][t0 + i:t0 + min(n, i + 256), h * G:(h + 1) * G].double()
                    got += torch.exp(z - lse[..., None]).sum((0, 1))
                else:
                    out[t0 + i:t0 + min(n, i + 256), h * G:(h + 1) * G] = torch.einsum(
                        "ngl,ld->ngd", torch.softmax(z, -1), rows("v", b, h, x))
            if c["op"] == "weights":
                got[:x - n] += c["decay"] * s["weights"][b, h, :x - n].double()
                out[b, h, :x] = got
        t0 += n
    return {"out": out}
