// How the attention of a ragged batch of new tokens is cut into work for a
// persistent grid, shared by the kernels that compute it.
//
// An item is one KV head of one group of P consecutive new tokens of one
// sequence (all query heads of the KV head: P * G query rows); it walks the
// KT-key tiles its rows can see. It counts its tiles plus `fixed` units of work
// (bringing the queries in and writing the rows out cost about as much as
// that many tiles: without it the CTA that got a prompt's first groups, of a
// tile each, took three times as long as the others). The items in the order
// (sequence, group, head) form one stream of units that is cut into equal
// contiguous ranges, one a CTA, so the load is even whatever the mix of long
// and short contexts, and a long cache with few queries is split over all CTAs
// by the same rule. An item inside one range is finished by its CTA; an item
// that crosses ranges leaves one partial (m, l, o) a CTA, merged in CTA order
// by a second kernel. A CTA has at most two such items (its first and its
// last), so two partial slots each. When no item can be longer than a few
// tiles (short tables) a CTA takes the items that begin in its range whole, and
// there is nothing to merge.
//
// Lengths live on the device, so every CTA finds its own range, one warp of it
// alone, 32 sequences or groups a step: no launch and no block-wide barrier.
#pragma once

#include "cvsa_common.cuh"
#include "cvsa_internal.h"

namespace cvsa {

struct ChunkGeo {
  int bs, hkv, G;
  int P;        // new tokens a group
  int KT;       // keys a tile
  int causal, window;
  int fixed;    // units an item counts beside its tiles
  int few, fixed_few;  // the same for items of at most `few` rows
  int split;    // items may cross ranges
};

struct SeqInfo {
  int tok0, n;     // rows of the packed token arrays
  int slot;        // row of the tables
  int start, ctx;  // position of the first new token; keys the sequence holds
};

// Sequence b; every field ends in range whatever the arrays hold.
__device__ __forceinline__ SeqInfo chunk_seq(const RaggedView& rg, int bs, int b,
                                             int32_t* dev_err) {
  // every load before the first check, so that they wait for one another only
  // where one names the next
  SeqInfo q;
  q.tok0 = rg.cu[b];
  const int end = rg.cu[b + 1];
  q.slot = rg.seq_ids ? rg.seq_ids[b] : b;
  const bool row_ok = q.slot >= 0 && q.slot < rg.num_seqs;
  q.ctx = row_ok ? rg.lens[q.slot] : 0;
  const int start = rg.starts ? rg.starts[b] : 0;
  q.n = end - q.tok0;
  q.start = rg.starts ? start : q.ctx - q.n;
  if (q.tok0 < 0 || end > rg.T || end < q.tok0) {  // whose tokens these are is not known
    set_dev_error(dev_err, CVSA_DEV_ERR_RAGGED);
    q.n = q.slot = q.start = q.ctx = 0;
    return q;
  }
  if (!row_ok) {  // its rows see no key
    set_dev_error(dev_err, CVSA_DEV_ERR_RAGGED);
    q.slot = q.start = q.ctx = 0;
    return q;
  }
  if (q.ctx < 0 || q.ctx > (int64_t)rg.W * bs) {
    set_dev_error(dev_err, CVSA_DEV_ERR_RAGGED);
    q.ctx = q.ctx < 0 ? 0 : rg.W * bs;
  }
  if (rg.starts && start < 0) q.start = q.ctx = 0;  // refused: its rows see no key
  return q;
}

__device__ __forceinline__ int chunk_groups(const SeqInfo& q, int P) { return (q.n + P - 1) / P; }

// Keys [lo, hi) some row of tokens [t0, t1) sees.
__device__ __forceinline__ void chunk_keys(const SeqInfo& q, const ChunkGeo& g, int t0, int t1,
                                           int& lo, int& hi) {
  hi = g.causal ? max(0, min(q.ctx, q.start + t1)) : q.ctx;
  lo = g.window > 0 ? max(0, q.start + t0 - g.window + 1) : 0;
}

__device__ __forceinline__ int chunk_tiles(int lo, int hi, int KT) {
  return hi > lo ? (hi + KT - 1) / KT - lo / KT : 0;
}

__device__ __forceinline__ int chunk_fixed(const ChunkGeo& g, int tokens) {
  return tokens * g.G <= g.few ? g.fixed_few : g.fixed;
}

__device__ __forceinline__ int chunk_units(const SeqInfo& q, const ChunkGeo& g, int i) {
  int lo, hi;
  chunk_keys(q, g, i * g.P, min(q.n, (i + 1) * g.P), lo, hi);
  return chunk_tiles(lo, hi, g.KT) + chunk_fixed(g, min(q.n - i * g.P, g.P));
}

// What a CTA does: units [u0, u1) of the stream, starting at unit `skip` of
// item (b, i, h). The host has checked that the units of sequences that share
// no token fit 31 bits.
struct ChunkRange {
  int u0, u1, per_cta;
  int b, i, h, skip;
};

__device__ __forceinline__ int warp_scan_incl(int v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, v, o);
    if ((int)(threadIdx.x & 31) >= o) v += t;
  }
  return v;
}

// Units of 32 sequences from b0, one a lane (all heads).
__device__ __forceinline__ int chunk_seq_units(const RaggedView& rg, const ChunkGeo& g, int b0,
                                               SeqInfo& q, int32_t* dev_err) {
  const int lane = threadIdx.x & 31;
  q.n = 0;
  if (b0 + lane < rg.B) q = chunk_seq(rg, g.bs, b0 + lane, dev_err);
  const int ng = chunk_groups(q, g.P);
  int units = ng == 1 ? chunk_units(q, g, 0) : 0;
  // sequences of several groups: the warp sums the groups of one at a time
  for (unsigned many = __ballot_sync(0xffffffffu, ng > 1); many; many &= many - 1) {
    const int src = __ffs(many) - 1;
    SeqInfo s;
    s.n = __shfl_sync(0xffffffffu, q.n, src);
    s.start = __shfl_sync(0xffffffffu, q.start, src);
    s.ctx = __shfl_sync(0xffffffffu, q.ctx, src);
    const int groups = chunk_groups(s, g.P);
    int sum = 0;
    for (int i = lane; i < groups; i += 32) sum += chunk_units(s, g, i);
    sum = warp_sum_i(sum);
    if (lane == src) units = sum;
  }
  return units * g.hkv;
}

// The range of CTA `cta`, by a whole warp; every lane returns it. Ranges are at
// least `min_units` long: a partial costs its write and its read by the merge,
// which a tile or two do not pay for.
__device__ __forceinline__ ChunkRange chunk_range(const RaggedView& rg, const ChunkGeo& g, int cta,
                                                  int ctas, int min_units, int32_t* dev_err) {
  const int lane = threadIdx.x & 31;
  SeqInfo q = {};
  ChunkRange r = {};
  int units = 0;
  int64_t sum = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < rg.B; b0 += 32) {
    units = chunk_seq_units(rg, g, b0, q, cta == 0 ? dev_err : nullptr);
    sum += __reduce_add_sync(0xffffffffu, (unsigned)units & 0xffff) +
           ((int64_t)__reduce_add_sync(0xffffffffu, (unsigned)units >> 16) << 16);
  }
  if (sum > 0x7fffffff) {  // offsets that name tokens again and again: nothing is done
    if (cta == 0) set_dev_error(dev_err, CVSA_DEV_ERR_RAGGED);
    return r;
  }
  const int total = (int)sum;
  r.per_cta = max(min_units, (total + ctas - 1) / ctas);
  r.u0 = (int)min((int64_t)total, (int64_t)cta * r.per_cta);
  r.u1 = min(total, r.u0 + r.per_cta);
  if (r.u0 >= r.u1) return r;
  int before = 0;  // units ahead of this step
#pragma unroll 1
  for (int b0 = 0; b0 < rg.B; b0 += 32) {
    if (rg.B > 32) units = chunk_seq_units(rg, g, b0, q, nullptr);  // else still in registers
    const int incl = warp_scan_incl(units) + before;
    const unsigned past = __ballot_sync(0xffffffffu, incl > r.u0);
    if (!past) {
      before = __shfl_sync(0xffffffffu, incl, 31);
      continue;
    }
    const int src = __ffs(past) - 1;
    before = __shfl_sync(0xffffffffu, incl - units, src);
    r.b = b0 + src;
    SeqInfo s;
    s.n = __shfl_sync(0xffffffffu, q.n, src);
    s.start = __shfl_sync(0xffffffffu, q.start, src);
    s.ctx = __shfl_sync(0xffffffffu, q.ctx, src);
    const int groups = chunk_groups(s, g.P);
#pragma unroll 1
    for (int i0 = 0; i0 < groups; i0 += 32) {
      const int per_head = i0 + lane < groups ? chunk_units(s, g, i0 + lane) : 0;
      const int in = warp_scan_incl(per_head * g.hkv) + before;
      const unsigned here = __ballot_sync(0xffffffffu, in > r.u0);
      if (!here) {
        before = __shfl_sync(0xffffffffu, in, 31);
        continue;
      }
      const int at = __ffs(here) - 1;
      const int ph = __shfl_sync(0xffffffffu, per_head, at);
      const int off = r.u0 - __shfl_sync(0xffffffffu, in - per_head * g.hkv, at);
      r.i = i0 + at;
      r.h = off / ph;
      r.skip = off - r.h * ph;
      break;
    }
    break;
  }
  return r;
}

// A CTA's walk over its items, identical in every thread that runs one.
struct ChunkItem {
  SeqInfo q;
  int h;
  int t0, t1;        // new tokens of the group
  int lo, hi;        // keys its rows see
  int tile0;         // first key tile of the item
  int k0, k1;        // tiles of it in this CTA's range, from tile0
  bool whole;        // all of them
  int slot;          // partial slot of the CTA (0: begun before its range)
  int parts;         // when it begins here: CTAs that share it
};

struct ChunkWalk {
  int u, b, i, h, skip, loaded;
  ChunkRange r;
  SeqInfo q;
  __device__ __forceinline__ explicit ChunkWalk(const ChunkRange& r_)
      : u(r_.u0), b(r_.b), i(r_.i), h(r_.h), skip(r_.skip), loaded(-1), r(r_) {}
  // false at the end of the range
  __device__ __forceinline__ bool next(const RaggedView& rg, const ChunkGeo& g, int cta,
                                       ChunkItem& it) {
    while (u < r.u1) {
      if (h == g.hkv) { h = 0; ++i; }
      if (loaded != b) {
        q = chunk_seq(rg, g.bs, b, nullptr);
        loaded = b;
      }
      if (i >= chunk_groups(q, g.P)) {
        i = 0;
        if (++b >= rg.B) return false;
        continue;
      }
      it.t0 = i * g.P;
      it.t1 = min(q.n, it.t0 + g.P);
      chunk_keys(q, g, it.t0, it.t1, it.lo, it.hi);
      const int tiles = chunk_tiles(it.lo, it.hi, g.KT), units = tiles + chunk_fixed(g, it.t1 - it.t0);
      const int k0 = skip, k1 = g.split ? min(units, skip + (r.u1 - u)) : units;
      const int first = u - skip;
      u += k1 - k0;
      skip = 0;
      it.h = h++;
      // of another CTA, or nothing but the end of the item's fixed part
      if (k0 > 0 && (!g.split || k0 >= tiles)) continue;
      it.q = q;
      it.tile0 = tiles ? it.lo / g.KT : 0;
      it.k0 = k0;
      it.k1 = min(k1, tiles);
      it.whole = k0 == 0 && k1 >= tiles;
      it.slot = first < r.u0 ? 0 : 1;
      it.parts = it.whole || k0 > 0 ? 0 : (first + tiles - 1) / r.per_cta - cta + 1;
      return true;
    }
    return false;
  }
};

// Partial slots. A slot holds m [ROWS], l [ROWS] and o as [D / 4][ROWS]
// float4 columns (lanes of a warp own neighbouring rows, so both sides are
// whole lines); l and o count in units of 2^m.
struct ChunkMergeDesc {
  int32_t parts;       // CTAs that share the item (0: none)
  int32_t tok, rows;   // its first packed token; query rows
  int32_t head;
};
__host__ __device__ constexpr size_t chunk_slot_floats(int rows, int d) {
  return (size_t)rows * (d + 2);
}

// CTAs of a call at most: the workspace has a descriptor for each ahead of the partial slots,
// and the merges hold a weight for each in shared memory.
constexpr int kMaxCtas = 320;
inline int chunk_grid(int per_sm) {
  const int n = per_sm * num_sms();
  return n < kMaxCtas ? n : kMaxCtas;
}

// Whether a call's units fit 31 bits, and whether its items may be split.
inline bool chunk_fits(const RaggedView& rg, const ChunkGeo& g) {
  const int64_t tiles = ((int64_t)rg.W * g.bs + g.KT - 1) / g.KT + 1;
  return ((int64_t)rg.T / g.P + rg.B + 1) * g.hkv * (tiles + g.fixed + g.fixed_few) < (int64_t(1) << 31);
}
inline int chunk_may_split(const RaggedView& rg, int bs, int KT) {
  // up to four tiles: less than the merge's launch and the partials' way
  return ((int64_t)rg.W * bs + KT - 1) / KT > 4;
}

// ---- chunk_attend_tc.cu ----
bool chunk_tc_eligible(const KvView& kv, const ChunkView& c);
ChunkGeo chunk_tc_geo(const KvView& kv, const RaggedView& rg, const ChunkView& c);
int chunk_tc_rows();  // query rows of an item at most (a partial slot's rows)
cudaError_t launch_chunk_tc(const KvView& kv, const RaggedView& rg, const ChunkView& c, int ctas,
                            float* parts, ChunkMergeDesc* desc, int32_t* dev_err, cudaStream_t s);

// ---- chunk_attend_few.cu ----
int chunk_few_rows(const KvView& kv, const RaggedView& rg, const ChunkView& c);
int chunk_few_ctas();
ChunkGeo chunk_few_geo(const KvView& kv, const RaggedView& rg, const ChunkView& c, int rows);
cudaError_t launch_chunk_few(const KvView& kv, const RaggedView& rg, const ChunkView& c, int rows,
                             int ctas, float* parts, ChunkMergeDesc* desc, int32_t* dev_err,
                             cudaStream_t s);

}  // namespace cvsa
