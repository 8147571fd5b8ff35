// How the attention of a ragged batch of new tokens is cut into work for a
// persistent grid, shared by the kernels that compute it.
//
// An item is one KV head of one group of P consecutive new tokens of one
// sequence (all query heads of the KV head: P * G query rows); it walks the
// KT-key tiles its rows can see, one unit of work a tile (an item that sees
// none counts one, so its rows are still written). The items in the order
// (sequence, group, head) form one stream of units that is cut into equal
// contiguous ranges, one a CTA, so the load is even whatever the mix of long
// and short contexts, and a long cache with few queries is split over all CTAs
// by the same rule. An item inside one range is finished by its CTA; an item
// that crosses ranges leaves one partial (m, l, o) a CTA, merged in CTA order
// by a second kernel. A CTA has at most two such items (its first and its
// last), so two partial slots each.
//
// Lengths live on the device, so every CTA finds its own range: the threads
// evaluate the groups of all sequences in parallel (a block scan a thousand
// groups), which costs about a microsecond and no extra launch.
#pragma once

#include "cvsa_common.cuh"
#include "cvsa_internal.h"

namespace cvsa {

struct ChunkGeo {
  int bs, hkv, G;
  int P;        // new tokens a group
  int KT;       // keys a tile
  int causal, window;
};

struct SeqInfo {
  int tok0, n;     // rows of the packed token arrays
  int slot;        // row of the tables
  int start, ctx;  // position of the first new token; keys the sequence holds
};

// Sequence b; every field ends in range whatever the arrays hold.
__device__ __forceinline__ SeqInfo chunk_seq(const RaggedView& rg, int bs, int b,
                                             int32_t* dev_err) {
  SeqInfo q;
  q.tok0 = rg.cu[b];
  const int end = rg.cu[b + 1];
  q.slot = rg.seq_ids ? rg.seq_ids[b] : b;
  q.n = end - q.tok0;
  q.start = q.ctx = 0;
  if (q.tok0 < 0 || end > rg.T || end < q.tok0 || q.slot < 0 || q.slot >= rg.num_seqs) {
    set_dev_error(dev_err, CVSA_DEV_ERR_RAGGED);
    q.n = 0;
    q.slot = 0;
    return q;
  }
  q.ctx = rg.lens[q.slot];
  q.start = rg.starts ? rg.starts[b] : q.ctx - q.n;
  if (q.ctx < 0 || q.ctx > (int64_t)rg.W * bs) {
    set_dev_error(dev_err, CVSA_DEV_ERR_RAGGED);
    q.ctx = q.ctx < 0 ? 0 : rg.W * bs;
  }
  if (rg.starts && q.start < 0) q.start = q.ctx = 0;  // refused: its rows see no key
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

__device__ __forceinline__ int chunk_units(const SeqInfo& q, const ChunkGeo& g, int i) {
  int lo, hi;
  chunk_keys(q, g, i * g.P, min(q.n, (i + 1) * g.P), lo, hi);
  return max(1, chunk_tiles(lo, hi, g.KT));
}

// What the CTA at `cta` of `ctas` does: units [u0, u1) of the stream, starting
// at unit `skip` of item (b, i, h).
struct ChunkRange {
  long long u0, u1, per_cta;
  int b, i, h, skip;
};

template <int NT>
struct ChunkPlanSmem {
  int incl[NT];            // inclusive sum of the groups of a round's sequences
  SeqInfo seq[NT];
  long long warp_sums[NT / 32];
  long long carry;
  int total;
  ChunkRange range;
};

template <int NT>
__device__ __forceinline__ long long chunk_scan_incl(long long v, long long* warp_sums) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  if (lane == 31) warp_sums[wid] = v;
  __syncthreads();
  long long before = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) before += w < wid ? warp_sums[w] : 0;
  __syncthreads();
  return v + before;
}

// Runs `visit(pair, b, i, units, incl)` for every group of the batch in
// stream order, NT at a time, all threads together (units = 0 and b = -1
// beyond the end; units already times the heads, incl = inclusive sum over
// the whole stream so far). Returns the stream's total.
template <int NT, typename Visit>
__device__ __forceinline__ long long chunk_enumerate(const RaggedView& rg, const ChunkGeo& g,
                                                     ChunkPlanSmem<NT>& sm, int32_t* dev_err,
                                                     Visit visit) {
  const int tid = threadIdx.x;
  long long base = 0;
  for (int b0 = 0; b0 < rg.B; b0 += NT) {
    int ng = 0;
    if (b0 + tid < rg.B) {
      const SeqInfo q = chunk_seq(rg, g.bs, b0 + tid, dev_err);
      sm.seq[tid] = q;
      ng = chunk_groups(q, g.P);
    }
    const long long in = chunk_scan_incl<NT>(ng, sm.warp_sums);
    sm.incl[tid] = (int)in;
    __syncthreads();
    const int total = sm.incl[NT - 1];
    for (int p0 = 0; p0 < total; p0 += NT) {
      const int p = p0 + tid;
      int b = -1, i = 0;
      long long units = 0;
      if (p < total) {
        int lo = 0, hi = NT - 1;
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (sm.incl[mid] > p) hi = mid; else lo = mid + 1;
        }
        i = p - (lo ? sm.incl[lo - 1] : 0);
        b = b0 + lo;
        units = (long long)chunk_units(sm.seq[lo], g, i) * g.hkv;
      }
      const long long incl = base + chunk_scan_incl<NT>(units, sm.warp_sums);
      visit(b, i, units, incl);
      if (tid == NT - 1) sm.carry = incl;
      __syncthreads();
      base = sm.carry;
    }
    __syncthreads();
  }
  return base;
}

// The range of CTA `cta`; every thread of the block returns it. Ranges are at
// least `min_units` long: a partial costs its write and its read by the merge,
// which a tile or two do not pay for.
template <int NT>
__device__ __forceinline__ ChunkRange chunk_range(const RaggedView& rg, const ChunkGeo& g,
                                                  ChunkPlanSmem<NT>& sm, int cta, int ctas,
                                                  int min_units, int32_t* dev_err) {
  int kb = -1, ki = 0, rounds = 0;
  long long kunits = 0, kincl = 0;
  const long long total = chunk_enumerate<NT>(
      rg, g, sm, cta == 0 ? dev_err : nullptr, [&](int b, int i, long long units, long long incl) {
        kb = b; ki = i; kunits = units; kincl = incl;
        ++rounds;
      });
  ChunkRange r;
  r.per_cta = max((long long)min_units, (total + ctas - 1) / ctas);
  r.u0 = min(total, cta * (long long)r.per_cta);
  r.u1 = min(total, r.u0 + r.per_cta);
  r.b = r.i = r.h = r.skip = 0;
  if (r.u0 >= r.u1) return r;
  auto find = [&](int b, int i, long long units, long long incl) {
    if (b >= 0 && incl > r.u0 && incl - units <= r.u0) {
      ChunkRange f = r;
      const int per_head = (int)(units / g.hkv);
      const int off = (int)(r.u0 - (incl - units));
      f.b = b; f.i = i; f.h = off / per_head; f.skip = off % per_head;
      sm.range = f;
    }
  };
  if (rounds == 1) {
    find(kb, ki, kunits, kincl);  // one round held every group: its values are still here
    __syncthreads();
  } else {
    chunk_enumerate<NT>(rg, g, sm, nullptr, find);
  }
  r = sm.range;
  __syncthreads();
  return r;
}

// A CTA's walk over its items, identical in every thread that runs one.
struct ChunkItem {
  SeqInfo q;
  int i, h;
  int t0, t1;        // new tokens of the group
  int lo, hi;        // keys its rows see
  int tile0;         // first key tile of the item
  int units;         // units of the whole item
  int k0, k1;        // units of it in this CTA's range
  long long first;   // stream position of its unit 0
};

struct ChunkWalk {
  long long u, u1;
  int b, i, h, skip, loaded;
  SeqInfo q;
  __device__ __forceinline__ explicit ChunkWalk(const ChunkRange& r)
      : u(r.u0), u1(r.u1), b(r.b), i(r.i), h(r.h), skip(r.skip), loaded(-1) {}
  // false at the end of the range
  __device__ __forceinline__ bool next(const RaggedView& rg, const ChunkGeo& g, ChunkItem& it) {
    if (u >= u1) return false;
    if (h == g.hkv) { h = 0; ++i; }
    for (;;) {
      if (loaded != b) {
        q = chunk_seq(rg, g.bs, b, nullptr);
        loaded = b;
      }
      if (i < chunk_groups(q, g.P)) break;
      i = 0;
      if (++b >= rg.B) return false;
    }
    it.q = q;
    it.i = i;
    it.h = h;
    it.t0 = i * g.P;
    it.t1 = min(q.n, it.t0 + g.P);
    chunk_keys(q, g, it.t0, it.t1, it.lo, it.hi);
    it.tile0 = it.hi > it.lo ? it.lo / g.KT : 0;
    it.units = max(1, chunk_tiles(it.lo, it.hi, g.KT));
    it.k0 = skip;
    it.k1 = (int)min((long long)it.units, skip + (u1 - u));
    it.first = u - skip;
    u += it.k1 - it.k0;
    skip = 0;
    ++h;
    return true;
  }
};

// Partial slots. A slot holds m [ROWS], l [ROWS] and o as [D / 4][ROWS]
// float4 columns (lanes of a warp own neighbouring rows, so both sides are
// whole lines); m is a maximum in the base-2 domain.
struct ChunkMergeDesc {
  int32_t parts;       // CTAs that share the item (0: none)
  int32_t tok, rows;   // its first packed token; query rows
  int32_t head;
};
__host__ __device__ constexpr size_t chunk_slot_floats(int rows, int d) {
  return (size_t)rows * (d + 2);
}
__device__ __forceinline__ int chunk_slot(const ChunkItem& it, long long u0, int cta) {
  return 2 * cta + (it.first < u0 ? 0 : 1);
}

// ---- chunk_attend_tc.cu ----
bool chunk_tc_eligible(const KvView& kv, const ChunkView& c);
int chunk_tc_rows();  // query rows of an item at most (a partial slot's rows)
cudaError_t launch_chunk_tc(const KvView& kv, const RaggedView& rg, const ChunkView& c, int ctas,
                            float* parts, ChunkMergeDesc* desc, int32_t* dev_err, cudaStream_t s);

}  // namespace cvsa
