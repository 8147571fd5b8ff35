// How key_weights is cut into work, shared by its kernels.
//
// An item is a tile of KT keys of one KV head of one sequence, with all rows that see
// any of them. It counts `fixed` units plus one for each `rows` query rows that do. The
// items in the order (sequence, head, tile) form one stream that is cut into equal
// ranges, one a worker (a CTA or a warp), which takes the items that begin in its range
// whole: a key's sum is one worker's. Lengths live on the device, so every worker finds
// its own range, a whole warp 32 sequences or tiles a step.
#pragma once

#include "chunk_plan.cuh"

namespace cvsa {

struct WeightGeo {
  int bs, hkv, G, KT;
  int rows, fixed;
  int causal, window;
};

__device__ __forceinline__ int weight_tiles(const SeqInfo& q, int KT) {
  return (q.ctx + KT - 1) / KT;
}

// Keys [lo, hi) of the sequence that some row sees. Others keep their decayed weight, and a page
// of such keys alone is not looked up, as in the attention.
__device__ __forceinline__ void weight_keys(const SeqInfo& q, int causal, int window, int& lo,
                                            int& hi) {
  const int64_t end = causal ? (int64_t)q.start + q.n : q.ctx;
  lo = window > 0 ? (int)max((int64_t)0, (int64_t)q.start - window + 1) : 0;
  hi = q.n > 0 ? (int)max((int64_t)0, min(end, (int64_t)q.ctx)) : 0;
}

// Tokens [t0, t1) of the sequence see some key of tile i.
__device__ __forceinline__ void weight_tokens(const SeqInfo& q, const WeightGeo& g, int i, int& t0,
                                              int& t1) {
  const int64_t first = (int64_t)i * g.KT, last = min(first + g.KT, (int64_t)q.ctx) - 1;
  t0 = g.causal ? (int)min((int64_t)q.n, max((int64_t)0, first - q.start)) : 0;
  t1 = g.window > 0 ? (int)max((int64_t)t0, min((int64_t)q.n, last + g.window - q.start)) : q.n;
}

// Whether the sequence's tiles all count the same (its rows are one step).
__device__ __forceinline__ bool weight_even(const SeqInfo& q, const WeightGeo& g) {
  return (int64_t)q.n * g.G <= g.rows;
}

__device__ __forceinline__ int weight_units(const SeqInfo& q, const WeightGeo& g, int i) {
  if (weight_even(q, g)) return g.fixed + (q.n > 0);
  int t0, t1;
  weight_tokens(q, g, i, t0, t1);
  return g.fixed + (int)(((int64_t)(t1 - t0) * g.G + g.rows - 1) / g.rows);
}

struct WeightRange {
  int64_t units;  // of items that begin in the range (0: nothing)
  int b, h, i;    // the first of them
};

// Units of one head of 32 sequences from b0, one a lane.
__device__ __forceinline__ int64_t weight_seq_units(const RaggedView& rg, const WeightGeo& g,
                                                    int b0, SeqInfo& q, int32_t* dev_err) {
  const int lane = threadIdx.x & 31;
  q.n = q.ctx = q.start = 0;
  if (b0 + lane < rg.B) q = chunk_seq(rg, g.bs, b0 + lane, dev_err);
  const int nt = weight_tiles(q, g.KT);
  const bool even = weight_even(q, g);
  int64_t units = even ? (int64_t)nt * weight_units(q, g, 0) : 0;
  for (unsigned many = __ballot_sync(0xffffffffu, !even && nt > 0); many; many &= many - 1) {
    const int src = __ffs(many) - 1;
    SeqInfo s;
    s.n = __shfl_sync(0xffffffffu, q.n, src);
    s.start = __shfl_sync(0xffffffffu, q.start, src);
    s.ctx = __shfl_sync(0xffffffffu, q.ctx, src);
    const int tiles = weight_tiles(s, g.KT);
    int64_t sum = 0;
    for (int i = lane; i < tiles; i += 32) sum += weight_units(s, g, i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == src) units = sum;
  }
  return units;
}

__device__ __forceinline__ int64_t warp_scan_incl64(int64_t v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, v, o);
    if ((int)(threadIdx.x & 31) >= o) v += t;
  }
  return v;
}

// The range of worker w of `workers`, by a whole warp; every lane returns it.
__device__ __forceinline__ WeightRange weight_range(const RaggedView& rg, const WeightGeo& g, int w,
                                                    int workers, int32_t* dev_err) {
  const int lane = threadIdx.x & 31;
  SeqInfo q = {};
  int64_t units = 0, total = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < rg.B; b0 += 32) {
    units = weight_seq_units(rg, g, b0, q, w == 0 ? dev_err : nullptr);
    int64_t sum = units;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    total += sum * g.hkv;
  }
  WeightRange r = {0, 0, 0, 0};
  const int64_t per = (total + workers - 1) / workers, u0 = min(total, w * per),
                u1 = min(total, u0 + per);
  if (u0 >= u1) return r;
  int64_t before = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < rg.B; b0 += 32) {
    if (rg.B > 32) units = weight_seq_units(rg, g, b0, q, nullptr);  // else still in registers
    const int64_t incl = warp_scan_incl64(units * g.hkv) + before;
    const unsigned past = __ballot_sync(0xffffffffu, incl > u0);
    if (!past) {
      before = __shfl_sync(0xffffffffu, incl, 31);
      continue;
    }
    const int src = __ffs(past) - 1;
    const int64_t per_head = __shfl_sync(0xffffffffu, units, src);
    int64_t off = u0 - __shfl_sync(0xffffffffu, incl - units * g.hkv, src);
    SeqInfo s;
    s.n = __shfl_sync(0xffffffffu, q.n, src);
    s.start = __shfl_sync(0xffffffffu, q.start, src);
    s.ctx = __shfl_sync(0xffffffffu, q.ctx, src);
    r.b = b0 + src;
    r.h = (int)(off / per_head);
    off -= r.h * per_head;
    // the first tile that begins at or past `off` units of the head
    const int tiles = weight_tiles(s, g.KT);
    int64_t at = 0;  // where tile r.i begins
    if (weight_even(s, g)) {
      const int each = weight_units(s, g, 0);
      r.i = (int)((off + each - 1) / each);
      at = (int64_t)r.i * each;
    } else {
      r.i = tiles;
      at = per_head;
      int64_t sum = 0;
#pragma unroll 1
      for (int i0 = 0; i0 < tiles; i0 += 32) {
        const int mine = i0 + lane < tiles ? weight_units(s, g, i0 + lane) : 0;
        const int64_t in = warp_scan_incl64(mine) + sum;
        const unsigned here = __ballot_sync(0xffffffffu, i0 + lane < tiles && in - mine >= off);
        if (here) {
          const int lead = __ffs(here) - 1;
          r.i = i0 + lead;
          at = __shfl_sync(0xffffffffu, in - mine, lead);
          break;
        }
        sum = __shfl_sync(0xffffffffu, in, 31);
      }
    }
    r.units = u1 - u0 - (at - off);  // may be <= 0: no item begins in the range
    break;
  }
  return r;
}

// A worker's items, the same in every thread that runs it.
struct WeightWalk {
  int64_t left;
  int b, h, i, loaded;
  SeqInfo q;
  __device__ __forceinline__ explicit WeightWalk(const WeightRange& r)
      : left(r.units), b(r.b), h(r.h), i(r.i), loaded(-1) {}
  // false at the end; else (b, h, i) is the item and `q` its sequence. `step` goes on.
  __device__ __forceinline__ bool next(const RaggedView& rg, const WeightGeo& g) {
    while (left > 0 && b < rg.B) {
      if (loaded != b) {
        q = chunk_seq(rg, g.bs, b, nullptr);
        loaded = b;
      }
      if (i < weight_tiles(q, g.KT) && h < g.hkv) {
        left -= weight_units(q, g, i);
        return true;
      }
      i = 0;
      if (++h >= g.hkv || q.ctx == 0) h = 0, ++b;
    }
    return false;
  }
  __device__ __forceinline__ void step() { ++i; }
};

// ---- key_weights_few.cu ----
int weights_few_rows(const KvView& kv, const RaggedView& rg, const KeyWeightsView& w);
cudaError_t launch_weights_few(const KvView& kv, const RaggedView& rg, const KeyWeightsView& w,
                               int rows, int32_t* dev_err, cudaStream_t s);

// ---- key_weights_tc.cu ----
bool weights_tc_eligible(const KvView& kv, const RaggedView& rg, const KeyWeightsView& w);
// cudaErrorNotSupported, with nothing launched, for queries whose strides no tensor map takes
cudaError_t launch_weights_tc(const KvView& kv, const RaggedView& rg, const KeyWeightsView& w,
                              int32_t* dev_err, cudaStream_t s);

}  // namespace cvsa
