// Eviction from the paged cache by accumulated attention weight.
//
// A sequence longer than `keep` keeps, for each KV head, its first `sink` keys, its
// last `recent` ones and those of largest weight between (equal weights: the earlier
// key; NaN below everything), `keep` in all, in their order. Their keys, values and
// weights move to the front: rows to new pages, so that no row is written over
// before it is read and all rows can move at once. In place, the weights behind the
// kept ones become 0, up to the old length.
//
// select: a cluster of 1 to 8 blocks a (sequence, KV head), each with a piece of the row
//   in shared memory. The cut, the n-th largest weight, is found by a radix select over
//   the weights' order-preserving keys, 11, 11 and 10 bits a pass, over the sum of the
//   blocks' histograms; a pass in order then writes the kept keys, placed by a prefix sum.
//   Bound by latency, a dozen rounds of block and cluster barriers: 32K keys of 8 heads
//   to 4096 take 25 us (one block a row 70).
// gather: one warp a new page and KV head; bound by bytes and, for few pages, by the three
//   loads that follow one another (kept key, table, row): 4096 keys of 8 heads 9 us. In an 8-bit cache a new
//   page gets the largest scale of the rows that go there, so none overflows; rows of
//   smaller scale move to it (exact but for values that become subnormal).
// reserve, commit: the page bookkeeping around them, one block each.
#include <cooperative_groups.h>

#include "block_scan.cuh"
#include "cvsa_common.cuh"
#include "cvsa_internal.h"
#include "cvsa_launch.cuh"
#include "fp8.cuh"

namespace cg = cooperative_groups;

namespace cvsa {
namespace {

constexpr int kThreads = 1024, kBins = 2048, kEach = 8;

struct SelectArgs {
  EvictView e;
  int hkv, bs;
  int parts;   // blocks a row
  int cached;  // keys of a piece that shared memory holds (all of it unless parts is 1)
  int32_t* dev_err;
};

// The sequence's length where it is evicted from, else 0.
__device__ __forceinline__ int evict_len(const EvictView& e, int bs, int s, int32_t* dev_err) {
  const int len = e.lens[s];
  if (len < 0 || len > (int64_t)e.W * bs) {
    set_dev_error(dev_err, CVSA_DEV_ERR_RAGGED);
    return 0;
  }
  return len > e.keep ? len : 0;
}

__global__ void __launch_bounds__(kThreads) evict_select_kernel(const __grid_constant__ SelectArgs a) {
  extern __shared__ float piece[];  // [cached]
  __shared__ int hist[2][kBins];
  __shared__ int sums[32];
  __shared__ int s_bin, s_left, s_all;
  __shared__ int counts[2];  // of this piece: taken above the cut or in any case, equal to it
  const cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, parts = a.parts, part = blockIdx.x % parts;
  const int s = blockIdx.x / parts / a.hkv, h = blockIdx.x / parts % a.hkv;
  const int len = evict_len(a.e, a.bs, s, tid == 0 && part == 0 && h == 0 ? a.dev_err : nullptr);
  int32_t* const kept = a.e.kept + ((int64_t)s * a.hkv + h) * a.e.keep;
  if (len == 0) {  // the same in all blocks of the row
    for (int i = part * kThreads + tid; i < a.e.keep; i += parts * kThreads) kept[i] = -1;
    return;
  }
  const float* const w = a.e.weights + ((int64_t)s * a.hkv + h) * a.e.w_stride;
  float* const out = a.e.out_weights + ((int64_t)s * a.hkv + h) * a.e.o_stride;
  const int lo = a.e.sink, hi = len - a.e.recent;
  const int size = (len + parts - 1) / parts, p0 = min(len, part * size), p1 = min(len, p0 + size);
  for (int i = p0 + tid; i < min(p1, p0 + a.cached); i += kThreads) piece[i - p0] = w[i];
  auto weight = [&](int i) { return i - p0 < a.cached ? piece[i - p0] : w[i]; };
  int left = a.e.keep - a.e.sink - a.e.recent;  // to take of [lo, hi)
  uint32_t cut = 0xffffffffu;  // keys above are taken
  int room = 0;                // and this many of those equal to it
  if (left > 0) {
    uint32_t prefix = 0, mask = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass < 2 ? 11 : 10;
      int* const mine = hist[pass & 1];
      for (int i = tid; i < kBins; i += kThreads) mine[i] = 0;
      __syncthreads();
      for (int i0 = p0; i0 < p1; i0 += kThreads) {
        const int i = i0 + tid;
        const bool in = i < p1 && i >= lo && i < hi;
        const uint32_t k = in ? float_key(weight(i)) : 0;
        const int bin = in && (k & mask) == prefix ? (int)(k >> shift & ((1 << bits) - 1)) : -1;
        // neighbouring keys share bins: one addition a warp and bin
        const unsigned same = __match_any_sync(0xffffffffu, bin);
        if (bin >= 0 && __ffs(same) - 1 == lane) atomicAdd(&mine[bin], __popc(same));
      }
      // Every block sums the row's histograms. (The other buffer is cleared a pass later,
      // when all blocks have passed this point and so are done with it.)
      if (parts > 1) cluster.sync(); else __syncthreads();
      // bin that holds the left-th key from the top: sums from the highest bin
      const int top = kBins - 1 - 2 * tid;
      int c0 = 0, c1 = 0;
      for (int p = 0; p < parts; ++p) {
        const int* const theirs = parts > 1 ? cluster.map_shared_rank(mine, p) : mine;
        c0 += theirs[top];
        c1 += theirs[top - 1];
      }
      const int incl = block_scan_incl(c0 + c1, sums);
      const int before = incl - c0 - c1;
      if (before < left && incl >= left) {
        const bool first = before + c0 >= left;
        s_bin = first ? top : top - 1;
        s_left = left - (first ? before : before + c0);
        s_all = s_left == (first ? c0 : c1);
      }
      __syncthreads();
      prefix |= (uint32_t)s_bin << shift;
      mask |= (uint32_t)((1 << bits) - 1) << shift;
      left = s_left;
      const bool all = s_all && prefix > 0;
      __syncthreads();
      cut = prefix;
      room = left;
      if (all) {  // the whole bin is taken (22 bits mostly tell weights apart): no more passes
        cut = prefix - 1;
        room = 0;
        break;
      }
    }
  } else {
    __syncthreads();
  }
  // kEach neighbours a thread from i0 on: which are taken in any case or above the cut,
  // and which are equal to it
  auto look = [&](int i0, float* x, uint32_t& above, uint32_t& same) {
    above = same = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = i0 + tid * kEach + j;
      x[j] = i < p1 ? weight(i) : 0.f;
      const uint32_t k = float_key(x[j]);
      const bool forced = i < lo || i >= hi;
      if (i < p1 && (forced || k > cut)) above |= 1u << j;
      if (i < p1 && !forced && k == cut && room > 0) same |= 1u << j;
    }
  };
  int taken = 0, equal = 0;  // before the keys at hand
  float x[kEach];
  uint32_t above, same;
  if (parts > 1) {
    if (tid < 2) counts[tid] = 0;
    __syncthreads();
    int n_above = 0, n_same = 0;
    for (int i0 = p0; i0 < p1; i0 += kThreads * kEach) {
      look(i0, x, above, same);
      n_above += __popc(above);
      n_same += __popc(same);
    }
    n_above = __reduce_add_sync(0xffffffffu, n_above);
    n_same = __reduce_add_sync(0xffffffffu, n_same);
    if (lane == 0) {
      atomicAdd(&counts[0], n_above);
      atomicAdd(&counts[1], n_same);
    }
    // beyond this point weights may be written over: every block holds its piece
    cluster.sync();
    for (int p = 0; p < part; ++p) {
      const int* const theirs = cluster.map_shared_rank(counts, p);
      taken += theirs[0];
      equal += theirs[1];
    }
    cluster.sync();  // the others' counts were read
  }
  // in order; a key's place is the number taken before it
  for (int i0 = p0; i0 < p1; i0 += kThreads * kEach) {
    const int base = i0 + tid * kEach;
    look(i0, x, above, same);
    // both counts in one scan: at most kThreads * kEach = 8192 of each
    const int mine = __popc(above) | __popc(same) << 16;
    const int incl = block_scan_incl(mine, sums);
    int a0 = taken + ((incl - mine) & 0xffff), q0 = equal + ((incl - mine) >> 16);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const bool is_above = above >> j & 1, is_same = same >> j & 1;
      if (is_above || (is_same && q0 < room)) {
        const int at = a0 + min(q0, room);
        kept[at] = base + j;
        out[at] = x[j];  // at <= base + j: held by a block, or read by this round or before
      }
      a0 += is_above;
      q0 += is_same;
    }
    if (tid == kThreads - 1) sums[0] = incl;
    __syncthreads();
    taken += sums[0] & 0xffff;
    equal += sums[0] >> 16;
    __syncthreads();
  }
  // In place, what stood behind the kept weights belongs to no key any more: a key that takes
  // such a slot without being counted begins at 0. (This piece was read by now, by its block.)
  if (out == w)
    for (int i = max(p0, a.e.keep) + tid; i < p1; i += kThreads) out[i] = 0.f;
  pdl_launch_dependents();
}

struct GatherArgs {
  EvictView e;
  KvView kv;
  int eb;        // bytes of an element
  int chunks;    // 16-byte chunks of a row
  int32_t* dev_err;
};

constexpr int kGatherWarps = 4, kBatch = 4;

template <bool F8>
__global__ void __launch_bounds__(kGatherWarps * 32) evict_gather_kernel(const __grid_constant__ GatherArgs a) {
  const int lane = threadIdx.x & 31, bs = a.kv.bs, hkv = a.kv.hkv;
  const int64_t warp = (int64_t)blockIdx.x * kGatherWarps + (threadIdx.x >> 5);
  const int h = (int)(warp % hkv), page = (int)(warp / hkv % a.e.new_pages);
  const int64_t s = warp / hkv / a.e.new_pages;
  if (s >= a.e.S) return;
  const int to = a.e.new_tables[s * a.e.new_pages + page];
  const int len = evict_len(a.e, bs, (int)s, nullptr);
  pdl_wait();  // the kept keys
  if (len == 0) return;
  if (to < 0 || to >= a.kv.num_blocks) {
    if (lane == 0) set_dev_error(a.dev_err, CVSA_DEV_ERR_BLOCK_RANGE);
    return;
  }
  const int n = (int)min((int64_t)bs, a.e.keep - (int64_t)page * bs);  // rows of the page
  const int32_t* const kept = a.e.kept + (s * hkv + h) * a.e.keep + (int64_t)page * bs;
  const uint8_t* const pk = static_cast<const uint8_t*>(a.kv.k);
  const uint8_t* const pv = static_cast<const uint8_t*>(a.kv.v);
  // lane i: byte offset of row r0 + i of the page (-1: none) and its block
  auto locate = [&](int r0, int& blk) -> int64_t {
    blk = -1;
    if (r0 + lane >= n) return -1;
    const int key = kept[r0 + lane];
    blk = a.e.tables[s * a.e.W + key / bs];
    if (blk < 0 || blk >= a.kv.num_blocks) {
      set_dev_error(a.dev_err, CVSA_DEV_ERR_BLOCK_RANGE);
      blk = -1;
      return -1;
    }
    return (blk * a.kv.sb + (key % bs) * a.kv.st + h * a.kv.sh) * a.eb;
  };
  int ek = kScaleMin, ev = kScaleMin;  // exponents of the new page
  int blk0;
  const int64_t off0 = locate(0, blk0);
  int mk = kScaleMin, mv = kScaleMin;  // of the lane's row's page
  if constexpr (F8) {
    for (int r0 = 0; r0 < n; r0 += 32) {
      int blk = blk0;
      if (r0 > 0) locate(r0, blk);
      if (blk >= 0) {
        mk = scale_exponent_of(a.kv.ks[(int64_t)blk * hkv + h]);
        mv = scale_exponent_of(a.kv.vs[(int64_t)blk * hkv + h]);
        ek = max(ek, mk);
        ev = max(ev, mv);
      }
    }
    ek = __reduce_max_sync(0xffffffffu, ek);
    ev = __reduce_max_sync(0xffffffffu, ev);
    if (lane == 0) {
      const_cast<float*>(a.kv.ks)[(int64_t)to * hkv + h] = pow2(ek);
      const_cast<float*>(a.kv.vs)[(int64_t)to * hkv + h] = pow2(ev);
    }
  }
  uint8_t* const base_k = const_cast<uint8_t*>(pk) + (to * a.kv.sb + h * a.kv.sh) * a.eb;
  uint8_t* const base_v = const_cast<uint8_t*>(pv) + (to * a.kv.sb + h * a.kv.sh) * a.eb;
  const int64_t st = a.kv.st * a.eb;
  for (int r0 = 0; r0 < n; r0 += 32) {
    int blk = blk0;
    const int64_t off = n > 32 ? locate(r0, blk) : off0;
    float fk = 1.f, fv = 1.f;
    if constexpr (F8) {
      if (n > 32 && blk >= 0) {
        mk = scale_exponent_of(a.kv.ks[(int64_t)blk * hkv + h]);
        mv = scale_exponent_of(a.kv.vs[(int64_t)blk * hkv + h]);
      }
      fk = pow2(mk - ek);
      fv = pow2(mv - ev);
    }
    const int pieces = min(32, n - r0) * a.chunks;
    for (int e0 = 0; e0 < pieces; e0 += 32 * kBatch) {
      uint4 xk[kBatch], xv[kBatch];
      int64_t from[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int e = e0 + i * 32 + lane, r = min(e / a.chunks, 31);
        from[i] = __shfl_sync(0xffffffffu, off, r);
        if (e >= pieces) from[i] = -1;
        if (from[i] < 0) continue;
        const int64_t at = from[i] + e % a.chunks * 16;
        xk[i] = *reinterpret_cast<const uint4*>(pk + at);
        xv[i] = *reinterpret_cast<const uint4*>(pv + at);
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int e = e0 + i * 32 + lane, r = min(e / a.chunks, 31);
        if constexpr (F8) {
          const float yk = __shfl_sync(0xffffffffu, fk, r), yv = __shfl_sync(0xffffffffu, fv, r);
          if (from[i] >= 0) {
            uint32_t* wk = reinterpret_cast<uint32_t*>(&xk[i]);
            uint32_t* wv = reinterpret_cast<uint32_t*>(&xv[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float f[4];
              e4m3x4_to_f4(wk[j], f);
              wk[j] = f4_to_e4m3x4(f[0] * yk, f[1] * yk, f[2] * yk, f[3] * yk);
              e4m3x4_to_f4(wv[j], f);
              wv[j] = f4_to_e4m3x4(f[0] * yv, f[1] * yv, f[2] * yv, f[3] * yv);
            }
          }
        }
        if (from[i] < 0) continue;
        const int64_t at = (r0 + e / a.chunks) * st + e % a.chunks * 16;
        *reinterpret_cast<uint4*>(base_k + at) = xk[i];
        *reinterpret_cast<uint4*>(base_v + at) = xv[i];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// pages: one block; the sequences' numbers are prefix sums in batch order
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kThreads) evict_reserve_kernel(const __grid_constant__ EvictPages p,
                                                                 int32_t* dev_err) {
  __shared__ int64_t sums[32];
  __shared__ int64_t s_first[kThreads];  // place of a sequence's first new page in the free list
  const int tid = threadIdx.x;
  const int64_t head = *p.free_head;
  // a sequence's pages to give back, or -1: it is not evicted from
  auto gives = [&](int b) {
    if (b >= p.S) return -1;
    const int len = p.lens[b], old = p.pages_alloc[b];
    if (len < 0 || len > (int64_t)p.W * p.bs || old < 0 || old > p.W) {
      set_dev_error(dev_err, CVSA_DEV_ERR_RAGGED);
      return -1;
    }
    return len > p.keep ? old : -1;
  };
  const int64_t most = head < 0 || head > p.free_len ? 0 : (p.free_len - head) / p.new_pages;
  // pages that come back from the sequences that get theirs: the first `most`
  int64_t want = 0, back = 0;
  for (int b0 = 0; b0 < p.S; b0 += kThreads) {
    const int g = gives(b0 + tid);
    const int64_t nth = want + block_scan_incl((int64_t)(g >= 0), sums);
    const int64_t came = block_scan_incl((int64_t)(g >= 0 && nth <= most ? g : 0), sums);
    if (tid == kThreads - 1) sums[0] = nth, sums[1] = came;
    __syncthreads();
    want = sums[0];
    back += sums[1];
    __syncthreads();
  }
  const int64_t got = min(want, most);
  // the list has no room for pages that it did not hand out: nothing is evicted
  const bool fits = back <= head + got * p.new_pages;
  if (tid == 0 && (want > most || (want > 0 && !fits))) set_dev_error(dev_err, CVSA_DEV_ERR_POOL);
  int64_t seen = 0;
  for (int b0 = 0; b0 < p.S; b0 += kThreads) {
    const int b = b0 + tid;
    const int g = gives(b);
    const int64_t nth = seen + block_scan_incl((int64_t)(g >= 0), sums);
    const bool ok = g >= 0 && fits && nth <= most;
    if (b < p.S) p.plan_lens[b] = ok ? p.lens[b] : 0;
    s_first[tid] = ok ? head + (nth - 1) * p.new_pages : -1;
    if (tid == kThreads - 1) sums[0] = nth;
    __syncthreads();
    seen = sums[0];
    const int rows = min(kThreads, p.S - b0);
    for (int64_t e = tid; e < (int64_t)rows * p.new_pages; e += kThreads) {
      const int64_t first = s_first[e / p.new_pages];
      p.new_tables[(int64_t)b0 * p.new_pages + e] =
          first >= 0 ? p.free_list[first + e % p.new_pages] : -1;
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kThreads) evict_commit_kernel(const __grid_constant__ EvictPages p) {
  __shared__ int64_t sums[32];
  __shared__ int64_t s_incl[kThreads];
  const int tid = threadIdx.x;
  const int64_t head = *p.free_head;
  int64_t got = 0, back = 0;
  for (int b0 = 0; b0 < p.S; b0 += kThreads) {
    const int b = b0 + tid;
    const bool ok = b < p.S && p.plan_lens[b] > 0;
    const int64_t n = block_scan_incl((int64_t)ok, sums);
    const int64_t g = block_scan_incl((int64_t)(ok ? p.pages_alloc[b] : 0), sums);
    if (tid == kThreads - 1) sums[0] = n, sums[1] = g;
    __syncthreads();
    got += sums[0];
    back += sums[1];
    __syncthreads();
  }
  int64_t at = head + got * p.new_pages - back;  // the list's new head
  const int64_t new_head = at;
  for (int b0 = 0; b0 < p.S; b0 += kThreads) {
    const int b = b0 + tid;
    const bool ok = b < p.S && p.plan_lens[b] > 0;
    s_incl[tid] = block_scan_incl((int64_t)(ok ? p.pages_alloc[b] : 0), sums);
    __syncthreads();
    const int64_t total = s_incl[kThreads - 1];
    for (int64_t e = tid; e < total; e += kThreads) {
      int lo = 0, hi = kThreads - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_incl[mid] > e) hi = mid; else lo = mid + 1;
      }
      p.free_list[at + e] = p.tables[(int64_t)(b0 + lo) * p.W + (e - (lo ? s_incl[lo - 1] : 0))];
    }
    at += total;
    __syncthreads();
    const int rows = min(kThreads, p.S - b0);
    for (int64_t e = tid; e < (int64_t)rows * p.new_pages; e += kThreads) {
      const int64_t row = b0 + e / p.new_pages;
      if (p.plan_lens[row] > 0)
        p.tables[row * p.W + e % p.new_pages] = p.new_tables[row * p.new_pages + e % p.new_pages];
    }
    if (ok) {
      p.evicted[b] += p.plan_lens[b] - p.keep;
      p.lens[b] = p.keep;
      p.pages_alloc[b] = p.new_pages;
    }
    __syncthreads();
  }
  if (tid == 0) *p.free_head = (int)new_head;
}

}  // namespace

bool evict_supported(const KvView& kv, const EvictView& e) {
  return (int64_t)e.S * kv.hkv < (int64_t(1) << 28) && (int64_t)e.W * kv.bs < (int64_t(1) << 30) &&
         (int64_t)e.S * e.new_pages * kv.hkv / kGatherWarps < (int64_t(1) << 31) - 1;
}

cudaError_t launch_evict(const KvView& kv, const EvictView& e, int32_t* dev_err, cudaStream_t s) {
  SelectArgs a;
  a.e = e;
  a.hkv = kv.hkv;
  a.bs = kv.bs;
  a.dev_err = dev_err;
  // Blocks a row: two for each SM in all while their pieces are of 8192 keys or more, and as
  // many as hold the row, if any do: alone, a block reads what it cannot hold again. The whole
  // call with 2, 4 and 8 blocks a row: 51, 39 and 43 us for 32K keys of 8 heads, for 131K
  // keys 88 us with 4 and 66 with 8.
  constexpr int kCached = 48 * 1024, kMost = 8;
  const int64_t row = (int64_t)e.W * kv.bs, rows = (int64_t)e.S * kv.hkv;
  a.parts = 1;
  while (a.parts < kMost && ((row > (int64_t)a.parts * 8192 && rows * a.parts < 2 * num_sms()) ||
                             row > (int64_t)a.parts * kCached))
    a.parts *= 2;
  if (row > (int64_t)a.parts * kCached) a.parts = 1;
  const int64_t size = (row + a.parts - 1) / a.parts;
  a.cached = size < kCached ? (int)size : kCached;
  if (rows * a.parts >= (int64_t(1) << 31)) return cudaErrorInvalidValue;
  cudaError_t err = cudaFuncSetAttribute(
      evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kCached * 4);
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * a.parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)a.cached * 4;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)a.parts, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  err = cudaLaunchKernelEx(&cfg, evict_select_kernel, a);
  if (err != cudaSuccess) return err;
  GatherArgs g;
  g.e = e;
  g.kv = kv;
  g.eb = dtype_bytes(kv.dtype);
  g.chunks = kv.d * g.eb / 16;
  g.dev_err = dev_err;
  const int64_t warps = (int64_t)e.S * e.new_pages * kv.hkv;
  const unsigned blocks = (unsigned)((warps + kGatherWarps - 1) / kGatherWarps);
  return launch_k(kv.dtype == CVSA_DTYPE_E4M3 ? evict_gather_kernel<true> : evict_gather_kernel<false>,
                  dim3(blocks), dim3(kGatherWarps * 32), 0, s, true, g);
}

cudaError_t launch_evict_reserve(const EvictPages& p, int32_t* dev_err, cudaStream_t s) {
  evict_reserve_kernel<<<1, kThreads, 0, s>>>(p, dev_err);
  return cudaGetLastError();
}

cudaError_t launch_evict_commit(const EvictPages& p, int32_t* dev_err, cudaStream_t s) {
  evict_commit_kernel<<<1, kThreads, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace cvsa
