// Key weights of many rows on the tensor cores: 16-bit queries over a cache of their type
// or of 8 bits, head_dim 64 or 128. Formula in key_weights.cu, work split as in
// weights_plan.cuh.
//
// A persistent CTA an SM. An item is 256 keys of one KV head, kept in shared memory as two
// tiles of M, against the rows that see them, 64 at a time (N):
//   S' = K Q'   (fp32 in tensor memory, two buffers of two tiles, each half of the elements
//                a sum of its own: the tensor core cuts where an addition rounds, and one sum
//                of 128 products left twice the error of fp32's own)
// so that a thread owns a key and its sum over rows never leaves it. The scores of the
// next rows form while these are summed; the next item's keys are loaded meanwhile. 8-bit
// keys are widened to the queries' type as they are copied, once an item.
// Roles: warps 0-3 and 4-7 sum the first and the second tile of an item's even steps, warps
// 8-15 of its odd ones, warps 16-19 load keys, warps 20 and 23 issue the products of the
// first and the second tile (one warp for both was the bottleneck: 164 us), warps 21 and 22
// load queries and their log-sum-exps. Each follows the same list of items on its own.
//
// 256 tokens of 32 heads at 32K 8-bit keys take 147 us: 41 us of products at the tensor
// cores' rate, 60 us of exponentials (16 a clock and SM). Bound by the way of a buffer: its
// group sums 64 rows in 2700 cycles of the 4700 from one use to the next, and waits for the
// next products the rest (clocks read in the kernel: 460 cycles to issue a tile's, some 300
// for each of the three waits before them). A third buffer does not fit in tensor memory.
// Measured with one issuing warp and not kept: one sum of all products (122 us, twice fp32's
// error), one tile of M and four buffers (231), one group of warps reading 32 columns at a time
// (184), 64 columns at a time or reads ahead of their use (slower).
#include <cstddef>
#include <type_traits>

#include "cvsa_common.cuh"
#include "cvsa_internal.h"
#include "fp8.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"
#include "weights_plan.cuh"

namespace cvsa {
namespace {

constexpr int kThreads = 768, kTile = 128, kKeys = 2 * kTile, kRows = 64;
constexpr int kQBufs = 4, kRing = 8;
constexpr float kLog2e = 1.4426950408889634f;

struct WMeta {
  uint64_t k_full[2], k_empty[2], q_full[kQBufs], q_copied[kQBufs], q_empty[kQBufs], drain[2];
  uint64_t s_full[2][2], s_free[2][2];  // buffer, tile
  uint64_t joined[2][2], taken[2][2];   // items in turn, tile: the second group's sums
  // rows of a step, in a ring: those of step n are written over once the products of step
  // n + 4 are done. By then they were read: one of the steps between waits for n's
  // buffer, which is given back behind the last read, or for group 0 to be done with a step of a
  // later item than n's.
  alignas(16) float c[kRing][kRows];  // minus the log-sum-exp
  uint32_t live[kRing][2];            // bit per row that takes part (is there, saw a key)
  float second[2][2][kTile];          // items in turn, tile: the second group's sums
  uint32_t tmem, abort;
};
static_assert(offsetof(WMeta, c) % 16 == 0, "wide loads");

struct WArgs {
  RaggedView rg;
  KvView kv;
  KeyWeightsView w;
  WeightGeo g;
  int P;  // tokens of a step
  int32_t* dev_err;
  uint32_t wait_limit;
  alignas(64) CUtensorMap q_map;  // tiles of P tokens of a KV head's group
};

// Bounded wait; false (with the CTA's abort flag and CVSA_DEV_ERR_TIMEOUT set) when the
// phase does not complete, or another warp gave up. Whole warp, one answer.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, WMeta* m, const WArgs& a) {
  bool ok = false;
  for (uint32_t i = 0; i < a.wait_limit && !ok; ++i) {
    ok = mbar_try_wait(bar, parity);
    if (!ok && (i & 15) == 15 && *reinterpret_cast<volatile uint32_t*>(&m->abort)) break;
  }
  if (!ok && !*reinterpret_cast<volatile uint32_t*>(&m->abort)) {
    *reinterpret_cast<volatile uint32_t*>(&m->abort) = 1;
    set_dev_error(a.dev_err, CVSA_DEV_ERR_TIMEOUT);
  }
  return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ float ex2(float x) {
  // weights below 2^-126 are flushed to 0, far below the rounding of any sum
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(ok ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void arrive_when_landed(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
// 16-byte piece `ch` of row `row` of a tile of 128 rows, 128-byte swizzle.
__device__ __forceinline__ uint32_t piece(uint32_t tile, int row, int ch) {
  return tile + (ch >> 3) * (kTile * 128) + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
}

template <int D>
struct WCfg {
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kQ = 4 * kTileBytes;                // two buffers of two K tiles first
  static constexpr int kQBytes = kRows * D * 2;
  static constexpr int kMeta = kQ + kQBufs * kQBytes;
  static constexpr int kSmem = kMeta + (int)sizeof(WMeta) + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

// 32 rows r0.. of a tile; lane i's row is off elements into src (< 0: zeros).
template <typename T, int D>
__device__ __forceinline__ void copy_rows(uint32_t tile, int r0, const void* src, int64_t off) {
  constexpr int kCh = D / 8, kRPI = 32 / kCh;
  const int lane = threadIdx.x & 31, ch = lane % kCh;
#pragma unroll 4
  for (int i = 0; i < 32 / kRPI; ++i) {
    const int r = i * kRPI + lane / kCh;
    const int64_t o = __shfl_sync(0xffffffffu, off, r);
    cp16(piece(tile, r0 + r, ch), static_cast<const T*>(src) + (o < 0 ? 0 : o + ch * 8), o >= 0);
  }
}

// The same of 8-bit codes, widened to T with the rows' factors.
template <typename T, int D>
__device__ __forceinline__ void widen_rows(uint32_t tile, int r0, const void* src, int64_t off,
                                           float scale) {
  constexpr int kCh = D / 16, kRPI = 32 / kCh, kN = 32 / kRPI;
  const int lane = threadIdx.x & 31, ch = lane % kCh;
  uint4 codes[kN];  // all loads before the first store
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int64_t o = __shfl_sync(0xffffffffu, off, i * kRPI + lane / kCh);
    codes[i] = o < 0 ? make_uint4(0, 0, 0, 0)
                     : ldg_stream16(static_cast<const char*>(src) + o + ch * 16);
  }
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int r = i * kRPI + lane / kCh;
    const float f = __shfl_sync(0xffffffffu, scale, r);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&codes[i]);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t y[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x[4];
        e4m3x4_to_f4(w[half * 2 + j], x);
        y[2 * j] = Mma<T>::pack(x[0] * f, x[1] * f);
        y[2 * j + 1] = Mma<T>::pack(x[2] * f, x[3] * f);
      }
      asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(piece(tile, r0 + r, ch * 2 + half)),
                   "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3])
                   : "memory");
    }
  }
}

template <typename T, int D, bool F8>
__device__ __forceinline__ void key_role(const WArgs& a, WMeta* m, uint32_t base, WeightWalk walk,
                                         int w) {
  using C = WCfg<D>;
  const int lane = threadIdx.x & 31;
  uint32_t n = 0;
  for (; walk.next(a.rg, a.g); walk.step()) {
    int t0, t1;
    weight_tokens(walk.q, a.g, walk.i, t0, t1);
    if (t0 >= t1) continue;
    const uint32_t buf = n & 1;
    const int32_t* const table = a.rg.tables + (int64_t)walk.q.slot * a.rg.W;
    int lo, hi;
    weight_keys(walk.q, a.g.causal, a.g.window, lo, hi);
    // keys w * 64 + 32 k + lane of the tiles
    int64_t off[2];
    float scale[2] = {1.f, 1.f};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int key = walk.i * kKeys + w * 64 + k * 32 + lane;
      off[k] = -1;
      if (key < lo || key >= hi) continue;
      const int page = key / a.g.bs, blk = table[page];
      if (blk < 0 || blk >= a.kv.num_blocks) {
        set_dev_error(a.dev_err, CVSA_DEV_ERR_BLOCK_RANGE);
        continue;
      }
      off[k] = blk * a.kv.sb + (key - page * a.g.bs) * a.kv.st + walk.h * a.kv.sh;
      if constexpr (F8)
        scale[k] = pow2(scale_exponent_of(a.kv.ks[(int64_t)blk * a.kv.hkv + walk.h]));
    }
    if (!warp_wait(&m->k_empty[buf], ((n >> 1) & 1) ^ 1, m, a)) break;
    const uint32_t tile = base + (buf * 2 + w / 2) * C::kTileBytes;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r0 = (w & 1) * 64 + k * 32;
      if constexpr (F8) widen_rows<T, D>(tile, r0, a.kv.k, off[k], scale[k]);
      else copy_rows<T, D>(tile, r0, a.kv.k, off[k]);
    }
    if constexpr (F8) mbar_arrive(&m->k_full[buf]);
    else arrive_when_landed(&m->k_full[buf]);
    ++n;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// A step's query rows, (token, head of the group) in order, are a tile of their array: one
// tensor copy for each 64 elements. What else a step needs of them is written by two
// warps, 32 rows each; the next step's is looked up while this step's is on its way.
template <int D>
__device__ __forceinline__ void query_role(const WArgs& a, WMeta* m, uint32_t base, WeightWalk walk,
                                           int w) {
  using C = WCfg<D>;
  const int lane = threadIdx.x & 31, G = a.g.G;
  const int r = w * 32 + lane, rt = r / G, rh = r - rt * G;  // row, its token and head
  int ta = 0, t0 = 0, t1 = 0;
  bool more = true, first = true;
  float lse = neg_inf();
  auto look = [&]() {  // the first step, or the next one; more: there is one
    if (!first) ta += a.P;
    while (more && ta >= t1) {
      if (!first) walk.step();
      first = false;
      more = walk.next(a.rg, a.g);
      if (more) {
        weight_tokens(walk.q, a.g, walk.i, t0, t1);
        ta = t0;
      }
    }
    lse = neg_inf();
    if (more && rt < min(a.P, t1 - ta))
      lse = a.w.lse[(int64_t)(walk.q.tok0 + ta + rt) * a.w.hq + walk.h * G + rh];
  };
  look();
  uint32_t n = 0;
  for (; more; ++n) {
    const uint32_t buf = n % kQBufs, slot = n % kRing;
    if (!warp_wait(&m->q_empty[buf], ((n / kQBufs) & 1) ^ 1, m, a)) break;
    if (w == 0 && elect_one()) {
      mbar_arrive_expect_tx(&m->q_copied[buf], a.P * G * D * 2);
#pragma unroll
      for (int x = 0; x < D; x += 64)
        token_load(base + C::kQ + buf * C::kQBytes + x / 64 * (kRows * 128), &a.q_map, x,
                   walk.h * G, walk.q.tok0 + ta, &m->q_copied[buf]);
    }
    __syncwarp();
    const bool live = lse != neg_inf();
    m->c[slot][r] = live ? -lse : neg_inf();
    const uint32_t bits = __ballot_sync(0xffffffffu, live);
    if (lane == 0) m->live[slot][w] = bits;
    mbar_arrive(&m->q_full[buf]);
    look();
  }
  // no copy outlives the CTA, whatever gave up
  if (w == 0)
    for (uint32_t i = n > kQBufs ? n - kQBufs : 0; i < n; ++i)
      mbar_wait_bounded(&m->q_copied[i % kQBufs], (i / kQBufs) & 1, 1u << 18);
  __syncwarp();
}

// The whole warp runs the loop, its conditions broadcast, so that the compiler keeps the
// descriptors in uniform registers, where the instruction wants them; one elected lane issues.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

template <typename T, int D>
__device__ __forceinline__ void mma_role(const WArgs& a, WMeta* m, uint32_t base, uint32_t tmem,
                                         WeightWalk walk, int mt) {
  using C = WCfg<D>;
  constexpr uint32_t kId = mma_idesc(!std::is_same<T, __half>::value, kTile, kRows, false);
  const uint64_t k_desc = smem_desc(base, 16, 1024), q_desc = smem_desc(base + C::kQ, 16, 1024);
  uint32_t nk = 0, n = 0, odd = 0;  // bit b: buffer b was used an odd number of times
  for (; uniform(walk.next(a.rg, a.g)); walk.step()) {
    int t0, t1;
    weight_tokens(walk.q, a.g, walk.i, t0, t1);
    const int steps = uniform((t1 - t0 + a.P - 1) / a.P);
    if (steps <= 0) continue;
    const uint32_t kb = nk & 1;
    if (!warp_wait(&m->k_full[kb], (nk >> 1) & 1, m, a)) goto out;
    fence_proxy_async_smem();  // the keys were written through the generic proxy
    for (int j = 0; j < steps; ++j, ++n) {
      const uint32_t b = j & 1, qb = n % kQBufs, turn = (n / kQBufs) & 1;
      if (!warp_wait(&m->q_full[qb], turn, m, a)) goto out;
      if (!warp_wait(&m->q_copied[qb], turn, m, a)) goto out;
      if (!warp_wait(&m->s_free[b][mt], (odd >> b & 1) ^ 1, m, a)) goto out;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t kd = k_desc + (((kb * 2 + mt) * C::kTileBytes) >> 4);
        const uint64_t qd = q_desc + ((qb * C::kQBytes) >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t ko = ((kk / 4) * (kTile * 128) + (kk % 4) * 32) >> 4;
          const uint32_t qo = ((kk / 4) * (kRows * 128) + (kk % 4) * 32) >> 4;
          constexpr int kHalf = D / 32;  // each half of the elements has a sum of its own
          mma_ss(tmem + (b * 2 + mt) * 2 * kRows + kk / kHalf * kRows, kd + ko, qd + qo, kId,
                 kk % kHalf > 0);
        }
        mma_commit(smem_u32(&m->s_full[b][mt]));
        mma_commit(smem_u32(&m->q_empty[qb]));
        if (j == steps - 1) mma_commit(smem_u32(&m->k_empty[kb]));
      }
      __syncwarp();
      odd ^= 1u << b;
    }
    ++nk;
  }
out:
  // nothing of this CTA may be in flight when its tensor memory is freed
  if (elect_one()) mma_commit(smem_u32(&m->drain[mt]));
  __syncwarp();
  mbar_wait_bounded(&m->drain[mt], 0, 1u << 18);
  __syncwarp();
}

// Bits e of [from, to) that lie in [x, x + 32), at e - x.
__device__ __forceinline__ uint32_t bits_of(int from, int to, int x) {
  const int a = max(from - x, 0), b = to - x;
  return a >= 32 || b <= a ? 0u : (b >= 32 ? ~0u : (1u << b) - 1) & (~0u << a);
}

// Two groups of warps take an item's steps in turn, each those of its own buffer of scores,
// so that one's waits fall beside the other's exponentials. (A buffer is one group's: a
// barrier's parity says which of two phases is done, so who waits on it may not leave out
// a phase.)
__device__ __forceinline__ void sum_role(const WArgs& a, WMeta* m, uint32_t tmem, WeightWalk walk,
                                         int mt, int group) {
  const int warp = threadIdx.x >> 5 & 3, lane = threadIdx.x & 31, G = a.g.G;
  const uint64_t sc = f2_pack(a.w.scale, a.w.scale), l2 = f2_pack(kLog2e, kLog2e);
  uint32_t n = 0, items = 0, turns = 0;  // turns: steps of this group
  for (; walk.next(a.rg, a.g); walk.step(), ++items) {
    const SeqInfo& q = walk.q;
    int t0, t1;
    weight_tokens(q, a.g, walk.i, t0, t1);
    const int first = walk.i * kKeys + mt * kTile, key = first + warp * 32 + lane;
    const int last = min(first + kTile, q.ctx) - 1;  // of the tile's keys
    const bool there = key < q.ctx;
    const int64_t at = ((int64_t)q.slot * a.kv.hkv + walk.h) * a.w.stride + key;
    // what the key had and its page, not looked at before the sums are done
    const float prior = group == 0 && there && key < q.start ? a.w.prior[at] : 0.f;
    const int blk = group == 0 && there ? a.rg.tables[(int64_t)q.slot * a.rg.W + key / a.g.bs] : -1;
    // the tokens that see the key: ta and those after it, up to tb
    const int see0 = a.g.causal ? key - q.start : 0;
    const int see1 = a.g.window > 0 ? see0 + a.g.window : q.n;
    float total = 0.f;
    int mine = group;  // 0: this step is the group's
    for (int ta = t0; ta < t1; ta += a.P, ++n, mine ^= 1) {
      if (mine) continue;
      const uint32_t b = group, slot = n % kRing;
      const int tokens = min(a.P, t1 - ta), rows = tokens * G;
      // some row does not see every key of the tile
      const bool partial = (a.g.causal && q.start + ta < last) ||
                           (a.g.window > 0 && first <= q.start + ta + tokens - 1 - a.g.window);
      // rows [from, to) see the key
      const int from = partial ? min(max(see0 - ta, 0), a.P) * G : 0;
      const int to = partial ? min(max(see1 - ta, 0), a.P) * G : kRows;
      if (!warp_wait(&m->s_full[b][mt], turns & 1, m, a)) return;
      ++turns;
      tc_fence_after();
      const uint32_t ts = tmem + (b * 2 + mt) * 2 * kRows + ((uint32_t)(warp * 32) << 16);
      uint64_t sum0 = 0, sum1 = 0;
#pragma unroll 1
      for (int x = 0; x < rows; x += 16) {
        float s[16], s2[16];
        tmem_ld16(ts + x, s);
        tmem_ld16(ts + kRows + x, s2);
        const uint32_t sees = (bits_of(from, to, x) & m->live[slot][x / 32] >> x % 32) & 0xffff;
        const bool all = __all_sync(0xffffffffu, sees == 0xffff);
        tmem_wait_ld();
        uint64_t y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          y[i] = f2_add(f2_pack(s[2 * i], s[2 * i + 1]), f2_pack(s2[2 * i], s2[2 * i + 1]));
        float4 c4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) c4[i] = reinterpret_cast<const float4*>(m->c[slot] + x)[i];
        if (x + 16 >= rows) {  // all was read: the next products may go there
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&m->s_free[b][mt]);
        }
        if (all) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 c = c4[i];
            float u, v;
            f2_unpack(f2_mul(f2_fma(y[2 * i], sc, f2_pack(c.x, c.y)), l2), u, v);
            sum0 = f2_add(sum0, f2_pack(ex2(u), ex2(v)));
            f2_unpack(f2_mul(f2_fma(y[2 * i + 1], sc, f2_pack(c.z, c.w)), l2), u, v);
            sum1 = f2_add(sum1, f2_pack(ex2(u), ex2(v)));
          }
        } else if (__any_sync(0xffffffffu, sees != 0)) {
          float add = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float4 c = c4[i / 4];
            const float z = i % 4 == 0 ? c.x : i % 4 == 1 ? c.y : i % 4 == 2 ? c.z : c.w;
            float u, v;
            f2_unpack(y[i / 2], u, v);
            const float e = ex2(fmaf(i & 1 ? v : u, a.w.scale, z) * kLog2e);
            add += sees >> i & 1 ? e : 0.f;
          }
          sum0 = f2_add(sum0, f2_pack(add, 0.f));
        }
      }
      float u, v;
      f2_unpack(f2_add(sum0, sum1), u, v);
      total += u + v;
    }
    const uint32_t ib = items & 1, turn = (items >> 1) & 1;
    float* const other = &m->second[ib][mt][warp * 32 + lane];
    if (group) {
      if (!warp_wait(&m->taken[ib][mt], turn ^ 1, m, a)) return;
      *other = total;
      __syncwarp();
      if (lane == 0) mbar_arrive(&m->joined[ib][mt]);
      continue;
    }
    if (!warp_wait(&m->joined[ib][mt], turn, m, a)) return;
    total += *other;
    __syncwarp();
    if (lane == 0) mbar_arrive(&m->taken[ib][mt]);
    if (there) {
      const float had = a.w.decay * prior;
      a.w.out[at] = blk >= 0 && blk < a.kv.num_blocks ? had + total : had;
    }
  }
}

template <typename T, int D, bool F8>
__global__ void __launch_bounds__(kThreads, 1) weights_tc_kernel(const __grid_constant__ WArgs a) {
  using C = WCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  WMeta* m = reinterpret_cast<WMeta*>(smem + C::kMeta);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&m->k_full[i], 128);
      mbar_init(&m->k_empty[i], 2);
      mbar_init(&m->drain[i], 1);
      for (int mt = 0; mt < 2; ++mt) {
        mbar_init(&m->s_full[i][mt], 1);
        mbar_init(&m->s_free[i][mt], 4);
        mbar_init(&m->joined[i][mt], 4);
        mbar_init(&m->taken[i][mt], 4);
      }
    }
    for (int i = 0; i < kQBufs; ++i) {
      mbar_init(&m->q_full[i], 64);  // the plain writes
      mbar_init(&m->q_copied[i], 1);
      mbar_init(&m->q_empty[i], 2);
    }
    m->abort = 0;
    fence_mbar_init();
  }
  if (warp == 20) tmem_alloc(smem_u32(&m->tmem), 512);
  const WeightRange r = weight_range(a.rg, a.g, blockIdx.x, gridDim.x,
                                     warp == 0 ? a.dev_err : nullptr);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t base = smem_u32(smem), tmem = __shfl_sync(0xffffffffu, m->tmem, 0);
  const WeightWalk walk(r);
  if (warp < 16) sum_role(a, m, tmem, walk, warp / 4 & 1, warp / 8);
  else if (warp < 20) key_role<T, D, F8>(a, m, base, walk, warp - 16);
  else if (warp == 20 || warp == 23) mma_role<T, D>(a, m, base, tmem, walk, warp == 23);
  else query_role<D>(a, m, base, walk, warp - 21);
  tc_fence_before();
  __syncthreads();
  if (warp == 20) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int D, bool F8>
cudaError_t launch_one(const WArgs& a, cudaStream_t s) {
  constexpr int kSmem = WCfg<D>::kSmem;
  const cudaError_t e = cudaFuncSetAttribute(weights_tc_kernel<T, D, F8>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  weights_tc_kernel<T, D, F8><<<num_sms(), kThreads, kSmem, s>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_t(const WArgs& a, cudaStream_t s) {
  const bool f8 = a.kv.dtype == CVSA_DTYPE_E4M3;
  if (a.kv.d == 64) return f8 ? launch_one<T, 64, true>(a, s) : launch_one<T, 64, false>(a, s);
  return f8 ? launch_one<T, 128, true>(a, s) : launch_one<T, 128, false>(a, s);
}

}  // namespace

bool weights_tc_eligible(const KvView& kv, const RaggedView& rg, const KeyWeightsView& w) {
  return rg.T > 0 && (kv.dtype == w.dtype || kv.dtype == CVSA_DTYPE_E4M3) && w.dtype != CVSA_DTYPE_F32 &&
         (kv.d == 64 || kv.d == 128);
}

cudaError_t launch_weights_tc(const KvView& kv, const RaggedView& rg, const KeyWeightsView& w,
                              int32_t* dev_err, cudaStream_t s) {
  WArgs a;
  a.rg = rg;
  a.kv = kv;
  a.w = w;
  a.g.bs = kv.bs;
  a.g.hkv = kv.hkv;
  a.g.G = w.hq / kv.hkv;
  a.g.KT = kKeys;
  a.P = kRows / a.g.G;
  a.g.rows = a.P * a.g.G;
  a.g.fixed = 1;
  a.g.causal = w.causal;
  a.g.window = w.window;
  a.dev_err = dev_err;
  if (!token_map(&a.q_map, w.q, w.dtype == CVSA_DTYPE_BF16, rg.T, w.hq, kv.d, w.q_st, w.q_sh, a.P,
                 a.g.G))
    return cudaErrorNotSupported;
  a.wait_limit = wait_limit() ? wait_limit() : 1u << 18;  // a poll waits about 4 us: a second
  return w.dtype == CVSA_DTYPE_BF16 ? launch_t<__nv_bfloat16>(a, s) : launch_t<__half>(a, s);
}

}  // namespace cvsa
