// Key weights of few new tokens a sequence (single tokens, drafts): 16-bit queries over a
// cache of their type or of 8 bits, head_dim 64 or 128, pages of a multiple of 16 tokens.
// Formula in key_weights.cu, work split as in weights_plan.cuh, a range a warp.
//
// Bound by the keys' bytes: 32 single tokens of 32 heads at 1 to 8192 bf16 keys take 70 us,
// 50 of them the bytes at the rate of a copy, the rest the first loads and the ranges'
// uneven ends (one at 128K keys 59 us, over 8 bits 49). Blocks of 16 keys that no row sees
// are not read, their weights are decayed beside (with a window of 16 keys: 14 us). As in
// chunk_attend_few.cu, keys go from memory to the operands of mma.sync in the registers of
// the lane that loads them: S' = K Q', 16 keys by 8 rows, lane (g, t) with 16-byte pieces
// of keys g and g + 8 and the same elements of query row g. A key's weights are summed over the two rows of a lane, the row tiles and
// the four lanes of its row, so nothing else is exchanged and a warp works on its own.
// 16-bit keys are used as they are; 8-bit ones are widened to f16, with queries scaled by
// row to fit. A sequence of more rows than a step holds (ROWS) goes over them in turn for
// each block of keys, reading its queries again.
#include <type_traits>

#include "cvsa_common.cuh"
#include "cvsa_internal.h"
#include "fp8.cuh"
#include "weights_plan.cuh"

namespace cvsa {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps, kTileKeys = 64;
constexpr float kLog2e = 1.4426950408889634f;

struct FewWeightArgs {
  RaggedView rg;
  KvView kv;
  KeyWeightsView w;
  WeightGeo g;
  int32_t* dev_err;
};

__device__ __forceinline__ float ex2(float x) {
  // weights below 2^-126 are flushed to 0, far below the rounding of any sum
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// TI: the queries' type; F8: an 8-bit cache
template <typename TI, int D, int ROWS, bool F8>
__global__ void __launch_bounds__(kThreads) weights_few_kernel(const __grid_constant__ FewWeightArgs a) {
  using T = typename std::conditional<F8, __half, TI>::type;  // of the operands
  constexpr int kNt = ROWS / 8, kSteps = D / 16;
  constexpr int kPieces = D * (F8 ? 1 : 2) / 64;  // 16-byte pieces of a key that a lane holds
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int worker = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int G = a.g.G, bs = a.kv.bs, hkv = a.kv.hkv;
  WeightWalk walk(weight_range(a.rg, a.g, worker, gridDim.x * kWarps, a.dev_err));
  bool more = walk.next(a.rg, a.g);
  const int64_t st = a.kv.st * (F8 ? 1 : 2);  // bytes between keys
  while (more) {
    // a run of tiles of one head
    const int b = walk.b, h = walk.h, first = walk.i * kTileKeys;
    const SeqInfo q = walk.q;
    int end = first;
    do {
      end = min(q.ctx, (walk.i + 1) * kTileKeys);
      walk.step();
      more = walk.next(a.rg, a.g);
    } while (more && walk.b == b && walk.h == h);
    const int rows = q.n * G;  // at most 2^31 by the call's check
    const int32_t* const table = a.rg.tables + (int64_t)q.slot * a.rg.W;
    const int64_t at_out = ((int64_t)q.slot * hkv + h) * a.w.stride;
    // n blocks of 16 keys from key0 on hold all keys of the run that some row sees
    int lo, stop;
    weight_keys(q, a.g.causal, a.g.window, lo, stop);
    lo = max(first, lo & ~15);
    stop = min(stop, end);
    const int n = lo < stop ? (stop - lo + 15) / 16 : 0, key0 = n ? lo : end;
    auto unseen = [&](int from, int to) {
      for (int key = from + lane; key < to; key += 32)
        a.w.out[at_out + key] = key < q.start ? a.w.decay * a.w.prior[at_out + key] : 0.f;
    };
    unseen(first, key0);
    unseen(key0 + 16 * n, end);
    if (n == 0) continue;
    // Queries r0.. as operands, their factors and what is subtracted; rows that are not
    // there or saw no key take no part.
    uint32_t qb[kNt][kSteps][2];
    float f[kNt][2], c[kNt][2];
    int pos[kNt][2];
    uint32_t live = 0;  // bits x * 2 + e
    auto queries = [&](int r0) {
      live = 0;
#pragma unroll
      for (int x = 0; x < kNt; ++x) {
        const int r = r0 + x * 8 + g;
        const bool there = r < rows;
        const TI* src = static_cast<const TI*>(a.w.q) +
                        (int64_t)(q.tok0 + (there ? r / G : 0)) * a.w.q_st +
                        (int64_t)(h * G + (there ? r % G : 0)) * a.w.q_sh;
        if constexpr (F8) {
          // codes t * 16.. of each 64 of a key: the same elements of the row
          uint4 raw[D / 64][2];
          float top = 0.f;
#pragma unroll
          for (int y = 0; y < D / 64; ++y)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              raw[y][i] = there ? *reinterpret_cast<const uint4*>(src + y * 64 + t * 16 + i * 8)
                                : make_uint4(0, 0, 0, 0);
              float e[8];
              Vec16<TI>::unpack(raw[y][i], e);
#pragma unroll
              for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(e[j]));
            }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int up = min(120, 13 + 127 - (__float_as_int(top) >> 23));
          const float by = pow2(up);
#pragma unroll
          for (int y = 0; y < D / 64; ++y)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float e[8];
              Vec16<TI>::unpack(raw[y][i], e);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                qb[x][y * 4 + i * 2 + j / 2][j % 2] =
                    Mma<__half>::pack(e[2 * j] * by, e[2 * j + 1] * by);
            }
#pragma unroll
          for (int e = 0; e < 2; ++e)
            f[x][e] = a.w.scale * pow2(-__shfl_sync(0xffffffffu, up, (2 * t + e) * 4));
        } else {
          // 8 elements t * 8.. of each 32 of a key: two steps
#pragma unroll
          for (int y = 0; y < D / 32; ++y) {
            const uint4 v = there ? *reinterpret_cast<const uint4*>(src + y * 32 + t * 8)
                                  : make_uint4(0, 0, 0, 0);
            qb[x][2 * y][0] = v.x, qb[x][2 * y][1] = v.y;
            qb[x][2 * y + 1][0] = v.z, qb[x][2 * y + 1][1] = v.w;
          }
          f[x][0] = f[x][1] = a.w.scale;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = r0 + x * 8 + 2 * t + e;
          const float lse = row < rows ? a.w.lse[(int64_t)(q.tok0 + row / G) * a.w.hq + h * G + row % G]
                                       : neg_inf();
          c[x][e] = -lse;
          pos[x][e] = q.start + (row < rows ? row / G : 0);
          if (lse != neg_inf()) live |= 1u << (x * 2 + e);
        }
      }
    };
    queries(0);
    // Lane i: page of block i0 + i (-1: out of range) and K's factor.
    auto find = [&](int i0, int& blk, float& ks) {
      const int key = key0 + (i0 + lane) * 16;
      blk = -1;
      ks = 1.f;
      if (key >= stop) return;
      blk = table[key / bs];
      if (blk < 0 || blk >= a.kv.num_blocks) {
        set_dev_error(a.dev_err, CVSA_DEV_ERR_BLOCK_RANGE);
        blk = -1;
      } else if constexpr (F8) {
        ks = a.kv.ks[(int64_t)blk * hkv + h];
      }
    };
    int blk0, blk1 = -1;
    float ks0, ks1 = 1.f;
    find(0, blk0, ks0);
    uint4 ck[2][kPieces];  // pieces of keys g, g + 8
    float had = 0.f;       // what key g + 8 t had, t < 2
    auto load = [&](int i) {
      if (i >= n) return;
      const int blk = max(0, __shfl_sync(0xffffffffu, i & 32 ? blk1 : blk0, i & 31));
      const int key = key0 + i * 16;
      // pages hold whole blocks, so keys past the context may be read
      const char* const p = static_cast<const char*>(a.kv.k) +
                            (blk * a.kv.sb + h * a.kv.sh) * (F8 ? 1 : 2) + (key % bs + g) * st + t * 16;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int x = 0; x < kPieces; ++x) ck[r][x] = ldg_stream16(p + r * 8 * st + x * 64);
      const int mine = key + g + 8 * t;
      had = t < 2 && mine < end && mine < q.start ? a.w.prior[at_out + mine] : 0.f;
    };
    load(0);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      if ((i & 31) == 16) {  // the next 32 blocks' pages, ahead of their loads
        if (i & 32) find((i & ~31) + 32, blk0, ks0);
        else find((i & ~31) + 32, blk1, ks1);
      }
      const bool good = __shfl_sync(0xffffffffu, i & 32 ? blk1 : blk0, i & 31) >= 0;
      const float ks =
          F8 ? pow2(scale_exponent_of(__shfl_sync(0xffffffffu, i & 32 ? ks1 : ks0, i & 31))) : 1.f;
      const int key = key0 + i * 16;
      uint32_t ka[kSteps][4];
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if constexpr (F8) {
            const uint4& v = ck[r][j / 4];
            e4m3x4_to_f16x4(j % 4 == 0 ? v.x : j % 4 == 1 ? v.y : j % 4 == 2 ? v.z : v.w, ka[j][r],
                            ka[j][2 + r]);
          } else {
            const uint4& v = ck[r][j / 2];
            ka[j][r] = j % 2 ? v.z : v.x;
            ka[j][2 + r] = j % 2 ? v.w : v.y;
          }
        }
      const float had_here = had;
      load(i + 1);
      float sum[2] = {0.f, 0.f};  // keys g, g + 8
#pragma unroll 1
      for (int r0 = 0;; r0 += ROWS) {
        if (r0 > 0 || (rows > ROWS && i > 0)) queries(r0);
        // some row does not see every key, or takes no part
        const int pos0 = q.start + r0 / G, pos1 = q.start + (min(rows, r0 + ROWS) - 1) / G;
        const bool partial = live != (1u << 2 * kNt) - 1 || (a.g.causal && key + 15 > pos0) ||
                             (a.g.window > 0 && key <= pos1 - a.g.window);
#pragma unroll
        for (int x = 0; x < kNt; ++x) {
          // The tensor core cuts its sums where an addition rounds them: pairs of steps, whose
          // sums are added (errors 2.0e-6 of the weights with one sum of 128 products, fp32's
          // own 1.1e-6).
          float s[4];
#pragma unroll
          for (int j = 0; j < kSteps; j += 2) {
            float y[4] = {0.f, 0.f, 0.f, 0.f};
            Mma<T>::m16n8k16(y, ka[j], qb[x][j][0], qb[x][j][1]);
            Mma<T>::m16n8k16(y, ka[j + 1], qb[x][j + 1][0], qb[x][j + 1][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = j ? s[e] + y[e] : y[e];
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // key g + 8 (e / 2), row 2t + e % 2
            const float u = ex2(fmaf(s[e], f[x][e & 1] * ks, c[x][e & 1]) * kLog2e);
            const int at = key + g + 8 * (e >> 1), p = pos[x][e & 1];
            const bool sees = !partial || ((live >> (x * 2 + (e & 1)) & 1) &&
                                           (!a.g.causal || at <= p) &&
                                           (a.g.window == 0 || at > p - a.g.window));
            sum[e >> 1] += sees ? u : 0.f;
          }
        }
        if (r0 + ROWS >= rows) break;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 1);
        sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 2);
      }
      const int mine = key + g + 8 * t;
      if (t < 2 && mine < end) {
        const float old = mine < q.start ? a.w.decay * had_here : 0.f;
        a.w.out[at_out + mine] = good ? old + (t ? sum[1] : sum[0]) : old;
      }
    }
  }
}

template <typename TI, int D, bool F8>
cudaError_t launch_rows(const FewWeightArgs& a, int rows, cudaStream_t s) {
  // blocks that an SM holds at once; all devices are of one kind
  auto resident = [](auto kernel) {
    int n = 0;
    return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kThreads, 0) == cudaSuccess && n > 0 ? n : 1;
  };
  if (rows == 8) {
    static const int per_sm = resident(weights_few_kernel<TI, D, 8, F8>);
    weights_few_kernel<TI, D, 8, F8><<<num_sms() * per_sm, kThreads, 0, s>>>(a);
  } else {
    static const int per_sm = resident(weights_few_kernel<TI, D, 16, F8>);
    weights_few_kernel<TI, D, 16, F8><<<num_sms() * per_sm, kThreads, 0, s>>>(a);
  }
  return cudaGetLastError();
}

template <typename TI>
cudaError_t launch_t(const FewWeightArgs& a, int rows, cudaStream_t s) {
  const bool f8 = a.kv.dtype == CVSA_DTYPE_E4M3;
  if (a.kv.d == 64) return f8 ? launch_rows<TI, 64, true>(a, rows, s) : launch_rows<TI, 64, false>(a, rows, s);
  return f8 ? launch_rows<TI, 128, true>(a, rows, s) : launch_rows<TI, 128, false>(a, rows, s);
}

}  // namespace

// Rows of a step, or 0 where the other kernels serve the call: by the batch's mean of
// rows a sequence, as in chunk_attend_few.cu. At 32 rows (8 tokens of 4 heads a KV head)
// two steps of 16 go over a block of keys; beyond, key_weights_tc.cu's tiles of 64 rows
// fill better.
int weights_few_rows(const KvView& kv, const RaggedView& rg, const KeyWeightsView& w) {
  if ((kv.dtype != w.dtype && kv.dtype != CVSA_DTYPE_E4M3) || w.dtype == CVSA_DTYPE_F32 ||
      (kv.d != 64 && kv.d != 128) || kv.bs % 16)
    return 0;
  const int64_t rows = ((int64_t)rg.T + rg.B - 1) / rg.B * (w.hq / kv.hkv);
  return rows <= 8 ? 8 : rows <= 32 ? 16 : 0;
}

cudaError_t launch_weights_few(const KvView& kv, const RaggedView& rg, const KeyWeightsView& w,
                               int rows, int32_t* dev_err, cudaStream_t s) {
  FewWeightArgs a;
  a.rg = rg;
  a.kv = kv;
  a.w = w;
  a.g.bs = kv.bs;
  a.g.hkv = kv.hkv;
  a.g.G = w.hq / kv.hkv;
  a.g.KT = kTileKeys;
  a.g.rows = rows;
  a.g.fixed = 1;
  a.g.causal = w.causal;
  a.g.window = w.window;
  a.dev_err = dev_err;
  return w.dtype == CVSA_DTYPE_BF16 ? launch_t<__nv_bfloat16>(a, rows, s) : launch_t<__half>(a, rows, s);
}

}  // namespace cvsa
