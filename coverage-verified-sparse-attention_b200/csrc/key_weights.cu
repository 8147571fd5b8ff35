// Attention weight that cached keys got from the new tokens of a ragged batch.
//
// For key j of a sequence and KV head h, over the rows (token t, query head of h's
// group) that see j:
//   out_j = decay prior_j + sum_rows e^(scale q . k_j - lse_row),
// lse the rows' log-sum-exp from the attention; the new tokens' own keys start from
// 0 whatever `prior` holds there. Rows without a key (lse -inf) add nothing, masked
// entries are left out by selection. Sums are fp32.
//
// General kernel (any mix of fp32, bf16, f16, and 8-bit pools; head_dim 64, 128,
// 256): a block owns 64 keys of one KV head and goes over the rows that see any of
// them, 64 at a time, on the FMA units. A key's sum is one block's, so there are no
// atomics and the order of the sum is fixed. Bound by the FMA units and the shared
// memory that feeds them; it serves what the two others do not take (fp32, pools of
// another 16-bit type, head_dim 256, small odd pages, queries that no tensor copy reads).
//
// Which kernel: key_weights_few.cu up to 32 rows a sequence and KV head in the batch's
// mean (32 single tokens of 32 heads, 1 to 8192 bf16 keys: 70 us, here 805), beyond it
// key_weights_tc.cu (256 tokens at 32K 8-bit keys: 147 us, here 2331).
#include "chunk_plan.cuh"
#include "cvsa_common.cuh"
#include "cvsa_internal.h"
#include "fp8.cuh"
#include "weights_plan.cuh"

namespace cvsa {
namespace {

constexpr int kKeys = 64, kRows = 64, kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

struct WeightArgs {
  RaggedView rg;
  KvView kv;
  KeyWeightsView w;
  int G, tiles;       // query heads a KV head; key tiles a table row can name
  int32_t* dev_err;
};

// Four neighbouring elements of a row as floats.
__device__ __forceinline__ void load4(const void* p, int64_t at, int dtype, float* f) {
  if (dtype == CVSA_DTYPE_F32) {
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
  } else if (dtype == CVSA_DTYPE_E4M3) {
    e4m3x4_to_f4(*reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(p) + at), f);
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at);
    if (dtype == CVSA_DTYPE_F16) {
      f16x2_to_f2(v.x, f[0], f[1]);
      f16x2_to_f2(v.y, f[2], f[3]);
    } else {
      bf16x2_to_f2(v.x, f[0], f[1]);
      bf16x2_to_f2(v.y, f[2], f[3]);
    }
  }
}

template <int D>
struct WeightSmem {
  float q[kRows][D + 4];
  float k[kKeys][D + 4];
  float lse[kRows];
  float red[16][kKeys];
  int64_t off[kKeys];
  float scale[kKeys];
  int8_t ok[kKeys];
};

template <int D>
__global__ void __launch_bounds__(kThreads) key_weights_kernel(const __grid_constant__ WeightArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  WeightSmem<D>& sm = *reinterpret_cast<WeightSmem<D>*>(smem_raw);
  const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16, G = a.G;
  const int tile = blockIdx.x % a.tiles, h = blockIdx.x / a.tiles % a.kv.hkv,
            b = blockIdx.x / a.tiles / a.kv.hkv;
  const SeqInfo q = chunk_seq(a.rg, a.kv.bs, b, tile == 0 && h == 0 && tid == 0 ? a.dev_err : nullptr);
  const int key0 = tile * kKeys;
  if (key0 >= q.ctx) return;
  if (tid < kKeys) {
    int lo, hi;
    weight_keys(q, a.w.causal, a.w.window, lo, hi);
    const int key = key0 + tid;
    bool ok = key >= lo && key < hi;
    int64_t off = 0;
    float scale = 1.f;
    if (ok) {
      const int blk = a.rg.tables[(int64_t)q.slot * a.rg.W + key / a.kv.bs];
      ok = blk >= 0 && blk < a.kv.num_blocks;
      if (!ok) set_dev_error(a.dev_err, CVSA_DEV_ERR_BLOCK_RANGE);
      if (ok) {
        off = blk * a.kv.sb + (key % a.kv.bs) * a.kv.st + h * a.kv.sh;
        if (a.kv.ks) scale = pow2(scale_exponent_of(a.kv.ks[(int64_t)blk * a.kv.hkv + h]));
      }
    }
    sm.off[tid] = off;
    sm.scale[tid] = scale;
    sm.ok[tid] = ok;
  }
  __syncthreads();
  for (int e = tid; e < kKeys * (D / 4); e += kThreads) {
    const int r = e / (D / 4), c = e % (D / 4);
    float f[4] = {0.f, 0.f, 0.f, 0.f};
    if (sm.ok[r]) {
      load4(a.kv.k, sm.off[r] + c * 4, a.kv.dtype, f);
      if (a.kv.ks) f[0] *= sm.scale[r], f[1] *= sm.scale[r], f[2] *= sm.scale[r], f[3] *= sm.scale[r];
    }
    *reinterpret_cast<float4*>(&sm.k[r][c * 4]) = make_float4(f[0], f[1], f[2], f[3]);
  }
  // tokens [t0, t1) of the sequence see some key of the tile
  const int last = min(key0 + kKeys, q.ctx) - 1;
  const int t0 = a.w.causal ? (int)min((int64_t)q.n, max((int64_t)0, (int64_t)key0 - q.start)) : 0;
  const int t1 = a.w.window > 0 ? (int)min((int64_t)q.n, (int64_t)last + a.w.window - q.start) : q.n;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int64_t r0 = (int64_t)t0 * G; r0 < (int64_t)t1 * G; r0 += kRows) {
    __syncthreads();
    for (int e = tid; e < kRows * (D / 4); e += kThreads) {
      const int r = e / (D / 4), c = e % (D / 4);
      float f[4] = {0.f, 0.f, 0.f, 0.f};
      if (r0 + r < (int64_t)t1 * G)
        load4(a.w.q, (q.tok0 + (r0 + r) / G) * a.w.q_st + (h * G + (r0 + r) % G) * a.w.q_sh + c * 4,
              a.w.dtype, f);
      *reinterpret_cast<float4*>(&sm.q[r][c * 4]) = make_float4(f[0], f[1], f[2], f[3]);
    }
    if (tid < kRows)
      sm.lse[tid] = r0 + tid < (int64_t)t1 * G
                        ? a.w.lse[(q.tok0 + (r0 + tid) / G) * a.w.hq + h * G + (r0 + tid) % G]
                        : neg_inf();
    __syncthreads();
    float s[4][4] = {};
#pragma unroll 2
    for (int d = 0; d < D; d += 4) {
      float4 qa[4], kb[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) qa[x] = *reinterpret_cast<float4*>(&sm.q[ty * 4 + x][d]);
#pragma unroll
      for (int y = 0; y < 4; ++y) kb[y] = *reinterpret_cast<float4*>(&sm.k[tx + 16 * y][d]);
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          s[x][y] = fmaf(qa[x].x, kb[y].x, s[x][y]);
          s[x][y] = fmaf(qa[x].y, kb[y].y, s[x][y]);
          s[x][y] = fmaf(qa[x].z, kb[y].z, s[x][y]);
          s[x][y] = fmaf(qa[x].w, kb[y].w, s[x][y]);
        }
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float lse = sm.lse[ty * 4 + x];
      const int64_t pos = q.start + (r0 + ty * 4 + x) / G;
      const int64_t hi = a.w.causal ? pos : q.ctx - 1, lo = a.w.window > 0 ? pos - a.w.window + 1 : 0;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int key = key0 + tx + 16 * y;
        if (key <= hi && key >= lo && lse != neg_inf())
          acc[y] += exp2f(fmaf(s[x][y], a.w.scale, -lse) * kLog2e);
      }
    }
  }
#pragma unroll
  for (int y = 0; y < 4; ++y) sm.red[ty][tx + 16 * y] = acc[y];
  __syncthreads();
  const int key = key0 + tid;
  if (tid >= kKeys || key >= q.ctx) return;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += sm.red[i][tid];
  const int64_t at = ((int64_t)q.slot * a.kv.hkv + h) * a.w.stride + key;
  const float had = key < q.start ? a.w.decay * a.w.prior[at] : 0.f;
  a.w.out[at] = sm.ok[tid] ? had + sum : had;
}

int64_t weight_blocks(const KvView& kv, const RaggedView& rg) {
  return ((int64_t)rg.W * kv.bs + kKeys - 1) / kKeys * kv.hkv * rg.B;
}

template <int D>
cudaError_t launch_d(const WeightArgs& a, int64_t blocks, cudaStream_t s) {
  cudaError_t e = cudaFuncSetAttribute(key_weights_kernel<D>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)sizeof(WeightSmem<D>));
  if (e != cudaSuccess) return e;
  key_weights_kernel<D><<<(unsigned)blocks, kThreads, sizeof(WeightSmem<D>), s>>>(a);
  return cudaGetLastError();
}

}  // namespace

bool key_weights_supported(const KvView& kv, const RaggedView& rg, const KeyWeightsView& w) {
  return (kv.d == 64 || kv.d == 128 || kv.d == 256) && w.hq / kv.hkv <= 64 &&
         (int64_t)rg.W * kv.bs < (int64_t(1) << 31) && weight_blocks(kv, rg) < (int64_t(1) << 31) &&
         (int64_t)rg.T * w.hq < (int64_t(1) << 31);
}

cudaError_t launch_key_weights(const KvView& kv, const RaggedView& rg, const KeyWeightsView& w,
                               int32_t* dev_err, cudaStream_t s) {
  if (const int rows = weights_few_rows(kv, rg, w))
    return launch_weights_few(kv, rg, w, rows, dev_err, s);
  if (weights_tc_eligible(kv, rg, w)) {
    const cudaError_t e = launch_weights_tc(kv, rg, w, dev_err, s);
    if (e != cudaErrorNotSupported) return e;
  }
  WeightArgs a;
  a.rg = rg;
  a.kv = kv;
  a.w = w;
  a.G = w.hq / kv.hkv;
  a.tiles = (int)(((int64_t)rg.W * kv.bs + kKeys - 1) / kKeys);
  a.dev_err = dev_err;
  const int64_t blocks = weight_blocks(kv, rg);
  switch (kv.d) {
    case 64: return launch_d<64>(a, blocks, s);
    case 128: return launch_d<128>(a, blocks, s);
    default: return launch_d<256>(a, blocks, s);
  }
}

}  // namespace cvsa
