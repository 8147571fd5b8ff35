// Attention of a ragged batch of new tokens over the paged cache: the general
// kernel (any mix of fp32, bf16, f16) and the merge of split items.
//
// Row (token t, query head h) at position p sees keys [lo, hi): hi = p + 1
// (causal) or the context length, lo = max(0, p - window + 1) or 0.
//   s_j = scale * q . k_j,  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),
//   lse = m + log sum_j e^(s_j - m); a row without a key: out 0, lse -inf.
// One pass over the keys with a running (m, l, o); a tile that raises m scales
// l and o once. Masked entries are excluded by selection, never by arithmetic,
// so values of keys a row does not see cannot reach it, NaN and infinities
// included.
//
// General kernel: a CTA walks its range of items (chunk_plan.cuh), 64 or 128
// query rows against tiles of 64 keys on the CUDA cores in fp32, each thread a
// block of 4 x 4 or 8 x 4 scores and as many rows by D/16 of the output. It is
// bound by fp32 FMA issue and serves fp32 caches, mixed types and 256-wide
// heads; 16-bit caches with 64- and 128-wide heads run in chunk_attend_tc.cu.
#include <type_traits>

#include "chunk_plan.cuh"
#include "cvsa_common.cuh"
#include "cvsa_internal.h"
#include "cvsa_launch.cuh"

namespace cvsa {
namespace {

constexpr int kKeys = 64, kThreads = 256;
// Query rows of an item: 64, 4 by 4 scores a thread, or, for 128-wide heads and
// sequences that fill them, 128, 8 by 4 (a thread's block sets how many FMAs a
// shared-memory load feeds: 1000 tokens at 8000 keys, fp32, 3.7 ms instead of
// 4.3; one token of 16 sequences 1.7 ms instead of 1.1).
int gen_rows(const RaggedView& rg, const KvView& kv, int G) {
  return kv.d == 128 && (int64_t)rg.T * G >= (int64_t)128 * rg.B ? 128 : 64;
}
constexpr int gen_max_rows(int d) { return d == 128 ? 128 : 64; }
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct GenArgs {
  RaggedView rg;
  KvView kv;
  ChunkView c;
  ChunkGeo g;
  float scale2;        // scale * log2(e)
  int min_units;
  float* parts;
  ChunkMergeDesc* desc;
  int32_t* dev_err;
};

template <typename T, int D>
__device__ __forceinline__ void load_row_piece(const T* src, float* dst) {  // 4 elements
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(src);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(src);
    float f[4];
    if constexpr (std::is_same<T, __half>::value) {
      f16x2_to_f2(w.x, f[0], f[1]);
      f16x2_to_f2(w.y, f[2], f[3]);
    } else {
      bf16x2_to_f2(w.x, f[0], f[1]);
      bf16x2_to_f2(w.y, f[2], f[3]);
    }
    *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
  }
}

// K and V have a buffer each: the next K is copied (asynchronously, from an
// fp32 pool) while the weights and the output are formed, the next V while the
// next scores are. 16-bit pools are converted on the way, through registers.
template <int D, int ROWS>
struct GenSmem {
  float q[ROWS][D + 4];
  float k[kKeys][D + 4];
  float v[kKeys][D + 4];
  float p[ROWS][kKeys + 4];
  int64_t key_off[2][kKeys];   // element offset of a key's row in the pools
  int8_t key_ok[2][kKeys];
  ChunkRange range;
};

template <typename T, typename C, int D, int kRows>
__global__ void __launch_bounds__(kThreads, D == 64 ? 2 : 1)
chunk_general_kernel(const __grid_constant__ GenArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  constexpr int kX = kRows / 16;  // rows of a thread
  GenSmem<D, kRows>& sm = *reinterpret_cast<GenSmem<D, kRows>*>(smem_raw);
  const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
  const int cta = blockIdx.x;
  if (tid < 32) {
    const ChunkRange r = chunk_range(a.rg, a.g, cta, gridDim.x, a.min_units, a.dev_err);
    if (tid == 0) {
      sm.range = r;
      a.desc[cta].parts = 0;
    }
  }
  __syncthreads();
  ChunkWalk walk(sm.range);
  ChunkItem it;
  const int G = a.g.G;
  while (walk.next(a.rg, a.g, cta, it)) {
    const int rows = (it.t1 - it.t0) * G;
    const bool busy = (ty & ~1) * kX < rows;  // a warp none of whose rows exist only copies
    // query rows: token t0 + r / G, head h * G + r % G
    for (int e = tid; e < kRows * (D / 4); e += kThreads) {
      const int r = e / (D / 4), c = e % (D / 4);
      float f[4] = {0.f, 0.f, 0.f, 0.f};
      if (r < rows) {
        const T* src = reinterpret_cast<const T*>(a.c.q) +
                       (int64_t)(it.q.tok0 + it.t0 + r / G) * a.c.q_st +
                       (int64_t)(it.h * G + r % G) * a.c.q_sh + c * 4;
        load_row_piece<T, D>(src, f);
      }
      *reinterpret_cast<float4*>(&sm.q[r][c * 4]) = make_float4(f[0], f[1], f[2], f[3]);
    }
    int lo[kX], hi[kX];
    float m[kX], l[kX], o[kX][D / 16];
#pragma unroll
    for (int x = 0; x < kX; ++x) {
      const int r = ty * kX + x;
      const int pos = it.q.start + it.t0 + r / G;
      hi[x] = r >= rows ? 0 : a.g.causal ? max(0, min(it.q.ctx, pos + 1)) : it.q.ctx;
      lo[x] = a.g.window > 0 ? max(0, pos - a.g.window + 1) : 0;
      m[x] = neg_inf();
      l[x] = 0.f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) o[x][d] = 0.f;
    }
    constexpr bool kAsync = sizeof(C) == 4;
    // where the keys of tile k are, to record k % 2
    auto locate = [&](int k) {
      if (tid >= kKeys) return;
      const int key = (it.tile0 + k) * kKeys + tid;
      bool ok = key >= it.lo && key < it.hi;
      int64_t off = 0;
      if (ok) {
        const int blk = a.rg.tables[(int64_t)it.q.slot * a.rg.W + key / a.kv.bs];
        ok = blk >= 0 && blk < a.kv.num_blocks;
        if (!ok) set_dev_error(a.dev_err, CVSA_DEV_ERR_BLOCK_RANGE);
        off = ok ? blk * a.kv.sb + (key % a.kv.bs) * a.kv.st + it.h * a.kv.sh : 0;
      }
      sm.key_off[k & 1][tid] = off;
      sm.key_ok[k & 1][tid] = ok;
    };
    auto copy = [&](int k, const void* pool, float (*to)[D + 4]) {
      if (k < it.k1) {
        for (int e = tid; e < kKeys * (D / 4); e += kThreads) {
          const int r = e / (D / 4), c = e % (D / 4);
          const bool ok = sm.key_ok[k & 1][r];
          const C* src = reinterpret_cast<const C*>(pool) + sm.key_off[k & 1][r] + c * 4;
          if constexpr (kAsync) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                             smem_u32(&to[r][c * 4])), "l"(src), "r"(ok ? 16 : 0) : "memory");
          } else {
            float f[4] = {0.f, 0.f, 0.f, 0.f};
            if (ok) load_row_piece<C, D>(src, f);
            *reinterpret_cast<float4*>(&to[r][c * 4]) = make_float4(f[0], f[1], f[2], f[3]);
          }
        }
      }
      if constexpr (kAsync) cp_async_commit();
    };
    if (it.k0 < it.k1) locate(it.k0);
    __syncthreads();
    copy(it.k0, a.kv.k, sm.k);
    copy(it.k0, a.kv.v, sm.v);
    for (int k = it.k0; k < it.k1; ++k) {
      const int base = (it.tile0 + k) * kKeys, rec = k & 1;
      if (k + 1 < it.k1) locate(k + 1);
      if constexpr (kAsync) cp_async_wait_dyn(1);  // K; V may be on its way
      __syncthreads();
      float s[kX][4];
#pragma unroll
      for (int x = 0; x < kX; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) s[x][y] = 0.f;
#pragma unroll 2
      for (int d = busy ? 0 : D; d < D; d += 4) {
        float4 qa[kX], kb[4];
#pragma unroll
        for (int x = 0; x < kX; ++x) qa[x] = *reinterpret_cast<float4*>(&sm.q[ty * kX + x][d]);
#pragma unroll
        for (int y = 0; y < 4; ++y) kb[y] = *reinterpret_cast<float4*>(&sm.k[tx + 16 * y][d]);
#pragma unroll
        for (int x = 0; x < kX; ++x)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            s[x][y] = fmaf(qa[x].x, kb[y].x, s[x][y]);
            s[x][y] = fmaf(qa[x].y, kb[y].y, s[x][y]);
            s[x][y] = fmaf(qa[x].z, kb[y].z, s[x][y]);
            s[x][y] = fmaf(qa[x].w, kb[y].w, s[x][y]);
          }
      }
      __syncthreads();  // K is done with
      copy(k + 1, a.kv.k, sm.k);
      // some row of the block does not see every key of the tile; rows past the item's
      // end see none, so items that do not fill the block take the selecting loop
      bool cut = false;
#pragma unroll
      for (int x = 0; x < kX; ++x) {
        float mx = m[x];
        bool see[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int c = tx + 16 * y, key = base + c;
          see[y] = key >= lo[x] && key < hi[x] && sm.key_ok[rec][c];
          cut |= !see[y];
          s[x][y] = see[y] ? s[x][y] * a.scale2 : neg_inf();
          if (see[y]) mx = fmaxf(mx, s[x][y]);
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
        const float ref = mx == neg_inf() ? 0.f : mx;
        const float fix = exp2f(m[x] - ref);  // 0 while the row has seen no key
        float sum = 0.f;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float p = see[y] ? exp2f(s[x][y] - ref) : 0.f;
          sum += p;
          // an unseen key is marked by a negative weight
          sm.p[ty * kX + x][tx + 16 * y] = see[y] ? p : -1.f;
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        l[x] = l[x] * fix + sum;
        m[x] = mx;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) o[x][d] *= fix;
      }
      if constexpr (kAsync) cp_async_wait_dyn(1);  // V; the next K may be on its way
      cut = __syncthreads_or(cut);
#pragma unroll 1
      for (int c = busy ? 0 : kKeys; c < kKeys; c += 4) {
        float p[kX][4];  // four keys at a time: one wide load a row
#pragma unroll
        for (int x = 0; x < kX; ++x)
          *reinterpret_cast<float4*>(p[x]) = *reinterpret_cast<float4*>(&sm.p[ty * kX + x][c]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v[D / 16];
#pragma unroll
          for (int y = 0; y < D / 64; ++y)
            *reinterpret_cast<float4*>(v + 4 * y) =
                *reinterpret_cast<float4*>(&sm.v[c + i][tx * 4 + 64 * y]);
          if (!cut) {
#pragma unroll
            for (int x = 0; x < kX; ++x)
#pragma unroll
              for (int d = 0; d < D / 16; ++d) o[x][d] = fmaf(p[x][i], v[d], o[x][d]);
          } else {
#pragma unroll
            for (int x = 0; x < kX; ++x)
#pragma unroll
              for (int d = 0; d < D / 16; ++d)
                o[x][d] = p[x][i] >= 0.f || p[x][i] != p[x][i] ? fmaf(p[x][i], v[d], o[x][d])
                                                               : o[x][d];
          }
        }
      }
      __syncthreads();  // V and the weights are done with
      copy(k + 1, a.kv.v, sm.v);
    }
    // whole items are finished here, pieces go to a partial slot
    if (it.whole) {
#pragma unroll
      for (int x = 0; x < kX; ++x) {
        const int r = ty * kX + x;
        if (r >= rows) continue;
        const int64_t tok = it.q.tok0 + it.t0 + r / G;
        const int head = it.h * G + r % G;
        const float inv = l[x] == 0.f ? 0.f : 1.f / l[x];
        T* dst = reinterpret_cast<T*>(a.c.out) + tok * a.c.o_st + head * a.c.o_sh;
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
          dst[(d / 4) * 64 + tx * 4 + d % 4] =
              Elem<T>::from_f(l[x] == 0.f ? 0.f : o[x][d] * inv);
        if (a.c.lse && tx == 0)
          a.c.lse[tok * a.c.hq + head] = l[x] == 0.f ? neg_inf() : (m[x] + log2f(l[x])) * kLn2;
      }
    } else {
      float* part = a.parts + (size_t)(2 * cta + it.slot) * chunk_slot_floats(kRows, D);
#pragma unroll
      for (int x = 0; x < kX; ++x) {
        const int r = ty * kX + x;
        if (r >= rows) continue;
        if (tx == 0) {
          part[r] = m[x];
          part[kRows + r] = l[x];
        }
        float4* po = reinterpret_cast<float4*>(part + 2 * kRows);
#pragma unroll
        for (int y = 0; y < D / 64; ++y)
          po[(size_t)(tx + 16 * y) * kRows + r] =
              make_float4(o[x][4 * y], o[x][4 * y + 1], o[x][4 * y + 2], o[x][4 * y + 3]);
      }
      if (tid == 0 && it.parts) {
        ChunkMergeDesc d;
        d.parts = it.parts;
        d.tok = it.q.tok0 + it.t0;
        d.rows = rows;
        d.head = it.h;
        a.desc[cta] = d;
      }
    }
    __syncthreads();
  }
}

template <typename T, typename C>
cudaError_t launch_general_d(const GenArgs& a, int rows, int ctas, cudaStream_t s) {
  auto go = [&](auto kernel, size_t smem) -> cudaError_t {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    if (e != cudaSuccess) return e;
    kernel<<<ctas, kThreads, smem, s>>>(a);
    return cudaGetLastError();
  };
  switch (a.kv.d) {
    case 64: return go(chunk_general_kernel<T, C, 64, 64>, sizeof(GenSmem<64, 64>));
    case 128:
      if (rows == 64) return go(chunk_general_kernel<T, C, 128, 64>, sizeof(GenSmem<128, 64>));
      return go(chunk_general_kernel<T, C, 128, 128>, sizeof(GenSmem<128, 128>));
    case 256: return go(chunk_general_kernel<T, C, 256, 64>, sizeof(GenSmem<256, 64>));
    default: return cudaErrorInvalidValue;
  }
}

template <typename T>
cudaError_t launch_general_c(const GenArgs& a, int rows, int ctas, cudaStream_t s) {
  switch (a.kv.dtype) {
    case CVSA_DTYPE_BF16: return launch_general_d<T, __nv_bfloat16>(a, rows, ctas, s);
    case CVSA_DTYPE_F16: return launch_general_d<T, __half>(a, rows, ctas, s);
    default: return launch_general_d<T, float>(a, rows, ctas, s);
  }
}

// ---------------------------------------------------------------------------
// merge of split items
// ---------------------------------------------------------------------------
// Block (x, y): rows [32 x, 32 x + 32) of the item that begins in CTA y's range
// and leaves it. Lanes own rows, warps own float4 columns. Parts are summed in
// CTA order. Most blocks find no item and leave at once.
constexpr int kMaxCtas = 320;

struct MergeArgs {
  const float* parts;
  const ChunkMergeDesc* desc;
  ChunkView c;
  int rows, G, d;
};

template <typename T>
__global__ void __launch_bounds__(256) chunk_merge_kernel(MergeArgs a) {
  __shared__ float w[kMaxCtas][32];  // weight of each part, then of the output
  __shared__ float red[8][32];
  pdl_launch_dependents();
  pdl_wait();
  const int cta = blockIdx.y;
  const ChunkMergeDesc ds = a.desc[cta];
  const int r0 = blockIdx.x * 32;
  if (ds.parts == 0 || r0 >= ds.rows) return;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int r = r0 + lane;
  const size_t slot_floats = chunk_slot_floats(a.rows, a.d);
  auto slot = [&](int p) {
    return a.parts + (size_t)(p == 0 ? 2 * cta + 1 : 2 * (cta + p)) * slot_floats;
  };
  const bool live = r < ds.rows;
  float mx = neg_inf();
  constexpr int kMine = 4;  // sums of this warp's first parts, loaded beside the maxima
  float sums[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i)
    sums[i] = live && wid + 8 * i < ds.parts ? slot(wid + 8 * i)[a.rows + r] : 0.f;
  for (int p = wid; p < ds.parts; p += 8) {
    const float m = live ? slot(p)[r] : neg_inf();
    w[p][lane] = m;
    mx = fmaxf(mx, m);
  }
  red[wid][lane] = mx;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) mx = fmaxf(mx, red[i][lane]);
  __syncthreads();
  const float ref = mx == neg_inf() ? 0.f : mx;
  float l = 0.f;
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int p = wid + 8 * i;
    if (p >= ds.parts) break;
    const float e = exp2f(w[p][lane] - ref);
    w[p][lane] = e;
    l += e * sums[i];
  }
  for (int p = wid + 8 * kMine; p < ds.parts; p += 8) {
    const float e = exp2f(w[p][lane] - ref);
    w[p][lane] = e;
    l += live ? e * slot(p)[a.rows + r] : 0.f;
  }
  red[wid][lane] = l;
  __syncthreads();
  l = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) l += red[i][lane];
  if (!live) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t tok = ds.tok + r / a.G;
  const int head = ds.head * a.G + r % a.G;
  T* dst = reinterpret_cast<T*>(a.c.out) + tok * a.c.o_st + head * a.c.o_sh;
  for (int c = wid; c < a.d / 4; c += 8) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int p = 0; p < ds.parts; ++p) {
      const float4 v = reinterpret_cast<const float4*>(slot(p) + 2 * a.rows)[(size_t)c * a.rows + r];
      const float e = w[p][lane];
      // a part whose rows saw no key holds o = 0 and weighs 0
      o.x = fmaf(e, v.x, o.x);
      o.y = fmaf(e, v.y, o.y);
      o.z = fmaf(e, v.z, o.z);
      o.w = fmaf(e, v.w, o.w);
    }
    if (l == 0.f) o = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<float4*>(dst + c * 4) =
          make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    else
      *reinterpret_cast<uint2*>(dst + c * 4) =
          make_uint2(Mma<T>::pack(o.x * inv, o.y * inv), Mma<T>::pack(o.z * inv, o.w * inv));
  }
  if (a.c.lse && wid == 0)
    a.c.lse[tok * a.c.hq + head] = l == 0.f ? neg_inf() : (mx + log2f(l)) * kLn2;
}

// ---------------------------------------------------------------------------
// workspace: [merge descriptors][partial slots]
// ---------------------------------------------------------------------------
constexpr size_t kDescBytes = ((kMaxCtas * sizeof(ChunkMergeDesc) + 255) / 256) * 256;

// One CTA an SM; the general kernel's two where shared memory and registers
// hold two (64-wide heads): one hides the other's barriers.
int chunk_ctas(const KvView& kv, bool tc) {
  const int n = num_sms() * (!tc && kv.d == 64 ? 2 : 1);
  return n < kMaxCtas ? n : kMaxCtas;
}

ChunkGeo general_geo(const KvView& kv, const RaggedView& rg, const ChunkView& c) {
  ChunkGeo g;
  g.bs = kv.bs;
  g.hkv = kv.hkv;
  g.G = c.hq / kv.hkv;
  g.P = gen_rows(rg, kv, g.G) / g.G;
  g.KT = kKeys;
  g.causal = c.causal;
  g.window = c.window;
  g.fixed = g.fixed_few = 1;
  g.few = 0;
  g.split = chunk_may_split(rg, kv.bs, kKeys);
  return g;
}

}  // namespace

bool chunk_attend_supported(const KvView& kv, const RaggedView& rg, const ChunkView& c) {
  return (kv.d == 64 || kv.d == 128 || kv.d == 256) && c.hq / kv.hkv <= 64 &&
         chunk_fits(rg, chunk_tc_eligible(kv, c) ? chunk_tc_geo(kv, rg, c)
                                                 : general_geo(kv, rg, c));
}

size_t chunk_attend_workspace_bytes(const KvView& kv, const RaggedView& rg, const ChunkView& c) {
  const int rows = chunk_tc_eligible(kv, c) ? chunk_tc_rows() : gen_max_rows(kv.d);
  return kDescBytes + 2 * (size_t)chunk_ctas(kv, chunk_tc_eligible(kv, c)) * chunk_slot_floats(rows, kv.d) * 4;
}

cudaError_t launch_chunk_attend(const KvView& kv, const RaggedView& rg, const ChunkView& c,
                                void* ws, int32_t* dev_err, cudaStream_t s) {
  const bool tc = chunk_tc_eligible(kv, c);
  const int ctas = chunk_ctas(kv, tc);
  const int rows = tc ? chunk_tc_rows() : gen_rows(rg, kv, c.hq / kv.hkv);  // of an item
  ChunkMergeDesc* desc = reinterpret_cast<ChunkMergeDesc*>(ws);
  float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kDescBytes);
  const bool split = tc ? chunk_tc_geo(kv, rg, c).split : general_geo(kv, rg, c).split;
  cudaError_t e;
  if (tc) {
    e = launch_chunk_tc(kv, rg, c, ctas, parts, desc, dev_err, s);
  } else {
    GenArgs a;
    a.rg = rg;
    a.kv = kv;
    a.c = c;
    a.g = general_geo(kv, rg, c);
    a.scale2 = c.scale * kLog2e;
    a.min_units = 2;
    a.desc = desc;
    a.parts = parts;
    a.dev_err = dev_err;
    switch (c.dtype) {
      case CVSA_DTYPE_BF16: e = launch_general_c<__nv_bfloat16>(a, rows, ctas, s); break;
      case CVSA_DTYPE_F16: e = launch_general_c<__half>(a, rows, ctas, s); break;
      default: e = launch_general_c<float>(a, rows, ctas, s); break;
    }
  }
  if (e != cudaSuccess || !split) return e;
  MergeArgs m;
  m.parts = parts;
  m.desc = desc;
  m.c = c;
  m.rows = rows;
  m.G = c.hq / kv.hkv;
  m.d = kv.d;
  const int64_t all = (int64_t)rg.T * m.G;
  const dim3 grid(((all < rows ? (int)all : rows) + 31) / 32, ctas);
  switch (c.dtype) {
    case CVSA_DTYPE_BF16:
      return launch_k(chunk_merge_kernel<__nv_bfloat16>, grid, dim3(256), 0, s, true, m);
    case CVSA_DTYPE_F16:
      return launch_k(chunk_merge_kernel<__half>, grid, dim3(256), 0, s, true, m);
    default: return launch_k(chunk_merge_kernel<float>, grid, dim3(256), 0, s, true, m);
  }
}

}  // namespace cvsa
