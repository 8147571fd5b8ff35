// New tokens of a ragged batch into the paged cache.
//
// reserve: page bookkeeping. Sequence b of the batch gets cu[b+1] - cu[b] new
// positions behind its context length; pages that start at or past the
// position and past the pages it owns are popped from the free list, in the
// order of the batch (a prefix sum, so the same state always gives the same
// tables), and the context length advances. One CTA: the work is a few
// integers a sequence.
//
// rope_append: per token and head, in fp32 with one rounding at the store:
//   x^ = x * rsqrt(mean(x^2) + eps) * w      (query and key rows, optional)
//   y_i = x^_i cos_i - x^_j sin_i,  y_j = x^_j cos_i + x^_i sin_i
// over the pairs (i, j) of the rotated part (j = i + R/2, or neighbouring
// elements), cos and sin from row `position` of a table; query rows go to
// q_out, key and value rows to the slot of their position in their page.
// Bound by bytes for long chunks (each row is read and written once) and by
// latency for a few tokens. A row is held by D/16 neighbouring lanes, 16
// elements (8 pairs) a lane, so a rotation never leaves its lane and a norm is
// a few shuffles; rows are independent, so there is no shared memory and no
// block-wide barrier. A block holds rows of one token, so that the lookup
// (sequence, position, block id) is uniform; the row's data loads are issued before it. It is bound by
// instruction issue and occupancy together: several rows a lane, or a lookup a
// token shared through shared memory, cost more in registers than they saved.
#include "cvsa_common.cuh"
#include "cvsa_internal.h"

namespace cvsa {
namespace {

// ---------------------------------------------------------------------------
// reserve
// ---------------------------------------------------------------------------
constexpr int kReserveThreads = 1024;

// Inclusive sum over the block; `warp_sums` holds one value a warp.
template <typename T>
__device__ __forceinline__ T block_scan_incl(T v, T* warp_sums) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  if (lane == 31) warp_sums[wid] = v;
  __syncthreads();
  if (wid == 0) {
    T w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T t = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += t;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  if (wid > 0) v += warp_sums[wid - 1];
  __syncthreads();
  return v;
}

__global__ void __launch_bounds__(kReserveThreads)
reserve_kernel(const int32_t* cu, const int32_t* seq_ids, int B, int num_seqs, int bs,
               int32_t* tables, int W, int32_t* lens, int32_t* pages_alloc,
               const int32_t* free_list, int free_len, int32_t* free_head, int32_t* starts,
               int32_t* dev_err) {
  __shared__ int64_t wanted_sums[32];
  __shared__ int warp_sums[32];
  __shared__ int s_incl[kReserveThreads];   // inclusive sum of the pages granted
  __shared__ int s_slot[kReserveThreads];   // table row and first new page of a granted sequence
  __shared__ int s_first[kReserveThreads];
  const int tid = threadIdx.x;
  const int64_t head0 = *free_head;
  int64_t wanted = 0, taken = 0;  // pages asked for / granted by earlier sequences
  __syncthreads();                // every thread holds free_head before it changes
  for (int b0 = 0; b0 < B; b0 += kReserveThreads) {
    const int b = b0 + tid;
    int need = 0, slot = 0, first = 0, start = -1;
    int64_t end = 0;
    bool ok = false;
    if (b < B) {
      const int64_t n = (int64_t)cu[b + 1] - cu[b];
      slot = seq_ids ? seq_ids[b] : b;
      if (n < 0 || slot < 0 || slot >= num_seqs) {
        set_dev_error(dev_err, CVSA_DEV_ERR_RAGGED);
      } else {
        const int len = lens[slot];
        end = len + n;
        if (len < 0 || end > (int64_t)W * bs) {
          set_dev_error(dev_err, CVSA_DEV_ERR_TABLE_FULL);
        } else {
          ok = true;
          start = len;
          first = max(pages_alloc[slot], (len + bs - 1) / bs);
          need = max(0, (int)((end + bs - 1) / bs) - first);
        }
      }
    }
    // 64 bits: offsets out of order can ask for the same pages again and again
    const int64_t incl = block_scan_incl((int64_t)need, wanted_sums);
    if (ok && need > 0 && (head0 < 0 || head0 + wanted + incl > free_len)) {
      set_dev_error(dev_err, CVSA_DEV_ERR_POOL);
      ok = false;
      need = 0;
    }
    if (tid == kReserveThreads - 1) wanted_sums[0] = incl;
    __syncthreads();
    wanted += wanted_sums[0];
    __syncthreads();
    if (b < B) {
      if (starts) starts[b] = ok ? start : -1;
      if (ok) {
        lens[slot] = (int)end;
        if (need > 0) pages_alloc[slot] = first + need;
      }
    }
    // the granted pages, spread over the block: entry e of this round belongs
    // to the first sequence whose inclusive sum passes e. Sequences refused for
    // want of pages come after all granted ones, so the sums stay contiguous.
    s_incl[tid] = block_scan_incl(need, warp_sums);
    s_slot[tid] = slot;
    s_first[tid] = first;
    __syncthreads();
    const int total = s_incl[kReserveThreads - 1];
    for (int e = tid; e < total; e += kReserveThreads) {
      int lo = 0, hi = kReserveThreads - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_incl[mid] > e) hi = mid; else lo = mid + 1;
      }
      const int before = lo ? s_incl[lo - 1] : 0;
      tables[(int64_t)s_slot[lo] * W + s_first[lo] + (e - before)] =
          free_list[head0 + taken + e];
    }
    taken += total;
    __syncthreads();
  }
  if (tid == 0 && taken) *free_head = (int)(head0 + taken);
}

// ---------------------------------------------------------------------------
// rope_append
// ---------------------------------------------------------------------------
struct RopeArgs {
  RaggedView rg;
  KvView kv;
  RopeView r;
  int rows_per_token;
  int q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh, c_st, c_sh;  // strides (31 bits)
  int bs_shift;   // log2 of the page size, or -1
  int32_t* dev_err;
};

// 8 consecutive elements as floats, and back.
template <typename T>
__device__ __forceinline__ void load8(const void* base, int64_t elem, float* f) {
  const T* p = reinterpret_cast<const T*>(base) + elem;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
    const uint4 w = *reinterpret_cast<const uint4*>(p + i * Vec16<T>::N);
    Vec16<T>::unpack(w, f + i * Vec16<T>::N);
  }
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return Mma<T>::pack(a, b);
}
template <typename T>
__device__ __forceinline__ void store8(void* base, int64_t elem, const float* f) {
  T* p = reinterpret_cast<T*>(base) + elem;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]),
                                              pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
  }
}

// The sequence that holds token t, by the whole warp: 32 probes a step of the
// offsets cu[0..B], so three dependent loads serve any batch up to 32768.
// -1 when no sequence holds it.
__device__ __forceinline__ int warp_find_seq(const int32_t* cu, int B, int t) {
  int lo = 0, n = B;  // the answer, if any, is in [lo, lo + n)
  const int lane = threadIdx.x & 31;
  if (t < cu[0] || t >= cu[B]) return -1;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lo + min(lane * step, n);          // lane 0 probes lo: cu[lo] <= t holds
    const bool below = lane * step < n && cu[at] <= t;
    const unsigned m = __ballot_sync(0xffffffffu, below);
    const int k = 31 - __clz(m | 1u);
    lo += k * step;
    n = min(step, n - k * step);
  }
  return lo;
}

template <typename T, typename C, int U>  // input type, cache type, lanes a row (head_dim / 16)
__global__ void __launch_bounds__(64) rope_append_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int D = U * 16;
  const int lane = threadIdx.x & 31, u = lane % U;
  // blockIdx.x is the token, so what is looked up is the same for the block
  const int tok = blockIdx.x, hq = a.r.hq, hkv = a.kv.hkv;
  const int row = (blockIdx.y * blockDim.x + threadIdx.x) / U;
  const bool live = row < a.rows_per_token;
  if (!__any_sync(0xffffffffu, live)) return;
  const int r = live ? row : 0;
  // kind 0: query head r, 1: key head, 2: value head
  const int kind = r < hq ? 0 : r < hq + hkv ? 1 : 2;
  const int h = kind == 0 ? r : kind == 1 ? r - hq : r - hq - hkv;
  // this lane's two runs of 8 elements: the halves of its 8 pairs, or, past the
  // rotated part and for neighbouring pairs, 16 elements in a row
  const int half = a.r.rot / 2;
  const bool in_rot = u * 16 < a.r.rot;
  const int e0 = in_rot && !a.r.interleaved ? u * 8 : u * 16;
  const int e1 = in_rot && !a.r.interleaved ? half + u * 8 : u * 16 + 8;
  float x[16];
  {
    const void* base = kind == 0 ? a.r.q : kind == 1 ? a.r.k : a.r.v;
    const int st = kind == 0 ? a.q_st : kind == 1 ? a.k_st : a.v_st;
    const int sh = kind == 0 ? a.q_sh : kind == 1 ? a.k_sh : a.v_sh;
    const int64_t at = (int64_t)tok * st + (int64_t)h * sh;
    load8<T>(base, at + e0, x);
    load8<T>(base, at + e1, x + 8);
  }
  const int b = warp_find_seq(a.rg.cu, a.rg.B, tok);
  const bool rotate = a.r.cos_sin != nullptr && kind != 2;
  int pos = -1, slot = -1, page = 0;
  bool good = live && b >= 0;
  if (good) {
    slot = a.rg.seq_ids ? a.rg.seq_ids[b] : b;
    if (slot < 0 || slot >= a.rg.num_seqs) {
      good = false;
      if (u == 0) set_dev_error(a.dev_err, CVSA_DEV_ERR_RAGGED);
    } else if (a.rg.starts) {
      const int s = a.rg.starts[b];
      good = s >= 0;  // refused by the reservation, which recorded why
      pos = s + (tok - a.rg.cu[b]);
    } else {
      pos = a.rg.lens[slot] - (a.rg.cu[b + 1] - tok);
    }
    page = a.bs_shift >= 0 ? pos >> a.bs_shift : pos / a.kv.bs;
    if (good && (pos < 0 || page >= a.rg.W ||
                 (a.r.cos_sin && pos >= a.r.max_positions))) {
      good = false;
      if (u == 0) set_dev_error(a.dev_err, CVSA_DEV_ERR_RAGGED);
    }
  }
  int blk = 0;
  if (good && kind != 0) blk = a.rg.tables[(int64_t)slot * a.rg.W + page];
  float cs[16];
  if (good && rotate && in_rot) {
    const float* c = a.r.cos_sin + (int64_t)pos * a.r.rot + u * 8;
    *reinterpret_cast<float4*>(cs) = *reinterpret_cast<const float4*>(c);
    *reinterpret_cast<float4*>(cs + 4) = *reinterpret_cast<const float4*>(c + 4);
    *reinterpret_cast<float4*>(cs + 8) = *reinterpret_cast<const float4*>(c + half);
    *reinterpret_cast<float4*>(cs + 12) = *reinterpret_cast<const float4*>(c + half + 4);
  }
  const void* wn = kind == 0 ? a.r.q_norm : kind == 1 ? a.r.k_norm : nullptr;
  float ss = 0.f;
  if (a.r.q_norm || a.r.k_norm) {  // every lane, for the shuffles
#pragma unroll
    for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = U / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  }
  if (wn) {
    float w[16];
    if (a.r.norm_f32) {
      load8<float>(wn, e0, w);
      load8<float>(wn, e1, w + 8);
    } else {
      load8<T>(wn, e0, w);
      load8<T>(wn, e1, w + 8);
    }
    const float inv = rsqrtf(ss / D + a.r.eps);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = x[i] * inv * w[i];
  }
  if (good && rotate && in_rot) {
    if (a.r.interleaved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = x[2 * i], q = x[2 * i + 1];
        x[2 * i] = p * cs[i] - q * cs[8 + i];
        x[2 * i + 1] = q * cs[i] + p * cs[8 + i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = x[i], q = x[8 + i];
        x[i] = p * cs[i] - q * cs[8 + i];
        x[8 + i] = q * cs[i] + p * cs[8 + i];
      }
    }
  }
  if (!live || b < 0) return;
  if (kind == 0) {
    if (!good) {  // a row without a position: a defined value, not the buffer's old one
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = 0.f;
    }
    const int64_t at = (int64_t)tok * a.qo_st + (int64_t)h * a.qo_sh;
    store8<T>(a.r.q_out, at + e0, x);
    store8<T>(a.r.q_out, at + e1, x + 8);
    return;
  }
  if (!good) return;
  if (blk < 0 || blk >= a.kv.num_blocks) {
    if (u == 0) set_dev_error(a.dev_err, CVSA_DEV_ERR_BLOCK_RANGE);
    return;
  }
  void* pool = const_cast<void*>(kind == 1 ? a.kv.k : a.kv.v);
  const int64_t at = blk * a.kv.sb + (int64_t)(pos - page * a.kv.bs) * a.c_st + (int64_t)h * a.c_sh;
  store8<C>(pool, at + e0, x);
  store8<C>(pool, at + e1, x + 8);
}

template <typename T, typename C>
cudaError_t launch_ru(const RopeArgs& a, cudaStream_t s) {
  const int lanes = a.rows_per_token * (a.kv.d / 16);
  // two warps a block: 8192 tokens of 48 heads 46 us, 49 with four, 63 with twelve
  const int parts = (lanes + 63) / 64;
  const dim3 grid(a.rg.T, parts), block(((lanes + parts - 1) / parts + 31) / 32 * 32);
  switch (a.kv.d) {
    case 64: rope_append_kernel<T, C, 4><<<grid, block, 0, s>>>(a); break;
    case 128: rope_append_kernel<T, C, 8><<<grid, block, 0, s>>>(a); break;
    case 256: rope_append_kernel<T, C, 16><<<grid, block, 0, s>>>(a); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_rc(const RopeArgs& a, cudaStream_t s) {
  switch (a.kv.dtype) {
    case CVSA_DTYPE_BF16: return launch_ru<T, __nv_bfloat16>(a, s);
    case CVSA_DTYPE_F16: return launch_ru<T, __half>(a, s);
    default: return launch_ru<T, float>(a, s);
  }
}

}  // namespace

cudaError_t launch_paged_reserve(const int32_t* cu, const int32_t* seq_ids, int B, int num_seqs,
                                 int bs, int32_t* tables, int W, int32_t* lens,
                                 int32_t* pages_alloc, const int32_t* free_list, int free_len,
                                 int32_t* free_head, int32_t* starts, int32_t* dev_err,
                                 cudaStream_t s) {
  reserve_kernel<<<1, kReserveThreads, 0, s>>>(cu, seq_ids, B, num_seqs, bs, tables, W, lens,
                                               pages_alloc, free_list, free_len, free_head, starts,
                                               dev_err);
  return cudaGetLastError();
}

bool rope_append_supported(const KvView& kv) {
  return kv.d == 64 || kv.d == 128 || kv.d == 256;
}

cudaError_t launch_rope_append(const RaggedView& rg, const KvView& kv, const RopeView& r,
                               int32_t* dev_err, cudaStream_t s) {
  RopeArgs a;
  a.rg = rg;
  a.kv = kv;
  a.r = r;
  a.rows_per_token = r.hq + 2 * kv.hkv;
  a.q_st = (int)r.q_st;
  a.q_sh = (int)r.q_sh;
  a.k_st = (int)r.k_st;
  a.k_sh = (int)r.k_sh;
  a.v_st = (int)r.v_st;
  a.v_sh = (int)r.v_sh;
  a.qo_st = (int)r.qo_st;
  a.qo_sh = (int)r.qo_sh;
  a.c_st = (int)kv.st;
  a.c_sh = (int)kv.sh;
  a.dev_err = dev_err;
  a.bs_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (kv.bs == 1 << i) a.bs_shift = i;
  switch (r.dtype) {
    case CVSA_DTYPE_BF16: return launch_rc<__nv_bfloat16>(a, s);
    case CVSA_DTYPE_F16: return launch_rc<__half>(a, s);
    default: return launch_rc<float>(a, s);
  }
}

}  // namespace cvsa
