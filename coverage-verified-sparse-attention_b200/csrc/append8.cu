// New tokens of a ragged batch into the 8-bit paged cache.
//
// Rows are normed and rotated as in rope_append.cu, in fp32, and rounded once: the
// queries to their type, a key or value x to the e4m3 code of x 2^-e. e belongs to
// the page and KV head, keys and values apart (fp8.cuh): for a page that begins
// with these tokens, the least that holds their largest absolute value; for a page
// that held tokens before, not less than it was, and when it grows the codes of the
// tokens in use move to the new scale. (Infinities do not count for the largest
// value; they saturate. NaN stays NaN.)
//
// A block of 128 threads has one page, KV head and kind (key or value), so the
// largest value is a block's and no atomics are needed; the blocks behind those
// have query rows. Which pages a batch touches is known on the device only: item i
// of the grid is looked up in cu[b] / page + 2 b, which leaves every sequence room
// for all its pages (n tokens touch at most n / page + 2) without a sum over the batch.
// Bound by bytes for long chunks and by latency for a few tokens.
#include "cvsa_common.cuh"
#include "cvsa_internal.h"
#include "fp8.cuh"
#include "rope_rows.cuh"

namespace cvsa {
namespace {

constexpr int kThreads = 128;

struct Append8Args {
  RaggedView rg;
  KvView kv;
  RopeView r;
  int page_blocks;  // blocks that have a page
  int q_parts;      // blocks a token's query rows take
  int32_t* dev_err;
};

// The sequence whose items hold item i: the last b with cu[b] / bs + 2 b <= i (0 if
// none), by the whole warp, 32 probes a step.
__device__ __forceinline__ int warp_find_item(const int32_t* cu, int B, int bs, int64_t i) {
  int lo = 0, n = B;
  const int lane = threadIdx.x & 31;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lo + min(lane * step, n - 1);
    const bool below = lane * step < n && cu[at] / bs + 2 * (int64_t)at <= i;
    const unsigned m = __ballot_sync(0xffffffffu, below);
    const int k = 31 - __clz(m | 1u);
    lo += k * step;
    n = min(step, n - k * step);
  }
  return lo;
}

// A lane's two runs of 8 elements of a row: the halves of its 8 pairs, or 16 elements.
struct Runs {
  int e0, e1;
  bool in_rot;
  __device__ __forceinline__ Runs(const RopeView& r, int u) {
    in_rot = u * 16 < r.rot;
    const bool halves = in_rot && !r.interleaved;
    e0 = halves ? u * 8 : u * 16;
    e1 = halves ? r.rot / 2 + u * 8 : u * 16 + 8;
  }
};

template <typename T, int U>
__device__ __forceinline__ void query_block(const Append8Args& a, int bid) {
  const int lane = threadIdx.x & 31, u = lane % U;
  const int tok = bid / a.q_parts;
  const int h = ((bid % a.q_parts) * kThreads + threadIdx.x) / U;
  const bool live = h < a.r.hq;
  const Runs e(a.r, u);
  float x[16];
  const int64_t at = (int64_t)tok * a.r.q_st + (int64_t)(live ? h : 0) * a.r.q_sh;
  load8<T>(a.r.q, at + e.e0, x);
  load8<T>(a.r.q, at + e.e1, x + 8);
  const int b = warp_find_seq(a.rg.cu, a.rg.B, tok);
  if (b < 0) return;  // a row no sequence owns
  const int slot = a.rg.seq_ids ? a.rg.seq_ids[b] : b;
  bool good = slot >= 0 && slot < a.rg.num_seqs;
  int turn = 0;
  if (good) {
    int64_t pos;
    if (a.rg.starts) {
      const int s = a.rg.starts[b];
      good = s >= 0;
      pos = (int64_t)s + (tok - a.rg.cu[b]);
    } else {
      pos = (int64_t)a.rg.lens[slot] - ((int64_t)a.rg.cu[b + 1] - tok);
    }
    good = good && pos >= 0 && pos < (int64_t)a.rg.W * a.kv.bs && pos <= 0x7fffffff;
    if (good) turn = a.r.shift ? rope_turn((int)pos, a.r.shift[slot]) : (int)pos;
    if (a.r.cos_sin && (turn < 0 || turn >= a.r.max_positions)) good = false;
    if (!good && !(a.rg.starts && a.rg.starts[b] < 0)) set_dev_error(a.dev_err, CVSA_DEV_ERR_RAGGED);
  } else {
    set_dev_error(a.dev_err, CVSA_DEV_ERR_RAGGED);
  }
  if (a.r.q_norm) norm_row<T, U>(x, a.r.q_norm, a.r.norm_f32, a.r.eps, e.e0, e.e1);
  if (good && a.r.cos_sin && e.in_rot) {
    float cs[16];
    load_turn(a.r.cos_sin + (int64_t)turn * a.r.rot + u * 8, a.r.rot / 2, cs);
    rotate_row(x, cs, a.r.interleaved);
  }
  if (!live) return;
  if (!good) {  // a row without a position: a defined value, not the buffer's old one
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 0.f;
  }
  const int64_t to = (int64_t)tok * a.r.qo_st + (int64_t)h * a.r.qo_sh;
  store8<T>(a.r.q_out, to + e.e0, x);
  store8<T>(a.r.q_out, to + e.e1, x + 8);
}

template <typename T, int U>
__device__ __forceinline__ void page_block(const Append8Args& a, int bid) {
  constexpr int kRows = kThreads / U, kWarps = kThreads / 32;
  __shared__ float s_max[kWarps];
  const int tid = threadIdx.x, u = tid % U, bs = a.kv.bs, hkv = a.kv.hkv;
  const bool is_k = bid % (2 * hkv) < hkv;
  const int h = bid % hkv;  // 2 hkv is a multiple of hkv
  const int64_t item = bid / (2 * hkv);
  const int b = warp_find_item(a.rg.cu, a.rg.B, bs, item);
  const int tok0 = a.rg.cu[b], end = a.rg.cu[b + 1], n = end - tok0;
  const int64_t ordinal = item - (tok0 / bs + 2 * (int64_t)b);
  const int slot = a.rg.seq_ids ? a.rg.seq_ids[b] : b;
  if (ordinal < 0) return;
  if (tok0 < 0 || end > a.rg.T || end < tok0 || slot < 0 || slot >= a.rg.num_seqs) {
    if (ordinal == 0 && tid == 0) set_dev_error(a.dev_err, CVSA_DEV_ERR_RAGGED);
    return;
  }
  if (n == 0) return;
  const int64_t start = a.rg.starts ? a.rg.starts[b] : (int64_t)a.rg.lens[slot] - n;
  if (a.rg.starts && start < 0) return;  // refused by the reservation, which recorded why
  if (start < 0 && tid == 0) set_dev_error(a.dev_err, CVSA_DEV_ERR_RAGGED);
  // positions [p0, p1) are written
  const int64_t p0 = start < 0 ? 0 : start, p1 = start + n, page = p0 / bs + ordinal;
  if (page * bs >= p1) return;
  if (page >= a.rg.W) {
    if (tid == 0) set_dev_error(a.dev_err, CVSA_DEV_ERR_RAGGED);
    return;
  }
  const int blk = a.rg.tables[(int64_t)slot * a.rg.W + page];  // looked at behind the rows' loads
  const int r0 = (int)max((int64_t)0, p0 - page * bs), r1 = (int)min((int64_t)bs, p1 - page * bs);
  // rows behind the written ones that hold tokens (an append in the middle of a sequence)
  const int used = (int)max((int64_t)r1, min((int64_t)bs, a.rg.lens[slot] - page * bs));
  const bool begun = r0 > 0 || used > r1;
  const int64_t shift = a.r.shift ? a.r.shift[slot] : 0;
  const Runs e(a.r, u);
  const void* const src = is_k ? a.r.k : a.r.v;
  const int64_t st = is_k ? a.r.k_st : a.r.v_st, sh = is_k ? a.r.k_sh : a.r.v_sh;
  // Row r of the page, normed and rotated; whether it is to be written.
  auto take = [&](int r, float* x) {
    bool ok = r < r1;
    const int64_t pos = page * bs + (ok ? r : r0);
    const int64_t at = (tok0 + (pos - start)) * st + h * sh;
    load8<T>(src, at + e.e0, x);
    load8<T>(src, at + e.e1, x + 8);
    const int64_t turn = pos + shift;
    if (a.r.cos_sin && (turn < 0 || turn >= a.r.max_positions)) {
      if (ok && u == 0) set_dev_error(a.dev_err, CVSA_DEV_ERR_RAGGED);
      ok = false;
    }
    if (is_k) {
      if (a.r.k_norm) norm_row<T, U>(x, a.r.k_norm, a.r.norm_f32, a.r.eps, e.e0, e.e1);
      if (ok && a.r.cos_sin && e.in_rot) {
        float cs[16];
        load_turn(a.r.cos_sin + turn * a.r.rot + u * 8, a.r.rot / 2, cs);
        rotate_row(x, cs, a.r.interleaved);
      }
    }
    return ok;
  };
  float x[16], top = 0.f;
  bool ok = false, some = false;
  // one round unless the page has more rows than the block; then the second sweep
  // takes the rows again
  const int rounds = (r1 - r0 + kRows - 1) / kRows;
  for (int i = 0; i < rounds; ++i) {
    ok = take(r0 + i * kRows + tid / U, x);
    some |= ok;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float m = fabsf(x[j]);
      top = ok && m <= 3.402823466e38f ? fmaxf(top, m) : top;
    }
  }
  if (blk < 0 || blk >= a.kv.num_blocks) {
    if (tid == 0) set_dev_error(a.dev_err, CVSA_DEV_ERR_BLOCK_RANGE);
    return;
  }
  float* const scale = const_cast<float*>(is_k ? a.kv.ks : a.kv.vs) + (int64_t)blk * hkv + h;
  const int had = begun ? scale_exponent_of(*scale) : kScaleMin;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (tid % 32 == 0) s_max[tid / 32] = top;
  if (!__syncthreads_or(some)) return;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_max[w]);
  const int now = max(had, scale_exponent(top));
  uint8_t* const rows = reinterpret_cast<uint8_t*>(const_cast<void*>(is_k ? a.kv.k : a.kv.v)) +
                        (int64_t)blk * a.kv.sb + (int64_t)h * a.kv.sh;
  if (tid == 0) *scale = pow2(now);  // every thread holds the old one
  if (now > had && begun) {
    const float f = pow2(had - now);
    for (int c = tid; c < (r0 + used - r1) * U; c += kThreads) {
      const int r = c / U < r0 ? c / U : c / U - r0 + r1;
      uint4* p = reinterpret_cast<uint4*>(rows + (int64_t)r * a.kv.st + (c % U) * 16);
      uint4 w = *p;
      uint32_t* words = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float y[4];
        e4m3x4_to_f4(words[i], y);
        words[i] = f4_to_e4m3x4(y[0] * f, y[1] * f, y[2] * f, y[3] * f);
      }
      *p = w;
    }
  }
  const float f = pow2(-now);
  for (int i = 0; i < rounds; ++i) {
    const int r = r0 + i * kRows + tid / U;
    if (rounds > 1) ok = take(r, x);
    if (!ok) continue;
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] *= f;
    uint8_t* p = rows + (int64_t)r * a.kv.st;
    *reinterpret_cast<uint2*>(p + e.e0) =
        make_uint2(f4_to_e4m3x4(x[0], x[1], x[2], x[3]), f4_to_e4m3x4(x[4], x[5], x[6], x[7]));
    *reinterpret_cast<uint2*>(p + e.e1) =
        make_uint2(f4_to_e4m3x4(x[8], x[9], x[10], x[11]), f4_to_e4m3x4(x[12], x[13], x[14], x[15]));
  }
}

template <typename T, int U>
__global__ void __launch_bounds__(kThreads, 10) append8_kernel(const __grid_constant__ Append8Args a) {
  if ((int)blockIdx.x < a.page_blocks)
    page_block<T, U>(a, blockIdx.x);
  else
    query_block<T, U>(a, blockIdx.x - a.page_blocks);
}

template <typename T>
cudaError_t launch_t(Append8Args& a, cudaStream_t s) {
  a.q_parts = (a.r.hq * (a.kv.d / 16) + kThreads - 1) / kThreads;
  const int64_t blocks = a.page_blocks + (int64_t)a.rg.T * a.q_parts;
  switch (a.kv.d) {
    case 64: append8_kernel<T, 4><<<(unsigned)blocks, kThreads, 0, s>>>(a); break;
    case 128: append8_kernel<T, 8><<<(unsigned)blocks, kThreads, 0, s>>>(a); break;
    case 256: append8_kernel<T, 16><<<(unsigned)blocks, kThreads, 0, s>>>(a); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

int64_t page_blocks(const RaggedView& rg, const KvView& kv) {
  return (rg.T / kv.bs + 2 * (int64_t)rg.B) * 2 * kv.hkv;
}

}  // namespace

bool append8_fits(const RaggedView& rg, const KvView& kv, const RopeView& r) {
  return page_blocks(rg, kv) + (int64_t)rg.T * (r.hq + 1) < (int64_t(1) << 31);
}

cudaError_t launch_append8(const RaggedView& rg, const KvView& kv, const RopeView& r,
                           int32_t* dev_err, cudaStream_t s) {
  Append8Args a;
  a.rg = rg;
  a.kv = kv;
  a.r = r;
  a.page_blocks = (int)page_blocks(rg, kv);
  a.dev_err = dev_err;
  switch (r.dtype) {
    case CVSA_DTYPE_BF16: return launch_t<__nv_bfloat16>(a, s);
    case CVSA_DTYPE_F16: return launch_t<__half>(a, s);
    default: return launch_t<float>(a, s);
  }
}

}  // namespace cvsa
