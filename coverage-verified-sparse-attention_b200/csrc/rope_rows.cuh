// A row of a new token, D/16 neighbouring lanes with 16 elements (8 pairs) each:
// its loads and stores, its norm and its rotation, and the search for the
// sequence that a token belongs to. Shared by the kernels that append.
#pragma once

#include "cvsa_common.cuh"

namespace cvsa {

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

// The position a key is turned by: its slot's plus what was evicted before it
// (-1 where the sum is out of range).
__device__ __forceinline__ int rope_turn(int pos, int shift) {
  const int64_t t = (int64_t)pos + shift;
  return t >= 0 && t <= 0x7fffffff ? (int)t : -1;
}

// Cosines and sines of a lane's 8 pairs.
__device__ __forceinline__ void load_turn(const float* c, int half, float* cs) {
  *reinterpret_cast<float4*>(cs) = *reinterpret_cast<const float4*>(c);
  *reinterpret_cast<float4*>(cs + 4) = *reinterpret_cast<const float4*>(c + 4);
  *reinterpret_cast<float4*>(cs + 8) = *reinterpret_cast<const float4*>(c + half);
  *reinterpret_cast<float4*>(cs + 12) = *reinterpret_cast<const float4*>(c + half + 4);
}

// x * rsqrt(mean(x^2) + eps) * w; rows without weights pass through. Every lane
// of the warp, for the shuffles.
template <typename T, int U>
__device__ __forceinline__ void norm_row(float* x, const void* wn, int norm_f32, float eps, int e0,
                                         int e1) {
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
  for (int o = U / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (wn) {
    float w[16];
    if (norm_f32) {
      load8<float>(wn, e0, w);
      load8<float>(wn, e1, w + 8);
    } else {
      load8<T>(wn, e0, w);
      load8<T>(wn, e1, w + 8);
    }
    const float inv = rsqrtf(ss / (U * 16) + eps);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = x[i] * inv * w[i];
  }
}

__device__ __forceinline__ void rotate_row(float* x, const float* cs, int interleaved) {
  if (interleaved) {
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

}  // namespace cvsa
