// Attention of few new tokens a sequence over the 8-bit paged cache: single tokens
// and drafts of at most 32 query rows a KV head, 16-bit queries, head_dim 64 or 128,
// pages of a multiple of 16 tokens. Formulas as in chunk_attend.cu, work split as in
// chunk_plan.cuh; the pieces of split items go to the same merge.
//
// Bound by the cache's bytes, 2 D a key, so everything else is kept off the way:
// codes become the operands of mma.sync in the registers of the lane that copied them, and
// a warp is on its own until the end of an item. (tcgen05 takes its operands from shared
// memory: the codes are widened there for all, as chunk_attend_tc.cu does, where 32 single
// tokens take 291 us.) The warps of a block take blocks of 16 keys in turn, each with a
// running maximum, sum and output of its own, joined in shared memory at the end of
// the item.
//
// Layouts. The products run transposed, so that 16 keys fill M of mma.sync m16n8k16
// and 8 query rows N. It sums over k in any order that both operands share, and rows
// of M may be any: so lane (g, t) = (lane / 4, lane % 4) of
//   S' = K Q' takes 16 consecutive codes t*16.. of keys g and g + 8, four to a k step,
//     and of query row g the same elements;
//   O' += V' P' takes D/8 consecutive codes from g*D/8 on of keys 2t, 2t+1, 2t+8, 2t+9,
//     two a tile of M; the codes of two keys are interleaved by byte permutation and
//     widened as pairs.
// P' is transposed in registers (movmatrix). K's scale goes to the scores, V's to the
// widened codes. f16 throughout: queries are scaled by row as in chunk_attend_tc.cu,
// weights carry 2^11 and the reference maximum follows rises of 2^4, for the reasons
// given there. Their sum is of the 32-bit weights: rounding one to f16 errs by at most 2^-11 of
// it, either way, so a row errs by less than that of its values' absolute moment. The next
// block's codes are loaded to registers as soon as this block's are operands, so nothing
// synchronises.
//
// 32 single tokens of 32 heads at 1 to 8192 keys take 72 us (50 of them the codes at the
// rate of a copy; the rest goes to the first loads and the join at the end of an item), one
// token at 128K keys 60 us, 8 drafts of 2 to 8 tokens of 64-wide heads 80 us. Measured and not
// kept: codes through a ring of asynchronous copies in shared memory (91 us), 32 keys a step
// of 12 warps (89), rows on M (125). The pieces of a split item are joined by a block a
// row, since 128K keys make 37 pieces (a warp a row: 47 us, now 9).
#include "chunk_plan.cuh"
#include "cvsa_common.cuh"
#include "cvsa_internal.h"
#include "cvsa_launch.cuh"
#include "fp8.cuh"

namespace cvsa {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kRaise = 4.f, kUp = 11.f;

// Warps of a block (two an SM), by the registers that a warp's O takes.
constexpr int few_warps(int d, int rows) { return d * rows <= 1024 ? 8 : d * rows <= 2048 ? 6 : 4; }
struct FewArgs {
  RaggedView rg;
  KvView kv;
  ChunkView c;
  ChunkGeo g;
  float scale2;
  int min_units;
  float* parts;
  ChunkMergeDesc* desc;
  int32_t* dev_err;
};

// A block of 16 keys: where it is in the pools, and what its scales multiply by. One that is
// not to be read (before the window, not in the pool) is at 0, with a V factor of 0.
struct alignas(16) BlockRec {
  int64_t off;
  float ks;
  uint32_t vs;
};

template <int D, int ROWS>
struct FewSmem {
  static constexpr int kWarps = few_warps(D, ROWS);
  float o[kWarps][ROWS][D + 4];
  BlockRec rec[kWarps][64];               // of a warp's blocks, mod 64
  uint2 q[ROWS / 8][D / 16][32];          // queries as operands, a lane's pair a step
  float f[ROWS];                          // what a score of the row is multiplied by
  float m[kWarps][ROWS], l[kWarps][ROWS];
  float out_m[ROWS], out_l[ROWS], weight[kWarps][ROWS];
  float p[kWarps][ROWS][16];              // weights of a block whose values are not all finite
  ChunkItem item[2];
  int more[2];
  alignas(8) uint8_t walk[sizeof(ChunkWalk)];
};

__device__ __forceinline__ float ex2(float x) {
  // weights below 2^-126 are flushed to 0, far below the rounding of any sum
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t hmul2(uint32_t x, uint32_t y) {
  const __half2 z = __hmul2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&y));
  return *reinterpret_cast<const uint32_t*>(&z);
}

template <typename TI, int D, int ROWS>
__global__ void __launch_bounds__(32 * few_warps(D, ROWS), 2)
chunk_few_kernel(const __grid_constant__ FewArgs a) {
  constexpr int kWarps = few_warps(D, ROWS), kThreads = 32 * kWarps, kKeys = 16 * kWarps;
  constexpr int kNt = ROWS / 8;                     // tiles of 8 rows
  constexpr int kSteps = D / 16, kTiles = D / 16, kCols = D / 8;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  using Smem = FewSmem<D, ROWS>;
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  ChunkWalk& walk = *reinterpret_cast<ChunkWalk*>(sm.walk);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int G = a.g.G, bs = a.kv.bs;
  if (warp == 0) {
    const ChunkRange r = chunk_range(a.rg, a.g, blockIdx.x, gridDim.x, a.min_units, a.dev_err);
    if (tid == 0) {
      a.desc[blockIdx.x].parts = 0;
      walk = ChunkWalk(r);
      sm.more[0] = walk.next(a.rg, a.g, blockIdx.x, sm.item[0]);
    }
  }
  __syncthreads();
  uint4 ck[2][D / 64];     // codes of keys g, g + 8
  uint32_t cv[4][D / 32];  // of values 2t, 2t + 1, 2t + 8, 2t + 9
  // This lane's first bytes of a block; pages hold whole blocks, so rows that nothing
  // sees may be read (values of such rows are cleared before use).
  const int64_t st = a.kv.st;
  const char* const at_k = static_cast<const char*>(a.kv.k) + g * st + t * 16;
  const char* const at_v = static_cast<const char*>(a.kv.v) + 2 * t * st + g * (D / 8);
  auto load_k = [&](int64_t off) {
    const char* const p = at_k + off;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int x = 0; x < D / 64; ++x) ck[i][x] = ldg_stream16(p + i * 8 * st + x * 64);
  };
  auto load_v = [&](int64_t off) {
    const char* const p = at_v + off;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const char* const row = p + ((i & 1) + 8 * (i >> 1)) * st;
      if constexpr (D == 128) {
        const uint4 w = ldg_stream16(row);
        cv[i][0] = w.x, cv[i][1] = w.y, cv[i][2] = w.z, cv[i][3] = w.w;
      } else {
        asm("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];"
            : "=r"(cv[i][0]), "=r"(cv[i][1]) : "l"(row));
      }
    }
  };
  // The warps' parts of an item, joined in warp order: its rows, or a piece of them.
  auto finish = [&](const ChunkItem& it) {
    const int rows = (it.t1 - it.t0) * G;
    for (int r = tid; r < rows; r += kThreads) {
      float top = neg_inf(), sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm.m[w][r]);
      const float ref = top == neg_inf() ? 0.f : top;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float e = exp2f(sm.m[w][r] - ref);
        sm.weight[w][r] = e;
        sum += sm.l[w][r] == 0.f ? 0.f : e * sm.l[w][r];
      }
      sm.out_m[r] = top;
      sm.out_l[r] = sum;
    }
    __syncthreads();
    float* const part = a.parts + (size_t)(2 * blockIdx.x + it.slot) *
                                      chunk_slot_floats(ROWS, D);
    for (int e = tid; e < rows * (D / 4); e += kThreads) {
      const int r = e / (D / 4), col = e % (D / 4);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (sm.l[w][r] == 0.f) continue;  // a warp that saw no key of the row
        const float4 y = *reinterpret_cast<const float4*>(&sm.o[w][r][col * 4]);
        const float k = sm.weight[w][r];
        x.x = fmaf(k, y.x, x.x);
        x.y = fmaf(k, y.y, x.y);
        x.z = fmaf(k, y.z, x.z);
        x.w = fmaf(k, y.w, x.w);
      }
      const float sum = sm.out_l[r];
      const int64_t tok = it.q.tok0 + it.t0 + r / G;
      const int qh = it.h * G + r % G;
      if (it.whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        TI* dst = reinterpret_cast<TI*>(a.c.out) + tok * a.c.o_st + qh * a.c.o_sh + col * 4;
        *reinterpret_cast<uint2*>(dst) =
            make_uint2(Mma<TI>::pack(x.x * inv, x.y * inv), Mma<TI>::pack(x.z * inv, x.w * inv));
        if (a.c.lse && col == 0)
          a.c.lse[tok * a.c.hq + qh] =
              sum == 0.f ? neg_inf() : (sm.out_m[r] + log2f(sum * exp2f(-kUp))) * kLn2;
      } else {
        *reinterpret_cast<float4*>(part + 2 * ROWS + r * D + col * 4) = x;
        if (col == 0) {
          part[r] = sum == 0.f ? neg_inf() : sm.out_m[r] - kUp;
          part[ROWS + r] = sum;
        }
      }
    }
    if (tid == 0 && it.parts) {
      ChunkMergeDesc d;
      d.parts = it.parts;
      d.tok = it.q.tok0 + it.t0;
      d.rows = rows;
      d.head = it.h;
      a.desc[blockIdx.x] = d;
    }
  };
  bool written = false;  // there are parts
  // An item is prepared (pages, first codes, queries) before the one ahead of it is
  // written out, so that its loads are on their way meanwhile.
#pragma unroll 1
  for (int turn = 0;; turn ^= 1) {
    const bool more = sm.more[turn];
    const ChunkItem& it = sm.item[turn];
    // this warp's blocks: 16 keys from base + kKeys i on, i < n
    int klo = 0, base = 0, end = 0, n = 0;
    const int32_t* table = nullptr;
    // Lane i: block i0 + i, its scales as they are (`record` makes factors of them).
    auto find = [&](int i0) {
      BlockRec r = {0, 0.f, 0};
      const int key = base + (i0 + lane) * kKeys;
      if (key >= end || key + 16 <= klo) return r;
      const int page = key / bs, blk = table[page];
      if (blk < 0 || blk >= a.kv.num_blocks) {
        set_dev_error(a.dev_err, CVSA_DEV_ERR_BLOCK_RANGE);
        return r;
      }
      r.off = blk * a.kv.sb + (key - page * bs) * a.kv.st + it.h * a.kv.sh;
      const int64_t at = (int64_t)blk * a.kv.hkv + it.h;
      r.ks = a.kv.ks[at];
      r.vs = __float_as_uint(a.kv.vs[at]) | 1u;  // not 0
      return r;
    };
    auto record = [&](int i0, BlockRec r) {
      r.ks = pow2(scale_exponent_of(r.ks));
      r.vs = r.vs ? widen_factor(__uint_as_float(r.vs)) : 0;
      sm.rec[warp][(i0 + lane) & 63] = r;
      __syncwarp();
    };
    if (more) {
      klo = it.lo;
      base = (it.tile0 + it.k0) * kKeys + warp * 16;
      end = min(it.hi, (it.tile0 + it.k1) * kKeys);
      n = base < end ? (end - base + kKeys - 1) / kKeys : 0;
      table = a.rg.tables + (int64_t)it.q.slot * a.rg.W;
      const BlockRec found = find(0);
      if (n > 0) {
        const int64_t off = __shfl_sync(0xffffffffu, found.off, 0);
        load_k(off);
        load_v(off);
      }
      if (warp < kNt) {  // query rows (row g of the warp's tile), scaled to f16
        const int rows = (it.t1 - it.t0) * G, r = warp * 8 + g;
        const bool live = r < rows;
        const int64_t at = (int64_t)(it.q.tok0 + it.t0 + (live ? r / G : 0)) * a.c.q_st +
                           (int64_t)(it.h * G + (live ? r % G : 0)) * a.c.q_sh + t * 16;
        float top = 0.f;
        uint4 raw[D / 64][2];
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            raw[c][i] = live ? *reinterpret_cast<const uint4*>(static_cast<const TI*>(a.c.q) + at +
                                                               c * 64 + i * 8)
                             : make_uint4(0, 0, 0, 0);
            float e[8];
            Vec16<TI>::unpack(raw[c][i], e);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(e[j]));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int up = min(120, 13 + 127 - (__float_as_int(top) >> 23));
        const float by = pow2(up);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float e[8];
            Vec16<TI>::unpack(raw[c][i], e);
#pragma unroll
            for (int j = 0; j < 4; j += 2)
              sm.q[warp][c * 4 + i * 2 + j / 2][lane] =
                  make_uint2(Mma<__half>::pack(e[2 * j] * by, e[2 * j + 1] * by),
                             Mma<__half>::pack(e[2 * j + 2] * by, e[2 * j + 3] * by));
          }
        if (t == 0) sm.f[r] = a.scale2 * pow2(-up);
      }
      record(0, found);
    }
    if (written) finish(sm.item[turn ^ 1]);
    if (!more) break;
    __syncthreads();  // the queries are there, the parts of the item before were read
    if (tid == kThreads - 32)  // beside the first loads
      sm.more[turn ^ 1] = walk.next(a.rg, a.g, blockIdx.x, sm.item[turn ^ 1]);
    const int rows = (it.t1 - it.t0) * G;
    BlockRec found, now = sm.rec[warp][0], next = sm.rec[warp][1];  // of blocks i, i + 1
    // Few rows keep their queries in registers, others read them again.
    constexpr bool kQRegs = D * ROWS <= 1024;
    uint2 qr[kQRegs ? kNt : 1][kQRegs ? kSteps : 1];
    if constexpr (kQRegs) {
#pragma unroll
      for (int x = 0; x < kNt; ++x)
#pragma unroll
        for (int j = 0; j < kSteps; ++j) qr[x][j] = sm.q[x][j][lane];
    }
    // S' of the block in ck: key g + 8 (e / 2), row 2t + e % 2
    auto scores = [&](float (*s)[4]) {
#pragma unroll
      for (int x = 0; x < kNt; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[x][e] = 0.f;
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        uint32_t ka[4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint4& w4 = ck[r][j / 4];
          e4m3x4_to_f16x4(j % 4 == 0 ? w4.x : j % 4 == 1 ? w4.y : j % 4 == 2 ? w4.z : w4.w, ka[r],
                          ka[2 + r]);
        }
#pragma unroll
        for (int x = 0; x < kNt; ++x) {
          const uint2 b = kQRegs ? qr[kQRegs ? x : 0][kQRegs ? j : 0] : sm.q[x][j][lane];
          Mma<__half>::m16n8k16(s[x], ka, b.x, b.y);
        }
      }
    };
    float f[kNt][2];
#pragma unroll
    for (int x = 0; x < kNt; ++x)
#pragma unroll
      for (int e = 0; e < 2; ++e) f[x][e] = sm.f[x * 8 + 2 * t + e];
    // keys that every row sees, and those that row 2t + e of tile x sees
    const int first_hi = a.g.causal ? min(it.q.ctx, it.q.start + it.t0 + 1) : it.q.ctx;
    const int last_lo = a.g.window > 0 ? it.q.start + it.t1 - a.g.window : 0;
    auto sees = [&](int x, int e, int key) {
      const int row = x * 8 + 2 * t + e, pos = it.q.start + it.t0 + (row < rows ? row / G : 0);
      return key < (a.g.causal ? min(it.q.ctx, pos + 1) : it.q.ctx) &&
             (a.g.window == 0 || key > pos - a.g.window);
    };
    // c: what goes to a scaled score for its weight, kUp less the reference maximum; beyond
    // any score's reach while the row has seen no key, so that the first one raises it
    constexpr float kNone = 3e38f;
    float m[kNt][2], c[kNt][2], l[kNt][2], o[kNt][kTiles][4];
#pragma unroll
    for (int x = 0; x < kNt; ++x) {
#pragma unroll
      for (int e = 0; e < 2; ++e) m[x][e] = neg_inf(), c[x][e] = kNone, l[x][e] = 0.f;
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[x][j][e] = 0.f;
    }
    float s[kNt][4];
    if (n > 0) {
      scores(s);
      if (n > 1) load_k(next.off);
    }
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      if ((i & 7) == 0) {
        if ((i & 31) == 0) found = find(i + 32);  // ahead of their loads
        if ((i & 31) == 24) record((i & ~31) + 32, found);
      }
      const int key = base + i * kKeys;
      float y[kNt][4];
#pragma unroll
      for (int x = 0; x < kNt; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[x][e] = fmaf(s[x][e], f[x][e & 1] * now.ks, c[x][e & 1]);
      uint32_t hidden = 0;  // bits x * 4 + e
      bool odd = false;
      if (key + 16 > first_hi || key < last_lo || now.vs == 0) {  // some row does not see all
        // values of keys that no row sees are 0 times whatever they hold; of a key that
        // some row sees and another does not, one that is not finite would be NaN in both,
        // so plain FMAs over the keys each row sees
#pragma unroll
        for (int x = 0; x < kNt; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (now.vs == 0 || !sees(x, e & 1, key + g + 8 * (e >> 1))) {
              y[x][e] = neg_inf();
              hidden |= 1u << (x * 4 + e);
            }
        bool nan = false;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int at = key + 2 * t + (r & 1) + 8 * (r >> 1);
          const bool none = at < klo || at >= end || now.vs == 0;
#pragma unroll
          for (int w = 0; w < D / 32; ++w) {
            if (none) cv[r][w] = 0;
            nan |= (((cv[r][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
          }
        }
        odd = __any_sync(0xffffffffu, nan);
      }
      // weights as they are if the maxima stay, and, beside them, the next block's scores
      float p[kNt][4], top = neg_inf();
      uint32_t pb[kNt][2];
#pragma unroll
      for (int x = 0; x < kNt; ++x) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          top = fmaxf(top, y[x][e]);
          p[x][e] = ex2(y[x][e]);
        }
        pb[x][0] = movmatrix_trans(Mma<__half>::pack(p[x][0], p[x][1]));
        pb[x][1] = movmatrix_trans(Mma<__half>::pack(p[x][2], p[x][3]));
      }
      const bool rises = __any_sync(0xffffffffu, top > kRaise + kUp);
      float sn[kNt][4];
      scores(sn);  // past the last block of whatever is there, unused
      const BlockRec after = sm.rec[warp][(i + 2) & 63];
      if (i + 2 < n) load_k(after.off);
      if (rises) {
#pragma unroll
        for (int x = 0; x < kNt; ++x) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float fr = f[x][e] * now.ks;
            const float z0 = hidden >> (x * 4 + e) & 1 ? neg_inf() : s[x][e] * fr;
            const float z1 = hidden >> (x * 4 + 2 + e) & 1 ? neg_inf() : s[x][2 + e] * fr;
            float most = fmaxf(z0, z1);
#pragma unroll
            for (int w = 4; w < 32; w <<= 1)
              most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, w));
            const float up = fmaxf(m[x][e], most);
            const float fix = m[x][e] == neg_inf() ? 0.f : ex2(m[x][e] - up);
            m[x][e] = up;
            c[x][e] = up == neg_inf() ? kNone : kUp - up;
            l[x][e] *= fix;  // NaN stays
#pragma unroll
            for (int j = 0; j < kTiles; ++j) o[x][j][e] *= fix, o[x][j][2 + e] *= fix;
            p[x][e] = ex2(z0 + c[x][e]);
            p[x][2 + e] = ex2(z1 + c[x][e]);
          }
          pb[x][0] = movmatrix_trans(Mma<__half>::pack(p[x][0], p[x][1]));
          pb[x][1] = movmatrix_trans(Mma<__half>::pack(p[x][2], p[x][3]));
        }
      }
#pragma unroll
      for (int x = 0; x < kNt; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) l[x][e & 1] += p[x][e];
      if (odd) {
        const float vf = __half2float(__ushort_as_half((unsigned short)(now.vs & 0xffffu)));
        __syncwarp();
#pragma unroll
        for (int x = 0; x < kNt; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sm.p[warp][x * 8 + 2 * t + (e & 1)][g + 8 * (e >> 1)] =
                hidden >> (x * 4 + e) & 1 ? -1.f : p[x][e];
        __syncwarp();
        const uint8_t* const pv = static_cast<const uint8_t*>(a.kv.v) + now.off + g * kCols;
#pragma unroll 1
        for (int col = 0; col < 16; ++col) {
          if (key + col < klo || key + col >= end) continue;
#pragma unroll
          for (int j = 0; j < kCols; ++j) {
            float w[4];
            e4m3x4_to_f4(pv[col * st + j], w);
#pragma unroll
            for (int x = 0; x < kNt; ++x)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float u = sm.p[warp][x * 8 + 2 * t + e][col];
                float& z = o[x][j / 2][(j & 1) * 2 + e];
                if (u >= 0.f || u != u) z = fmaf(u, w[0] * vf, z);
              }
          }
        }
      } else {
#pragma unroll
        for (int w = 0; w < D / 32; ++w)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x7362 : 0x5140;
            uint32_t va[4];
            e4m3x4_to_f16x4(__byte_perm(cv[0][w], cv[1][w], sel), va[0], va[1]);
            e4m3x4_to_f16x4(__byte_perm(cv[2][w], cv[3][w], sel), va[2], va[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) va[e] = hmul2(va[e], now.vs);
#pragma unroll
            for (int x = 0; x < kNt; ++x)
              Mma<__half>::m16n8k16(o[x][w * 2 + half], va, pb[x][0], pb[x][1]);
          }
      }
      if (i + 1 < n) load_v(next.off);
      now = next;
      next = after;
#pragma unroll
      for (int x = 0; x < kNt; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[x][e] = sn[x][e];
    }
    // the warps' parts, joined in warp order
#pragma unroll
    for (int x = 0; x < kNt; ++x)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = x * 8 + 2 * t + e;
        float sum = l[x][e];
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        if (g == 0) {
          sm.m[warp][r] = m[x][e];
          sm.l[warp][r] = sum;
        }
#pragma unroll
        for (int j = 0; j < kCols; j += 4)
          *reinterpret_cast<float4*>(&sm.o[warp][r][g * kCols + j]) =
              make_float4(o[x][j / 2][e], o[x][j / 2][2 + e], o[x][j / 2 + 1][e],
                          o[x][j / 2 + 1][2 + e]);
      }
    written = true;
    __syncthreads();
  }
  pdl_launch_dependents();  // the merge
}

// Joins the pieces of the item that begins in CTA y's range: block (x, y) its row x.
// Warps take pieces in turn, lanes columns; sums in a fixed order. A slot is
// m [rows], l [rows], o [rows][D].
constexpr int kJoin = 4;
template <typename TI, int D>
__global__ void __launch_bounds__(32 * kJoin) few_merge_kernel(const float* parts,
                                                               const ChunkMergeDesc* desc,
                                                               ChunkView c, int slot_rows, int G) {
  __shared__ float weight[kMaxCtas];
  __shared__ float red[kJoin][2];
  __shared__ float sums[kJoin][D];
  const int cta = blockIdx.y, r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  const ChunkMergeDesc ds = desc[cta];
  if (r >= ds.rows || ds.parts == 0) return;
  auto slot = [&](int p) {
    return parts + (size_t)(p == 0 ? 2 * cta + 1 : 2 * (cta + p)) * chunk_slot_floats(slot_rows, D);
  };
  float top = neg_inf(), sum = 0.f;
  for (int p = tid; p < ds.parts; p += 32 * kJoin) top = fmaxf(top, weight[p] = slot(p)[r]);
  top = warp_max(top);
  if (lane == 0) red[warp][0] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoin; ++w) top = fmaxf(top, red[w][0]);
  const float ref = top == neg_inf() ? 0.f : top;
  for (int p = tid; p < ds.parts; p += 32 * kJoin) {
    const float l = slot(p)[slot_rows + r], e = exp2f(weight[p] - ref);
    // a piece that saw no key of the row holds nothing; NaN stays
    weight[p] = l == 0.f ? 0.f : e;
    sum += l == 0.f ? 0.f : e * l;
  }
  sum = warp_sum(sum);
  if (lane == 0) red[warp][1] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kJoin; ++w) sum += red[w][1];
  constexpr int kPer = D / 32;  // columns a lane
  float o[kPer] = {};
#pragma unroll 4
  for (int p = warp; p < ds.parts; p += kJoin) {
    const float* const src = slot(p) + 2 * slot_rows + r * D + lane * kPer;
    float x[kPer];
    if constexpr (kPer == 4) *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(src);
    else *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(src);
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = fmaf(weight[p], x[i], o[i]);
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) sums[warp][lane * kPer + i] = o[i];
  __syncthreads();
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t tok = ds.tok + r / G;
  const int qh = ds.head * G + r % G;
  if (tid < D / 4) {
    float x[4] = {};
#pragma unroll
    for (int w = 0; w < kJoin; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] += sums[w][tid * 4 + i];
    *reinterpret_cast<uint2*>(reinterpret_cast<TI*>(c.out) + tok * c.o_st + qh * c.o_sh + tid * 4) =
        make_uint2(Mma<TI>::pack(x[0] * inv, x[1] * inv), Mma<TI>::pack(x[2] * inv, x[3] * inv));
  }
  if (c.lse && tid == 0)
    c.lse[tok * c.hq + qh] = sum == 0.f ? neg_inf() : (top + log2f(sum)) * kLn2;
}

template <typename TI, int D, int ROWS>
cudaError_t launch_few(const FewArgs& a, int ctas, cudaStream_t s) {
  constexpr int kSmem = (int)sizeof(FewSmem<D, ROWS>);
  static_assert(kSmem <= 113 * 1024, "two blocks an SM");
  cudaError_t e = cudaFuncSetAttribute(chunk_few_kernel<TI, D, ROWS>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  chunk_few_kernel<TI, D, ROWS><<<ctas, 32 * few_warps(D, ROWS), kSmem, s>>>(a);
  e = cudaGetLastError();
  if (e != cudaSuccess || !a.g.split) return e;
  return launch_k(few_merge_kernel<TI, D>, dim3(ROWS, ctas), dim3(32 * kJoin), 0, s, true,
                  (const float*)a.parts, (const ChunkMergeDesc*)a.desc, a.c, ROWS, a.g.G);
}

template <typename TI, int D>
cudaError_t launch_rows(const FewArgs& a, int rows, int ctas, cudaStream_t s) {
  if (rows == 8) return launch_few<TI, D, 8>(a, ctas, s);
  if (rows == 16) return launch_few<TI, D, 16>(a, ctas, s);
  return launch_few<TI, D, 32>(a, ctas, s);
}

}  // namespace

// Rows of an item, or 0 where the other kernels serve the call: never fewer than one token's.
// By the batch's mean of rows a sequence, rounded up: longer sequences take several items,
// which read its cache again each, so batches that hold a prompt are left to the tensor cores.
// Here against there:
// 32 single tokens 72 and 291 us, 8 drafts of 2 to 8 tokens 80 and 101 us (64-wide heads),
// 115 and 157 us (128-wide).
int chunk_few_rows(const KvView& kv, const RaggedView& rg, const ChunkView& c) {
  if (kv.dtype != CVSA_DTYPE_E4M3 || c.dtype == CVSA_DTYPE_F32 || (kv.d != 64 && kv.d != 128) ||
      kv.bs % 16)
    return 0;
  const int64_t mean = rg.B > 0 ? ((int64_t)rg.T + rg.B - 1) / rg.B : rg.T;
  const int64_t rows = (mean > 0 ? mean : 1) * (c.hq / kv.hkv);
  return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 0;
}

// Blocks: two an SM.
int chunk_few_ctas() { return chunk_grid(2); }

ChunkGeo chunk_few_geo(const KvView& kv, const RaggedView& rg, const ChunkView& c, int rows) {
  ChunkGeo g;
  g.bs = kv.bs;
  g.hkv = kv.hkv;
  g.G = c.hq / kv.hkv;
  g.P = rows / g.G;
  g.KT = 16 * few_warps(kv.d, rows);
  g.causal = c.causal;
  g.window = c.window;
  g.fixed = g.fixed_few = 2;
  g.few = 0;
  g.split = chunk_may_split(rg, kv.bs, g.KT);
  return g;
}

cudaError_t launch_chunk_few(const KvView& kv, const RaggedView& rg, const ChunkView& c, int rows,
                             int ctas, float* parts, ChunkMergeDesc* desc, int32_t* dev_err,
                             cudaStream_t s) {
  FewArgs a;
  a.rg = rg;
  a.kv = kv;
  a.c = c;
  a.g = chunk_few_geo(kv, rg, c, rows);
  a.scale2 = c.scale * kLog2e;
  a.min_units = 4;
  a.parts = parts;
  a.desc = desc;
  a.dev_err = dev_err;
  if (c.dtype == CVSA_DTYPE_BF16)
    return kv.d == 64 ? launch_rows<__nv_bfloat16, 64>(a, rows, ctas, s)
                      : launch_rows<__nv_bfloat16, 128>(a, rows, ctas, s);
  return kv.d == 64 ? launch_rows<__half, 64>(a, rows, ctas, s)
                    : launch_rows<__half, 128>(a, rows, ctas, s);
}

}  // namespace cvsa
