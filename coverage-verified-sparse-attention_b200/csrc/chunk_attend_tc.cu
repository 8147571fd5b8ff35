// Attention of a ragged batch of new tokens over the paged cache on the tensor
// cores: 16-bit pools of q's dtype, head_dim 64 or 128. Formulas as in
// chunk_attend.cu, work split as in chunk_plan.cuh.
//
// A persistent CTA an SM. An item's query rows (token, head of the group) are
// packed into one or two tiles of 128 rows, so a KV tile of 128 keys, brought
// in once, serves up to 256 rows. Per tile and Q tile:
//   S = Q K^T   (both from shared memory, fp32 in tensor memory)
//   P = exp2(scale2 S - m) in registers, one row a thread, back to tensor
//       memory in 16 bits over S
//   O += P V    (P from tensor memory, V from shared memory)
// Roles: warps 0-3 and 4-7 the softmax of Q tile 0 and 1 (and the rescaling
// and output of its O), warps 8-11 the loads, warp 12 issues the MMAs. The
// two Q tiles take turns on the tensor core: while one is in its softmax the
// other's products run. A row is one thread's, so its maximum and sum need no
// exchange.
//
// Loads: a page holds 16 tokens of one head 2 KB or 4 KB apart, so a tensor
// copy would be many small boxes; 16-byte asynchronous copies per lane,
// straight into the 128-byte-swizzled layout, take any page size and stride.
// Keys outside the item's range and bad blocks are zero-filled.
//
// The running maximum is only raised when it grows by more than 2^8 in the
// weights' domain (weights up to 256 are exact enough in fp32 sums and in
// 16 bits), so O is rarely rescaled. Weights are rounded to the 16-bit type for
// the second product (the tensor core's operand type); their sum is taken
// before the rounding, in fp32, and the error this adds is of the size of the
// output's own rounding.
//
// A masked weight is exactly 0, but 0 times a non-finite V is NaN: the loading
// warps check the V rows of tiles some row sees only in part, and a tile with
// a non-finite value is added by the softmax warps with plain FMAs over the
// keys each row sees. Rows that see the value get it, others do not.
#include <type_traits>

#include "chunk_plan.cuh"
#include "cvsa_common.cuh"
#include "cvsa_internal.h"
#include "tcgen05.cuh"

namespace cvsa {
namespace {

constexpr int kThreads = 512, kTile = 128, kKT = 128;
// Tile records: one is rewritten when a tile kSlots later is loaded, whose buffer
// is free only once the softmax of the tile kSlots - kStages / 2 - 1 or more
// before it has been handed over.
constexpr int kSlots = 8;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kRaise = 8.f;  // log2 growth of the maximum that triggers a rescale

template <int D>
struct Cfg {
  static constexpr int kStage = kKT * D * 2;            // bytes of a K or V tile
  static constexpr int kStages = D == 128 ? 4 : 8;
  static constexpr int kQTile = kTile * D * 2;
  static constexpr int kPanel = kKT * 128;              // bytes of a panel
  static constexpr int kRing = 2 * kQTile;              // offset of the ring
  static constexpr int kMeta = kRing + kStages * kStage;
};

struct TcMeta {
  uint64_t kv_full[8], kv_empty[8];
  uint64_t q_full, q_empty;
  uint64_t s_full[2], p_full[2], o_full[2];
  uint64_t drain;
  uint32_t key_bad[kSlots][4];  // per tile (mod kSlots): bit per key no row may see
  uint32_t v_odd[kSlots][4];    // per tile and loading warp: a V value is not finite
  uint32_t tmem;
  uint32_t abort;
};

struct TcArgs {
  RaggedView rg;
  KvView kv;
  ChunkView c;
  ChunkGeo g;
  int TQ;               // tokens of a Q tile
  int bs_shift;         // log2 of the page size, or -1
  float scale2;
  int min_units;
  float* parts;
  ChunkMergeDesc* desc;
  int32_t* dev_err;
  uint32_t wait_limit;
};

// Bounded wait; false (with the CTA's abort flag and CVSA_DEV_ERR_TIMEOUT set)
// when the phase does not complete, or another warp gave up.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, TcMeta* m,
                                         const TcArgs& a) {
  for (uint32_t i = 0; i < a.wait_limit; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 15) == 15 && *reinterpret_cast<volatile uint32_t*>(&m->abort)) return false;
  }
  *reinterpret_cast<volatile uint32_t*>(&m->abort) = 1;
  set_dev_error(a.dev_err, CVSA_DEV_ERR_TIMEOUT);
  return false;
}

// The same by a whole warp, with one answer for all lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, TcMeta* m,
                                          const TcArgs& a) {
  return __all_sync(0xffffffffu, wait_for(bar, parity, m, a));
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

// Whether some row of the item does not see all keys [base, base + KT).
__device__ __forceinline__ bool tile_partial(const ChunkItem& it, const ChunkGeo& g, int base) {
  const int first_hi = g.causal ? min(it.q.ctx, it.q.start + it.t0 + 1) : it.q.ctx;
  const int last_lo = g.window > 0 ? it.q.start + it.t1 - g.window : 0;
  return base + kKT > first_hi || base < last_lo;
}

// ---------------------------------------------------------------------------
// loading warps
// ---------------------------------------------------------------------------
// A copy's arrival on its buffer's barrier is left to the hardware
// (cp.async.mbarrier.arrive), so these warps never wait for their own copies,
// and the proxy fence the tensor core needs is the MMA thread's: a fence in a
// thread with copies in flight waits for all of them (2500 cycles a buffer).
__device__ __forceinline__ void arrive_when_landed(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

template <typename T, int D>
struct Loader {
  using C = Cfg<D>;
  static constexpr int kCh = D / 8;           // 16-byte chunks a row
  static constexpr int kRPI = 32 / kCh;       // rows a warp instruction
  const TcArgs& a;
  TcMeta* m;
  uint32_t base;    // shared memory base
  int w, lane;

  __device__ Loader(const TcArgs& a_, TcMeta* m_, uint32_t base_, int w_, int lane_)
      : a(a_), m(m_), base(base_), w(w_), lane(lane_) {}

  __device__ __forceinline__ uint32_t dst(uint32_t tile, int row, int ch) const {
    return tile + (ch >> 3) * C::kPanel + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
  }
  // Whether this warp's rows of a V tile hold a value that is not finite.
  __device__ __forceinline__ bool has_odd(uint32_t tile) const {
    bool odd = false;
    const int ch = lane % kCh;
    for (int i = 0; i < 32 / kRPI; ++i) {
      const int row = w * 32 + i * kRPI + lane / kCh;
      uint32_t x[4];
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                   : "r"(dst(tile, row, ch)));
      constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
#pragma unroll
      for (int j = 0; j < 4; ++j) odd |= __vcmpgeu2(x[j] & 0x7fff7fffu, kExp) != 0;
    }
    return __any_sync(0xffffffffu, odd);
  }
  // 32 rows of this warp; `off` is each lane's row offset in elements, < 0: zeros
  __device__ __forceinline__ void copy_rows(uint32_t tile, const void* src, int64_t off) {
    const int ch = lane % kCh;
#pragma unroll 8
    for (int i = 0; i < 32 / kRPI; ++i) {
      const int r = i * kRPI + lane / kCh;
      const int64_t o = __shfl_sync(0xffffffffu, off, r);
      const bool ok = o >= 0;
      cp16(dst(tile, w * 32 + r, ch), reinterpret_cast<const T*>(src) + (ok ? o + ch * 8 : 0), ok);
    }
  }

  __device__ void run(const ChunkRange& rng) {
    ChunkWalk walk(rng);
    ChunkItem it;
    uint32_t op = 0, items = 0;
    while (walk.next(a.rg, a.g, it)) {
      if (it.hi <= it.lo) continue;
      const int G = a.g.G;
      // queries
      if (!warp_wait(&m->q_empty, (items & 1) ^ 1, m, a)) break;
      const int ntok = it.t1 - it.t0;
      const int nq = ntok > a.TQ ? 2 : 1;
      for (int q = 0; q < nq; ++q) {
        const int r = w * 32 + lane;
        const int rows = min(a.TQ, ntok - q * a.TQ) * G;
        int64_t off = -1;
        if (r < rows)
          off = (int64_t)(it.q.tok0 + it.t0 + q * a.TQ + r / G) * a.c.q_st +
                (int64_t)(it.h * G + r % G) * a.c.q_sh;
        copy_rows(base + q * C::kQTile, a.c.q, off);
      }
      arrive_when_landed(&m->q_full);
      ++items;
      // keys and values
      const int32_t* table = a.rg.tables + (int64_t)it.q.slot * a.rg.W;
      auto block_of = [&](int key) {  // -1: not an item key
        if (key < it.lo || key >= it.hi) return -1;
        return table[a.bs_shift >= 0 ? key >> a.bs_shift : key / a.kv.bs];
      };
      int key = (it.tile0 + it.k0) * kKT + w * 32 + lane;
      int blk = block_of(key);
      for (int k = it.k0; k < it.k1; ++k, key += kKT) {
        const int next = k + 1 < it.k1 ? block_of(key + kKT) : -1;
        int64_t off = -1;
        if (key >= it.lo && key < it.hi) {
          if (blk >= 0 && blk < a.kv.num_blocks) {
            const int in = a.bs_shift >= 0 ? key & (a.kv.bs - 1) : key % a.kv.bs;
            off = blk * a.kv.sb + in * a.kv.st + it.h * a.kv.sh;
          } else {
            set_dev_error(a.dev_err, CVSA_DEV_ERR_BLOCK_RANGE);
          }
        }
        blk = next;
        const uint32_t slot = (op >> 1) % kSlots;
        uint32_t st = op % C::kStages;
        if (!warp_wait(&m->kv_empty[st], ((op / C::kStages) & 1) ^ 1, m, a)) goto out;
        const uint32_t bad = __ballot_sync(0xffffffffu, off < 0);
        if (lane == 0) {
          m->key_bad[slot][w] = bad;
          mbar_arrive(&m->kv_full[st]);  // a plain arrival, behind the plain write
        }
        copy_rows(base + C::kRing + st * C::kStage, a.kv.k, off);
        arrive_when_landed(&m->kv_full[st]);
        ++op;
        st = op % C::kStages;
        if (!warp_wait(&m->kv_empty[st], ((op / C::kStages) & 1) ^ 1, m, a)) goto out;
        const uint32_t v = base + C::kRing + st * C::kStage;
        copy_rows(v, a.kv.v, off);
        if (tile_partial(it, a.g, (it.tile0 + k) * kKT)) {
          asm volatile("cp.async.wait_all;" ::: "memory");
          __syncwarp();
          const bool odd = has_odd(v);
          if (lane == 0) m->v_odd[slot][w] = odd;
          mbar_arrive(&m->kv_full[st]);
        } else {
          arrive_when_landed(&m->kv_full[st]);
        }
        ++op;
      }
    }
  out:
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
};

// ---------------------------------------------------------------------------
// MMA issue (one warp, one elected lane)
// ---------------------------------------------------------------------------
// The whole warp runs the loop, with its trip counts broadcast, so that the
// compiler keeps descriptors in uniform registers, where the instruction
// wants them: issued from a single-lane branch each MMA cost about 95 cycles
// of moves, against the 64 that it runs.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

template <typename T, int D>
__device__ __forceinline__ void mma_role(const TcArgs& a, TcMeta* m, uint32_t base, uint32_t tmem,
                                         const ChunkRange& rng) {
  using C = Cfg<D>;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  constexpr uint32_t kIdS = mma_idesc(kBf16, kTile, kKT, false);
  constexpr uint32_t kIdO = mma_idesc(kBf16, kTile, D, true);
  const uint32_t ring = base + C::kRing;
  const uint64_t q_desc = smem_desc(base, 16, 1024), k_desc = smem_desc(ring, 16, 1024),
                 v_desc = smem_desc(ring, C::kPanel, 1024);
  ChunkWalk walk(rng);
  ChunkItem it;
  uint32_t op = 0, items = 0, turn0 = 0, turn1 = 0;
  auto scores = [&](int q, uint32_t st) {  // S_q = Q_q K^T
    if (elect_one()) {
      const uint32_t d = tmem + q * kKT;
      const uint64_t qd = q_desc + ((q * C::kQTile) >> 4), kd = k_desc + ((st * C::kStage) >> 4);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t o = ((kk / 4) * C::kPanel + (kk % 4) * 32) >> 4;
        mma_ss(d, qd + o, kd + o, kIdS, kk > 0);
      }
      mma_commit(smem_u32(&m->s_full[q]));
      mbar_arrive(&m->s_full[q]);  // orders the loaders' plain writes before the softmax too
    }
    __syncwarp();
  };
  auto outputs = [&](int q, uint32_t st, bool acc) {  // O_q (+)= P_q V
    if (elect_one()) {
      const uint32_t d = tmem + 2 * kKT + q * D, p = tmem + q * kKT;
      const uint64_t vd = v_desc + ((st * C::kStage) >> 4);
#pragma unroll
      for (int kk = 0; kk < kKT / 16; ++kk)
        mma_ts(d, p + kk * 8, vd + ((kk * 2048) >> 4), kIdO, acc || kk > 0);
    }
    __syncwarp();
  };
  auto commit = [&](uint64_t* bar) {
    if (elect_one()) mma_commit(smem_u32(bar));
    __syncwarp();
  };
  while (walk.next(a.rg, a.g, it)) {
    if (it.hi <= it.lo) continue;
    const int nq = uniform(it.t1 - it.t0 > a.TQ ? 2 : 1);
    const int nt = uniform(it.k1 - it.k0);
    if (!warp_wait(&m->q_full, items & 1, m, a)) break;
    ++items;
    for (int j = 0; j <= nt; ++j) {
      const uint32_t kop = op + 2 * j, vop = kop - 1;
      const uint32_t kst = kop % C::kStages, vst = vop % C::kStages;
      if (j < nt && !warp_wait(&m->kv_full[kst], (kop / C::kStages) & 1, m, a)) goto out;
      bool skip = false;
      if (j > 0) {
        if (!warp_wait(&m->kv_full[vst], (vop / C::kStages) & 1, m, a)) goto out;
        if (tile_partial(it, a.g, (it.tile0 + it.k0 + j - 1) * kKT)) {
          const uint32_t slot = (vop >> 1) % kSlots;
          skip = uniform(m->v_odd[slot][0] | m->v_odd[slot][1] | m->v_odd[slot][2] |
                         m->v_odd[slot][3]);
        }
      }
      fence_proxy_async_smem();  // the tiles were written through the generic proxy
      tc_fence_after();
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (q >= nq) break;
        if (j > 0) {
          uint32_t& turn = q ? turn1 : turn0;
          if (!warp_wait(&m->p_full[q], turn & 1, m, a)) goto out;
          ++turn;
          tc_fence_after();
          if (!skip) outputs(q, vst, j > 1);
          if (j == nt) commit(&m->o_full[q]);
        }
        if (j < nt) scores(q, kst);
      }
      if (j < nt) commit(&m->kv_empty[kst]);
      if (j > 0) commit(&m->kv_empty[vst]);
      if (j == nt - 1) commit(&m->q_empty);
    }
    op += 2 * nt;
  }
out:
  // nothing of this CTA may be in flight when its tensor memory is freed
  commit(&m->drain);
  mbar_wait_bounded(&m->drain, 0, 1u << 22);
  __syncwarp();
}

// ---------------------------------------------------------------------------
// softmax, rescaling and output of one Q tile
// ---------------------------------------------------------------------------
template <typename T, int D>
__device__ __forceinline__ void softmax_role(const TcArgs& a, TcMeta* m, uint32_t base,
                                             uint32_t tmem, const ChunkRange& rng, int q) {
  using C = Cfg<D>;
  const int r = threadIdx.x & 127, warp = r >> 5;
  const uint32_t lanes = (uint32_t)(warp * 32) << 16;
  const uint32_t ts = tmem + q * kKT + lanes, to = tmem + 2 * kKT + q * D + lanes;
  const int G = a.g.G;
  ChunkWalk walk(rng);
  ChunkItem it;
  uint32_t op = 0, turns = 0, ends = 0;
  while (walk.next(a.rg, a.g, it)) {
    const int ntok = min(a.TQ, it.t1 - it.t0 - q * a.TQ);
    const bool empty = it.hi <= it.lo;
    const int nt = empty ? 0 : it.k1 - it.k0;
    if (ntok <= 0) {
      op += 2 * nt;
      continue;
    }
    const int rows = ntok * G;
    const bool active = warp * 32 < rows;
    const int pos = it.q.start + it.t0 + q * a.TQ + r / G;
    const int hi = a.g.causal ? min(it.q.ctx, pos + 1) : it.q.ctx;
    const int lo = a.g.window > 0 ? pos - a.g.window + 1 : 0;
    float mx = neg_inf(), l = 0.f;
    for (int j = 0; j < nt; ++j, op += 2) {
      if (!warp_wait(&m->s_full[q], turns & 1, m, a)) return;
      ++turns;
      tc_fence_after();
      const int kbase = (it.tile0 + it.k0 + j) * kKT;
      const uint32_t slot = (op >> 1) % kSlots;
      const bool partial = tile_partial(it, a.g, kbase);
      bool odd = false;
      if (partial) {
        const uint32_t vop = op + 1;
        if (!warp_wait(&m->kv_full[vop % C::kStages], (vop / C::kStages) & 1, m, a)) return;
        odd = m->v_odd[slot][0] | m->v_odd[slot][1] | m->v_odd[slot][2] | m->v_odd[slot][3];
      }
      if (active) {
        float s[kKT];
#pragma unroll
        for (int c = 0; c < kKT; c += 32) tmem_ld32(ts + c, s + c);
        uint32_t bad[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) bad[i] = m->key_bad[slot][i];
        const bool masked = partial || (bad[0] | bad[1] | bad[2] | bad[3]);
        tmem_wait_ld();
        if (masked) {
          // bit c of see[c / 32]: this row sees key kbase + c
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int h = hi - kbase - 32 * i, b = lo - kbase - 32 * i;
            const uint32_t upto = h >= 32 ? 0xffffffffu : h <= 0 ? 0u : (1u << h) - 1;
            const uint32_t from = b <= 0 ? 0xffffffffu : b >= 32 ? 0u : 0xffffffffu << b;
            bad[i] = ~(upto & from) | bad[i];
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (bad[i] >> c & 1) s[32 * i + c] = neg_inf();
          }
        }
        float t4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c < kKT; c += 4) {
#pragma unroll
          for (int i = 0; i < 4; ++i) t4[i] = fmaxf(t4[i], s[c + i]);
        }
        const float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
        float fix = 1.f;
        if ((top - mx) * a.scale2 > kRaise || mx == neg_inf()) {
          const float raised = fmaxf(mx, top);
          if (mx != neg_inf()) fix = ex2((mx - raised) * a.scale2);
          mx = raised;
        }
        if (j > 0 && __any_sync(0xffffffffu, fix != 1.f)) {
          // O of all earlier tiles is complete: S of this tile was issued behind it
#pragma unroll 1
          for (int c = 0; c < D; c += 8) {
            float o[8];
            tmem_ld8(to + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] *= fix;
            tmem_st8(to + c, o);
          }
        }
        l *= fix;
        const float ref = mx == neg_inf() ? 0.f : -mx * a.scale2;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        if (!odd) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t p[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const float x = ex2(fmaf(s[64 * half + 2 * c], a.scale2, ref));
              const float y = ex2(fmaf(s[64 * half + 2 * c + 1], a.scale2, ref));
              sum[(2 * c) & 3] += x;
              sum[(2 * c + 1) & 3] += y;
              p[c] = Mma<T>::pack(x, y);
            }
            tmem_st32(ts + 32 * half, p);
          }
        } else {
          // a value of V is not finite and some row does not see it: plain FMAs.
          // The weights go over S in fp32, -1 for an unseen key.
#pragma unroll
          for (int c = 0; c < kKT; c += 32) {
            uint32_t p[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float x = ex2(fmaf(s[c + i], a.scale2, ref));
              const bool see = !(bad[c / 32] >> i & 1);
              sum[i & 3] += x;
              p[i] = __float_as_uint(see ? x : -1.f);
            }
            tmem_st32(ts + c, p);
          }
          tmem_wait_st();
          const uint32_t v = base + C::kRing + ((op + 1) % C::kStages) * C::kStage;
#pragma unroll 1
          for (int ch = 0; ch < D / 8; ++ch) {
            float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (j > 0) {
              tmem_ld8(to + ch * 8, o);
              tmem_wait_ld();
            }
#pragma unroll 1
            for (int c = 0; c < kKT; c += 8) {
              float p[8];
              tmem_ld8(ts + c, p);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int row = c + i;
                uint4 x;
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                             : "r"(v + (ch >> 3) * C::kPanel + row * 128 +
                                   (((ch & 7) ^ (row & 7)) << 4)));
                float f[8];
                Vec16<T>::unpack(x, f);
                if (p[i] >= 0.f || p[i] != p[i]) {
#pragma unroll
                  for (int e = 0; e < 8; ++e) o[e] = fmaf(p[i], f[e], o[e]);
                }
              }
            }
            tmem_st8(to + ch * 8, o);
          }
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_wait_st();
      }
      tc_fence_before();
      mbar_arrive(&m->p_full[q]);
    }
    // the item's rows, or this range's part of them
    if (nt > 0) {
      if (!warp_wait(&m->o_full[q], ends & 1, m, a)) return;
      ++ends;
      tc_fence_after();
    }
    const bool whole = it.k0 == 0 && it.k1 == it.units;
    const int cta = blockIdx.x;
    if (active) {
      const bool live = r < rows;
      const int64_t tok = it.q.tok0 + it.t0 + q * a.TQ + r / G;
      const int head = it.h * G + r % G;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      T* dst = reinterpret_cast<T*>(a.c.out) + tok * a.c.o_st + head * a.c.o_sh;
      const int R = 2 * kTile, rr = q * a.TQ * G + r;
      float* part = a.parts + (size_t)chunk_slot(it, rng.u0, cta) * chunk_slot_floats(R, D);
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        float o[32];
        if (nt > 0) {
          tmem_ld32(to + c, o);
          tmem_wait_ld();
        }
        if (l == 0.f) {  // a row without a key (or without any so far)
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
        }
        if (live && whole) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 x;
            x.x = Mma<T>::pack(o[i] * inv, o[i + 1] * inv);
            x.y = Mma<T>::pack(o[i + 2] * inv, o[i + 3] * inv);
            x.z = Mma<T>::pack(o[i + 4] * inv, o[i + 5] * inv);
            x.w = Mma<T>::pack(o[i + 6] * inv, o[i + 7] * inv);
            *reinterpret_cast<uint4*>(dst + c + i) = x;
          }
        } else if (live) {
          float4* po = reinterpret_cast<float4*>(part + 2 * R) + (size_t)(c / 4) * R + rr;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            po[(size_t)i * R] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
        __syncwarp();
      }
      if (live) {
        const float m2 = mx * a.scale2;
        if (whole) {
          if (a.c.lse)
            a.c.lse[tok * a.c.hq + head] = l == 0.f ? neg_inf() : (m2 + log2f(l)) * kLn2;
        } else {
          part[rr] = l == 0.f ? neg_inf() : m2;
          part[R + rr] = l;
        }
      }
    }
    if (threadIdx.x == 0 && !whole && it.k0 == 0) {
      ChunkMergeDesc d;
      d.parts = (int)((it.first + it.units - 1) / rng.per_cta) - cta + 1;
      d.tok = it.q.tok0 + it.t0;
      d.rows = (it.t1 - it.t0) * G;
      d.head = it.h;
      a.desc[cta] = d;
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) chunk_tc_kernel(const __grid_constant__ TcArgs a) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  TcMeta* m = reinterpret_cast<TcMeta*>(smem + C::kMeta);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&m->kv_full[i], i % 2 ? 128 : 128 + 4);  // K (even): and the key_bad writers
      mbar_init(&m->kv_empty[i], 1);
    }
    mbar_init(&m->q_full, 128);
    mbar_init(&m->q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&m->s_full[i], 2);
      mbar_init(&m->p_full[i], 128);
      mbar_init(&m->o_full[i], 1);
    }
    mbar_init(&m->drain, 1);
    m->abort = 0;
    fence_mbar_init();
    a.desc[blockIdx.x].parts = 0;
  }
  if (warp == 12) tmem_alloc(smem_u32(&m->tmem), 512);
  // the plan's scratch is the ring's memory
  const ChunkRange rng = chunk_range<kThreads>(
      a.rg, a.g, *reinterpret_cast<ChunkPlanSmem<kThreads>*>(smem + C::kRing), blockIdx.x,
      gridDim.x, a.min_units, a.dev_err);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t base = smem_u32(smem), tmem = __shfl_sync(0xffffffffu, m->tmem, 0);
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    softmax_role<T, D>(a, m, base, tmem, rng, warp / 4);
  } else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    Loader<T, D>(a, m, base, warp - 8, lane).run(rng);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 12) mma_role<T, D>(a, m, base, tmem, rng);
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int D>
cudaError_t launch_tc(const TcArgs& a, int ctas, cudaStream_t s) {
  using C = Cfg<D>;
  static_assert(sizeof(ChunkPlanSmem<kThreads>) <= C::kStages * C::kStage, "plan scratch");
  constexpr int kSmem = C::kMeta + (int)sizeof(TcMeta) + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory");
  cudaError_t e = cudaFuncSetAttribute(chunk_tc_kernel<T, D>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  chunk_tc_kernel<T, D><<<ctas, kThreads, kSmem, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

bool chunk_tc_eligible(const KvView& kv, const ChunkView& c) {
  return c.dtype == kv.dtype && kv.dtype != CVSA_DTYPE_F32 && (kv.d == 64 || kv.d == 128) &&
         c.hq / kv.hkv <= kTile;
}

int chunk_tc_rows() { return 2 * kTile; }

cudaError_t launch_chunk_tc(const KvView& kv, const RaggedView& rg, const ChunkView& c, int ctas,
                            float* parts, ChunkMergeDesc* desc, int32_t* dev_err, cudaStream_t s) {
  TcArgs a;
  a.rg = rg;
  a.kv = kv;
  a.c = c;
  a.TQ = kTile / (c.hq / kv.hkv);
  a.g.bs = kv.bs;
  a.g.hkv = kv.hkv;
  a.g.G = c.hq / kv.hkv;
  a.g.P = 2 * a.TQ;
  a.g.KT = kKT;
  a.g.causal = c.causal;
  a.g.window = c.window;
  a.bs_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (kv.bs == 1 << i) a.bs_shift = i;
  a.scale2 = c.scale * kLog2e;
  a.min_units = 2;
  a.parts = parts;
  a.desc = desc;
  a.dev_err = dev_err;
  a.wait_limit = wait_limit() ? wait_limit() : 1u << 22;
  if (kv.dtype == CVSA_DTYPE_BF16)
    return kv.d == 64 ? launch_tc<__nv_bfloat16, 64>(a, ctas, s)
                      : launch_tc<__nv_bfloat16, 128>(a, ctas, s);
  return kv.d == 64 ? launch_tc<__half, 64>(a, ctas, s) : launch_tc<__half, 128>(a, ctas, s);
}

}  // namespace cvsa
