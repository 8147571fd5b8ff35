// Attention of a ragged batch of new tokens over the paged cache on the tensor
// cores: 16-bit pools of q's dtype or 8-bit pools, head_dim 64 or 128. Formulas as in
// chunk_attend.cu, work split as in chunk_plan.cuh.
//
// A persistent CTA an SM. An item's query rows (token, head of the group) are
// packed into one or two tiles of 128 rows, so a KV tile of 128 keys, brought
// in once, serves up to 256 rows. Per tile and Q tile:
//   S = Q K^T   (both from shared memory, fp32 in tensor memory)
//   P = exp2(scale2 S - m) in registers, one row a thread, back to tensor
//       memory in 16 bits over S
//   O += P V    (P from tensor memory, V from shared memory)
// The two Q tiles take turns: while one is in its softmax the other's products
// run. (Tiles of 64 keys with two S buffers, so that scores never wait, were
// slower: what a tile costs beside its weights, barriers, maximum, checks, is
// then paid twice as often.)
// Roles: warps 0-3 and 4-7 the softmax of slot 0 and 1 (and the rescaling and
// output of its O), warps 8-11 the loads, warps 12 and 14 issue the MMAs of
// slot 0 and 1 (one warp for both was the bottleneck: it waits, issues and
// commits in turn), warp 13 resolves the CTA's items into records in shared
// memory (so that the others hold no walk state in registers). A slot is a Q
// tile; for an item of one Q tile of at most 64 rows (single tokens, drafts),
// where the chain of products and softmax is the limit, the slots take the KV
// tiles in turn, each with its own O, and join them in shared memory at the
// end. A row is one thread's, so its maximum and sum need no exchange.
//
// Code is kept short on purpose: eight warps of three roles share the SM's
// instruction caches. A tile's scores are read from tensor memory 64 columns at
// a time in a loop, the last 64 twice (maximum, then weights), not held in
// registers by unrolled code. The first 64 weights of a row are handed over
// before the rest is computed, so the second product starts earlier, and the
// next tile's last 64 scores are formed as soon as this tile's were read for
// the last time (1024 tokens at 32K keys, 64 heads: 1.44 -> 1.34 ms when it was
// made). That case takes 1.28 ms now in ten calls after a pause, 845 TFLOP/s, and
// 1.45 ms, 749 TFLOP/s, in a second of calls, whose power lowers the clock.
//
// Loads: a page holds 16 tokens of one head 2 KB or 4 KB apart, so a tensor
// copy would be many small boxes; 16-byte asynchronous copies per lane,
// straight into the 128-byte-swizzled layout, take any page size and stride.
// Keys outside the item's range and bad blocks are zero-filled.
//
// The reference maximum is only raised when the row's maximum passes it by more
// than 2^kRaise in the weights' domain, so O is rarely rescaled. Weights are
// rounded to the 16-bit type for the second product (the tensor core's operand
// type); their sum is taken before the rounding, in fp32, so what the rounding
// loses is missing from the output. In bf16 that is at most 2^-8 of a weight,
// whatever its size. In f16 a weight below 2^-25 would vanish, and many small weights
// behind one large one (an early key that takes most of the weight) are most of
// the output when that key's value is small: 65536 of them at 2^-27 of the largest
// were lost whole. So f16 weights carry 2^11: at most 2^15 of the type's 65504,
// 11 bits each down to 2^-25 of the reference and none lost above 2^-36 of it
// (2^7 with a raise of 2^8 would lose 0.5 % of weights at 2^-25.1). The factor is
// exact and leaves again in the log-sum-exp and in the partials' maxima.
//
// A masked weight is exactly 0, but 0 times a non-finite V is NaN: the loading
// warps check the V rows of tiles some row sees only in part, and a tile with
// a non-finite value is added by the softmax warps with plain FMAs over the
// keys each row sees. Rows that see the value get it, others do not.
#include <type_traits>

#include "chunk_plan.cuh"
#include "cvsa_common.cuh"
#include "cvsa_internal.h"
#include "cvsa_launch.cuh"
#include "fp8.cuh"
#include "tcgen05.cuh"

namespace cvsa {
namespace {

constexpr int kThreads = 512, kTile = 128, kKT = 128;
// Tile records: the record of tile j is rewritten for tile j + kSlots, whose K
// buffer is free only when the scores of tile j + kSlots - kStages / 2 were
// taken, and these wait for the weights of an earlier tile of their slot, four
// tiles before at most: j or a later one.
constexpr int kSlots = 16;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// log2: growth of the maximum that triggers a rescale, and the weights' factor
template <typename T> struct Weight { static constexpr float kRaise = 8.f, kUp = 0.f; };
template <> struct Weight<__half> { static constexpr float kRaise = 4.f, kUp = 11.f; };

template <int D>
struct Cfg {
  static constexpr int kStage = kKT * D * 2;            // bytes of a K or V tile
  static constexpr int kStages = D == 128 ? 4 : 8;
  static_assert(kStages / 2 + 4 <= kSlots, "tile records");
  static constexpr int kQTile = kTile * D * 2;
  static constexpr int kPanel = kKT * 128;              // bytes of a 64-column panel
  static_assert(kTile == kKT, "Q tiles and KV tiles share the copy code");
  static constexpr int kRing = 2 * kQTile;              // offset of the ring
  static constexpr int kMeta = kRing + kStages * kStage;
  // 8-bit pools: a K and a V tile's codes, 128-byte lines of 8 lanes
  static constexpr int kRaw8 = kKT * D;
};

// What the roles need of an item.
struct ItemRec {
  int nt;                  // tiles (-1: no more items; 0: its rows see no key)
  int tok, ntok, h;        // packed tokens [tok, tok + ntok), KV head
  int kbase;               // first key of the first tile
  int lo, hi;              // keys any row sees
  int pos0, ctx, slot;     // position of the first token, keys held, table row
  int first_hi, last_lo;   // keys [last_lo, first_hi) every row sees
  int nq, pair;            // Q tiles; the slots take the KV tiles of one Q tile in turn
  int whole, pslot, parts; // complete here, or the partial slot (and how many parts)
};
constexpr int kItems = 4;
constexpr int kPairRows = 64;  // rows whose fp32 O fits the second Q tile's memory

struct alignas(8) TcMeta {
  uint64_t kv_full[8], kv_empty[8];
  uint64_t q_full, q_empty;
  uint64_t q_second;                    // a second Q tile is there (its softmax group skips
                                        // items without one, so q_full's parity misleads it)
  uint64_t q_ready[2];                  // Q tiles that are scaled first: they were
  uint64_t s_full[2], s_free[2], p_half[2], p_full[2], o_full[2];  // per slot
  uint64_t it_full[kItems], it_empty[kItems];
  uint64_t joined, join_free;           // paired items: slot 1's part is there; was read
  uint64_t drain[2];
  uint32_t key_bad[kSlots][4];  // per tile (mod kSlots): bit per key no row may see
  uint8_t v_odd[kSlots][4];     // per tile and loading warp: a V value is not finite
  ItemRec item[kItems];
  float pair_m[kPairRows], pair_l[kPairRows];
  int8_t pair_exp[kPairRows];   // rows' powers of two (scale_query)
  uint32_t tmem;
  uint32_t abort;
};

constexpr int kMetaBytes = ((int)sizeof(TcMeta) + 15) / 16 * 16;

struct TcArgs {
  RaggedView rg;
  KvView kv;
  ChunkView c;
  ChunkGeo g;
  int TQ;               // tokens of a Q tile
  int bs_shift;         // log2 of the page size, or -1
  int pages16;          // the page size is a multiple of 16
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

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(ok ? 16 : 0)
               : "memory");
}

// Order of an item's K and V tiles in the ring: V of tile j behind K of tile
// j + lag, the order in which a slot's MMAs take them (scores of its next tile,
// then the product of this one); lag 2 when the slots take tiles in turn, else 1.
__device__ __forceinline__ uint32_t ring_v(int j, int lag, int nt) {
  return min(j + lag + 1, nt) + j;
}

__device__ __forceinline__ bool tile_partial(const ItemRec& it, int base) {
  return base + kKT > it.first_hi || base < it.last_lo;
}

__device__ __forceinline__ uint32_t any_odd(const TcMeta* m, uint32_t slot) {
  return *reinterpret_cast<const uint32_t*>(m->v_odd[slot]);
}

// A role's side of the item records. `next` is false at the end (or after a
// timeout); the record may be read until `done`.
struct ItemReader {
  TcMeta* m;
  const TcArgs& a;
  uint32_t n;
  __device__ __forceinline__ ItemReader(TcMeta* m_, const TcArgs& a_) : m(m_), a(a_), n(0) {}
  __device__ __forceinline__ const ItemRec* next() {
    if (!warp_wait(&m->it_full[n % kItems], (n / kItems) & 1, m, a)) return nullptr;
    const ItemRec* r = &m->item[n % kItems];
    return __shfl_sync(0xffffffffu, r->nt, 0) < 0 ? nullptr : r;
  }
  __device__ __forceinline__ void done() {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&m->it_empty[n % kItems]);
    ++n;
  }
};
constexpr int kReaders = 14;  // warps that read the records

// ---------------------------------------------------------------------------
// items (one warp finds the range, one lane walks it)
// ---------------------------------------------------------------------------
__device__ __forceinline__ void item_role(const TcArgs& a, TcMeta* m, const ChunkRange& rng) {
  if ((threadIdx.x & 31) != 0) return;
  ChunkWalk walk(rng);
  ChunkItem it;
  uint32_t n = 0;
  bool more = true;
  while (more) {
    more = walk.next(a.rg, a.g, blockIdx.x, it);
    if (!wait_for(&m->it_empty[n % kItems], ((n / kItems) & 1) ^ 1, m, a)) return;
    ItemRec& r = m->item[n % kItems];
    if (more) {
      r.nt = it.k1 - it.k0;
      r.tok = it.q.tok0 + it.t0;
      r.ntok = it.t1 - it.t0;
      r.h = it.h;
      r.kbase = (it.tile0 + it.k0) * kKT;
      r.lo = it.lo;
      r.hi = it.hi;
      r.pos0 = it.q.start + it.t0;
      r.ctx = it.q.ctx;
      r.slot = it.q.slot;
      r.first_hi = a.g.causal ? min(it.q.ctx, it.q.start + it.t0 + 1) : it.q.ctx;
      r.last_lo = a.g.window > 0 ? it.q.start + it.t1 - a.g.window : 0;
      r.nq = r.ntok > a.TQ ? 2 : 1;
      r.pair = r.nq == 1 && r.ntok * a.g.G <= kPairRows && r.nt > 1;
      r.whole = it.whole;
      r.pslot = 2 * blockIdx.x + it.slot;
      r.parts = it.parts;
    } else {
      r.nt = -1;
    }
    mbar_arrive(&m->it_full[n % kItems]);
    ++n;
  }
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
  // This warp's 32 rows of a tile; lane i holds row i's offset in elements, < 0: zeros
  __device__ __forceinline__ void copy_rows(uint32_t tile, const void* src, int64_t off) {
    const int ch = lane % kCh;
#pragma unroll 4
    for (int i = 0; i < 32 / kRPI; ++i) {
      const int r = i * kRPI + lane / kCh;
      const int64_t o = __shfl_sync(0xffffffffu, off, r);
      const bool ok = o >= 0;
      cp16(dst(tile, w * 32 + r, ch), reinterpret_cast<const T*>(src) + (ok ? o + ch * 8 : 0), ok);
    }
  }
  // The same when all rows exist and each 16 of them share a page: two
  // addresses and a constant stride, three instructions a copy instead of about
  // 25. The copies share their schedulers with the softmax warps, so the
  // difference is the softmax's.
  __device__ __forceinline__ void copy(uint32_t tile, const void* src, int64_t off, bool pages) {
    if (!pages) {
      copy_rows(tile, src, off);
      return;
    }
    const int ch = lane % kCh, sub = lane / kCh;
    const int64_t step = (int64_t)kRPI * a.kv.st * sizeof(T);
    uint32_t d[8 / kRPI];  // the swizzle repeats every 8 rows
#pragma unroll
    for (int i = 0; i < 8 / kRPI; ++i) d[i] = dst(tile, w * 32 + i * kRPI + sub, ch);
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
      const int64_t o = __shfl_sync(0xffffffffu, off, 16 * pg + sub);
      const char* p = reinterpret_cast<const char*>(reinterpret_cast<const T*>(src) + o + ch * 8);
#pragma unroll
      for (int i = 0; i < 16 / kRPI; ++i) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                         d[i % (8 / kRPI)] + (pg * 16 + i * kRPI) / 8 * 1024),
                     "l"(p)
                     : "memory");
        p += step;
      }
    }
  }

  __device__ void run() {
    ItemReader items(m, a);
    uint32_t op = 0, tiles = 0, loads = 0, joins = 0;
    const int G = a.g.G;
    while (const ItemRec* it = items.next()) {
      const int nt = it->nt;
      if (nt == 0) {
        items.done();
        continue;
      }
      const int lag = it->pair ? 2 : 1;
      const int lo = it->lo, hi = it->hi;
      const int32_t* table = a.rg.tables + (int64_t)it->slot * a.rg.W;
      const int64_t head = it->h * a.kv.sh;
      auto block_of = [&](int key) {  // only of an item key
        return key >= lo && key < hi ? table[a.bs_shift >= 0 ? key >> a.bs_shift : key / a.kv.bs]
                                     : -1;
      };
      int key = it->kbase + w * 32 + lane;
      int blk = block_of(key);
      int64_t off0 = -1, off1 = -1, off2 = -1;  // rows of tiles j, j - 1, j - 2
      uint32_t pages = 0;                       // bit i: tile j - i is of whole pages
      for (int j = 0; j < nt + lag; ++j) {
        off2 = off1;
        off1 = off0;
        pages <<= 1;
        if (j < nt) {
          const int next = j + 1 < nt ? block_of(key + kKT) : -1;
          off0 = -1;
          if (key >= lo && key < hi) {
            if (blk >= 0 && blk < a.kv.num_blocks) {
              const int in = a.bs_shift >= 0 ? key & (a.kv.bs - 1) : key % a.kv.bs;
              off0 = blk * a.kv.sb + in * a.kv.st + head;
            } else {
              set_dev_error(a.dev_err, CVSA_DEV_ERR_BLOCK_RANGE);
            }
          }
          blk = next;
          key += kKT;
          const uint32_t st = op % C::kStages, slot = (tiles + j) % kSlots;
          if (!warp_wait(&m->kv_empty[st], ((op / C::kStages) & 1) ^ 1, m, a)) goto out;
          const uint32_t bad = __ballot_sync(0xffffffffu, off0 < 0);
          if (lane == 0) {
            m->key_bad[slot][w] = bad;
            mbar_arrive(&m->kv_full[st]);  // a plain arrival, behind the plain write
          }
          pages |= bad == 0 && a.pages16;
          copy(base + C::kRing + st * C::kStage, a.kv.k, off0, pages & 1);
          arrive_when_landed(&m->kv_full[st]);
          ++op;
        }
        if (j == lag - 1) {
          // the queries, behind the first K tiles: those are on their way while the
          // item before still holds the queries' memory
          if (!warp_wait(&m->q_empty, (loads & 1) ^ 1, m, a)) goto out;
          ++loads;
          if (joins && !warp_wait(&m->join_free, (joins - 1) & 1, m, a)) goto out;
          joins += it->pair;
          for (int q = 0; q < it->nq; ++q) {
            const int r = w * 32 + lane;
            const int rows = min(a.TQ, it->ntok - q * a.TQ) * G;
            int64_t off = -1;
            if (r < rows)
              off = (int64_t)(it->tok + q * a.TQ + r / G) * a.c.q_st +
                    (int64_t)(it->h * G + r % G) * a.c.q_sh;
            copy_rows(base + q * C::kQTile, a.c.q, off);
          }
          arrive_when_landed(&m->q_full);
        }
        if (j >= lag) {
          const uint32_t st = op % C::kStages, slot = (tiles + j - lag) % kSlots;
          if (!warp_wait(&m->kv_empty[st], ((op / C::kStages) & 1) ^ 1, m, a)) goto out;
          const uint32_t v = base + C::kRing + st * C::kStage;
          copy(v, a.kv.v, lag == 1 ? off1 : off2, pages >> lag & 1);
          if (tile_partial(*it, it->kbase + (j - lag) * kKT)) {
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncwarp();
            const bool odd = has_odd(v);
            if (lane == 0) m->v_odd[slot][w] = odd;
            mbar_arrive(&m->kv_full[st]);
          } else {
            arrive_when_landed(&m->kv_full[st]);
          }
          if (lane == 0) mbar_arrive(&m->kv_full[st]);
          ++op;
        }
      }
      tiles += nt;
      items.done();
    }
  out:
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
};

// 8-bit pools. A tile's codes are copied (asynchronously) to a buffer of their own, one
// for K and one for V, and widened from there to the 16-bit tile: each thread widens
// the pieces that it copied, so it waits for nobody's copies but its own. V of one tile
// is on its way while K of another is widened, and the other way round.
//
// The tensor cores take f16 whatever the queries' type: an instruction widens two codes
// to f16, where bf16 takes thirteen for four (1024 tokens at 32K keys 975 us in bf16,
// 739 in f16), and the weights keep 11 bits. Widening is exact (fp8.cuh). bf16 queries
// are scaled by row (scale_query).
template <int D>
struct Loader8 : Loader<__half, D> {
  using T = __half;
  using L = Loader<T, D>;
  using C = Cfg<D>;
  using L::a; using L::m; using L::base; using L::w; using L::lane;
  static constexpr int kCh = D / 16;           // 16-byte pieces of a row's codes
  static constexpr int kRPI = 32 / kCh;        // rows a warp instruction
  static constexpr int kPieces = 32 / kRPI;    // pieces a lane of a tile
  uint32_t raw;                                // this thread's pieces: 512 bytes apart

  __device__ Loader8(const TcArgs& a_, TcMeta* m_, uint32_t base_, uint32_t raw_, int w_, int lane_)
      : L(a_, m_, base_, w_, lane_), raw(raw_ + w_ * kPieces * 512 + lane_ * 16) {}

  // Lane i's row is off bytes into the pool (< 0: zeros); v: the V tile's buffer.
  __device__ __forceinline__ void fetch(const void* src, int64_t off, int v) {
    const int ch = lane % kCh;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int64_t o = __shfl_sync(0xffffffffu, off, i * kRPI + lane / kCh);
      cp16(raw + v * C::kRaw8 + i * 512, static_cast<const char*>(src) + (o < 0 ? 0 : o + ch * 16),
           o >= 0);
    }
    cp_async_commit();
  }
  // To the 16-bit tile; lane i holds row i's factor. Whether a code was NaN, if asked.
  __device__ __forceinline__ bool widen(uint32_t tile, uint32_t factor, int v, bool ask) {
    const int ch = lane % kCh;
    const bool swap = ch >= 4;  // the two stores of a row's lanes then fall on different banks
    bool nan = false;
#pragma unroll 2
    for (int i = 0; i < kPieces; ++i) {
      const int r = i * kRPI + lane / kCh;
      uint4 codes, x[2];
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(codes.x), "=r"(codes.y), "=r"(codes.z), "=r"(codes.w)
                   : "r"(raw + v * C::kRaw8 + i * 512));
      widen16(codes, __shfl_sync(0xffffffffu, factor, r), x);
      if (ask) nan |= any_nan8(codes);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int e = swap ? 1 - half : half;
        const uint4 y = e ? x[1] : x[0];
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(
                         this->dst(tile, w * 32 + r, ch * 2 + e)),
                     "r"(y.x), "r"(y.y), "r"(y.z), "r"(y.w)
                     : "memory");
      }
    }
    return ask && __any_sync(0xffffffffu, nan);
  }

  __device__ void run() {
    ItemReader items(m, a);
    uint32_t op = 0, tiles = 0, loads = 0, joins = 0;
    const int G = a.g.G;
    while (const ItemRec* it = items.next()) {
      const int nt = it->nt;
      if (nt == 0) {
        items.done();
        continue;
      }
      const int lag = it->pair ? 2 : 1;
      const int lo = it->lo, hi = it->hi, h = it->h;
      const int32_t* table = a.rg.tables + (int64_t)it->slot * a.rg.W;
      auto block_of = [&](int key) {  // only of an item key
        return key >= lo && key < hi ? table[a.bs_shift >= 0 ? key >> a.bs_shift : key / a.kv.bs]
                                     : -1;
      };
      int key = it->kbase + w * 32 + lane;  // of the tile that is located next
      int blk = block_of(key);
      // rows and V factors of tiles j, j - 1, j - 2 at turn j; K's factor of tile j
      int64_t off[4] = {-1, -1, -1, -1};
      uint32_t fv[4] = {0, 0, 0, 0}, fk = 0;
      // Finds tile j's rows and starts its K copies; the others move up.
      auto locate = [&]() {
#pragma unroll
        for (int i = 3; i > 0; --i) off[i] = off[i - 1], fv[i] = fv[i - 1];
        const int next = block_of(key + kKT);
        off[0] = -1;
        fk = fv[0] = 0;
        if (key >= lo && key < hi) {
          if (blk >= 0 && blk < a.kv.num_blocks) {
            const int in = a.bs_shift >= 0 ? key & (a.kv.bs - 1) : key % a.kv.bs;
            off[0] = blk * a.kv.sb + in * a.kv.st + h * a.kv.sh;
            const int64_t at = (int64_t)blk * a.kv.hkv + h;
            fk = widen_factor(a.kv.ks[at]);
            fv[0] = widen_factor(a.kv.vs[at]);
          } else {
            set_dev_error(a.dev_err, CVSA_DEV_ERR_BLOCK_RANGE);
          }
        }
        blk = next;
        key += kKT;
        fetch(a.kv.k, off[0], 0);
      };
      locate();
      for (int j = 0; j < nt + lag; ++j) {
        // before tile j + 1 is located its predecessors are at 0, 1, ...; from nt on
        // nothing is located, so tile j - lag stays where it was at turn nt - 1
        const int back = lag - max(0, j - (nt - 1));
        const uint32_t fvj = back == 0 ? fv[0] : back == 1 ? fv[1] : fv[2];
        if (j >= lag) fetch(a.kv.v, back == 0 ? off[0] : back == 1 ? off[1] : off[2], 1);
        if (j < nt) {
          const uint32_t st = op % C::kStages, slot = (tiles + j) % kSlots;
          if (!warp_wait(&m->kv_empty[st], ((op / C::kStages) & 1) ^ 1, m, a)) goto out;
          const uint32_t bad = __ballot_sync(0xffffffffu, off[0] < 0);
          if (lane == 0) m->key_bad[slot][w] = bad;
          cp_async_wait_dyn(j >= lag ? 1 : 0);
          widen(base + C::kRing + st * C::kStage, fk, 0, false);
          mbar_arrive(&m->kv_full[st]);
          if (lane == 0) mbar_arrive(&m->kv_full[st]);
          ++op;
          if (j + 1 < nt) locate();
        }
        if (j == lag - 1) {
          // the queries; a group of their own behind the K tile on its way
          if (!warp_wait(&m->q_empty, (loads & 1) ^ 1, m, a)) goto out;
          ++loads;
          if (joins && !warp_wait(&m->join_free, (joins - 1) & 1, m, a)) goto out;
          joins += it->pair;
          for (int q = 0; q < it->nq; ++q) {
            const int r = w * 32 + lane;
            const int rows = min(a.TQ, it->ntok - q * a.TQ) * G;
            int64_t qo = -1;
            if (r < rows)
              qo = (int64_t)(it->tok + q * a.TQ + r / G) * a.c.q_st +
                   (int64_t)(h * G + r % G) * a.c.q_sh;
            this->copy_rows(base + q * C::kQTile, a.c.q, qo);
          }
          arrive_when_landed(&m->q_full);
          if (it->nq > 1) arrive_when_landed(&m->q_second);
        }
        if (j >= lag) {
          const uint32_t st = op % C::kStages, slot = (tiles + j - lag) % kSlots;
          if (!warp_wait(&m->kv_empty[st], ((op / C::kStages) & 1) ^ 1, m, a)) goto out;
          cp_async_wait_dyn(j + 1 < nt ? 1 : 0);
          const bool partial = tile_partial(*it, it->kbase + (j - lag) * kKT);
          const bool odd = widen(base + C::kRing + st * C::kStage, fvj, 1, partial);
          if (partial && lane == 0) m->v_odd[slot][w] = odd;
          mbar_arrive(&m->kv_full[st]);
          if (lane == 0) mbar_arrive(&m->kv_full[st]);
          ++op;
        }
      }
      tiles += nt;
      items.done();
    }
  out:
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
};

// ---------------------------------------------------------------------------
// MMA issue (a warp a slot, one elected lane)
// ---------------------------------------------------------------------------
// The whole warp runs the loop, with its trip counts broadcast, so that the
// compiler keeps descriptors in uniform registers, where the instruction
// wants them: issued from a single-lane branch each MMA cost about 95 cycles
// of moves, against the 64 that it runs.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

template <typename T, int D, bool kScaled>
__device__ __forceinline__ void mma_role(const TcArgs& a, TcMeta* m, uint32_t base, uint32_t tmem,
                                         const int s) {
  using C = Cfg<D>;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  constexpr uint32_t kIdS = mma_idesc(kBf16, kTile, kKT, false);
  constexpr uint32_t kIdHalf = mma_idesc(kBf16, kTile, kKT / 2, false);
  constexpr uint32_t kIdO = mma_idesc(kBf16, kTile, D, true);
  const uint32_t ring = base + C::kRing;
  const uint64_t q_desc = smem_desc(base, 16, 1024), k_desc = smem_desc(ring, 16, 1024),
                 v_desc = smem_desc(ring, C::kPanel, 1024);
  const uint32_t ts = tmem + s * kKT, to = tmem + 2 * kKT + s * D;
  // Scores of the keys from byte `row` of a K tile, as many as the descriptor says.
  auto scores = [&](uint32_t d, uint64_t qd, uint32_t st, uint32_t row, uint32_t idesc) {
    const uint64_t kd = k_desc + ((st * C::kStage + row) >> 4);
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const uint32_t o = ((kk / 4) * C::kPanel + (kk % 4) * 32) >> 4;
      mma_ss(d, qd + o, kd + o, idesc, kk > 0);
    }
  };
  // Both slots take every buffer of the ring in order, used or not, and free it:
  // a barrier's parity says which of two phases is done, so no one may lag or
  // lead by more.
  ItemReader items(m, a);
  uint32_t op = 0, tiles = 0, loads = 0, second = 0;
  uint32_t turn = 0;  // tiles of this slot before this item
  while (const ItemRec* it = items.next()) {
    const int nt = uniform(it->nt), nq = uniform(it->nq), kbase = uniform(it->kbase);
    const int pair = uniform(it->pair), lag = pair ? 2 : 1;
    if (nt == 0) {
      items.done();
      continue;
    }
    const int n = pair ? (nt + 1 - s) / 2 : s < nq ? nt : 0;  // tiles of this slot
    if (!warp_wait(&m->q_full, loads & 1, m, a)) break;
    if (kScaled && n > 0) {
      const bool one = s == 1 && !pair;  // the second Q tile
      if (!warp_wait(&m->q_ready[one], (one ? second : loads) & 1, m, a)) break;
      second += one;
    }
    ++loads;
    if (n == 0 && elect_one()) mbar_arrive(&m->q_empty);
    const uint64_t qd = q_desc + (((pair ? 0 : s) * C::kQTile) >> 4);
    int i = 0, iv = 0;  // this slot's scores and products so far
    for (int j = 0; j < nt + lag; ++j) {
      // K of tile j and V of tile j - lag, which is of the same slot
      const int jv = j - lag;
      const bool mine = n && (!pair || (j & 1) == s);
      const uint32_t kst = op % C::kStages;
      if (j < nt) {
        if (!warp_wait(&m->kv_full[kst], (op / C::kStages) & 1, m, a)) goto out;
        ++op;
      }
      const uint32_t vst = op % C::kStages;
      if (jv >= 0) {
        if (!warp_wait(&m->kv_full[vst], (op / C::kStages) & 1, m, a)) goto out;
        ++op;
      }
      if (!mine) {
        if (elect_one()) {
          if (j < nt) mbar_arrive(&m->kv_empty[kst]);
          if (jv >= 0) mbar_arrive(&m->kv_empty[vst]);
        }
        __syncwarp();
        continue;
      }
      fence_proxy_async_smem();  // the tiles were written through the generic proxy
      if (jv >= 0) {
        bool skip = false;
        if (tile_partial(*it, kbase + jv * kKT))
          skip = uniform(any_odd(m, (tiles + jv) % kSlots));
        const uint64_t vd = v_desc + ((vst * C::kStage) >> 4);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (half && j < nt && !pair) {
            // the scores of the next tile's last 64 keys, behind the softmax's last
            // look at this tile's: the weights cover only the first 64 columns. (Not for
            // paired items, which wait for memory: two products of 64 keys cost more
            // than one of 128.)
            if (!warp_wait(&m->s_free[s], (turn + iv) & 1, m, a)) goto out;
            tc_fence_after();
            if (elect_one()) scores(ts + 64, qd, kst, 64 * 128, kIdHalf);
            __syncwarp();
          }
          if (!warp_wait(half ? &m->p_full[s] : &m->p_half[s], (turn + iv) & 1, m, a)) goto out;
          tc_fence_after();
          if (!skip && elect_one()) {
#pragma unroll
            for (int kk = half * 4; kk < half * 4 + 4; ++kk)
              mma_ts(to, ts + kk * 8, vd + ((kk * 2048) >> 4), kIdO, iv > 0 || kk > 0);
          }
          __syncwarp();
        }
        ++iv;
      }
      if (elect_one()) {
        if (jv >= 0) {
          if (iv == n) mma_commit(smem_u32(&m->o_full[s]));
          if (j >= nt) mma_commit(smem_u32(&m->kv_empty[vst]));
        }
        if (j < nt) {  // over the weights that the product before reads: MMAs run in order
          scores(ts, qd, kst, 0, jv >= 0 && !pair ? kIdHalf : kIdS);
          mma_commit(smem_u32(&m->s_full[s]));
          mbar_arrive(&m->s_full[s]);  // orders the loaders' plain writes before it too
          mma_commit(smem_u32(&m->kv_empty[kst]));
          if (jv >= 0) mma_commit(smem_u32(&m->kv_empty[vst]));
          if (i + 1 == n) mma_commit(smem_u32(&m->q_empty));
        }
      }
      __syncwarp();
      if (j < nt) ++i;
    }
    tiles += nt;
    turn += n;
    items.done();
  }
out:
  // nothing of this CTA may be in flight when its tensor memory is freed
  if (elect_one()) mma_commit(smem_u32(&m->drain[s]));
  __syncwarp();
  mbar_wait_bounded(&m->drain[s], 0, 1u << 18);
  __syncwarp();
}

// ---------------------------------------------------------------------------
// softmax, rescaling and output of one Q tile
// ---------------------------------------------------------------------------
// Bit c: the row whose keys are [lo, hi) does not see key base + c.
__device__ __forceinline__ uint32_t hidden(int lo, int hi, int base) {
  const int h = hi - base, b = lo - base;
  const uint32_t upto = h >= 32 ? ~0u : h <= 0 ? 0u : (1u << h) - 1;
  const uint32_t from = b <= 0 ? ~0u : b >= 32 ? 0u : ~0u << b;
  return ~(upto & from);
}

// Piece j of lane i's x and piece i of lane j's change places, i, j < 4 within
// each group of 4 lanes.
__device__ __forceinline__ void transpose4(uint4* x) {
#pragma unroll
  for (int step = 1; step <= 2; step <<= 1) {
    const bool up = (threadIdx.x & step) != 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i & step) continue;
      uint4 &lo = x[i], &hi = x[i | step];
      uint4 give = up ? lo : hi;
      give.x = __shfl_xor_sync(0xffffffffu, give.x, step);
      give.y = __shfl_xor_sync(0xffffffffu, give.y, step);
      give.z = __shfl_xor_sync(0xffffffffu, give.z, step);
      give.w = __shfl_xor_sync(0xffffffffu, give.w, step);
      if (up) lo = give; else hi = give;
    }
  }
}

// bf16 queries for f16 tensor cores, one row a thread, in place: each row is brought to
// a largest value in [2^13, 2^14) by a power of two, 2^-e of which is returned as e and
// goes to the row's softmax scale. bf16's 8 bits fit f16's 11 down to 2^-27 of the
// largest; what lies below errs by at most 2^-38 of it, far below the rounding of a
// product's sum. (Where a row holds an infinity, its scores are that or NaN whatever
// its other values are.)
template <typename TI, int D>
__device__ __forceinline__ int scale_query(uint32_t tile, int row) {
  constexpr int kPanel = Cfg<D>::kPanel;
  auto at = [&](int ch) {
    return tile + (ch >> 3) * kPanel + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
  };
  auto load = [&](int ch, float* f) {
    uint4 x;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                 : "r"(at(ch)));
    Vec16<TI>::unpack(x, f);
  };
  float top = 0.f;
#pragma unroll 2
  for (int ch = 0; ch < D / 8; ++ch) {
    float f[8];
    load(ch, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[e]));
  }
  const int up = min(120, 13 + 127 - (__float_as_int(top) >> 23));  // >= -115
  const float by = pow2(up);
#pragma unroll 2
  for (int ch = 0; ch < D / 8; ++ch) {
    float f[8];
    load(ch, f);
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at(ch)),
                 "r"(Mma<__half>::pack(f[0] * by, f[1] * by)),
                 "r"(Mma<__half>::pack(f[2] * by, f[3] * by)),
                 "r"(Mma<__half>::pack(f[4] * by, f[5] * by)),
                 "r"(Mma<__half>::pack(f[6] * by, f[7] * by))
                 : "memory");
  }
  return -up;
}

template <typename TI, typename T, int D>  // T: of the tensor cores' operands
__device__ __forceinline__ void softmax_role(const TcArgs& a, TcMeta* m, uint32_t base,
                                             uint32_t tmem, const int g) {
  using C = Cfg<D>;
  constexpr float kRaise = Weight<T>::kRaise, kUp = Weight<T>::kUp;
  constexpr bool kScaled = !std::is_same<TI, T>::value;
  const int r = threadIdx.x & 127, warp = r >> 5;
  const uint32_t lanes = (uint32_t)(warp * 32) << 16;
  const uint32_t ts = tmem + g * kKT + lanes, to = tmem + 2 * kKT + g * D + lanes;
  const int G = a.g.G;
  float scale2 = a.scale2;
  ItemReader items(m, a);
  uint32_t op = 0, tiles = 0, turn = 0, ends = 0, joins = 0, loads = 0, seconds = 0;
  while (const ItemRec* it = items.next()) {
    loads += it->nt > 0;
    const int nt = it->nt, pair = it->pair, q = pair ? 0 : g, step = pair ? 2 : 1;
    const int rows = min(a.TQ, it->ntok - q * a.TQ) * G;
    if (rows <= 0) {
      op += 2 * nt;
      tiles += nt;
      items.done();
      continue;
    }
    const bool active = warp * 32 < rows;
    if (kScaled && nt > 0 && !(pair && g == 1)) {
      ++seconds;
      if (!warp_wait(g ? &m->q_second : &m->q_full, ((g ? seconds : loads) - 1) & 1, m, a)) return;
      if (active) {
        const int e = scale_query<TI, D>(base + g * C::kQTile, r);
        scale2 = a.scale2 * pow2(e);
        if (pair && r < kPairRows) m->pair_exp[r] = (int8_t)e;  // for the other slot's softmax
      }
      mbar_arrive(&m->q_ready[g]);
    }
    const int pos = it->pos0 + q * a.TQ + r / G;
    const int hi = a.g.causal ? min(it->ctx, pos + 1) : it->ctx;
    const int lo = a.g.window > 0 ? pos - a.g.window + 1 : 0;
    float mx = neg_inf(), l = 0.f;
    const int first = pair ? g : 0;
    for (int j = first; j < nt; j += step, ++turn) {
      if (!warp_wait(&m->s_full[g], turn & 1, m, a)) return;
      tc_fence_after();
      if (kScaled && j == 1 && first == 1 && r < kPairRows) scale2 = a.scale2 * pow2(m->pair_exp[r]);
      const int kbase = it->kbase + j * kKT;
      const uint32_t slot = (tiles + j) % kSlots;
      const bool partial = tile_partial(*it, kbase);
      bool odd = false;
      uint32_t vst = 0;
      if (partial) {
        const uint32_t vop = op + ring_v(j, step, nt);
        vst = vop % C::kStages;
        if (!warp_wait(&m->kv_full[vst], (vop / C::kStages) & 1, m, a)) return;
        odd = any_odd(m, slot) != 0;
      }
      if (active) {
        const uint32_t* const bad = m->key_bad[slot];
        const bool masked = partial || (bad[0] | bad[1] | bad[2] | bad[3]);
        float top = neg_inf();
        float s[64];  // ends with the first 64 scores
#pragma unroll 1
        for (int c = kKT - 64; c >= 0; c -= 64) {
          tmem_ld32(ts + c, s);
          tmem_ld32(ts + c + 32, s + 32);
          tmem_wait_ld();
          if (masked) {  // hidden keys' scores become -inf, here and in tensor memory
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int at = c + 32 * i;
              const uint32_t hide = hidden(lo, hi, kbase + at) | bad[at / 32];
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (hide >> e & 1) s[32 * i + e] = neg_inf();
              tmem_st32(ts + at, reinterpret_cast<const uint32_t*>(s + 32 * i));
            }
          }
          float t4[4] = {top, top, top, top};
#pragma unroll
          for (int x = 0; x < 64; x += 8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) t4[i] = max3_nan(t4[i], s[x + i], s[x + 4 + i]);
          }
          top = max3_nan(max3_nan(t4[0], t4[1], t4[2]), t4[3], t4[3]);
        }
        if (masked) tmem_wait_st();
        float fix = 1.f;
        if ((top - mx) * scale2 > kRaise || mx == neg_inf() || top != top) {
          const float raised = top != top ? top : fmaxf(mx, top);  // NaN: so is the row
          if (mx != neg_inf()) fix = ex2((mx - raised) * scale2);
          mx = raised;
        }
        if (j > first && __any_sync(0xffffffffu, fix != 1.f)) {
          // O of this slot's earlier tiles is complete: S was issued behind it
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
        const float ref = mx == neg_inf() ? 0.f : fmaf(-mx, scale2, kUp);
        if (odd) {
          // a value of V is not finite and some row does not see it: plain FMAs.
          // The weights go over S in fp32, -1 for an unseen key.
#pragma unroll 1
          for (int c = 0; c < kKT; c += 8) {
            const uint32_t hide = (hidden(lo, hi, kbase + c / 32 * 32) | bad[c / 32]) >> (c % 32);
            float p[8];
            tmem_ld8(ts + c, p);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const bool see = !(hide >> e & 1);
              const float x = ex2(fmaf(p[e], scale2, ref));
              l += see ? x : 0.f;
              p[e] = see ? x : -1.f;
            }
            tmem_st8(ts + c, p);
          }
          tmem_wait_st();
          const uint32_t v = base + C::kRing + vst * C::kStage;
#pragma unroll 1
          for (int ch = 0; ch < D / 8; ++ch) {
            float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (j > first) {
              tmem_ld8(to + ch * 8, o);
              tmem_wait_ld();
            }
#pragma unroll 1
            for (int c = 0; c < kKT; c += 8) {
              float p[8];
              tmem_ld8(ts + c, p);
              tmem_wait_ld();
#pragma unroll 1
              for (int i = 0; i < 8; ++i) {
                const int row = c + i;
                uint4 x;
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                             : "r"(v + (ch >> 3) * C::kPanel + row * 128 +
                                   (((ch & 7) ^ (row & 7)) << 4)));
                float f[8];
                Vec16<T>::unpack(x, f);
                const float w = p[0];
#pragma unroll
                for (int e = 0; e < 7; ++e) p[e] = p[e + 1];
                if (w >= 0.f || w != w) {
#pragma unroll
                  for (int e = 0; e < 8; ++e) o[e] = fmaf(w, f[e], o[e]);
                }
              }
              __syncwarp();
            }
            tmem_st8(to + ch * 8, o);
          }
          tc_fence_before();
          mbar_arrive(&m->s_free[g]);
          mbar_arrive(&m->p_half[g]);
        } else {
          const uint64_t sc = f2_pack(scale2, scale2), rf = f2_pack(ref, ref);
          uint64_t sum0 = 0, sum1 = 0;
#pragma unroll 1
          for (int c = 0; c < kKT; c += 64) {
            uint32_t p[32];
            if (c) {
              tmem_ld32(ts + c, s);
              tmem_ld32(ts + c + 32, s + 32);
              tmem_wait_ld();
              tc_fence_before();
              mbar_arrive(&m->s_free[g]);  // the next tile's scores may go there
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float u, v;
              f2_unpack(f2_fma(f2_pack(s[2 * i], s[2 * i + 1]), sc, rf), u, v);
              u = ex2(u);
              v = ex2(v);
              uint64_t& sum = i & 1 ? sum1 : sum0;
              sum = f2_add(sum, f2_pack(u, v));
              p[i] = Mma<T>::pack(u, v);
            }
            tmem_st32(ts + c / 2, p);
            if (c == 0) {
              tmem_wait_st();
              tc_fence_before();
              mbar_arrive(&m->p_half[g]);
            }
          }
          float u, v;
          f2_unpack(f2_add(sum0, sum1), u, v);
          l += u + v;
        }
        tmem_wait_st();
      } else {
        mbar_arrive(&m->s_free[g]);
        mbar_arrive(&m->p_half[g]);
      }
      tc_fence_before();
      mbar_arrive(&m->p_full[g]);
    }
    op += 2 * nt;
    tiles += nt;
    // the item's rows, or this range's part of them
    if (nt > 0) {
      if (!warp_wait(&m->o_full[g], ends & 1, m, a)) return;
      ++ends;
      tc_fence_after();
    }
    const bool live = r < rows;
    float4* shared_o = reinterpret_cast<float4*>(
        __cvta_shared_to_generic(base + C::kQTile));  // paired items: [D / 4][kPairRows]
    if (pair && g == 1) {  // hand this slot's part over
      if (active) {
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float o[32];
          tmem_ld32(to + c, o);
          tmem_wait_ld();
          if (live) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              shared_o[(c / 4 + i) * kPairRows + r] =
                  l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                           : make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
          __syncwarp();
        }
        if (live) {
          m->pair_m[r] = mx;
          m->pair_l[r] = l;
        }
      }
      tc_fence_before();
      mbar_arrive(&m->joined);
      items.done();
      continue;
    }
    float w0 = 1.f, w1 = 0.f;  // weights of this slot's and the other's part
    if (pair) {
      if (!warp_wait(&m->joined, joins & 1, m, a)) return;
      ++joins;
      if (active && live) {
        const float m1 = m->pair_m[r], l1 = m->pair_l[r];
        const float top = mx != mx || m1 != m1 ? mx + m1 : fmaxf(mx, m1);
        w0 = mx == neg_inf() ? 0.f : ex2((mx - top) * scale2);
        w1 = m1 == neg_inf() ? 0.f : ex2((m1 - top) * scale2);
        l = l * w0 + l1 * w1;
        mx = top;
      }
    }
    const bool whole = it->whole;
    if (active) {
      const int64_t tok = it->tok + q * a.TQ + r / G;
      const int head = it->h * G + r % G;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int R = 2 * kTile, rr = q * a.TQ * G + r;
      float* part = a.parts + (size_t)it->pslot * chunk_slot_floats(R, D);
      const int64_t own = tok * a.c.o_st + head * a.c.o_sh;
      TI* dst[4];  // this lane's pieces of the rows of its 4 lanes
#pragma unroll
      for (int i = 0; i < 4; ++i)
        dst[i] = reinterpret_cast<TI*>(a.c.out) + (r & 3) * 8 +
                 __shfl_sync(0xffffffffu, own, (r & 28) + i);
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        float o[32];
        if (nt > 0) {
          tmem_ld32(to + c, o);
          tmem_wait_ld();
        }
        if (pair && live) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            // a slot that has seen no key of the row holds nothing of it
            const float4 x = shared_o[(c / 4 + i) * kPairRows + r];
            o[4 * i] = (w0 == 0.f ? 0.f : o[4 * i] * w0) + x.x * w1;
            o[4 * i + 1] = (w0 == 0.f ? 0.f : o[4 * i + 1] * w0) + x.y * w1;
            o[4 * i + 2] = (w0 == 0.f ? 0.f : o[4 * i + 2] * w0) + x.z * w1;
            o[4 * i + 3] = (w0 == 0.f ? 0.f : o[4 * i + 3] * w0) + x.w * w1;
          }
        }
        if (l == 0.f) {  // a row without a key (or without any so far)
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
        }
        if (whole) {
          // 4 lanes own 4 rows of 4 16-byte pieces: transposed among them, an
          // instruction writes 64 consecutive bytes of 8 rows, not 16 of 32
          uint4 x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i].x = Mma<TI>::pack(o[8 * i] * inv, o[8 * i + 1] * inv);
            x[i].y = Mma<TI>::pack(o[8 * i + 2] * inv, o[8 * i + 3] * inv);
            x[i].z = Mma<TI>::pack(o[8 * i + 4] * inv, o[8 * i + 5] * inv);
            x[i].w = Mma<TI>::pack(o[8 * i + 6] * inv, o[8 * i + 7] * inv);
          }
          transpose4(x);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if ((r & ~3) + i < rows) *reinterpret_cast<uint4*>(dst[i] + c) = x[i];
        } else if (live) {
          float4* po = reinterpret_cast<float4*>(part + 2 * R) + (size_t)(c / 4) * R + rr;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            po[(size_t)i * R] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
        __syncwarp();
      }
      if (live) {
        const float m2 = mx * scale2;
        if (whole) {
          if (a.c.lse)
            a.c.lse[tok * a.c.hq + head] =
                l == 0.f ? neg_inf() : (m2 + log2f(l * exp2f(-kUp))) * kLn2;
        } else {
          part[rr] = l == 0.f ? neg_inf() : m2 - kUp;
          part[R + rr] = l;
        }
      }
    }
    if (threadIdx.x == 0 && it->parts) {
      ChunkMergeDesc d;
      d.parts = it->parts;
      d.tok = it->tok;
      d.rows = it->ntok * G;
      d.head = it->h;
      a.desc[blockIdx.x] = d;
    }
    __syncwarp();
    if (pair && (threadIdx.x & 31) == 0) mbar_arrive(&m->join_free);
    items.done();
  }
}

template <typename TI, int D, bool F8>  // the queries' type; F8: an 8-bit pool
__global__ void __launch_bounds__(kThreads, 1)
chunk_tc_kernel(const __grid_constant__ TcArgs a) {
  using C = Cfg<D>;
  using T = typename std::conditional<F8, __half, TI>::type;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  TcMeta* m = reinterpret_cast<TcMeta*>(smem + C::kMeta);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&m->kv_full[i], 128 + 4);  // copies, and the writers of the tile's record
      mbar_init(&m->kv_empty[i], 2);
    }
    mbar_init(&m->q_full, 128);
    mbar_init(&m->q_second, 128);
    mbar_init(&m->q_empty, 2);
    for (int i = 0; i < 2; ++i) mbar_init(&m->q_ready[i], 128);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&m->s_full[i], 2);
      mbar_init(&m->s_free[i], 128);
      mbar_init(&m->p_half[i], 128);
      mbar_init(&m->p_full[i], 128);
      mbar_init(&m->o_full[i], 1);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&m->it_full[i], 1);
      mbar_init(&m->it_empty[i], kReaders);
    }
    mbar_init(&m->joined, 128);
    mbar_init(&m->join_free, 4);
    for (int i = 0; i < 2; ++i) mbar_init(&m->drain[i], 1);
    m->abort = 0;
    fence_mbar_init();
  }
  pdl_launch_dependents();  // the merge's blocks wait for this grid's end on the SMs it leaves
  if (warp == 12) tmem_alloc(smem_u32(&m->tmem), 512);
  // launched early too: nothing global is touched before the work ahead is complete
  pdl_wait();
  if (threadIdx.x == 0) a.desc[blockIdx.x].parts = 0;
  ChunkRange rng = {};
  if (warp == 13)  // beside the set-up
    rng = chunk_range(a.rg, a.g, blockIdx.x, gridDim.x, a.min_units, a.dev_err);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t base = smem_u32(smem), tmem = __shfl_sync(0xffffffffu, m->tmem, 0);
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    softmax_role<TI, T, D>(a, m, base, tmem, warp / 4);
  } else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if constexpr (F8)
      Loader8<D>(a, m, base, base + C::kMeta + kMetaBytes, warp - 8, lane).run();
    else
      Loader<T, D>(a, m, base, warp - 8, lane).run();
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 12 || warp == 14) mma_role<T, D, F8 && !std::is_same<TI, T>::value>(a, m, base, tmem, (warp - 12) / 2);
    if (warp == 13) item_role(a, m, rng);
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int D, bool F8>
cudaError_t launch_tc(const TcArgs& a, int ctas, cudaStream_t s) {
  using C = Cfg<D>;
  constexpr int kSmem = C::kMeta + (F8 ? kMetaBytes + 2 * C::kRaw8 : (int)sizeof(TcMeta)) + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory");
  cudaError_t e = cudaFuncSetAttribute(chunk_tc_kernel<T, D, F8>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  return launch_k(chunk_tc_kernel<T, D, F8>, dim3(ctas), dim3(kThreads), kSmem, s, true, a);
}

template <typename T, int D>
cudaError_t launch_tc(const TcArgs& a, int ctas, cudaStream_t s) {
  return a.kv.dtype == CVSA_DTYPE_E4M3 ? launch_tc<T, D, true>(a, ctas, s)
                                       : launch_tc<T, D, false>(a, ctas, s);
}

}  // namespace

bool chunk_tc_eligible(const KvView& kv, const ChunkView& c) {
  return (c.dtype == kv.dtype || kv.dtype == CVSA_DTYPE_E4M3) && c.dtype != CVSA_DTYPE_F32 &&
         (kv.d == 64 || kv.d == 128) && c.hq / kv.hkv <= kTile;
}

int chunk_tc_rows() { return 2 * kTile; }

ChunkGeo chunk_tc_geo(const KvView& kv, const RaggedView& rg, const ChunkView& c) {
  ChunkGeo g;
  g.bs = kv.bs;
  g.hkv = kv.hkv;
  g.G = c.hq / kv.hkv;
  g.P = 2 * (kTile / g.G);
  g.KT = kKT;
  g.causal = c.causal;
  g.window = c.window;
  g.fixed = 2;
  g.few = kPairRows;
  g.fixed_few = 4;
  g.split = chunk_may_split(rg, kv.bs, kKT);
  return g;
}

cudaError_t launch_chunk_tc(const KvView& kv, const RaggedView& rg, const ChunkView& c, int ctas,
                            float* parts, ChunkMergeDesc* desc, int32_t* dev_err, cudaStream_t s) {
  TcArgs a;
  a.rg = rg;
  a.kv = kv;
  a.c = c;
  a.TQ = kTile / (c.hq / kv.hkv);
  a.g = chunk_tc_geo(kv, rg, c);
  a.bs_shift = -1;
  a.pages16 = kv.bs % 16 == 0;
  for (int i = 0; i < 31; ++i)
    if (kv.bs == 1 << i) a.bs_shift = i;
  a.scale2 = c.scale * kLog2e;
  a.min_units = 2;
  a.parts = parts;
  a.desc = desc;
  a.dev_err = dev_err;
  a.wait_limit = wait_limit() ? wait_limit() : 1u << 18;  // a poll waits about 4 us: a second
  if (c.dtype == CVSA_DTYPE_BF16)
    return kv.d == 64 ? launch_tc<__nv_bfloat16, 64>(a, ctas, s)
                      : launch_tc<__nv_bfloat16, 128>(a, ctas, s);
  return kv.d == 64 ? launch_tc<__half, 64>(a, ctas, s) : launch_tc<__half, 128>(a, ctas, s);
}

}  // namespace cvsa
