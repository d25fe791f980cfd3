// Attention over the paged 8-bit K/V cache for many rows a sequence: prompt
// chunks (nh_paged_attention's tiled form), on the 5th-generation tensor cores.
//
// A CTA takes 128 queries (rows x heads of one KV head) of one sequence and
// walks the visible positions in tiles of 128:
//   warps 8-11 (K) and 12-15 (V) read a tile's codes and write them as f16
//   operands (exact);
//   warp 16 issues S = Qhi K + Qlo K and O += Phi V + Plo V (tcgen05.mma
//   kind::f16; accumulators, Q and P in tensor memory);
//   warps 0-3 and 4-7 hold a row a lane and take the tiles in turn: scores,
//   running maximum (handed from tile to tile) and sum, weights split into two
//   f16 parts that take the scores' place.
// Two or three score tiles rotate (what the tensor memory holds), so that the
// tensor cores form the scores ahead while weights are in the making.
// What bounds it.  The products: f32 queries and weights as two f16 parts each
// make 8 hd operations a score where one f16 pass would make 4, 2,048 cycles a
// tile of 128 dimensions; the exponentials, 1,024 cycles a tile.  At present the
// way of a tile from its scores to its weights (tensor memory's loads, the
// exponentials, the hand-over) is longer than either, although the two groups of
// warps share it: 2.6 us a tile of 128 dimensions (5,100 cycles at 1,965 MHz),
// 1.4 us (2,750) of 64, and some 12 us of a launch of one CTA to an SM belong to
// none (nine sequences of 128 rows, 16 heads, 1 to 64 tiles each: 15 to 177 us,
// 14 to 102 of 64 dimensions).  2,048 rows after 2,048 others, 16 heads of 128:
// 123 us (half of the tensor cores' measured rate with both parts counted); four
// prompts of up to 4,000 rows, 16 heads of 64 over 8, window 1,024: 244 us.
// Measured and left, beside 125 and 240 to 247 us of the states they were tried in:
// both groups on one tile, half of its columns each, 137 and 274; walking a tile
// in loops instead of unrolled, 129 and 251; narrow heads as two CTAs to an SM,
// each with one group of softmax warps and one score tile, which would hide the
// starts, 253 for 247, and 91 for 76 with one prompt, as each tile then waits for
// its own products.  A CTA's start is mostly its queries': 16 copies by each of
// eight warps 240 us, 32 by four 245, 128 by one 281, 16-byte copies 253, loads
// into registers 248.
// Operand tiles lie in shared memory as rows of 64 dimensions, 128 bytes swizzled:
// the same image serves K (K-major) and V (MN-major), and eight lanes write to
// different banks.
// (Unswizzled operands are read at half the rate: with Q in shared memory too, a
// 16-wide step of the scores took 138 cycles for 64, and the softmax warps'
// own accesses waited.)
// The tensor cores' own additions cut off, which over a long sequence pulls every
// sum towards zero (9e-6 of it at 4,096 positions): the sums of every few tiles
// leave tensor memory and are added up in shared memory, rounded.  (Every third:
// 1.1e-6 against the f32 formula's 1.4e-6 on 2,048 rows after 2,048 others;
// every seventh would save 5% of the time at 2.1e-6.  With values of one sign,
// where nothing cancels what is cut off, 2.5e-6.)
// All waits are bounded; an expired one records NH_E_TIMEOUT and makes the rows NaN.
#include <cooperative_groups.h>

#include "paged_attention.cuh"

namespace cg = cooperative_groups;

namespace nh {

namespace {

constexpr int kTileQ = 128;     // queries of a CTA = tensor-memory lanes
constexpr int kTileK = 128;     // positions of a step
constexpr int kSub = 16;        // positions that certainly share a page
constexpr int kSubs = kTileK / kSub;
constexpr int kTileThreads = 640;
constexpr int kSoftThreads = 256;
constexpr float kLeast = 1.17549435e-38f;  // factor of the scores at least: a hidden one, -inf, stays that
constexpr int kHidden = -1000;     // V's exponent where no position is seen
constexpr int kHalfBytes = kTileK * 128;  // 64 dimensions of an operand tile
constexpr int kTileShift = 7;   // weights are 2^7 times [0, 2^8], of the maximum in use: 22 bits of those from 2^-10 on
constexpr int kFlush = 3;       // tiles whose products are added up in tensor memory
constexpr int kScalePlaces = 8;
constexpr int kLowest = -60;    // least power of two of a part's weights that products take
constexpr float kGrow = 8.f;    // the maximum in use lags the true one by at most 2^8

constexpr uint32_t kTmemCols = 512;

// Tensor-memory columns: the score tiles, O, Q (high parts, then low ones).
template <int HD>
struct TileTmem {
  static constexpr int kScoreTiles = HD <= 64 ? 3 : 2;
  static constexpr uint32_t kS = 0, kO = kScoreTiles * kTileK, kQ = kO + HD;
  static_assert(kQ + HD <= kTmemCols, "tensor memory");
};

template <int HD>
struct TileShared {
  static constexpr int kOperand = (HD + 63) / 64 * kHalfBytes, kScoreTiles = TileTmem<HD>::kScoreTiles;
  static constexpr int kRow = HD + 4;  // floats of a joined row, padded against bank conflicts
  uint8_t ring[2][2][kOperand];        // K, V: two stages each
  // Q on its way to tensor memory; the joined values once the products are done.
  float rows[kTileQ][kRow];
  float ks[kScalePlaces][kSubs];  // scales of a tile's 16-position parts
  int ve[kScalePlaces][kSubs];    // exponents of V's, or kHidden
  // A row's maximum in use and V's exponent in use (as bits; of the parts that the row sees), after an even and an odd tile.
  float2 ref[2][kTileQ];
  float2 at_flush[kTileQ];   // the same, of the sums in `rows`
  float top[2][kTileQ];      // largest magnitudes of the query's halves
  int64_t row_at[kTileQ];  // where a query's row starts in q and out
  uint64_t full[2][2], empty[2][2], scales[kScalePlaces], q_rows, q_full, drained;
  uint64_t s_full[kScoreTiles], p_full[kScoreTiles], pv_done[kScoreTiles];
  float m[kTileQ], sum[kTileQ], l[2][kTileQ], lm[2][kTileQ];
  uint32_t tmem;
  int failed;
};

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar))
               : "memory");
}

// Shared-memory operand descriptor, 128-byte swizzle, version 1: 8-row groups
// 1024 bytes apart (K's rows of the score product, V's positions); `lead`: from
// 64 columns of an MN-major operand to the next.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(lead >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor: D f32, A and B f16, M = 128; B MN-major for V.
__host__ __device__ constexpr uint32_t idesc(int n, bool mn_major) {
  return (1u << 4) | (mn_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (128u >> 4 << 24);
}
// D (+)= A B with A in tensor memory; a 16-wide step of B is a constant added to
// its descriptor's low word.
template <uint32_t kIdesc>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(kIdesc), "r"(add)
      : "memory");
}
// One lane of the warp, always the same.
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(is));
  return is != 0u;
}

#define NH_R8(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), "=r"(a[i + 4]), "=r"(a[i + 5]), \
                    "=r"(a[i + 6]), "=r"(a[i + 7])
#define NH_W8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), "r"(a[i + 4]), "r"(a[i + 5]), "r"(a[i + 6]), \
                    "r"(a[i + 7])
#define NH_RW8(a, i) "+r"(a[i]), "+r"(a[i + 1]), "+r"(a[i + 2]), "+r"(a[i + 3]), "+r"(a[i + 4]), "+r"(a[i + 5]), \
                     "+r"(a[i + 6]), "+r"(a[i + 7])
// 32 columns of the warp's lanes; the registers hold them after tc_wait_ld, and
// tc_loaded keeps the compiler from using them before it.
__device__ __forceinline__ void tc_ld32(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : NH_R8(v, 0), NH_R8(v, 8), NH_R8(v, 16), NH_R8(v, 24)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};\n" ::NH_W8(v, 0),
      NH_W8(v, 8), NH_W8(v, 16), NH_W8(v, 24), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : NH_R8(v, 0), NH_R8(v, 8)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};\n" ::NH_W8(
          v, 0),
      NH_W8(v, 8), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tc_st8(uint32_t addr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};\n" ::NH_W8(v, 0), "r"(addr)
               : "memory");
}
__device__ __forceinline__ void tc_loaded16(uint32_t* v) { asm volatile("" : NH_RW8(v, 0), NH_RW8(v, 8)); }
__device__ __forceinline__ void tc_loaded(uint32_t* v) {
  asm volatile("" : NH_RW8(v, 0), NH_RW8(v, 8), NH_RW8(v, 16), NH_RW8(v, 24));
}
#undef NH_R8
#undef NH_W8
#undef NH_RW8
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Tiles of a sequence in this form.
__device__ __forceinline__ int tiles_of(const PagedAttnArgs& p, const SeqRows& r) {
  const int64_t n_q = static_cast<int64_t>(r.n) * p.group;
  return n_q > p.few ? static_cast<int>((n_q + kTileQ - 1) / kTileQ) : 0;
}

// The rows and tile of `item`, later tiles (which see more positions) first;
// false when there are not that many.  Warp-wide, 32 sequences at a time, from
// the last one on.
__device__ __forceinline__ bool find_tile(const PagedAttnArgs& p, int64_t cap, int64_t item, int lane, int& seq, int& tile,
                                          SeqRows& rows) {
  for (int s0 = (p.rows.n_seq - 1) & ~31; s0 >= 0; s0 -= 32) {
    const int s = s0 + lane;
    SeqRows r{0, 0, 0};
    if (s < p.rows.n_seq) r = seq_rows(p.rows, s, cap);
    if (r.n < 0 && blockIdx.x == 0) paged_error(p.rows);
    const int mine = tiles_of(p, r);
    int inc = mine;  // tiles of this sequence and the later ones of the 32
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int down = __shfl_down_sync(0xffffffffu, inc, o);
      if (lane + o < 32) inc += down;
    }
    const int sum = __shfl_sync(0xffffffffu, inc, 0);
    if (item < sum) {
      const int l = 31 - __clz(__ballot_sync(0xffffffffu, inc > item));
      seq = s0 + l;
      tile = __shfl_sync(0xffffffffu, inc, l) - 1 - static_cast<int>(item);
      rows.r0 = __shfl_sync(0xffffffffu, r.r0, l);
      rows.n = __shfl_sync(0xffffffffu, r.n, l);
      rows.p0 = __shfl_sync(0xffffffffu, r.p0, l);
      return true;
    }
    item -= sum;
  }
  return false;
}

template <int HD>
__global__ void __launch_bounds__(kTileThreads, 1) paged_tile_kernel(const PagedAttnArgs p) {
  constexpr int kItems = HD / 16;  // 16-byte pieces a converting lane takes of a tile
  extern __shared__ __align__(1024) uint8_t tile_smem[];
  auto& sh = *reinterpret_cast<TileShared<HD>*>(tile_smem);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), nrank = static_cast<int>(cluster.num_blocks());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int page = p.kv.page, lg = p.kv.page_log2;
  constexpr int kScoreTiles = TileTmem<HD>::kScoreTiles;
  if (tid == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sh.full[i >> 1][i & 1], 4);
      mbar_init(&sh.empty[i >> 1][i & 1], 1);
    }
    for (int i = 0; i < kScalePlaces; ++i) mbar_init(&sh.scales[i], 4);
    mbar_init(&sh.q_rows, 8);
    mbar_init(&sh.q_full, 8);
    for (int i = 0; i < kScoreTiles; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], 4);
      mbar_init(&sh.pv_done[i], 1);
    }
    mbar_init(&sh.drained, 1);
    sh.failed = 0;
    fence_barrier_init();
  }
  if (warp == 16) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&sh.tmem)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  pdl_wait();
  pdl_trigger();
  const int64_t cap = static_cast<int64_t>(p.rows.max_blocks) * page;
  const int64_t item = static_cast<int64_t>(blockIdx.x) / nrank;
  const int kh = static_cast<int>(item % p.kv.n_kv);
  int s = 0, qt = 0;
  SeqRows sq{0, 0, 0};
  const bool work = find_tile(p, cap, item / p.kv.n_kv, lane, s, qt, sq);  // every CTA of the cluster alike
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = sh.tmem;
  if (!work) {
    if (warp == 16)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kTmemCols) : "memory");
    return;
  }
  const int n_q = sq.n * p.group, q0 = qt * kTileQ, nq = min(kTileQ, n_q - q0);
  const int first_pos = sq.p0 + q0 / p.group, last_pos = sq.p0 + (q0 + nq - 1) / p.group;
  // Visible tiles: the sinks', then those from `lo` on; this CTA's share of them.
  const int lo = p.window > 0 ? max(0, first_pos - p.window + 1) / kTileK : 0;
  const int n_sink = p.window > 0 ? min((min(p.n_sink, last_pos + 1) + kTileK - 1) / kTileK, lo) : 0;
  const int n_all = n_sink + last_pos / kTileK + 1 - lo;
  const int share = n_all / nrank, rest = n_all % nrank;
  const int j0 = rank * share + min(rank, rest), n = share + (rank < rest ? 1 : 0);
  auto tile_pos = [&](int j) { return (j0 + j < n_sink ? j0 + j : j0 + j - n_sink + lo) * kTileK; };

  // Barriers.  A wait tells a phase's parity from the next one's only, so none may run two phases ahead of a waiter: one
  // barrier a place (score tile, operand stage), whose next phase needs what the waiter does after this one.
  auto products_done = [&](int j) {
    return mbar_wait(&sh.pv_done[j % kScoreTiles], static_cast<uint32_t>(j / kScoreTiles) & 1u);
  };
  auto all = [](bool lane_ok) { return __all_sync(0xffffffffu, lane_ok) != 0; };
  bool ok = true;
  if (warp >= 8 && warp < 16) {
    // ---------------------------------------------------------------- codes to operands
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
    // Lanes: row r of eight, 16-byte column c of four.  (Rows across neighbouring lanes instead cost eight times the load
    // wavefronts, and with them a third of the kernel's time: they delay the softmax warps' tensor-memory loads.)
    const int of_v = (warp - 8) >> 2, w = warp & 3, r = lane >> 2, c = lane & 3;
    const uint8_t* codes = (of_v ? p.kv.v_codes : p.kv.k_codes) + static_cast<uint64_t>(kh) * static_cast<uint32_t>(page * HD);
    const uint32_t page_bytes = static_cast<uint32_t>(p.kv.n_kv) * static_cast<uint32_t>(page * HD);  // at most 2^30
    const int32_t* table = p.rows.page_table + static_cast<int64_t>(s) * p.rows.max_blocks;
    // Pages of this warp's two 16-position parts of 16 tiles: lane l has part l & 1 of tile f + (l >> 1).  -1: none (past
    // the last position, or between the sinks and the window of every query: its page may have been given up), -2: out
    // of range.
    auto ids_of = [&](int f) {
      const int j = f + (lane >> 1);
      int id = -1;
      if (j < n) {
        const int t = tile_pos(j) + w * 32 + (lane & 1) * kSub;
        if (t <= last_pos && (p.window == 0 || t + kSub - 1 > first_pos - p.window || t < p.n_sink)) {
          id = __ldcg(table + (t >> lg));
          if (id < 0 || id >= p.kv.n_pages) id = -2;
        }
      }
      return id;
    };
    // Piece i of a lane: 16 codes of row `rg` * 8 + r of the warp's 32, from column `col` * 16 on.
    auto rg_of = [&](int i) {
      return HD == 128 ? i >> 1 : HD == 64 ? i : HD == 32 ? 2 * i + (c >> 1) : (i * 4 + c) / kItems;
    };
    auto col_of = [&](int i) {
      return HD == 128 ? (i & 1) * 4 + c : HD == 64 ? c : HD == 32 ? c & 1 : (i * 4 + c) % kItems;
    };
    uint4 raw[kItems];
    int id0 = 0, id1 = 0, ids = ids_of(0), ids_next = ids_of(16);
    float ks = 1.f, vs = 0.f;
    bool seen = false;
    auto load = [&](int j) {
      id0 = __shfl_sync(0xffffffffu, ids, (j & 15) * 2);
      id1 = __shfl_sync(0xffffffffu, ids, (j & 15) * 2 + 1);
      if ((j & 15) == 15) {
        ids = ids_next;
        ids_next = ids_of(j + 17);
      }
      const int slot = (tile_pos(j) + w * 32 + r) & (page - 1);
      const uint8_t* p0 = codes + static_cast<uint64_t>(static_cast<uint32_t>(max(id0, 0))) * page_bytes + slot * HD;
      const uint8_t* p1 = codes + static_cast<uint64_t>(static_cast<uint32_t>(max(id1, 0))) * page_bytes +
                          ((slot + kSub) & (page - 1)) * HD;
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int rg = rg_of(i);
        raw[i] = __ldcg(reinterpret_cast<const uint4*>((rg < 2 ? p0 : p1) + (rg & 1) * 8 * HD + col_of(i) * 16));
      }
      if (!of_v) {
        const int mine = lane == 0 ? id0 : id1;
        seen = mine >= 0;
        if (lane < 2 && seen) {
          ks = __ldcg(p.kv.k_scales + static_cast<int64_t>(mine) * p.kv.n_kv + kh);
          vs = __ldcg(p.kv.v_scales + static_cast<int64_t>(mine) * p.kv.n_kv + kh);
        }
      }
    };
    bool lost = false;
    if (n > 0) load(0);
    for (int j = 0; j < n; ++j) {
      lost |= id0 == -2 || id1 == -2;
      ok = all(mbar_wait(&sh.empty[of_v][j & 1], static_cast<uint32_t>((j >> 1) & 1) ^ 1u));
      if (!ok) break;
      uint8_t* to = sh.ring[of_v][j & 1] + (w * 32 + r) * 128;
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        // Two 8-dimension pieces of the row, which the swizzle moves by the row's place among eight.
        const int col = col_of(i), piece = col * 2 & 7;
        uint8_t* d = to + rg_of(i) * 1024 + (col >> 2) * kHalfBytes;
        *reinterpret_cast<uint4*>(d + (piece ^ r) * 16) =
            make_uint4(codes_lo(raw[i].x), codes_hi(raw[i].x), codes_lo(raw[i].y), codes_hi(raw[i].y));
        *reinterpret_cast<uint4*>(d + ((piece + 1) ^ r) * 16) =
            make_uint4(codes_lo(raw[i].z), codes_hi(raw[i].z), codes_lo(raw[i].w), codes_hi(raw[i].w));
      }
      // The scales' place was last read for tile j - 8, whose weights were in use before K of tile j found its stage free
      // (the scores of tile j - 2 follow the products of j - 5 at the latest).
      if (!of_v && lane < 2) {
        sh.ks[j & (kScalePlaces - 1)][w * 2 + lane] = seen ? ks : 1.f;
        sh.ve[j & (kScalePlaces - 1)][w * 2 + lane] = seen ? exponent_of(vs) : kHidden;
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sh.full[of_v][j & 1]);
        if (!of_v) mbar_arrive(&sh.scales[j & (kScalePlaces - 1)]);
      }
      if (j + 1 < n) load(j + 1);
    }
    if (lost && lane == 0) paged_error(p.rows);
    if (!ok) sh.failed = 1;
  } else if (warp >= 16) {
    // ---------------------------------------------------------------- products
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;\n");
    if (warp == 16 && n > 0) {
      constexpr uint32_t kOp = TileShared<HD>::kOperand;
      // 16 dimensions of K (step k of its 64), 16 positions of V.
      auto step_k = [](int k) { return static_cast<uint64_t>((k >> 2) * kHalfBytes + (k & 3) * 32) >> 4; };
      constexpr uint64_t kStepV = 2048 >> 4;
      const bool one = elect_one();
      const uint64_t kd = operand(smem_u32(sh.ring[0][0]), 16);
      const uint64_t vd = operand(smem_u32(sh.ring[1][0]), kHalfBytes);
      const uint32_t qa = tmem + TileTmem<HD>::kQ, oa = tmem + TileTmem<HD>::kO;
      auto scores = [&](int j) {
        if (!all(mbar_wait(&sh.full[0][j & 1], static_cast<uint32_t>(j >> 1) & 1u))) return false;
        tc_after();
        const uint64_t b = kd + ((j & 1) * kOp >> 4);
        const uint32_t d = tmem + TileTmem<HD>::kS + (j % kScoreTiles) * kTileK;
        if (one) {
#pragma unroll
          for (int k = 0; k < HD / 8; ++k) {  // the low parts' steps first, while the sums they cut are small
            const int step = k % (HD / 16), part = k < HD / 16 ? HD / 2 : 0;
            mma_ts<idesc(kTileK, false)>(d, qa + part + step * 8, b + step_k(step), k > 0 ? 1u : 0u);
          }
          tc_commit(&sh.empty[0][j & 1]);
          tc_commit(&sh.s_full[j % kScoreTiles]);
        }
        __syncwarp();
        return true;
      };
      ok = all(mbar_wait(&sh.q_full, 0)) && scores(0) && (n < 2 || scores(1));
      for (int j = 0; j < n && ok; ++j) {
        // With three score tiles those of j + 2 take the place of tile j - 1's weights, before the products of j.
        if (kScoreTiles == 3 && j + 2 < n) ok = (j == 0 || all(products_done(j - 1))) && scores(j + 2);
        if (!ok) break;
        ok = all(mbar_wait(&sh.full[1][j & 1], static_cast<uint32_t>(j >> 1) & 1u) &&
                 mbar_wait(&sh.p_full[j % kScoreTiles], static_cast<uint32_t>(j / kScoreTiles) & 1u));
        if (!ok) break;
        tc_after();
        const uint64_t b = vd + ((j & 1) * kOp >> 4);
        const uint32_t a = tmem + TileTmem<HD>::kS + (j % kScoreTiles) * kTileK;
        if (one) {
#pragma unroll
          for (int k = 0; k < kTileK / 8; ++k) {
            const int step = k % (kTileK / 16), part = k < kTileK / 16 ? 16 : 0;  // low, high
            mma_ts<idesc(HD, true)>(oa, a + (step >> 1) * 32 + part + (step & 1) * 8, b + step * kStepV,
                                    k > 0 || j % kFlush > 0 ? 1u : 0u);
          }
          tc_commit(&sh.empty[1][j & 1]);
          tc_commit(&sh.pv_done[j % kScoreTiles]);
        }
        __syncwarp();
        if (kScoreTiles == 2 && j + 2 < n) ok = all(products_done(j)) && scores(j + 2);  // with two, that of this one's
      }
      // No product is left in flight when the operands and the tensor memory are given up, whatever ended the loop.
      if (one) tc_commit(&sh.drained);
      __syncwarp();
      ok = mbar_wait(&sh.drained, 0) && ok;
      if (!ok) sh.failed = 1;
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax: a row a lane, every second tile
    asm volatile("setmaxnreg.inc.sync.aligned.u32 144;\n");
    float row_m = -INFINITY, row_l = 0.f;  // the row's maximum in use, sum of its weights
    int eref = -200;                       // O is in units of 2^(eref - kTileShift + kCodeShift)
    const int half = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const int pos = row < nq ? sq.p0 + (q0 + row) / p.group : -1;
    const bool idle = quad * 32 >= nq;  // no row of this warp is a query
    float fq;
    {
      // The rows, copied whole, sixteen by a warp (the copies are sent one after the other); then the two lanes of a row
      // scale half of it each so that the largest magnitude is in [2^13, 2^14), and split it.  A negative factor of the
      // scores changes the query's sign.
      {
        const int mine = warp * 16 + lane;
        if (lane == 0) mbar_expect_tx(&sh.q_rows, static_cast<uint32_t>(max(0, min(nq - warp * 16, 16))) * HD * 4);
        __syncwarp();
        if (lane < 16 && mine < nq) {
          const int qr = (q0 + mine) / p.group, qh = q0 + mine - qr * p.group;
          const int64_t at = (static_cast<int64_t>(sq.r0 + qr) * p.n_head + kh * p.group + qh) * HD;
          bulk_g2s(sh.rows[mine], p.q + at, HD * 4, &sh.q_rows);
          sh.row_at[mine] = at;
        }
      }
      ok = mbar_wait(&sh.q_rows, 0);
      __syncwarp();
      float4 x[HD / 8];
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        x[i] = row < nq ? reinterpret_cast<const float4*>(sh.rows[row])[half * (HD / 8) + i] : make_float4(0.f, 0.f, 0.f, 0.f);
        top = max3(top, max3(fabsf(x[i].x), fabsf(x[i].y), fabsf(x[i].z)), fabsf(x[i].w));
      }
      sh.top[half][row] = top;
      asm volatile("bar.sync %0, 64;\n" ::"r"(10 + quad) : "memory");
      top = fmaxf(top, sh.top[half ^ 1][row]);
      const int e = min(max(exponent_of(top), -100), 127);
      const float up = p.scale < 0.f ? -pow2i(13 - e) : pow2i(13 - e);
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        uint32_t h[8], l[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4& y = x[i * 4 + k];
          split2(y.x * up, y.y * up, h[2 * k], l[2 * k]);
          split2(y.z * up, y.w * up, h[2 * k + 1], l[2 * k + 1]);
        }
        const uint32_t to = tmem + TileTmem<HD>::kQ + lanes + half * (HD / 4) + i * 8;
        tc_st8(to, h);
        tc_st8(to + HD / 2, l);
      }
      fq = fabsf(p.scale) * kLog2e * pow2i(e - 13 + kCodeShift);
      tc_wait_st();
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.q_full);
    }
    // Sums of the row in shared memory (when `more`) times f, plus those in tensor memory times g, 16 columns a step;
    // `done` is applied to the results.
    auto add_sums = [&](int i0, int i1, bool more, float f, float g, auto done) {
#pragma unroll 1
      for (int i = i0; i < i1; i += 2) {
        uint32_t o[2][16];
        float4 v[2][4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (i + e >= i1) break;
          tc_ld16(tmem + TileTmem<HD>::kO + lanes + (i + e) * 16, o[e]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (i + e >= i1) break;
          const float4* from = reinterpret_cast<const float4*>(&sh.rows[row][(i + e) * 16]);
#pragma unroll
          for (int k = 0; k < 4; ++k) v[e][k] = more ? from[k] : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        tc_wait_ld();
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (i + e >= i1) break;
          tc_loaded16(o[e]);
          float4* to = reinterpret_cast<float4*>(&sh.rows[row][(i + e) * 16]);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            to[k] = make_float4(done(fmaf(v[e][k].x, f, __uint_as_float(o[e][4 * k]) * g)),
                                done(fmaf(v[e][k].y, f, __uint_as_float(o[e][4 * k + 1]) * g)),
                                done(fmaf(v[e][k].z, f, __uint_as_float(o[e][4 * k + 2]) * g)),
                                done(fmaf(v[e][k].w, f, __uint_as_float(o[e][4 * k + 3]) * g)));
        }
      }
    };
    // From one maximum in use to another (-inf: nothing has been seen, and the sums are zero).
    auto factor = [](float from, float to) { return from == to ? 1.f : exp2_fast(from - to); };
    // The warps of a row take turns: one forms the maximum of its tile while the other forms the weights of the tile
    // before.  Maximum and exponent in use go from tile to tile through shared memory, each row's sum of weights stays
    // with the warp.  No warp leaves the loop early, so that the pairs' barriers stay matched: after an expired wait it
    // runs on without waiting.
    for (int j = half; j < n; j += 2) {
      ok = ok && mbar_wait(&sh.s_full[j % kScoreTiles], static_cast<uint32_t>(j / kScoreTiles) & 1u);
      __syncwarp();
      if (idle) {
        if (lane == 0) mbar_arrive(&sh.p_full[j % kScoreTiles]);
        continue;
      }
      tc_after();
      const uint32_t scol = tmem + TileTmem<HD>::kS + (j % kScoreTiles) * kTileK + lanes;
      const int place = j & (kScalePlaces - 1);
      ok = ok && mbar_wait(&sh.scales[place], static_cast<uint32_t>(j / kScalePlaces) & 1u);
      const int t0 = tile_pos(j);
      // The tile's 16-position parts: V's exponents, what K's scale makes of a product.
      int ve[kSubs];
      float ka[kSubs];
#pragma unroll
      for (int i = 0; i < kSubs; i += 4) {
        *reinterpret_cast<int4*>(ve + i) = *reinterpret_cast<const int4*>(&sh.ve[place][i]);
        *reinterpret_cast<float4*>(ka + i) = *reinterpret_cast<const float4*>(&sh.ks[place][i]);
      }
      bool whole = true;
#pragma unroll
      for (int i = 0; i < kSubs; ++i) {
        ka[i] = fmaxf(fq * ka[i], kLeast);
        whole &= ve[i] != kHidden;
      }
      const bool plain = whole && t0 + kTileK - 1 <= first_pos &&
                         (p.window == 0 || t0 > last_pos - p.window || t0 + kTileK <= p.n_sink);
      if (!plain) {
        // Scores that the row does not see become -inf in tensor memory, 32 columns a step.
#pragma unroll 1
        for (int c = 0; c < kTileK / 32; ++c) {
          const int h0 = t0 + c * 32;
          auto up_to = [](int i) { return i < 0 ? 0u : i >= 31 ? ~0u : (2u << i) - 1u; };
          uint32_t see = up_to(pos - h0);
          if (p.window > 0) see &= ~up_to(pos - p.window - h0) | up_to(p.n_sink - 1 - h0);
          if (sh.ve[place][2 * c] == kHidden) see &= 0xffff0000u;
          if (sh.ve[place][2 * c + 1] == kHidden) see &= 0xffffu;
          if (__all_sync(0xffffffffu, see == ~0u)) continue;
          uint32_t x[32];
          tc_ld32(scol + c * 32, x);
          tc_wait_ld();
          tc_loaded(x);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if ((see & (1u << i)) == 0u) x[i] = 0xff800000u;
          tc_st32(scol + c * 32, x);
        }
        tc_wait_st();
        // Parts of which the row sees nothing: their scales must not count for it.
#pragma unroll
        for (int i = 0; i < kSubs; ++i) {
          const int a = t0 + i * kSub;
          if (a > pos || (p.window > 0 && a + kSub - 1 <= pos - p.window && a >= p.n_sink)) ve[i] = kHidden;
        }
      }
      int ev = kHidden, low_e = 1000;  // the row's largest exponent of V in the tile, and the least
#pragma unroll
      for (int i = 0; i < kSubs; ++i) {
        ev = max(ev, ve[i]);
        if (ve[i] != kHidden) low_e = min(low_e, ve[i]);
      }
      uint32_t u[2][32];
      tc_ld32(scol, u[0]);
      tc_ld32(scol + 32, u[1]);
      float top = -INFINITY;
      auto maximum = [&](int c, const uint32_t* x) {
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          float t = fmaxf(__uint_as_float(x[d * kSub]), __uint_as_float(x[d * kSub + 1]));
#pragma unroll
          for (int i = 2; i < kSub; i += 2) t = max3(t, __uint_as_float(x[d * kSub + i]), __uint_as_float(x[d * kSub + i + 1]));
          top = fmaxf(top, t * ka[2 * c + d]);
        }
      };
      __syncwarp();
      tc_wait_ld();
      tc_loaded(u[0]);
      tc_loaded(u[1]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        maximum(c, u[c]);
        tc_ld32(scol + (c + 2) * 32, u[c]);
      }
      tc_wait_ld();
      tc_loaded(u[0]);
      tc_loaded(u[1]);
#pragma unroll
      for (int c = 0; c < 2; ++c) maximum(c + 2, u[c]);
      float2 before = make_float2(-INFINITY, __int_as_float(-200));
      if (j > 0) {
        asm volatile("bar.sync %0, 64;\n" ::"r"(2 + half * 4 + quad) : "memory");  // the tile before's
        before = sh.ref[half ^ 1][row];
      }
      row_l *= factor(row_m, before.x);
      row_m = before.x;
      eref = __float_as_int(before.y);
      // The maximum in use follows the true one only when that is 2^8 above it; O follows then, and when V's scale grows.
      const bool grow = top > (row_m == -INFINITY ? row_m : row_m + kGrow);
      const bool flush = j > 0 && j % kFlush == 0;
      const bool move = __any_sync(0xffffffffu, grow || ev > eref);
      float alpha = 1.f;
      if (grow) {
        alpha = factor(row_m, top);
        row_m = top;
        row_l *= alpha;
      }
      const int en = max(eref, ev);
      alpha *= pow2i(max(eref - en, -200));
      eref = en;
      sh.ref[half][row] = make_float2(row_m, __int_as_float(eref));
      if (j + 1 < n) asm volatile("bar.arrive %0, 64;\n" ::"r"(2 + (half ^ 1) * 4 + quad) : "memory");
      const float base = row_m == -INFINITY ? 0.f : row_m;
      const bool low = low_e - eref + kTileShift < kLowest;
      // Weights, in pairs as high and low f16 parts: of every 32 columns the first 16 hold the high ones.
      auto weights = [&](int c, const uint32_t* x) {
        uint32_t w[32];
        if (low) {
          // Parts whose scale is 2^60 below the largest: the weights count for the sum alone.
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            if (ve[2 * c + d] == kHidden || ve[2 * c + d] - eref + kTileShift >= kLowest) continue;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < kSub; ++i) sum += exp2_fast(fmaf(__uint_as_float(x[d * kSub + i]), ka[2 * c + d], -base));
            row_l += sum;
          }
        }
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const int eb = ve[2 * c + d] - eref + kTileShift;
          const float a = ka[2 * c + d], off = eb < kLowest ? -INFINITY : static_cast<float>(eb) - base;
          float2 sum2 = make_float2(0.f, 0.f);
          const float2 a2 = make_float2(a, a), off2 = make_float2(off, off);
#pragma unroll
          for (int i = 0; i < kSub / 2; ++i) {
            const int k = d * kSub + 2 * i;
            const float2 y = fma2(make_float2(__uint_as_float(x[k]), __uint_as_float(x[k + 1])), a2, off2);
            const float2 e = make_float2(exp2_fast(y.x), exp2_fast(y.y));
            sum2 = add2(sum2, e);
            const __half2 h = __floats2half2_rn(e.x, e.y);
            const float2 g = __half22float2(h), rest = fma2(g, make_float2(-1.f, -1.f), e);
            const __half2 l = __floats2half2_rn(rest.x, rest.y);
            w[d * 8 + i] = *reinterpret_cast<const uint32_t*>(&h);
            w[16 + d * 8 + i] = *reinterpret_cast<const uint32_t*>(&l);
          }
          const float sum = sum2.x + sum2.y;
          row_l += sum * pow2i(min(-eb, -kLowest));
        }
        tc_st32(scol + c * 32, w);
      };
      // The last two quarters are at hand; the first two come back while these are worked on.
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        weights(c + 2, u[c]);
        tc_ld32(scol + c * 32, u[c]);
      }
      tc_wait_ld();
      tc_loaded(u[0]);
      tc_loaded(u[1]);
#pragma unroll
      for (int c = 0; c < 2; ++c) weights(c, u[c]);
      if (flush || (move && j > 0)) {
        ok = ok && products_done(j - 1);
        __syncwarp();
        tc_after();
        if (flush) {
          // The tiles' sums so far, in this tile's units; its own products start from zero.
          const float2 at = sh.at_flush[row];
          const float f = j > kFlush ? factor(at.x, row_m) * pow2i(max(__float_as_int(at.y) - eref, -200)) : 0.f;
          add_sums(0, HD / 16, j > kFlush, f, alpha, [](float x) { return x; });
          sh.at_flush[row] = make_float2(row_m, __int_as_float(eref));
        } else {
#pragma unroll 1
          for (int i = 0; i < HD / 16; ++i) {
            uint32_t o[16];
            tc_ld16(tmem + TileTmem<HD>::kO + lanes + i * 16, o);
            tc_wait_ld();
            tc_loaded16(o);
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            tc_st16(tmem + TileTmem<HD>::kO + lanes + i * 16, o);
          }
        }
      }
      tc_wait_st();
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_full[j % kScoreTiles]);
    }
    if (n > 0 && ok) ok = products_done(n - 1);
    const bool expired = __any_sync(0xffffffffu, !ok) != 0;
    if (expired && lane == 0) sh.failed = 1;
    // Every product is done: the row's values in their own units.  The group that did not take the last tile may not
    // have seen the phase before the one that it has waited for, whose parity then lets it through at once; the other
    // group's wait is sure, so the reads of O come after the barrier of both and a fence behind it.
    __syncwarp();
    sh.l[half][row] = expired ? __int_as_float(0x7fc00000) : row_l;  // an expired wait leaves no number in its rows
    sh.lm[half][row] = row_m;
    tc_before();
    asm volatile("bar.sync 1, 256;\n" ::: "memory");
    tc_after();
    const float2 last = n > 0 && !idle ? sh.ref[(n - 1) & 1][row] : make_float2(-INFINITY, __int_as_float(-200));
    const float unit = pow2i(max(__float_as_int(last.y), -126));
    const float l = sh.l[0][row] * factor(sh.lm[0][row], last.x) + sh.l[1][row] * factor(sh.lm[1][row], last.x);
    const float inv = nrank > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
    if (half == 0) {
      sh.m[row] = last.x;
      sh.sum[row] = l;
    }
    if (n == 0) {
      for (int i = half * (HD / 8); i < (half + 1) * (HD / 8); ++i)
        reinterpret_cast<float4*>(sh.rows[row])[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    } else if (!idle) {
      const float2 at = n > kFlush ? sh.at_flush[row] : last;
      add_sums(half * (HD / 32), (half + 1) * (HD / 32), n > kFlush,
               factor(at.x, last.x) * pow2i(max(__float_as_int(at.y) - __float_as_int(last.y), -200)), 1.f,
               [=](float x) { return x * inv * (pow2i(kCodeShift - kTileShift - (nrank > 1 ? kRoom : 0)) * unit); });
    }
    tc_before();
  }
  if (nrank > 1)
    cluster.sync();
  else
    __syncthreads();
  if (warp < 8) {
    constexpr int kQuads = HD / 4;
    if (nrank == 1) {
#pragma unroll 4
      for (int i = tid; i < nq * kQuads; i += kSoftThreads) {
        const int row = i / kQuads, d = i % kQuads;
        reinterpret_cast<float4*>(p.out + sh.row_at[row])[d] = reinterpret_cast<const float4*>(sh.rows[row])[d];
      }
    } else {
      // Rows of the tile in turn over the ranks, joined in rank order.
      for (int i = rank * kSoftThreads + tid; i < nq * kQuads; i += nrank * kSoftThreads) {
        const int row = i / kQuads, d = i % kQuads;
        float top = -INFINITY, sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r = 0; r < nrank; ++r) top = fmaxf(top, cluster.map_shared_rank(sh.m, r)[row]);
        for (int r = 0; r < nrank; ++r) {
          const TileShared<HD>* o = cluster.map_shared_rank(&sh, r);
          const float a = o->m[row] == -INFINITY ? 0.f : exp2_fast(o->m[row] - top);
          const float4 y = reinterpret_cast<const float4*>(o->rows[row])[d];
          sum += a * o->sum[row];
          v.x += a * y.x;
          v.y += a * y.y;
          v.z += a * y.z;
          v.w += a * y.w;
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum * pow2i(kRoom);
        reinterpret_cast<float4*>(p.out + sh.row_at[row])[d] = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
      }
    }
  }
  if (nrank > 1) cluster.sync();  // no CTA leaves while another reads its part
  if (tid == 0 && sh.failed != 0 && p.rows.err != nullptr) atomicCAS(p.rows.err, 0, NH_E_TIMEOUT);
  if (warp == 16) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

template <int HD>
int launch_tiles(const PagedAttnArgs& p, int64_t tiles, cudaStream_t s) {
  // One CTA to an SM (it takes all of the tensor memory).
  const size_t smem = std::max<size_t>(sizeof(TileShared<HD>), 120 * 1024);
  static SmemLimit configured;
  if (!ensure_smem(paged_tile_kernel<HD>, smem, configured)) return NH_E_CUDA;
  const int64_t items = tiles * p.kv.n_kv, steps = static_cast<int64_t>(p.rows.max_blocks) * p.kv.page / kTileK;
  int ranks = 1;
  while (ranks < 8 && items * ranks * 2 <= device_sm_count() && steps >= 4 * ranks) ranks *= 2;
  return launch_cluster(paged_tile_kernel<HD>, dim3(static_cast<unsigned>(items * ranks)), dim3(kTileThreads), ranks, smem,
                        s, p);
}

}  // namespace

int launch_paged_tiles(const PagedAttnArgs& p, cudaStream_t s) {
  static_assert(kTileQ == 128, "paged_tiles");
  const int64_t tiles = paged_tiles(p);
  switch (p.kv.hd) {
    case 32:
      return launch_tiles<32>(p, tiles, s);
    case 64:
      return launch_tiles<64>(p, tiles, s);
    case 96:
      return launch_tiles<96>(p, tiles, s);
    default:
      return launch_tiles<128>(p, tiles, s);
  }
}

}  // namespace nh
