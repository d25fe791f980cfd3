// Attention over the paged 8-bit K/V cache for many rows a sequence: prompt
// chunks (nh_paged_attention's tiled form), on the 5th-generation tensor cores.
//
// A CTA takes 128 queries (rows x heads of one KV head) of one sequence and
// walks the visible positions in tiles of 128:
//   warps 8-11 read a tile's codes and write them as f16 operands (exact);
//   warp 12 issues S = Qhi K + Qlo K and O += Phi V + Plo V (tcgen05.mma
//   kind::f16, accumulators and P in tensor memory);
//   warps 0-3 and 4-7 hold a row a lane and half of the tile's positions each:
//   scores, running maximum (exchanged) and sum, weights split into two f16
//   parts that take the scores' place.  The next tile's scores are formed
//   meanwhile.
// What bounds it: the two-part products make 8 hd products a score and row
// where one f16 pass would make 4 (the price of f32 queries and weights); beside
// them some 8 operations a score for the softmax.  Operands lie in shared
// memory as [8-dimension chunk][row][16 bytes], unswizzled: the same image
// serves K (K-major) and V (MN-major), and eight lanes write 128 contiguous
// bytes.
// All waits are bounded; an expired one records NH_E_TIMEOUT.
#include <cooperative_groups.h>

#include "paged_attention.cuh"

namespace cg = cooperative_groups;

namespace nh {

namespace {

constexpr int kTileQ = 128;     // queries of a CTA = tensor-memory lanes
constexpr int kTileK = 128;     // positions of a step
constexpr int kSub = 16;        // positions that certainly share a page
constexpr int kSubs = kTileK / kSub;
constexpr int kTileStages = 4;  // operand tiles in flight (K and V alternate)
constexpr int kTileThreads = 416;
constexpr int kHalf = kTileK / 2;  // positions of a tile that one softmax warp takes
constexpr float kLeast = 1.17549435e-38f;  // factor of the scores at least: a hidden one, -inf, stays that
constexpr int kHidden = -1000;     // V's exponent where no position is seen
constexpr int kChunkBytes = kTileK * 16;  // one 8-dimension chunk of an operand tile
constexpr int kTileShift = 7;   // weights are 2^7 times [0, 2^8]
constexpr float kGrow = 8.f;    // the maximum in use lags the true one by at most 2^8

constexpr uint32_t kColS = 0, kColO = 256, kTmemCols = 512;

template <int HD>
struct TileShared {
  static constexpr int kOperand = HD / 8 * kChunkBytes;
  uint8_t q[2][kOperand];  // high, low parts
  uint8_t ring[kTileStages][kOperand];
  float ks[4][kSubs];  // scales of a tile's 16-position parts (four tiles)
  int ve[4][kSubs];    // exponents of V's, or kHidden
  float top[2][2][kTileQ];  // the halves' maxima of a row (two tiles)
  uint64_t full[kTileStages], empty[kTileStages], scales[4], q_full, s_full[2], p_full, pv_done, drained, maxima[4];
  float m[kTileQ], l[2][kTileQ], b[2][kTileQ];
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

// Shared-memory operand descriptor, no swizzle, version 1.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead, uint32_t stride) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(lead >> 4) << 16) |
         (static_cast<uint64_t>(stride >> 4) << 32) | (1ull << 46);
}
// Instruction descriptor: D f32, A and B f16, M = 128; B MN-major for V.
__host__ __device__ constexpr uint32_t idesc(int n, bool mn_major) {
  return (1u << 4) | (mn_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (128u >> 4 << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(add ? 1 : 0)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(add ? 1 : 0)
      : "memory");
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
__device__ __forceinline__ void tc_loaded16(uint32_t* v) { asm volatile("" : NH_RW8(v, 0), NH_RW8(v, 8)); }
__device__ __forceinline__ void tc_loaded(uint32_t* v) {
  asm volatile("" : NH_RW8(v, 0), NH_RW8(v, 8), NH_RW8(v, 16), NH_RW8(v, 24));
}
#undef NH_R8
#undef NH_W8
#undef NH_RW8
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

// Tiles of a sequence in this form.
__device__ __forceinline__ int tiles_of(const PagedAttnArgs& p, int s, int64_t cap) {
  const int64_t n_q = static_cast<int64_t>(seq_rows(p.rows, s, cap).n) * p.group;
  return n_q > p.few ? static_cast<int>((n_q + kTileQ - 1) / kTileQ) : 0;
}

// The sequence and tile of `item`, later tiles (which see more positions)
// first; false when there are not that many.  Warp-wide.
__device__ __forceinline__ bool find_tile(const PagedAttnArgs& p, int64_t cap, int64_t item, int lane, int& seq, int& tile) {
  int64_t total = 0;
  for (int s0 = 0; s0 < p.rows.n_seq; s0 += 32) {
    int n = s0 + lane < p.rows.n_seq ? tiles_of(p, s0 + lane, cap) : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    total += n;
  }
  if (item >= total) return false;
  const int64_t want = total - 1 - item;
  int64_t base = 0;
  for (int s0 = 0; s0 < p.rows.n_seq; s0 += 32) {
    const int mine = s0 + lane < p.rows.n_seq ? tiles_of(p, s0 + lane, cap) : 0;
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    const int sum = __shfl_sync(0xffffffffu, inc, 31);
    if (want < base + sum) {
      const unsigned over = __ballot_sync(0xffffffffu, base + inc > want);
      const int l = __ffs(over) - 1;
      seq = s0 + l;
      tile = static_cast<int>(want - base) - __shfl_sync(0xffffffffu, inc - mine, l);
      return true;
    }
    base += sum;
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
  pdl_wait();
  pdl_trigger();
  const int64_t cap = static_cast<int64_t>(p.rows.max_blocks) * page;
  const int64_t item = static_cast<int64_t>(blockIdx.x) / nrank;
  const int kh = static_cast<int>(item % p.kv.n_kv);
  int s = 0, qt = 0;
  if (!find_tile(p, cap, item / p.kv.n_kv, lane, s, qt)) return;  // every CTA of the cluster alike
  const SeqRows sq = seq_rows(p.rows, s, cap);
  const int n_q = sq.n * p.group, q0 = qt * kTileQ, nq = min(kTileQ, n_q - q0);
  const int first_pos = sq.p0 + q0 / p.group, last_pos = sq.p0 + (q0 + nq - 1) / p.group;
  // Visible tiles: the sinks', then those from `lo` on; this CTA's share of them.
  const int lo = p.window > 0 ? max(0, first_pos - p.window + 1) / kTileK : 0;
  const int n_sink = p.window > 0 ? min((min(p.n_sink, last_pos + 1) + kTileK - 1) / kTileK, lo) : 0;
  const int n_all = n_sink + last_pos / kTileK + 1 - lo;
  const int j0 = static_cast<int>(static_cast<int64_t>(n_all) * rank / nrank);
  const int n = static_cast<int>(static_cast<int64_t>(n_all) * (rank + 1) / nrank) - j0;
  auto tile_pos = [&](int j) { return (j0 + j < n_sink ? j0 + j : j0 + j - n_sink + lo) * kTileK; };

  if (tid == 0) {
    for (int i = 0; i < kTileStages; ++i) {
      mbar_init(&sh.full[i], 4);
      mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&sh.scales[i], 4);
    for (int i = 0; i < 4; ++i) mbar_init(&sh.maxima[i], 2);
    mbar_init(&sh.q_full, 8);
    mbar_init(&sh.s_full[0], 1);
    mbar_init(&sh.s_full[1], 1);
    mbar_init(&sh.p_full, 8);
    mbar_init(&sh.pv_done, 1);
    mbar_init(&sh.drained, 1);
    sh.failed = 0;
    fence_barrier_init();
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&sh.tmem)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = sh.tmem;

  float row_m = -INFINITY, row_l = 0.f, row_b = 0.f;  // a softmax lane's row: maximum in use, sum, sum in units of V
  int eref = -200;                                    // O is in units of 2^(eref - kTileShift)
  bool ok = true, lost = false;

  if (warp >= 8 && warp < 12) {
    // ---------------------------------------------------------------- codes to operands
    const int w = warp - 8, r = lane & 7, c = lane >> 3;
    const int32_t* table = p.rows.page_table + static_cast<int64_t>(s) * p.rows.max_blocks;
    const uint64_t page_bytes = static_cast<uint64_t>(p.kv.n_kv) * static_cast<uint64_t>(page * HD);
    const uint64_t head_off = static_cast<uint64_t>(kh) * static_cast<uint64_t>(page * HD);
    // Pages of this warp's two 16-position parts of tile j; -1: none (past the last position), -2: out of range.
    auto ids_of = [&](int j, int (&id)[2]) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        id[b] = -1;
        if (j < n) {
          const int t = tile_pos(j) + w * 32 + b * kSub;
          if (t <= last_pos) {
            const int pg = __ldcg(table + (t >> lg));
            id[b] = pg >= 0 && pg < p.kv.n_pages ? pg : -2;
          }
        }
      }
    };
    auto load = [&](const uint8_t* codes, int j, const int (&id)[2], uint4 (&raw)[kItems]) {
      const int t0 = tile_pos(j) + w * 32;
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int it = i * 4 + c, rg = it / kItems, col = it % kItems, pg = rg < 2 ? id[0] : id[1];
        raw[i] = pg >= 0 ? __ldcg(reinterpret_cast<const uint4*>(codes + static_cast<uint64_t>(pg) * page_bytes + head_off +
                                                                 ((t0 + rg * 8 + r) & (page - 1)) * HD + col * 16))
                         : make_uint4(0u, 0u, 0u, 0u);
      }
    };
    auto put = [&](int use, const uint4 (&raw)[kItems]) {  // the use-th operand tile
      const int st = use % kTileStages;
      if (!mbar_wait(&sh.empty[st], static_cast<uint32_t>((use / kTileStages) & 1) ^ 1u)) return false;
      uint8_t* to = sh.ring[st] + (w * 32 + r) * 16;
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int it = i * 4 + c, rg = it / kItems, col = it % kItems;
        uint8_t* d = to + rg * 128 + col * 2 * kChunkBytes;
        *reinterpret_cast<uint4*>(d) =
            make_uint4(codes_lo(raw[i].x), codes_hi(raw[i].x), codes_lo(raw[i].y), codes_hi(raw[i].y));
        *reinterpret_cast<uint4*>(d + kChunkBytes) =
            make_uint4(codes_lo(raw[i].z), codes_hi(raw[i].z), codes_lo(raw[i].w), codes_hi(raw[i].w));
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.full[st]);
      return true;
    };
    int id[2], id_next[2];
    uint4 rk[kItems], rv[kItems];
    ids_of(0, id);
    if (n > 0) load(p.kv.k_codes, 0, id, rk);
    for (int j = 0; j < n && ok; ++j) {
      ids_of(j + 1, id_next);
      lost |= id[0] == -2 || id[1] == -2;
      float ks = 1.f;
      int ve = kHidden;
      const int mine = lane == 0 ? id[0] : id[1];
      if (lane < 2 && mine >= 0) {
        ks = __ldcg(p.kv.k_scales + static_cast<int64_t>(mine) * p.kv.n_kv + kh);
        ve = exponent_of(__ldcg(p.kv.v_scales + static_cast<int64_t>(mine) * p.kv.n_kv + kh));
      }
      load(p.kv.v_codes, j, id, rv);
      ok = put(2 * j, rk);
      // The scales' place was last read for tile j - 4, whose weights are in use before K of tile j finds its stage free.
      if (ok) {
        if (lane < 2) {
          sh.ks[j & 3][w * 2 + lane] = ks;
          sh.ve[j & 3][w * 2 + lane] = ve;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.scales[j & 3]);
        if (j + 1 < n) load(p.kv.k_codes, j + 1, id_next, rk);
        ok = put(2 * j + 1, rv);
      }
      id[0] = id_next[0];
      id[1] = id_next[1];
    }
  } else if (warp == 12) {
    // ---------------------------------------------------------------- products
    if (lane == 0 && n > 0) {
      const uint32_t ring = smem_u32(sh.ring[0]), qh = smem_u32(sh.q[0]), ql = smem_u32(sh.q[1]);
      constexpr uint32_t kOp = TileShared<HD>::kOperand;
      auto scores = [&](int j) {
        const int use = 2 * j, st = use % kTileStages;
        if (!mbar_wait(&sh.full[st], static_cast<uint32_t>((use / kTileStages) & 1))) return false;
        tc_after();
        const uint32_t kb = ring + st * kOp, d = tmem + kColS + (j & 1) * kTileK;
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int k = 0; k < HD / 16; ++k)
            mma_ss(d, operand((part == 0 ? qh : ql) + k * 2 * kChunkBytes, kChunkBytes, 128),
                   operand(kb + k * 2 * kChunkBytes, kChunkBytes, 128), idesc(kTileK, false), part + k > 0);
        tc_commit(&sh.empty[st]);
        tc_commit(&sh.s_full[j & 1]);
        return true;
      };
      ok = mbar_wait(&sh.q_full, 0) && scores(0);
      for (int j = 0; j < n && ok; ++j) {
        // S of tile j + 1 takes the place of tile j - 1's weights.
        if (j > 0) ok = mbar_wait(&sh.pv_done, static_cast<uint32_t>(j - 1) & 1u);
        if (ok && j + 1 < n) ok = scores(j + 1);
        const int use = 2 * j + 1, st = use % kTileStages;
        ok = ok && mbar_wait(&sh.full[st], static_cast<uint32_t>((use / kTileStages) & 1)) &&
             mbar_wait(&sh.p_full, static_cast<uint32_t>(j & 1));
        if (!ok) break;
        tc_after();
        const uint32_t vb = ring + st * kOp;
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int k = 0; k < kTileK / 16; ++k)
            mma_ts(tmem + kColO, tmem + kColS + (j & 1) * kTileK + (k >> 1) * 32 + part * 16 + (k & 1) * 8, operand(vb + k * 256, 128, kChunkBytes),
                   idesc(HD, true), j + part + k > 0);
        tc_commit(&sh.empty[st]);
        tc_commit(&sh.pv_done);
      }
      // No product is left in flight when the operands and the tensor memory are given up, whatever ended the loop.
      tc_commit(&sh.drained);
      ok = mbar_wait(&sh.drained, 0) && ok;
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax: a row a lane, half of the positions
    const int half = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const bool row_ok = row < nq;
    const int qi = q0 + (row_ok ? row : 0), pos = row_ok ? sq.p0 + qi / p.group : -1;
    const bool idle = quad * 32 >= nq;  // no row of this warp is a query
    float fq, hq;
    {
      const float4* q = reinterpret_cast<const float4*>(
          p.q + (static_cast<int64_t>(sq.r0 + qi / p.group) * p.n_head + kh * p.group + qi % p.group) * HD);
      float top = 0.f, sum = 0.f;
#pragma unroll 8
      for (int i = 0; i < HD / 4; ++i) {
        const float4 x = row_ok ? __ldcg(q + i) : make_float4(0.f, 0.f, 0.f, 0.f);
        top = fmaxf(top, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
        sum += (x.x + x.y) + (x.z + x.w);
      }
      // The largest magnitude goes to [2^13, 2^14); a negative factor of the scores changes the query's sign.
      const int e = min(max(exponent_of(top), -100), 126);
      const float up = p.scale < 0.f ? -pow2i(13 - e) : pow2i(13 - e);
#pragma unroll 4
      for (int i = half * (HD / 16); i < (half + 1) * (HD / 16); ++i) {
        const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 a = row_ok ? __ldcg(q + 2 * i) : z, b = row_ok ? __ldcg(q + 2 * i + 1) : z;
        uint4 h, l;
        split2(a.x * up, a.y * up, h.x, l.x);
        split2(a.z * up, a.w * up, h.y, l.y);
        split2(b.x * up, b.y * up, h.z, l.z);
        split2(b.z * up, b.w * up, h.w, l.w);
        *reinterpret_cast<uint4*>(sh.q[0] + i * kChunkBytes + row * 16) = h;
        *reinterpret_cast<uint4*>(sh.q[1] + i * kChunkBytes + row * 16) = l;
      }
      hq = 0.5f * up * sum;
      fq = fabsf(p.scale) * kLog2e * pow2i(e - 13);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.q_full);
    }
    for (int j = 0; j < n && ok; ++j) {
      if (idle) {
        // In step with the others: the phase before must be over.
        ok = j == 0 || mbar_wait(&sh.pv_done, static_cast<uint32_t>(j - 1) & 1u);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full);
        continue;
      }
      ok = mbar_wait(&sh.scales[j & 3], static_cast<uint32_t>(j >> 2) & 1u) &&
           mbar_wait(&sh.s_full[j & 1], static_cast<uint32_t>(j >> 1) & 1u);
      if (__any_sync(0xffffffffu, !ok)) {
        ok = false;
        break;
      }
      tc_after();
      const uint32_t scol = tmem + kColS + (j & 1) * kTileK + lanes + half * kHalf;
      uint32_t u[kHalf];
      tc_ld32(scol, u);
      tc_ld32(scol + 32, u + 32);
      const int t0 = tile_pos(j);
      // Scales: K's of this half's four parts, V's exponents of these and of the others.
      const float4 k4 = *reinterpret_cast<const float4*>(&sh.ks[j & 3][half * 4]);
      const int4 v4 = *reinterpret_cast<const int4*>(&sh.ve[j & 3][half * 4]);
      const int4 w4 = *reinterpret_cast<const int4*>(&sh.ve[j & 3][(half ^ 1) * 4]);
      const float ks[4] = {k4.x, k4.y, k4.z, k4.w};
      const int ve[4] = {v4.x, v4.y, v4.z, v4.w};
      const int low_e = min(min(min(v4.x, v4.y), min(v4.z, v4.w)), min(min(w4.x, w4.y), min(w4.z, w4.w)));
      const int ev = max(max(max(v4.x, v4.y), max(v4.z, v4.w)), max(max(w4.x, w4.y), max(w4.z, w4.w)));
      tc_wait_ld();
      tc_loaded(u);
      tc_loaded(u + 32);
      float* x = reinterpret_cast<float*>(u);
      const bool plain = low_e != kHidden && t0 + kTileK - 1 <= first_pos &&
                         (p.window == 0 || t0 > last_pos - p.window || t0 + kTileK <= p.n_sink);
      if (!plain) {
        const int h0 = t0 + half * kHalf;
        const int hi = pos - h0;                                                       // columns above it are hidden,
        const int low = p.window > 0 ? pos - p.window - h0 : -1, sk = p.n_sink - h0;  // up to `low` unless below `sk`
#pragma unroll
        for (int i = 0; i < kHalf; ++i)
          if (i > hi || (i <= low && i >= sk) || ve[i / kSub] == kHidden) x[i] = -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        float t = x[b * kSub];
#pragma unroll
        for (int i = 1; i < kSub; ++i) t = fmaxf(t, x[b * kSub + i]);
        top = fmaxf(top, (t + hq) * fmaxf(fq * ks[b], kLeast));
      }
      sh.top[j & 1][half][row] = top;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.maxima[quad]);
      ok = mbar_wait(&sh.maxima[quad], static_cast<uint32_t>(j) & 1u);
      if (__any_sync(0xffffffffu, !ok)) {
        ok = false;
        break;
      }
      top = fmaxf(top, sh.top[j & 1][half ^ 1][row]);
      // The maximum in use follows the true one only when that is 2^8 above it; O follows then, and when V's scale grows.
      const bool grow = top > (row_m == -INFINITY ? row_m : row_m + kGrow);
      if (__any_sync(0xffffffffu, grow) || ev > eref) {
        const int en = max(eref, ev);
        float alpha = 1.f;
        if (grow) {
          alpha = row_m == -INFINITY ? 0.f : exp2_fast(row_m - top);
          row_m = top;
          row_l *= alpha;
        }
        alpha *= pow2i(max(eref - en, -200));
        row_b *= alpha;
        eref = en;
        if (j > 0) {
          ok = mbar_wait(&sh.pv_done, static_cast<uint32_t>(j - 1) & 1u);
          if (__any_sync(0xffffffffu, !ok)) {
            ok = false;
            break;
          }
          tc_after();
#pragma unroll
          for (int i = half * (HD / 32); i < (half + 1) * (HD / 32); ++i) {
            uint32_t o[16];
            tc_ld16(tmem + kColO + lanes + i * 16, o);
            tc_wait_ld();
            tc_loaded16(o);
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            tc_st16(tmem + kColO + lanes + i * 16, o);
          }
        }
      }
      const float base = row_m == -INFINITY ? 0.f : row_m;
      // Weights, in pairs as high and low f16 parts: of every 32 columns the first 16 hold the high ones.
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t w[32];
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const int b = 2 * c + d, eb = ve[b] - eref + kTileShift;
          const float a = fmaxf(fq * ks[b], kLeast);
          float off = hq * a - base;
          if (eb < -60) {
            // Hidden, or a scale 2^60 below the largest: the weights count for the sum alone.
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < kSub; ++i) sum += exp2_fast(fmaf(x[b * kSub + i], a, off));
            row_l += sum;
            off = -INFINITY;
          } else {
            off += static_cast<float>(eb);
          }
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < kSub / 2; ++i) {
            const int k = b * kSub + 2 * i;
            const float w0 = exp2_fast(fmaf(x[k], a, off)), w1 = exp2_fast(fmaf(x[k + 1], a, off));
            sum += w0 + w1;
            split2(w0, w1, w[d * 8 + i], w[16 + d * 8 + i]);
          }
          row_l += sum * pow2i(min(-eb, 60));
          row_b += sum;
        }
        tc_st32(scol + c * 32, w);
      }
      tc_wait_st();
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_full);
    }
    if (n > 0 && ok) ok = mbar_wait(&sh.pv_done, static_cast<uint32_t>(n - 1) & 1u);
    sh.l[half][row] = row_l;
    sh.b[half][row] = row_b;
    tc_after();
  }
  if (!ok) sh.failed = 1;
  if (lost && lane == 0) paged_error(p.rows);
  // Every product is done (the softmax lanes waited for the last one); the operands' place holds the joined values.
  tc_before();
  __syncthreads();
  tc_after();
  float* part = reinterpret_cast<float*>(nrank > 1 ? sh.ring[0] : nullptr);  // [kTileQ][HD]
  if (warp < 8) {
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int qi = q0 + row;
    float* out = p.out + (static_cast<int64_t>(sq.r0 + qi / p.group) * p.n_head + kh * p.group + qi % p.group) * HD;
    const float l = sh.l[0][row] + sh.l[1][row], b = 0.5f * (sh.b[0][row] + sh.b[1][row]);
    const float unit = pow2i(max(eref, -126));
    const float inv = nrank > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
    if (nrank > 1 && half == 0) sh.m[row] = row_m;
#pragma unroll
    for (int i = half * (HD / 32); i < (half + 1) * (HD / 32); ++i) {
      uint32_t o[16];
      if (n > 0) {
        tc_ld16(tmem + kColO + lanes + i * 16, o);
        tc_wait_ld();
        tc_loaded16(o);
      }
      float4* to = reinterpret_cast<float4*>(nrank > 1 ? part + row * HD + i * 16 : out + i * 16);
      if (row < nq) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = n > 0 ? (__uint_as_float(o[4 * k + e]) + b) * pow2i(-kTileShift) * unit * inv : 0.f;
          to[k] = make_float4(v[0], v[1], v[2], v[3]);
        }
      }
    }
    tc_before();
  }
  if (nrank > 1) {
    cluster.sync();
    // Rows of the tile in turn over the ranks, joined in rank order.
    for (int i = rank * kTileThreads + tid; i < nq * HD / 4; i += nrank * kTileThreads) {
      const int row = i / (HD / 4), d = i % (HD / 4), qi = q0 + row;
      float top = -INFINITY, sum = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int r = 0; r < nrank; ++r) top = fmaxf(top, cluster.map_shared_rank(sh.m, r)[row]);
      for (int r = 0; r < nrank; ++r) {
        const float mr = cluster.map_shared_rank(sh.m, r)[row];
        const float a = mr == -INFINITY ? 0.f : exp2_fast(mr - top);
        const float4 y = reinterpret_cast<const float4*>(cluster.map_shared_rank(part, r))[i];
        const float* lr = cluster.map_shared_rank(&sh.l[0][0], r);
        sum += a * (lr[row] + lr[kTileQ + row]);
        v.x += a * y.x;
        v.y += a * y.y;
        v.z += a * y.z;
        v.w += a * y.w;
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      reinterpret_cast<float4*>(p.out + (static_cast<int64_t>(sq.r0 + qi / p.group) * p.n_head + kh * p.group +
                                         qi % p.group) * HD)[d] = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    }
    cluster.sync();  // no CTA leaves while another reads its part
  } else {
    __syncthreads();
  }
  if (tid == 0 && sh.failed != 0 && p.rows.err != nullptr) atomicCAS(p.rows.err, 0, NH_E_TIMEOUT);
  if (warp == 12) {
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
  if (items * ranks > INT32_MAX) return NH_E_ARG;
  return launch_cluster(paged_tile_kernel<HD>, dim3(static_cast<unsigned>(items * ranks)), dim3(kTileThreads), ranks, smem,
                        s, p);
}

}  // namespace

int launch_paged_tiles(const PagedAttnArgs& p, cudaStream_t s) {
  const int64_t most = static_cast<int64_t>(p.rows.max_rows) * p.group;
  // No more tiles than whole ones of all rows and a part of one for each sequence, nor than every sequence's most.
  const int64_t tiles = std::min(static_cast<int64_t>(p.rows.n_rows) * p.group / kTileQ + p.rows.n_seq,
                                 p.rows.n_seq * ((most + kTileQ - 1) / kTileQ));
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
