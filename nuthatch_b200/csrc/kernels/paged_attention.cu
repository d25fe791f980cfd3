// Attention over the paged 8-bit K/V cache for few rows a sequence: decode
// positions and drafted ones (nh_paged_attention's split form).
//
// A CTA takes up to 2, 4, 8 or 16 queries of one (sequence, KV head) and a
// contiguous part of the positions; a cluster's CTAs split the positions and
// join their (maximum, sum, weighted values) through distributed shared memory
// in rank order.  A warp takes units of 16 positions, always inside one page,
// through a ring of stages of its own in shared memory (cp.async, no barrier
// between warps), and reads them in the operand layout of mma.m16n8k16: both the
// dimensions of K and those of V may be permuted freely, so each lane reads
// whole 16-byte pieces.
//   2 queries: the scores by integer products (m16n8k32), K's codes as they
//   are: a query is scaled to 23-bit whole numbers, whose three balanced base-256
//   digits are columns of B; sums exact, joined in f32.  Weights as below.
//   4 queries: the codes are the A operand, the queries' (and weights') high
//   and low parts the 8 columns of B; half the products and accumulators of the
//   next form, four shuffles to bring the weights into place.
//   8 queries: rows 0-7 of the A operand are the high parts, 8-15 the low ones,
//   the codes are B; the score accumulators are the weights' operand layout.
//   16 queries: two A operands (the query's wait in shared memory), the codes'
//   conversion shared by twice the queries.
// What bounds it: every cached byte is read once, so the copy rate of HBM; with
// more queries the instructions of the codes' conversion and of the products'
// operands.  Measured (16 KV heads of 128, one query each): 64 sequences of up
// to 4,096 positions 127 us (5.4 TB/s of a copy's 6.5; the reads alone take 114,
// unequal lengths on 296 places for CTAs), one of 131,001 positions 133 us
// (4.0 TB/s: 256 CTAs on 148 SMs); 16 of up to 6,001, 8 heads of 128, 20 queries
// each 78 us, 32 queries 93.  Measured and left: CTAs in order of length (129
// us), two stages and three CTAs to an SM (156), page ids fetched in the units'
// loop.
#include <cooperative_groups.h>

#include <cmath>
#include <cstddef>

#include "paged_attention.cuh"

namespace cg = cooperative_groups;

namespace nh {

namespace {

constexpr int kUnit = 16;  // positions of one warp step
// Sequences with at most this many queries a KV head take this form, others the tiled one, whose time hardly depends on
// the queries: 16 sequences of up to 6,001 positions, 8 KV heads of 128, take 93 us here and 129 tiled with 32 queries,
// 130 and 130 with 48, 171 and 129 with 64; one of 8,000 positions and 16 KV heads 35 and 53 with 32.
constexpr int kFewQueries = 32;
// Warps of a CTA: sixteen to an SM either way by their registers, in fewer and larger CTAs for up to four queries (one
// long sequence 158 -> 135 us, the decode batch 134 -> 127 us against four warps a CTA).
template <int NQ>
constexpr int kWarpsOf = NQ <= 4 ? 8 : 4;

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_u8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// N consecutive 32-bit words of shared memory, in the widest pieces their
// alignment (4 * N bytes, at most 16) allows.
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 x = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = x.x;
      w[4 * i + 1] = x.y;
      w[4 * i + 2] = x.z;
      w[4 * i + 3] = x.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint2 x = reinterpret_cast<const uint2*>(p)[i];
      w[2 * i] = x.x;
      w[2 * i + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
  }
}

__device__ __forceinline__ void copy16(uint32_t smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(smem), "l"(gmem) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t smem, const void* gmem) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(smem), "l"(gmem) : "memory");
}

__device__ __forceinline__ void add_to(float (&o)[4], const float (&d)[4]) {
  const float2 a = add2(make_float2(o[0], o[1]), make_float2(d[0], d[1]));
  const float2 b = add2(make_float2(o[2], o[3]), make_float2(d[2], d[3]));
  o[0] = a.x;
  o[1] = a.y;
  o[2] = b.x;
  o[3] = b.y;
}

// One unit of a warp's ring.  Rows of V are padded so that the four rows that a
// quarter of a warp reads at once lie in different banks; rows of K need that
// at 128 bytes only, where odd rows swap their halves.
template <int HD>
struct SplitStage {
  uint8_t k[kUnit][HD];
  uint8_t v[kUnit][HD + 16];
  float scale[4];  // of K, of V
};
constexpr int kSplitStages = 3;

// The values that the warps and the CTAs of a cluster join ([0] holds the CTA's
// after the join); they take the rings' place once the units are done.  Within a
// query dimension a * (HD / 8) + i, which lane `a` of eight holds, lies at place
// i * 8 + a, and rows are padded by 8: no two lanes of a store share a bank.
template <int HD, int NQ>
struct SplitShared {
  static constexpr int kSplitWarps = kWarpsOf<NQ>;
  union {
    SplitStage<HD> ring[kSplitWarps][kSplitStages];
    float o[kSplitWarps][NQ][HD + 8];
  };
  float m[kSplitWarps][NQ], l[kSplitWarps][NQ];
  float cm[NQ], cl[NQ];
  uint4 qa[NQ == 16 ? HD / 16 : 1][2][32];  // A operands of the 16-query form: high, low
  uint32_t qd[NQ == 2 ? HD / 16 : 1][32];   // digits of the 2-query form
};

// Unit `i` of the visible ones: the sinks' units, then those from `lo` on.
struct Units {
  int n_sink, lo, n;
  __device__ __forceinline__ int at(int i) const { return i < n_sink ? i : i - n_sink + lo; }
};

// Up to NQ queries of the CTA's sequence and KV head, from a multiple of STEP on.
template <int HD, int NQ, int STEP>
__device__ __forceinline__ void split_queries(const PagedAttnArgs& p) {
  constexpr int kSplitWarps = kWarpsOf<NQ>, kSplitThreads = kSplitWarps * 32;
  constexpr int KS = HD / 16;                    // k-steps of the score product
  constexpr int KV = HD % 64 == 0 ? 16 : 8;      // contiguous bytes of K a lane loads at once
  constexpr int KW = KV / 4, KN = HD / (4 * KV);  // words of such a piece, pieces a row
  constexpr int VW = HD / 32;                    // words of V a lane loads a row
  constexpr int QT = NQ == 16 ? 2 : 1;           // queries a lane holds scores of
  constexpr bool kSmall = NQ <= 4;               // the codes are the A operand
  constexpr int ST = kSmall ? 2 : 4;             // scores a lane holds of each, a unit
  constexpr int ON = kSmall ? HD / 16 : HD / 8;  // accumulator tiles
  extern __shared__ __align__(16) uint8_t split_smem[];
  auto& sh = *reinterpret_cast<SplitShared<HD, NQ>*>(split_smem);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), nrank = static_cast<int>(cluster.num_blocks());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int s = blockIdx.z, kh = static_cast<int>(blockIdx.y) % p.kv.n_kv, q0 = static_cast<int>(blockIdx.y) / p.kv.n_kv * STEP;
  const int page = p.kv.page, lg = p.kv.page_log2;
  pdl_wait();
  pdl_trigger();
  const SeqRows sq = seq_rows(p.rows, s, static_cast<int64_t>(p.rows.max_blocks) * page);
  if (sq.n < 0 && blockIdx.y == 0 && rank == 0 && tid == 0) paged_error(p.rows);
  const int n_q = sq.n * p.group;  // query j: row j / group, head kh * group + j % group
  if (n_q <= q0 || n_q > p.few) return;  // every CTA of the cluster alike
  const int nq = min(NQ, n_q - q0);

  // Positions that any of these queries sees.
  const int first_pos = sq.p0 + q0 / p.group, last_pos = sq.p0 + (q0 + nq - 1) / p.group;
  Units un{0, 0, 0};
  if (p.window > 0) {
    un.lo = max(0, first_pos - p.window + 1) / kUnit;
    un.n_sink = min((min(p.n_sink, last_pos + 1) + kUnit - 1) / kUnit, un.lo);
  }
  un.n = un.n_sink + last_pos / kUnit + 1 - un.lo;
  const int u0 = static_cast<int>(static_cast<int64_t>(un.n) * rank / nrank);
  const int u1 = static_cast<int>(static_cast<int64_t>(un.n) * (rank + 1) / nrank);

  const int32_t* table = p.rows.page_table + static_cast<int64_t>(s) * p.rows.max_blocks;
  // Copies of 16 bytes: lane l takes chunks l, l + 32, ... of a unit's 16 rows, constant steps apart in both memories.
  constexpr unsigned kChunks = HD / 16;  // chunks of a row
  const unsigned c_row = static_cast<unsigned>(lane) / kChunks, c_col = static_cast<unsigned>(lane) % kChunks;
  const uint32_t page_bytes = static_cast<uint32_t>(p.kv.n_kv) * static_cast<uint32_t>(page * HD);  // below 2^30
  const uint8_t* const k_lane = p.kv.k_codes + static_cast<uint32_t>(kh * page * HD + lane * 16);
  const uint8_t* const v_lane = p.kv.v_codes + static_cast<uint32_t>(kh * page * HD + lane * 16);
  const float* const s_lane = (lane == 0 ? p.kv.k_scales : p.kv.v_scales) + kh;
  const uint32_t ring = smem_u32(&sh.ring[warp][0]);
  const uint32_t k_to = ring + static_cast<uint32_t>(offsetof(SplitStage<HD>, k)) + c_row * HD +
                        (HD == 128 ? c_col ^ ((c_row & 1u) * 4u) : c_col) * 16u;
  const uint32_t v_to = ring + static_cast<uint32_t>(offsetof(SplitStage<HD>, v)) + c_row * (HD + 16) + c_col * 16u;
  const uint32_t s_to = ring + static_cast<uint32_t>(offsetof(SplitStage<HD>, scale)) + lane * 4u;
  // Unit i into stage st.  A page out of range reads page 0 and hides its positions.
  auto fetch = [&](int i, int st, int pg) {
    const uint64_t off = static_cast<uint64_t>(static_cast<uint32_t>(pg)) * page_bytes +
                         static_cast<uint32_t>(((un.at(i) * kUnit) & (page - 1)) * HD);
    const uint32_t to = static_cast<uint32_t>(st) * static_cast<uint32_t>(sizeof(SplitStage<HD>));
#pragma unroll
    for (unsigned j = 0; j < HD / 32; ++j) {
      if constexpr (32 % kChunks == 0) {
        constexpr unsigned kRows = 32 / kChunks;  // an even number wherever odd rows swap halves
        copy16(k_to + to + j * kRows * HD, k_lane + off + j * 512);
        copy16(v_to + to + j * kRows * (HD + 16), v_lane + off + j * 512);
      } else {
        const unsigned c = static_cast<unsigned>(lane) + 32 * j, row = c / kChunks, col = c % kChunks;
        copy16(k_to + to + (row - c_row) * HD + (col - c_col) * 16, k_lane + off + j * 512);
        copy16(v_to + to + (row - c_row) * (HD + 16) + (col - c_col) * 16, v_lane + off + j * 512);
      }
    }
    if (lane < 2) copy4(s_to + to, s_lane + static_cast<uint64_t>(static_cast<uint32_t>(pg)) * static_cast<uint32_t>(p.kv.n_kv));
  };

  // The pages of this warp's units, 32 ahead of the fetches: lane l holds that of unit i0 + (f0 + l) * kSplitWarps, or
  // -1 where there is none.
  const int i0 = u0 + warp;
  auto page_ids = [&](int f0) {
    const int i = i0 + (f0 + lane) * kSplitWarps;
    int pg = -1;
    if (i < u1) {
      pg = __ldcg(table + ((un.at(i) * kUnit) >> lg));
      if (pg >= p.kv.n_pages) pg = -1;
    }
    return pg;
  };
  int ids = page_ids(0), ids_next = page_ids(32), fetched = 0;
  uint32_t here = 0u;  // bit j: the page of the j-th unit from here is known
  bool lost = false;
  auto fetch_next = [&](int i, int st, int bit) {
    if (i < u1) {
      const int pg = __shfl_sync(0xffffffffu, ids, fetched & 31);
      here |= (pg >= 0 ? 1u : 0u) << bit;
      fetch(i, st, max(pg, 0));
      if ((++fetched & 31) == 0) {
        ids = ids_next;
        ids_next = page_ids(fetched + 32);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int j = 0; j < kSplitStages - 1; ++j) fetch_next(i0 + j * kSplitWarps, j, j);

  // The query's operand: word w of lane t holds dimensions dim(w) .. dim(w)+3.
  auto dim = [&](int w) { return (w / KW) * (4 * KV) + t * KV + (w % KW) * 4; };
  uint32_t qa[NQ == 4 || NQ == 8 ? KS : 1][4], qd[NQ == 2 ? KS : 1];
  int h0 = 0, h1 = 0;            // 2 queries: 255 times the digit sums of this lane's two columns,
  float m0 = 0.f, m1 = 0.f;      // and half of what their digits stand for
  float fq[QT], nan_q = 0.f;  // nan_q: 2 queries, see below
  int pos[QT];
#pragma unroll
  for (int k = 0; k < QT; ++k) {
    const int jq = NQ == 2 ? (g >> 1) & 1 : NQ == 4 ? g >> 1 : g + 8 * k;  // the query whose operand this lane holds
    const int j = q0 + jq;
    const bool ok = jq < nq;
    const int row = sq.r0 + (ok ? j / p.group : 0), head = kh * p.group + (ok ? j % p.group : 0);
    pos[k] = ok ? sq.p0 + j / p.group : -1;
    const float* q = p.q + (static_cast<int64_t>(row) * p.n_head + head) * HD;
    float4 x[KS];
    float top = 0.f;
#pragma unroll
    for (int w = 0; w < KS; ++w) {
      x[w] = ok ? __ldcg(reinterpret_cast<const float4*>(q + dim(w))) : make_float4(0.f, 0.f, 0.f, 0.f);
      top = fmaxf(top, fmaxf(fmaxf(fabsf(x[w].x), fabsf(x[w].y)), fmaxf(fabsf(x[w].z), fabsf(x[w].w))));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = min(max(exponent_of(top), -100), 127);
    if constexpr (NQ == 2) {
      // Whole numbers of at most 2^22, column g: digit 0 or 1 of query (g / 2) % 2 for g < 4, else 2 (even) or none.  A
      // warp forms its share of the words for all of them.
      const float up = pow2i(21 - e);
      // nan_q: a NaN where the query holds a value that is not finite (which whole numbers do not show).
      const int digit = g < 4 ? g & 1 : 2;
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        nan_q += (x[w].x * 0.f + x[w].y * 0.f) + (x[w].z * 0.f + x[w].w * 0.f);
        if (w % kSplitWarps == warp) {
          const float y[4] = {x[w].x, x[w].y, x[w].z, x[w].w};
          uint32_t word = 0u;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            int v = __float2int_rn(y[i] * up);
            const int d2 = static_cast<int8_t>(v & 255);
            v = (v - d2) >> 8;
            const int d1 = static_cast<int8_t>(v & 255);
            const int d0 = (v - d1) >> 8;
            const int d = g > 3 && (g & 1) != 0 ? 0 : digit == 0 ? d0 : digit == 1 ? d1 : d2;
            word |= static_cast<uint32_t>(d & 255) << (8 * i);
          }
          sh.qd[w][lane] = word;
        }
      }
      __syncthreads();
      int sum = 0;
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        qd[w] = sh.qd[w][lane];
        sum = __dp4a(static_cast<int>(qd[w]), 0x01010101, sum);
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      nan_q += __shfl_xor_sync(0xffffffffu, nan_q, 1);
      nan_q += __shfl_xor_sync(0xffffffffu, nan_q, 2);
      // Scores: columns 2 t and 2 t + 1, query t % 2.
      h0 = 255 * __shfl_sync(0xffffffffu, sum, 8 * t);
      h1 = 255 * __shfl_sync(0xffffffffu, sum, 8 * t + 4);
      m0 = t < 2 ? 32768.f : 0.5f;
      m1 = t < 2 ? 128.f : 0.f;
      nan_q = __shfl_sync(0xffffffffu, nan_q, 8 * (t & 1));
      fq[k] = __shfl_sync(0xffffffffu, p.scale * kLog2e * pow2i(e - 21), 8 * (t & 1));
      pos[k] = __shfl_sync(0xffffffffu, pos[k], 8 * (t & 1));
      continue;
    }
    // The largest magnitude goes to [2^13, 2^14).
    const float up = pow2i(13 - e);
#pragma unroll
    for (int w = 0; w < KS; ++w) {
      uint32_t h0, l0, h1, l1;
      split2(x[w].x * up, x[w].y * up, h0, l0);
      split2(x[w].z * up, x[w].w * up, h1, l1);
      if constexpr (NQ == 4) {
        qa[w][0] = g & 1 ? l0 : h0;
        qa[w][1] = g & 1 ? l1 : h1;
      } else if constexpr (NQ == 8) {
        qa[w][0] = h0;
        qa[w][1] = l0;
        qa[w][2] = h1;
        qa[w][3] = l1;
      } else if (w % kSplitWarps == warp) {  // the warps share the words
        uint32_t* hi = reinterpret_cast<uint32_t*>(&sh.qa[w][0][lane]);
        uint32_t* lo = reinterpret_cast<uint32_t*>(&sh.qa[w][1][lane]);
        hi[k] = h0;
        hi[2 + k] = h1;
        lo[k] = l0;
        lo[2 + k] = l1;
      }
    }
    fq[k] = p.scale * kLog2e * pow2i(e - 13 + kCodeShift);
    if constexpr (NQ == 4) {  // scores: query t, whose operand lanes 8 t hold
      fq[k] = __shfl_sync(0xffffffffu, fq[k], 8 * t);
      pos[k] = __shfl_sync(0xffffffffu, pos[k], 8 * t);
    }
  }
  if constexpr (NQ == 16) __syncthreads();

  float o[ON][4];
#pragma unroll
  for (int i = 0; i < ON; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[QT], l[QT];  // running maximum; sum of the weights
  int eref[QT];  // a query's sums are in units of 2^(eref - kWeightShift + kCodeShift), of the scales that it sees
#pragma unroll
  for (int k = 0; k < QT; ++k) {
    m[k] = -INFINITY;
    l[k] = 0.f;
    eref[k] = -200;
  }

  int st = 0;
  for (int i = i0; i < u1; i += kSplitWarps) {
    const int t0 = un.at(i) * kUnit;
    cp_async_wait<kSplitStages - 2>();
    __syncwarp();  // every lane's copies of this unit have landed; the stage of the unit before it is free
    fetch_next(i + (kSplitStages - 1) * kSplitWarps, st == 0 ? kSplitStages - 1 : st - 1, kSplitStages - 1);
    const SplitStage<HD>& un_st = sh.ring[warp][st];
    st = st + 1 == kSplitStages ? 0 : st + 1;
    const bool seen_here = (here & 1u) != 0u;
    here >>= 1;
    lost |= !seen_here;
    const float k_scale = un_st.scale[0], v_scale = un_st.scale[1];
    uint32_t kw[2][KS], vw[4][VW];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int c = 0; c < KN; ++c)
        load_words<KW>(&un_st.k[8 * j + g][(HD == 128 ? c ^ (g & 1) : c) * 4 * KV + t * KV], &kw[j][c * KW]);
    float c[2][4];  // two chains of products: of even and odd k-steps (4 queries), of positions 0-7 and 8-15 (others)
#pragma unroll
    for (int j = 0; j < 2; ++j) c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.f;
    if constexpr (NQ == 2) {
      int ci[4] = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < KS; w += 2) mma_u8s8(ci, kw[0][w], kw[1][w], kw[0][w + 1], kw[1][w + 1], qd[w], qd[w + 1]);
      // Twice the digits' products with the codes' own values (u - 127.5), whole and exact; then the digits' weights.
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float part = fmaf(static_cast<float>(2 * ci[2 * e] - h0), m0, static_cast<float>(2 * ci[2 * e + 1] - h1) * m1);
        c[0][e] = part + __shfl_xor_sync(0xffffffffu, part, 2);
      }
    }
#pragma unroll
    for (int w = 0; w < (NQ == 2 ? 0 : KS); ++w) {
      const uint32_t a0 = codes_lo(kw[0][w]), a1 = codes_hi(kw[0][w]), b0 = codes_lo(kw[1][w]), b1 = codes_hi(kw[1][w]);
      if constexpr (NQ == 4) {
        mma_f16(c[w & 1], a0, b0, a1, b1, qa[w][0], qa[w][1]);
      } else if constexpr (NQ == 8) {
        mma_f16(c[0], qa[w][0], qa[w][1], qa[w][2], qa[w][3], a0, a1);
        mma_f16(c[1], qa[w][0], qa[w][1], qa[w][2], qa[w][3], b0, b1);
      } else {
        const uint4 hi = sh.qa[w][0][lane], lo = sh.qa[w][1][lane];
        mma_f16(c[0], hi.x, hi.y, hi.z, hi.w, a0, a1);
        mma_f16(c[1], hi.x, hi.y, hi.z, hi.w, b0, b1);
        mma_f16(c[0], lo.x, lo.y, lo.z, lo.w, a0, a1);
        mma_f16(c[1], lo.x, lo.y, lo.z, lo.w, b0, b1);
      }
    }
    // Scores of this lane's queries: at positions t0 + g, t0 + g + 8 (4 queries), t0 + 8 j + 2 t + e (others).
    const bool plain = seen_here && t0 + kUnit - 1 <= first_pos &&
                       (p.window == 0 || t0 > last_pos - p.window || t0 + kUnit <= p.n_sink);  // all of them see all
    float x[QT][ST], top[QT];
    int ev[QT];  // the exponent of V's scale where the query sees any of the unit
    bool grew = false;
#pragma unroll
    for (int k = 0; k < QT; ++k) {
      const float f = fq[k] * k_scale;
#pragma unroll
      for (int e = 0; e < ST; ++e) {
        const float d = NQ == 2   ? c[0][e]
                        : NQ == 4 ? (c[0][2 * e] + c[1][2 * e]) + (c[0][2 * e + 1] + c[1][2 * e + 1])
                        : NQ == 8 ? c[e >> 1][e & 1] + c[e >> 1][(e & 1) + 2]
                                  : c[e >> 1][2 * k + (e & 1)];
        x[k][e] = (NQ == 2 ? d + nan_q : d) * f;
      }
      ev[k] = exponent_of(v_scale);
      if (!plain) {
        if (!seen_here || t0 > pos[k] || (p.window != 0 && t0 + kUnit - 1 <= pos[k] - p.window && t0 >= p.n_sink))
          ev[k] = eref[k];
#pragma unroll
        for (int e = 0; e < ST; ++e) {
          const int tk = t0 + (kSmall ? g + 8 * e : 8 * (e >> 1) + 2 * t + (e & 1));
          if (!seen_here || tk > pos[k] || (p.window != 0 && tk <= pos[k] - p.window && tk >= p.n_sink))
            x[k][e] = -INFINITY;
        }
      }
      top[k] = m[k];
#pragma unroll
      for (int e = 0; e < ST; ++e) top[k] = fmaxf(top[k], x[k][e]);
#pragma unroll
      for (int e = kSmall ? 4 : 1; e <= (kSmall ? 16 : 2); e <<= 1)
        top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], e));
      grew |= top[k] > m[k] || ev[k] > eref[k];
    }
    // Rarely after the first units: a larger score, or a larger scale of V.
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int k = 0; k < QT; ++k) {
        const int en = max(eref[k], ev[k]);
        const float fe = pow2i(max(eref[k] - en, -200));
        eref[k] = en;
        const float a = m[k] == -INFINITY ? 0.f : exp2_fast(m[k] - top[k]);
        m[k] = top[k];
        l[k] *= a;
#pragma unroll
        for (int n = 0; n < ON; ++n) {
          if constexpr (NQ <= 8) {
            o[n][0] *= a * fe;
            o[n][1] *= a * fe;
            o[n][2] *= a * fe;
            o[n][3] *= a * fe;
          } else {
            o[n][2 * k] *= a * fe;
            o[n][2 * k + 1] *= a * fe;
          }
        }
      }
    }
    uint32_t hi[QT][2], lo[QT][2];
#pragma unroll
    for (int k = 0; k < QT; ++k) {
      const float base = m[k] == -INFINITY ? 0.f : m[k], fw = pow2i(ev[k] - eref[k] + kWeightShift);
      float w[4];
#pragma unroll
      for (int e = 0; e < ST; ++e) {
        w[e] = exp2_fast(x[k][e] - base);
        l[k] += w[e];
        w[e] *= fw;
      }
      if constexpr (kSmall) {
        // Column g of B: query g / 2's weights at positions 2 t, 2 t + 1 and 8 further, from the lanes that hold them.
        const int from = 8 * t + (g >> 1);
        const float w0 = __shfl_sync(0xffffffffu, w[0], from), w1 = __shfl_sync(0xffffffffu, w[0], from + 4);
        const float w2 = __shfl_sync(0xffffffffu, w[1], from), w3 = __shfl_sync(0xffffffffu, w[1], from + 4);
        const bool used = NQ == 4 || g < 4;
        w[0] = used ? w0 : 0.f;
        w[1] = used ? w1 : 0.f;
        w[2] = used ? w2 : 0.f;
        w[3] = used ? w3 : 0.f;
      }
      split2(w[0], w[1], hi[k][0], lo[k][0]);
      split2(w[2], w[3], hi[k][1], lo[k][1]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) load_words<VW>(&un_st.v[2 * t + (j & 1) + (j >> 1) * 8][g * VW * 4], vw[j]);
    const uint32_t b0 = g & 1 ? lo[0][0] : hi[0][0], b1 = g & 1 ? lo[0][1] : hi[0][1];  // 4 queries
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      // Positions 2 t, 2 t + 1 (a) and 8 further (b) side by side, for dimensions 0, 1 and 2, 3 of the word.
      const uint32_t a01 = __byte_perm(vw[0][w], vw[1][w], 0x5140), a23 = __byte_perm(vw[0][w], vw[1][w], 0x7362);
      const uint32_t b01 = __byte_perm(vw[2][w], vw[3][w], 0x5140), b23 = __byte_perm(vw[2][w], vw[3][w], 0x7362);
      const uint32_t va[4] = {codes_lo(a01), codes_hi(a01), codes_lo(a23), codes_hi(a23)};
      const uint32_t vb[4] = {codes_lo(b01), codes_hi(b01), codes_lo(b23), codes_hi(b23)};
      // A unit's products start from zero and join the sums by rounded additions: the tensor cores' own additions cut
      // off, which over thousands of units would pull every sum towards zero.
      if constexpr (kSmall) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          mma_f16(d, va[2 * e], va[2 * e + 1], vb[2 * e], vb[2 * e + 1], b0, b1);
          add_to(o[2 * w + e], d);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          if constexpr (NQ == 8) {
            mma_f16(d, hi[0][0], lo[0][0], hi[0][1], lo[0][1], va[e], vb[e]);
          } else {
            mma_f16(d, hi[0][0], hi[1][0], hi[0][1], hi[1][1], va[e], vb[e]);
            mma_f16(d, lo[0][0], lo[1][0], lo[0][1], lo[1][1], va[e], vb[e]);
          }
          add_to(o[4 * w + e], d);
        }
      }
    }
  }
  if (lost && lane == 0) paged_error(p.rows);

  // This warp's values in their own units, then the CTA's and the cluster's.
  cp_async_wait<0>();
  __syncthreads();
#pragma unroll
  for (int k = 0; k < QT; ++k) {
    const float unit = pow2i(max(eref[k], -126));
#pragma unroll
    for (int e = kSmall ? 4 : 1; e <= (kSmall ? 16 : 2); e <<= 1) {
      l[k] += __shfl_xor_sync(0xffffffffu, l[k], e);
    }
    const int qk = kSmall ? t : g + 8 * k;
    if (kSmall && t >= NQ) continue;  // columns without a query
    if (kSmall ? g == 0 : t == 0) {
      sh.m[warp][qk] = m[k];
      sh.l[warp][qk] = l[k];
    }
#pragma unroll
    for (int n = 0; n < ON; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float v = kSmall ? o[n][2 * e] + o[n][2 * e + 1] : NQ == 8 ? o[n][e] + o[n][e + 2] : o[n][2 * k + e];
        sh.o[warp][qk][kSmall ? (2 * n + e) * 8 + g : n * 8 + 2 * t + e] = v * pow2i(kCodeShift - kWeightShift - kRoom) * unit;
      }
  }
  __syncthreads();
  for (int j = tid; j < NQ; j += kSplitThreads) {
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < kSplitWarps; ++w) top = fmaxf(top, sh.m[w][j]);
    for (int w = 0; w < kSplitWarps; ++w) {
      const float a = sh.m[w][j] == -INFINITY ? 0.f : exp2_fast(sh.m[w][j] - top);
      sh.m[w][j] = a;  // from here on the warp's factor
      sum += a * sh.l[w][j];
    }
    sh.cm[j] = top;
    sh.cl[j] = sum;
  }
  __syncthreads();
  for (int j = tid; j < nq * HD; j += kSplitThreads) {
    const int q = j / HD, d = j % HD;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) v += sh.m[w][q] * sh.o[w][q][d];
    sh.o[0][q][d] = v;
  }
  if (nrank > 1)
    cluster.sync();
  else
    __syncthreads();
  const int per = (nq * HD + nrank - 1) / nrank;
  for (int j = rank * per + tid; j < min((rank + 1) * per, nq * HD); j += kSplitThreads) {
    const int q = j / HD, d = j % HD, qi = q0 + q, place = d % (HD / 8) * 8 + d / (HD / 8);
    float top = -INFINITY, sum = 0.f, v = 0.f;
    for (int r = 0; r < nrank; ++r) top = fmaxf(top, cluster.map_shared_rank(sh.cm, r)[q]);
    for (int r = 0; r < nrank; ++r) {
      const float mr = cluster.map_shared_rank(sh.cm, r)[q];
      const float a = mr == -INFINITY ? 0.f : exp2_fast(mr - top);
      sum += a * cluster.map_shared_rank(sh.cl, r)[q];
      v += a * cluster.map_shared_rank(&sh.o[0][q][0], r)[place];
    }
    const int row = sq.r0 + qi / p.group, head = kh * p.group + qi % p.group;
    p.out[(static_cast<int64_t>(row) * p.n_head + head) * HD + d] = sum == 0.f ? 0.f : v / sum * pow2i(kRoom);
  }
  if (nrank > 1) cluster.sync();  // no CTA leaves while another reads its part
}

template <int HD, int NQ>
__global__ void __launch_bounds__(kWarpsOf<NQ> * 32, NQ >= 8 ? 3 : 2) paged_split_kernel(const PagedAttnArgs p) {
  if constexpr (NQ == 16) {
    // The rest of a sequence's queries, or a sequence with few in a batch of others: half the products (20 queries of 16
    // sequences 83 -> 78 us).
    static_assert(kWarpsOf<8> == kWarpsOf<16> && sizeof(SplitShared<HD, 8>) <= sizeof(SplitShared<HD, 16>));
    pdl_wait();
    const int64_t rows = p.rows.row_off[blockIdx.z + 1] - static_cast<int64_t>(p.rows.row_off[blockIdx.z]);
    if (rows * p.group - static_cast<int>(blockIdx.y) / p.kv.n_kv * NQ <= 8) return split_queries<HD, 8, NQ>(p);
  }
  split_queries<HD, NQ, NQ>(p);
}

template <int HD, int NQ>
int launch_split(const PagedAttnArgs& p, int groups, int ranks, cudaStream_t s) {
  static SmemLimit configured;
  static WideCluster wide;
  constexpr size_t kSmem = sizeof(SplitShared<HD, NQ>), kApart = NQ == 16 && kSmem < 76 * 1024 ? 76 * 1024 : kSmem;
  if (!ensure_smem(paged_split_kernel<HD, NQ>, kApart, configured)) return NH_E_CUDA;
  if (ranks > 8 && !ensure_wide_cluster(paged_split_kernel<HD, NQ>, dim3(kWarpsOf<NQ> * 32), kApart, wide)) ranks = 8;
  // Few CTAs are spread out: two to an SM where that holds them all (32 queries over 8,000 positions, 16 heads: 35 us,
  // with three to an SM 41).
  const bool apart = static_cast<int64_t>(ranks) * p.kv.n_kv * groups * p.rows.n_seq <= 2 * device_sm_count();
  const size_t smem = apart ? kApart : kSmem;
  return launch_cluster(paged_split_kernel<HD, NQ>, dim3(ranks, p.kv.n_kv * groups, p.rows.n_seq),
                        dim3(kWarpsOf<NQ> * 32), ranks, smem, s, p);
}

// CTAs of a (sequence, KV head, query group): one, unless the groups alone leave less than eight warps to an SM, or, with
// the 16-query form, twelve (three CTAs of 168 registers; a last group of eight queries or fewer counts half, as it has
// half of the work, or none where the sequence is shorter).  16 sequences and 8 KV heads, 32 queries each: 93 us with 2
// CTAs a group, 105 with 4, 114 with 4 and two CTAs to an SM; 20 queries: 88 with 2, 78 with 4.  More
// are not free (each forms the query's operand and joins what it has), so a warp keeps a unit, and a cluster
// larger than the portable eight, which is slow to start, has more: one sequence's 8,000 positions of 16 heads take
// 17.6 us with 8 CTAs a head and 22.6 with 16, 131,001 positions 150 and 133.  The length is taken to be the page
// table's width, the only one that the host knows.
template <int HD, int NQ>
int launch_group(const PagedAttnArgs& p, int most, cudaStream_t s) {
  const int groups = (most + NQ - 1) / NQ, halves = 2 * groups - (NQ == 16 && most - (groups - 1) * NQ <= 8 ? 1 : 0);
  if (static_cast<int64_t>(p.kv.n_kv) * groups > 65535) return NH_E_ARG;
  constexpr int kWarps = kWarpsOf<NQ>, kFill = NQ == 16 ? 12 : 8;
  const int64_t items = static_cast<int64_t>(p.rows.n_seq) * p.kv.n_kv * halves;  // in halves
  const int64_t units = static_cast<int64_t>(p.rows.max_blocks) * p.kv.page / kUnit;
  int ranks = 1;
  while (ranks < 16 && items * ranks * kWarps < 2 * kFill * device_sm_count() &&
         units >= (ranks < 8 ? 1 : 16) * kWarps * 2 * ranks)
    ranks *= 2;
  return launch_split<HD, NQ>(p, groups, ranks, s);
}

template <int HD>
int launch_split_hd(const PagedAttnArgs& p, cudaStream_t s) {
  const int most = static_cast<int>(std::min<int64_t>(p.few, static_cast<int64_t>(p.rows.max_rows) * p.group));
  return most <= 2   ? launch_group<HD, 2>(p, most, s)
         : most <= 4 ? launch_group<HD, 4>(p, most, s)
         : most <= 8 ? launch_group<HD, 8>(p, most, s)
                     : launch_group<HD, 16>(p, most, s);
}

}  // namespace

int launch_paged_split(const PagedAttnArgs& p, cudaStream_t s) {
  switch (p.kv.hd) {
    case 32:
      return launch_split_hd<32>(p, s);
    case 64:
      return launch_split_hd<64>(p, s);
    case 96:
      return launch_split_hd<96>(p, s);
    default:
      return launch_split_hd<128>(p, s);
  }
}

}  // namespace nh

using namespace nh;

extern "C" int nh_paged_attention(const NhPagedKv* kv, const NhPagedRows* rows, const float* qr, int n_head,
                                  float kq_scale, int window, int n_sink, float* out, void* stream) {
  PagedAttnArgs p;
  const int rc = paged_args(kv, rows, p.kv, p.rows);
  if (rc != NH_OK) return rc;
  if (qr == nullptr || out == nullptr || !paged_aligned(qr) || !paged_aligned(out) || n_head <= 0 || n_head > 65535 ||
      n_head % p.kv.n_kv != 0 || window < 0 || n_sink < 0 || !std::isfinite(kq_scale) ||
      static_cast<int64_t>(p.rows.max_rows) * (n_head / p.kv.n_kv) > INT32_MAX)  // queries are counted in 32 bits
    return NH_E_ARG;
  if (p.rows.max_rows == 0) return NH_OK;
  p.q = qr;
  p.out = out;
  p.n_head = n_head;
  p.group = n_head / p.kv.n_kv;
  p.window = window;
  p.n_sink = n_sink;
  p.scale = kq_scale;
  p.few = INT32_MAX;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (static_cast<int64_t>(p.rows.max_rows) * p.group <= kFewQueries) return launch_paged_split(p, st);
  if (paged_tiles(p) * p.kv.n_kv > INT32_MAX) return NH_E_ARG;
  if (p.rows.n_seq == 1) {
    p.few = 0;
    return launch_paged_tiles(p, st);
  }
  // Sequences of either kind may be in the call: each form passes over the other's.
  p.few = kFewQueries;
  const int split_rc = launch_paged_split(p, st);
  return split_rc != NH_OK ? split_rc : launch_paged_tiles(p, st);
}
