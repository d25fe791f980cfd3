// The paged 8-bit K/V cache: rows into it (nh_paged_append) and values out of
// it (nh_paged_read).
//
// Append.  K and V of a row are coded with their page's scale, which needs the
// largest magnitude over the page's rows, and K is known only after the
// RMSNorm over the row's full width.  So a cluster owns one page of one
// sequence and its CTAs share the heads: each sums the squares of its heads'
// columns for every row of the page and writes the sums to all CTAs (distributed
// shared memory); from there each works on whole (page, head) pairs alone: a
// few warps a head, four rows of K and V a warp held in registers from the load
// (issued before the norm's barrier) to the codes.  q's arithmetic is
// nh_prefill_qk's, but for the order in which the 64-bit sum of squares is added
// up (by heads over the CTAs); K's norm and rotation are in 64 bits, rounded to
// f32 once, so that a value next to a code's border falls on the side where it belongs.
//
// What bounds it: one row a sequence, the chain of dependent loads and the
// cluster's barrier (one sequence 6.6 us on the GPU, 64 sequences 7.7, each among
// others in a graph); prompts (16 of up to 600 rows, 16 heads of 128: 95 us where
// the bytes take 37), not HBM nor the issue slots, which are 36% busy with 47% of
// the warps' places taken (counters): the loads before that barrier and what
// follows it lie one after the other.  q and K are read a second time, out of L2,
// after the norm is known.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <cstring>

#include "common.cuh"
#include "paged.cuh"

namespace cg = cooperative_groups;

namespace nh {

namespace {

constexpr int kMaxRanks = 8;

struct AppendArgs {
  PagedKv kv;
  PagedRows rows;
  const float* q;
  const float* k;
  const float* v;
  int64_t q_stride, k_stride, v_stride;
  const float* q_norm;
  const float* k_norm;
  float eps;
  int n_head, rope_len, kv_per, q_per;  // heads of a CTA
  const float* rope_cs;
  float* qr;
};

// The scale of a page's head whose largest finite magnitude has these bits, as
// a biased exponent: 2^(E-6), at least 2^-106.
__device__ __forceinline__ int scale_exponent(uint32_t amax_bits) {
  return max(static_cast<int>(amax_bits >> 23), 27) - 6;
}
__device__ __forceinline__ float exponent_float(int biased) { return __int_as_float(biased << 23); }

// floor(x * inv) + 128 in the low byte, for a finite x within the scale: the
// sum with 1.5 * 2^23, rounded down, holds the floor in its low bits.  (The
// product is exact, or below the subnormals and rounded down too: a negative
// x has floor -1 however small it is.)
__device__ __forceinline__ uint32_t code_bits(float x, float inv) {
  return __float_as_uint(__fadd_rd(__fmul_rd(x, inv), 12582912.f + 128.f));
}
// The same for any x: the nearest end of the range, a NaN as its middle.
__device__ __forceinline__ uint32_t code_of(float x, float inv) {
  return static_cast<uint32_t>(min(max(__float2int_rd(__fmul_rd(x, inv)), -128), 127) + 128);
}

// Warps a head, rows a warp and threads for a page size.
template <int PAGE>
struct AppendShape {
  static constexpr int kRows = 4, kHeadWarps = PAGE / kRows;
  static constexpr int kThreads = PAGE == 16 ? 256 : PAGE == 128 ? 1024 : 512;
  static constexpr int kWarps = kThreads / 32, kHeads = kWarps / kHeadWarps;
};

template <int PAGE>
struct AppendShared {
  double sums[kMaxRanks][PAGE][2];              // every CTA's sums of squares of each row's q, k
  double sck[PAGE];                             // each row's RMSNorm factor of k, of q
  float scq[PAGE];
  uint32_t top[2][AppendShape<PAGE>::kHeads][2];  // bits of the largest magnitude of a head's K, V (two rounds)
};

// The sum of squares of n4 four-column pieces, as f32 products added in 64 bits; this lane's share.
__device__ __forceinline__ double squares(const float* x, int n4, int lane) {
  double s = 0.0;
#pragma unroll 4
  for (int i = lane; i < n4; i += 32) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(x) + i);
    s += (static_cast<double>(__fmul_rn(v.x, v.x)) + static_cast<double>(__fmul_rn(v.y, v.y))) +
         (static_cast<double>(__fmul_rn(v.z, v.z)) + static_cast<double>(__fmul_rn(v.w, v.w)));
  }
  return s;
}

// The same with the products in 64 bits.
__device__ __forceinline__ double squares64(const float* x, int n4, int lane) {
  double s = 0.0;
#pragma unroll 4
  for (int i = lane; i < n4; i += 32) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(x) + i);
    const double a = v.x, b = v.y, c = v.z, d = v.w;
    s = fma(a, a, s);
    s = fma(b, b, s);
    s = fma(c, c, s);
    s = fma(d, d, s);
  }
  return s;
}

// The columns i .. i+N-1 of both halves of a head's row that a lane holds.
template <int N>
struct Pair {
  float lo[N], hi[N];
};
template <int N>
__device__ __forceinline__ Pair<N> load_pair(const float* x, int i, int half) {
  Pair<N> r;
  if constexpr (N == 2) {
    const float2 a = __ldg(reinterpret_cast<const float2*>(x + i)), b = __ldg(reinterpret_cast<const float2*>(x + i + half));
    r.lo[0] = a.x;
    r.lo[1] = a.y;
    r.hi[0] = b.x;
    r.hi[1] = b.y;
  } else {
    r.lo[0] = __ldg(x + i);
    r.hi[0] = __ldg(x + i + half);
  }
  return r;
}

// Norm (factor sc, weights w, when norm) and rotation by cs[i].
template <int N>
__device__ __forceinline__ void turn(Pair<N>& x, bool norm, float sc, const Pair<N>& w, const float (&cs)[2 * N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    float x0 = x.lo[e], x1 = x.hi[e];
    if (norm) {
      x0 = __fmul_rn(__fmul_rn(x0, sc), w.lo[e]);
      x1 = __fmul_rn(__fmul_rn(x1, sc), w.hi[e]);
    }
    x.lo[e] = __fsub_rn(__fmul_rn(x0, cs[2 * e]), __fmul_rn(x1, cs[2 * e + 1]));
    x.hi[e] = __fadd_rn(__fmul_rn(x0, cs[2 * e + 1]), __fmul_rn(x1, cs[2 * e]));
  }
}
// The same in 64 bits, rounded once.
template <int N>
__device__ __forceinline__ void turn64(Pair<N>& x, bool norm, double sc, const Pair<N>& w, const float (&cs)[2 * N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    double x0 = x.lo[e], x1 = x.hi[e];
    if (norm) {
      x0 *= sc * static_cast<double>(w.lo[e]);
      x1 *= sc * static_cast<double>(w.hi[e]);
    }
    const double c = cs[2 * e], s = cs[2 * e + 1];
    x.lo[e] = static_cast<float>(fma(x0, c, -(x1 * s)));
    x.hi[e] = static_cast<float>(fma(x0, s, x1 * c));
  }
}
template <int N>
__device__ __forceinline__ void load_cs(const float* cs, int i, float (&o)[2 * N]) {
  if constexpr (N == 2) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(cs + 2 * i));
    o[0] = v.x;
    o[1] = v.y;
    o[2] = v.z;
    o[3] = v.w;
  } else {
    const float2 v = __ldg(reinterpret_cast<const float2*>(cs + 2 * i));
    o[0] = v.x;
    o[1] = v.y;
  }
}
template <int N, bool kOdd>
__device__ __forceinline__ void store_codes(uint8_t* to, const float (&x)[N], float inv) {
  uint32_t c[N];
#pragma unroll
  for (int e = 0; e < N; ++e) c[e] = kOdd ? code_of(x[e], inv) : code_bits(x[e], inv);
  if constexpr (N == 2)
    *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(__byte_perm(c[0], c[1], 0x40));
  else
    *to = static_cast<uint8_t>(c[0]);
}

// Twice the largest magnitude's bits; 0xFF000000 and above: not finite.
template <int N>
__device__ __forceinline__ uint32_t top_of(const Pair<N>& x, uint32_t m) {
#pragma unroll
  for (int e = 0; e < N; ++e) m = max(m, max(__float_as_uint(x.lo[e]) << 1, __float_as_uint(x.hi[e]) << 1));
  return m;
}
template <int N>
__device__ __forceinline__ uint32_t finite_top_of(const Pair<N>& x, uint32_t m) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const uint32_t a = __float_as_uint(x.lo[e]) << 1, b = __float_as_uint(x.hi[e]) << 1;
    m = max(m, max(a < 0xFF000000u ? a : 0u, b < 0xFF000000u ? b : 0u));
  }
  return m;
}

template <int HD, int PAGE>
__global__ void __launch_bounds__(AppendShape<PAGE>::kThreads, 1024 / AppendShape<PAGE>::kThreads) paged_append_kernel(const AppendArgs p) {
  using S = AppendShape<PAGE>;
  constexpr int N = HD % 96 == 0 || HD == 128 ? 2 : 1, half = HD / 2, kLanes = half / N;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), nrank = static_cast<int>(cluster.num_blocks());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int s = blockIdx.z;
  __shared__ AppendShared<PAGE> sh;
  pdl_wait();
  pdl_trigger();
  const int64_t cap = static_cast<int64_t>(p.rows.max_blocks) * PAGE;
  const SeqRows sq = seq_rows(p.rows, s, min(cap, static_cast<int64_t>(p.rope_len)));
  if (sq.n < 0 && blockIdx.y == 0 && rank == 0 && tid == 0) paged_error(p.rows);
  if (sq.n <= 0) return;
  const int b = sq.p0 / PAGE + static_cast<int>(blockIdx.y);
  const int t0 = max(sq.p0, b * PAGE), t1 = min(sq.p0 + sq.n, (b + 1) * PAGE);
  if (t0 >= t1) return;  // every CTA of the cluster alike
  const int nt = t1 - t0, row0 = sq.r0 + (t0 - sq.p0);
  const float* const q0 = p.q + row0 * p.q_stride;  // this page's rows: 32-bit offsets from here
  const float* const k0 = p.k + row0 * p.k_stride;
  const float* const v0 = p.v + row0 * p.v_stride;
  const float* const cs0 = p.rope_cs + static_cast<int64_t>(t0) * HD;
  const int qs = static_cast<int>(p.q_stride), ks = static_cast<int>(p.k_stride), vs = static_cast<int>(p.v_stride);
  const int pg = p.rows.page_table[static_cast<int64_t>(s) * p.rows.max_blocks + b];
  const bool page_ok = pg >= 0 && pg < p.kv.n_pages;
  if (!page_ok && rank == 0 && tid == 0) paged_error(p.rows);

  // This CTA's heads.
  const int kv_per = p.kv_per, q_per = p.q_per;
  const int kh0 = min(rank * kv_per, p.kv.n_kv), kh1 = min(kh0 + kv_per, p.kv.n_kv);
  const int qh0 = min(rank * q_per, p.n_head), qh1 = min(qh0 + q_per, p.n_head);
  const bool has_q = p.q != nullptr, norm = p.k_norm != nullptr;
  const int dq = p.n_head * HD, dkv = p.kv.n_kv * HD;
  if (tid < 2 * S::kHeads * 2) (&sh.top[0][0][0])[tid] = 0u;
  const int i = lane * N;
  const bool on = lane < kLanes;
  const int hw = warp / S::kHeadWarps, w0 = warp % S::kHeadWarps;
  // This warp's rows of a head: rows w0, w0 + kHeadWarps, ... of the page's new ones.
  Pair<N> k[S::kRows], v[S::kRows];
  auto load_rows = [&](int h) {
    if (h < kh1 && on) {
#pragma unroll
      for (int r = 0; r < S::kRows; ++r) {
        const int t = w0 + r * S::kHeadWarps;
        if (t < nt) {
          k[r] = load_pair<N>(k0 + t * ks + h * HD, i, half);
          v[r] = load_pair<N>(v0 + t * vs + h * HD, i, half);
        }
      }
    }
  };
  load_rows(kh0 + hw);

  if (norm) {
    cluster.barrier_arrive();  // the others must have started before their shared memory is written
    bool started = false;
    for (int t = warp; t < nt; t += S::kWarps) {
      double a = has_q ? squares(q0 + t * qs + qh0 * HD, (qh1 - qh0) * (HD / 4), lane) : 0.0;
      double c = squares64(k0 + t * ks + kh0 * HD, (kh1 - kh0) * (HD / 4), lane);
      a = warp_sum_d(a);
      c = warp_sum_d(c);
      if (!started) {
        cluster.barrier_wait();
        started = true;
      }
      if (lane < nrank) {
        double* to = cluster.map_shared_rank(&sh.sums[0][0][0], lane) + (rank * PAGE + t) * 2;
        to[0] = a;
        to[1] = c;
      }
    }
    if (!started) cluster.barrier_wait();
    cluster.sync();
    for (int t = tid; t < nt; t += S::kThreads) {
      double a = 0.0, c = 0.0;
      for (int r = 0; r < nrank; ++r) {
        a += sh.sums[r][t][0];
        c += sh.sums[r][t][1];
      }
      sh.scq[t] = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(static_cast<float>(div_count(a, dq)), p.eps)));
      sh.sck[t] = 1.0 / sqrt(c / dkv + static_cast<double>(p.eps));
    }
  }
  __syncthreads();

  if (has_q && on) {
    float* const o0 = p.qr + static_cast<int64_t>(row0) * dq;
#pragma unroll 1
    for (int t = w0; t < nt; t += S::kHeadWarps) {
      float cs[2 * N];
      load_cs<N>(cs0 + t * HD, i, cs);
      const float sc = norm ? sh.scq[t] : 1.f;
#pragma unroll 4
      for (int h = qh0 + hw; h < qh1; h += S::kHeads) {
        Pair<N> x = load_pair<N>(q0 + t * qs + h * HD, i, half), w = x;
        if (norm) w = load_pair<N>(p.q_norm + h * HD, i, half);
        turn<N>(x, norm, sc, w, cs);
        float* o = o0 + t * dq + h * HD + i;
        if constexpr (N == 2) {
          *reinterpret_cast<float2*>(o) = make_float2(x.lo[0], x.lo[1]);
          *reinterpret_cast<float2*>(o + half) = make_float2(x.hi[0], x.hi[1]);
        } else {
          o[0] = x.lo[0];
          o[half] = x.hi[0];
        }
      }
    }
  }
  if (!page_ok) return;

  bool bad = false;
  const int held = t0 - b * PAGE;  // positions of this page that earlier calls wrote
  for (int h0 = kh0, round = 0; h0 < kh1; h0 += S::kHeads, round ^= 1) {
    const int h = h0 + hw;
    const bool mine = h < kh1;
    const int64_t at = static_cast<int64_t>(pg) * p.kv.n_kv + (mine ? h : kh0);
    float old[2] = {0.f, 0.f};
    uint32_t mk = 0u, mv = 0u;
    if (h0 > kh0) load_rows(h);
    if (mine) {
      if (held > 0) {
        old[0] = p.kv.k_scales[at];
        old[1] = p.kv.v_scales[at];
      }
      if (on) {
        Pair<N> w = {};
        if (norm) w = load_pair<N>(p.k_norm + h * HD, i, half);
#pragma unroll
        for (int r = 0; r < S::kRows; ++r) {
          const int t = w0 + r * S::kHeadWarps;
          if (t < nt) {
            float cs[2 * N];
            load_cs<N>(cs0 + t * HD, i, cs);
            turn64<N>(k[r], norm, norm ? sh.sck[t] : 1.0, w, cs);
            mk = top_of<N>(k[r], mk);
            mv = top_of<N>(v[r], mv);
          }
        }
      }
      if (max(mk, mv) >= 0xFF000000u) {  // a value that is not finite sets no scale
        bad = true;
        mk = mv = 0u;
#pragma unroll
        for (int r = 0; r < S::kRows; ++r)
          if (w0 + r * S::kHeadWarps < nt) {
            mk = finite_top_of<N>(k[r], mk);
            mv = finite_top_of<N>(v[r], mv);
          }
      }
      mk = __reduce_max_sync(0xffffffffu, mk);
      mv = __reduce_max_sync(0xffffffffu, mv);
      if (lane == 0 && w0 < nt) {
        atomicMax(&sh.top[round][hw][0], mk >> 1);
        atomicMax(&sh.top[round][hw][1], mv >> 1);
      }
    }
    __syncthreads();  // every warp has the old scales and its share of the maxima
    if (mine) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint8_t* codes = (q == 0 ? p.kv.k_codes : p.kv.v_codes) + at * PAGE * HD;
        int e = scale_exponent(sh.top[round][hw][q]);
        if (held > 0) {
          const int was = min(max((__float_as_int(old[q]) >> 23) & 255, 21), 248);
          if (was >= e) {
            e = was;
          } else {
            const int down = min(e - was, 31);
            for (int j = w0 * 32 + lane; j < held * HD / 4; j += S::kHeadWarps * 32) {
              uint32_t c4 = reinterpret_cast<uint32_t*>(codes)[j], o4 = 0u;
#pragma unroll
              for (int l = 0; l < 4; ++l) {
                const int c = static_cast<int>((c4 >> (8 * l)) & 255u) - 128;
                o4 |= static_cast<uint32_t>((c >> down) + 128) << (8 * l);
              }
              reinterpret_cast<uint32_t*>(codes)[j] = o4;
            }
          }
        }
        const float inv = exponent_float(254 - e);
        if (on) {
          if (!bad) {
#pragma unroll
            for (int r = 0; r < S::kRows; ++r) {
              const int t = w0 + r * S::kHeadWarps;
              if (t < nt) {
                const Pair<N>& x = q == 0 ? k[r] : v[r];
                store_codes<N, false>(codes + (held + t) * HD + i, x.lo, inv);
                store_codes<N, false>(codes + (held + t) * HD + i + half, x.hi, inv);
              }
            }
          } else {
#pragma unroll
            for (int r = 0; r < S::kRows; ++r) {
              const int t = w0 + r * S::kHeadWarps;
              if (t < nt) {
                const Pair<N>& x = q == 0 ? k[r] : v[r];
                store_codes<N, true>(codes + (held + t) * HD + i, x.lo, inv);
                store_codes<N, true>(codes + (held + t) * HD + i + half, x.hi, inv);
              }
            }
          }
        }
        if (w0 == 0 && lane == 0) (q == 0 ? p.kv.k_scales : p.kv.v_scales)[at] = exponent_float(e);
      }
    }
    if (h0 + S::kHeads < kh1) {
      __syncthreads();
      if (tid < S::kHeads * 2) (&sh.top[round][0][0])[tid] = 0u;
    }
  }
  if (bad) paged_error(p.rows);
}

struct ReadArgs {
  PagedKv kv;
  PagedRows rows;
  int bf16;
  void* k_out;
  void* v_out;
};

// The values of sixteen codes: 2^15 + u as bits, less 2^15 + 127.5, times the scale (all exact).
__device__ __forceinline__ void store_values(void* out, int bf16, int64_t i16, const uint4& c16, float scale) {
  const uint32_t w[4] = {c16.x, c16.y, c16.z, c16.w};
  float v[16];
#pragma unroll
  for (int j = 0; j < 16; ++j)
    v[j] = (__uint_as_float(__byte_perm(w[j >> 2], 0x47000000u, 0x7604 | (j & 3) << 4)) - 32895.5f) * scale;
  if (bf16 != 0) {
    uint32_t o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      memcpy(&o[j], &b, 4);
    }
    uint4* to = static_cast<uint4*>(out) + 2 * i16;
    to[0] = make_uint4(o[0], o[1], o[2], o[3]);
    to[1] = make_uint4(o[4], o[5], o[6], o[7]);
  } else {
    float4* to = static_cast<float4*>(out) + 4 * i16;
#pragma unroll
    for (int j = 0; j < 4; ++j) to[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  }
}

constexpr int kReadThreads = 256;
constexpr int kReadRows = 4;  // rows of a CTA, a quarter of its threads each
constexpr int kReadAhead = 2;

// CTA (c, s): rows c * kReadRows .. of sequence s, sixteen values a thread at a time.  Bound by its stores, a thread's 64
// (f32) or 32 bytes apart from its neighbour's: 32,000 rows of 16 heads of 128 take 148 us as f32 (4.4 TB/s), 76 as bf16
// (5.2 TB/s).
__global__ void __launch_bounds__(kReadThreads) paged_read_kernel(const ReadArgs p) {
  constexpr int kPart = kReadThreads / kReadRows;
  pdl_wait();
  pdl_trigger();
  const int s = blockIdx.y, page = p.kv.page, hd = p.kv.hd;
  const SeqRows sq = seq_rows(p.rows, s, static_cast<int64_t>(p.rows.max_blocks) * page);
  if (sq.n < 0 && blockIdx.x == 0 && threadIdx.x == 0) paged_error(p.rows);
  const int r = static_cast<int>(blockIdx.x) * kReadRows + static_cast<int>(threadIdx.x) / kPart;
  if (r >= sq.n) return;
  const int h16 = hd / 16, n16 = p.kv.n_kv * h16, pos = sq.p0 + r;
  const int pg = p.rows.page_table[static_cast<int64_t>(s) * p.rows.max_blocks + (pos >> p.kv.page_log2)];
  const bool ok = pg >= 0 && pg < p.kv.n_pages;
  const int64_t out = static_cast<int64_t>(sq.r0 + r) * n16, at0 = static_cast<int64_t>(ok ? pg : 0) * p.kv.n_kv;
  const int first = threadIdx.x % kPart;
  for (int i0 = first; i0 < n16; i0 += kReadAhead * kPart) {
    uint4 k[kReadAhead], v[kReadAhead];
    float ks[kReadAhead], vs[kReadAhead];
#pragma unroll
    for (int j = 0; j < kReadAhead; ++j) {
      const int i = i0 + j * kPart;
      if (i < n16) {
        const int h = i / h16, c = i - h * h16;
        const int64_t at = at0 + h, off = (at * page + (pos & (page - 1))) * h16 + c;
        k[j] = __ldg(reinterpret_cast<const uint4*>(p.kv.k_codes) + off);
        v[j] = __ldg(reinterpret_cast<const uint4*>(p.kv.v_codes) + off);
        ks[j] = ok ? __ldg(p.kv.k_scales + at) : 0.f;
        vs[j] = ok ? __ldg(p.kv.v_scales + at) : 0.f;
      }
    }
#pragma unroll
    for (int j = 0; j < kReadAhead; ++j) {
      const int i = i0 + j * kPart;
      if (i < n16 && p.k_out != nullptr) store_values(p.k_out, p.bf16, out + i, k[j], ks[j]);
      if (i < n16 && p.v_out != nullptr) store_values(p.v_out, p.bf16, out + i, v[j], vs[j]);
    }
  }
  if (!ok && first == 0) paged_error(p.rows);
}

template <int HD, int PAGE>
int launch_append(const AppendArgs& p, int ranks, unsigned pages, cudaStream_t s) {
  return launch_cluster(paged_append_kernel<HD, PAGE>, dim3(ranks, pages, p.rows.n_seq),
                        dim3(AppendShape<PAGE>::kThreads), ranks, 0, s, p);
}
template <int HD>
int launch_append_hd(const AppendArgs& p, int ranks, unsigned pages, cudaStream_t s) {
  switch (p.kv.page) {
    case 16:
      return launch_append<HD, 16>(p, ranks, pages, s);
    case 32:
      return launch_append<HD, 32>(p, ranks, pages, s);
    case 64:
      return launch_append<HD, 64>(p, ranks, pages, s);
    default:
      return launch_append<HD, 128>(p, ranks, pages, s);
  }
}

}  // namespace

}  // namespace nh

using namespace nh;

extern "C" int nh_paged_append(const NhPagedKv* kv, const NhPagedRows* rows, const float* q, int64_t q_stride,
                               const float* k, int64_t k_stride, const float* v, int64_t v_stride,
                               const float* q_norm, const float* k_norm, float eps, int n_head, const float* rope_cs,
                               int rope_len, float* qr, void* stream) {
  AppendArgs p;
  const int rc = paged_args(kv, rows, p.kv, p.rows);
  if (rc != NH_OK) return rc;
  const int64_t dq = static_cast<int64_t>(n_head) * p.kv.hd, dkv = static_cast<int64_t>(p.kv.n_kv) * p.kv.hd;
  if (k == nullptr || v == nullptr || rope_cs == nullptr || rope_len <= 0 || n_head <= 0 || n_head > 65535 ||
      n_head % p.kv.n_kv != 0 || (q == nullptr) != (qr == nullptr) || (q_norm == nullptr) != (k_norm == nullptr) ||
      k_stride < dkv || v_stride < dkv || (q != nullptr && q_stride < dq))
    return NH_E_ARG;
  if (!paged_aligned(k) || !paged_aligned(v) || !paged_aligned(q) || !paged_aligned(qr) || !paged_aligned(rope_cs) ||
      !paged_aligned(q_norm) || !paged_aligned(k_norm) || k_stride % 4 != 0 || v_stride % 4 != 0 ||
      (q != nullptr && q_stride % 4 != 0) || std::max(std::max(k_stride, v_stride), q != nullptr ? q_stride : 0) > 1 << 23)
    return NH_E_ARG;
  if (p.rows.max_rows == 0) return NH_OK;
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_stride = q != nullptr ? q_stride : 0;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.q_norm = q_norm;
  p.k_norm = k_norm;
  p.eps = eps;
  p.n_head = n_head;
  p.rope_len = rope_len;
  p.rope_cs = rope_cs;
  p.qr = qr;
  const int64_t pages = std::min<int64_t>((static_cast<int64_t>(p.rows.max_rows) + p.kv.page - 2) / p.kv.page + 1,
                                          p.rows.max_blocks);
  if (pages > 65535) return NH_E_ARG;
  // CTAs of a page: more heads each where the pages alone fill the machine (the sums and the barrier cost a CTA the same
  // for any number of heads): the prompts above take 121 us with eight CTAs a page, 95 with four, 106 with two; one
  // page alone is quickest with eight.
  int ranks = std::min(kMaxRanks, p.kv.n_kv);
  if (ranks == kMaxRanks && pages * p.rows.n_seq > 200) ranks = 4;
  p.kv_per = (p.kv.n_kv + ranks - 1) / ranks;
  p.q_per = (n_head + ranks - 1) / ranks;
  const unsigned np = static_cast<unsigned>(pages);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (p.kv.hd) {
    case 32:
      return launch_append_hd<32>(p, ranks, np, st);
    case 64:
      return launch_append_hd<64>(p, ranks, np, st);
    case 96:
      return launch_append_hd<96>(p, ranks, np, st);
    default:
      return launch_append_hd<128>(p, ranks, np, st);
  }
}

extern "C" int nh_paged_read(const NhPagedKv* kv, const NhPagedRows* rows, int32_t out_type, void* k_out, void* v_out,
                             void* stream) {
  ReadArgs p;
  const int rc = paged_args(kv, rows, p.kv, p.rows);
  if (rc != NH_OK) return rc;
  if (out_type != NH_TYPE_F32 && out_type != NH_TYPE_BF16) return NH_E_TYPE;
  if (!paged_aligned(k_out) || !paged_aligned(v_out)) return NH_E_ARG;
  if (p.rows.max_rows == 0 || (k_out == nullptr && v_out == nullptr)) return NH_OK;
  p.bf16 = out_type == NH_TYPE_BF16 ? 1 : 0;
  p.k_out = k_out;
  p.v_out = v_out;
  return launch_pdl(paged_read_kernel, dim3((p.rows.max_rows + kReadRows - 1) / kReadRows, p.rows.n_seq),
                    dim3(kReadThreads), 0, static_cast<cudaStream_t>(stream), p);
}
