// The paged 8-bit K/V cache: rows into it (nh_paged_append) and values out of
// it (nh_paged_read).
//
// Append.  K and V of a row are coded with their page's scale, which needs the
// largest magnitude over the page's rows, and K is known only after the
// RMSNorm over the row's full width.  So a cluster owns one page of one
// sequence and its CTAs share the heads: each sums the squares of its heads'
// columns for every row of the page, the sums are added over the cluster
// through distributed shared memory, and from there each CTA works on whole
// (page, head) pairs alone.  Per row the arithmetic is nh_prefill_qk's.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <cstring>

#include "common.cuh"
#include "paged.cuh"

namespace cg = cooperative_groups;

namespace nh {

namespace {

constexpr int kAppendThreads = 256;
constexpr int kMaxPage = 128;

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
  int n_head, rope_len;
  const float* rope_cs;
  float* qr;
};

// The scale of a page's head whose largest finite magnitude has these bits, as
// a biased exponent: 2^(E-6), at least 2^-106.
__device__ __forceinline__ int scale_exponent(uint32_t amax_bits) {
  return max(static_cast<int>(amax_bits >> 23), 27) - 6;
}
__device__ __forceinline__ float exponent_float(int biased) { return __int_as_float(biased << 23); }

// floor(x / 2^(e-127)) + 128 within the byte; a NaN gives 128.
__device__ __forceinline__ uint32_t code_of(float x, float inv) {
  return static_cast<uint32_t>(min(max(__float2int_rd(x * inv), -128), 127) + 128);
}

__device__ __forceinline__ uint32_t finite_magnitude(float x, bool& bad) {
  const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
  if (b >= 0x7F800000u) {
    bad = true;
    return 0u;
  }
  return b;
}

struct AppendShared {
  double ssq[kMaxPage], ssk[kMaxPage];  // this CTA's sums of squares of each row's q, k
  float scq[kMaxPage], sck[kMaxPage];   // each row's RMSNorm factors
  uint32_t top[4];                      // bits of the largest magnitude of K, V
};
static_assert(sizeof(AppendShared) % 16 == 0, "the staged rows follow it");

__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendArgs p) {
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), nrank = static_cast<int>(cluster.num_blocks());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nw = kAppendThreads / 32;
  const int s = blockIdx.z, hd = p.kv.hd, half = hd / 2, page = p.kv.page;
  extern __shared__ __align__(16) uint8_t append_smem[];
  AppendShared& sh = *reinterpret_cast<AppendShared*>(append_smem);
  float* const stage = reinterpret_cast<float*>(append_smem + sizeof(AppendShared));  // [page][hd] of K, then of V
  pdl_wait();
  pdl_trigger();
  const int64_t cap = static_cast<int64_t>(p.rows.max_blocks) * page;
  const SeqRows sq = seq_rows(p.rows, s, min(cap, static_cast<int64_t>(p.rope_len)));
  if (sq.n < 0 && blockIdx.y == 0 && rank == 0 && tid == 0) paged_error(p.rows);
  if (sq.n <= 0) return;
  const int b = (sq.p0 >> p.kv.page_log2) + static_cast<int>(blockIdx.y);
  const int t0 = max(sq.p0, b * page), t1 = min(sq.p0 + sq.n, (b + 1) * page);
  if (t0 >= t1) return;  // every CTA of the cluster alike
  const int nt = t1 - t0, row0 = sq.r0 + (t0 - sq.p0);
  const int pg = p.rows.page_table[static_cast<int64_t>(s) * p.rows.max_blocks + b];
  const bool page_ok = pg >= 0 && pg < p.kv.n_pages;
  if (!page_ok && rank == 0 && tid == 0) paged_error(p.rows);

  // This CTA's heads.
  const int kv_per = (p.kv.n_kv + nrank - 1) / nrank, q_per = (p.n_head + nrank - 1) / nrank;
  const int kh0 = min(rank * kv_per, p.kv.n_kv), kh1 = min(kh0 + kv_per, p.kv.n_kv);
  const int qh0 = min(rank * q_per, p.n_head), qh1 = min(qh0 + q_per, p.n_head);
  const bool has_q = p.q != nullptr, norm = p.k_norm != nullptr;
  const int dq = p.n_head * hd, dkv = p.kv.n_kv * hd;

  if (norm) {
    for (int t = warp; t < nt; t += nw) {
      double a = 0.0, c = 0.0;
      if (has_q) {
        const float* qb = p.q + (row0 + t) * p.q_stride;
        for (int i = qh0 * hd + lane; i < qh1 * hd; i += 32) a += static_cast<double>(__fmul_rn(qb[i], qb[i]));
      }
      const float* kb = p.k + (row0 + t) * p.k_stride;
      for (int i = kh0 * hd + lane; i < kh1 * hd; i += 32) c += static_cast<double>(__fmul_rn(kb[i], kb[i]));
      a = warp_sum_d(a);
      c = warp_sum_d(c);
      if (lane == 0) {
        sh.ssq[t] = a;
        sh.ssk[t] = c;
      }
    }
    cluster.sync();
    for (int t = tid; t < nt; t += kAppendThreads) {
      double a = 0.0, c = 0.0;
      for (int r = 0; r < nrank; ++r) {
        a += cluster.map_shared_rank(sh.ssq, r)[t];
        c += cluster.map_shared_rank(sh.ssk, r)[t];
      }
      sh.scq[t] = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(static_cast<float>(div_count(a, dq)), p.eps)));
      sh.sck[t] = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(static_cast<float>(div_count(c, dkv)), p.eps)));
    }
    cluster.sync();  // no CTA leaves while another reads its sums
  }

  if (has_q) {
    for (int j = warp; j < nt * (qh1 - qh0); j += nw) {
      const int t = j / (qh1 - qh0), h = qh0 + j % (qh1 - qh0);
      const float* x = p.q + (row0 + t) * p.q_stride + h * hd;
      float* o = p.qr + static_cast<int64_t>(row0 + t) * dq + h * hd;
      const float* cs = p.rope_cs + static_cast<int64_t>(t0 + t) * hd;
      for (int i = lane; i < half; i += 32) {
        float x0 = x[i], x1 = x[i + half];
        if (norm) {
          x0 = __fmul_rn(__fmul_rn(x0, sh.scq[t]), p.q_norm[h * hd + i]);
          x1 = __fmul_rn(__fmul_rn(x1, sh.scq[t]), p.q_norm[h * hd + i + half]);
        }
        const float c = cs[2 * i], sn = cs[2 * i + 1];
        o[i] = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, sn));
        o[i + half] = __fadd_rn(__fmul_rn(x0, sn), __fmul_rn(x1, c));
      }
    }
  }
  if (!page_ok) return;

  float* ks = stage;
  float* vs = stage + page * hd;
  bool bad = false;
  for (int h = kh0; h < kh1; ++h) {
    if (tid < 2) sh.top[tid] = 0u;
    __syncthreads();
    uint32_t mk = 0u, mv = 0u;
    for (int t = warp; t < nt; t += nw) {
      const float* x = p.k + (row0 + t) * p.k_stride + h * hd;
      const float* y = p.v + (row0 + t) * p.v_stride + h * hd;
      const float* cs = p.rope_cs + static_cast<int64_t>(t0 + t) * hd;
      for (int i = lane; i < half; i += 32) {
        float x0 = x[i], x1 = x[i + half];
        if (norm) {
          x0 = __fmul_rn(__fmul_rn(x0, sh.sck[t]), p.k_norm[h * hd + i]);
          x1 = __fmul_rn(__fmul_rn(x1, sh.sck[t]), p.k_norm[h * hd + i + half]);
        }
        const float c = cs[2 * i], sn = cs[2 * i + 1];
        const float r0 = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, sn));
        const float r1 = __fadd_rn(__fmul_rn(x0, sn), __fmul_rn(x1, c));
        const float y0 = y[i], y1 = y[i + half];
        ks[t * hd + i] = r0;
        ks[t * hd + i + half] = r1;
        vs[t * hd + i] = y0;
        vs[t * hd + i + half] = y1;
        mk = max(mk, max(finite_magnitude(r0, bad), finite_magnitude(r1, bad)));
        mv = max(mv, max(finite_magnitude(y0, bad), finite_magnitude(y1, bad)));
      }
    }
    mk = __reduce_max_sync(0xffffffffu, mk);
    mv = __reduce_max_sync(0xffffffffu, mv);
    if (lane == 0) {
      atomicMax(&sh.top[0], mk);
      atomicMax(&sh.top[1], mv);
    }
    __syncthreads();
    const int held = t0 - b * page;  // positions of this page that earlier calls wrote
    const int64_t at = static_cast<int64_t>(pg) * p.kv.n_kv + h;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float* scales = w == 0 ? p.kv.k_scales : p.kv.v_scales;
      uint8_t* codes = (w == 0 ? p.kv.k_codes : p.kv.v_codes) + at * page * hd;
      const float* src = w == 0 ? ks : vs;
      int e = scale_exponent(sh.top[w]);
      if (held > 0) {
        const int old = min(max((__float_as_int(scales[at]) >> 23) & 255, 21), 248);
        if (old >= e) {
          e = old;
        } else {
          const int sh = min(e - old, 31);
          for (int i = tid; i < held * hd / 4; i += kAppendThreads) {
            uint32_t c4 = reinterpret_cast<uint32_t*>(codes)[i], o4 = 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int c = static_cast<int>((c4 >> (8 * j)) & 255u) - 128;
              o4 |= static_cast<uint32_t>((c >> sh) + 128) << (8 * j);
            }
            reinterpret_cast<uint32_t*>(codes)[i] = o4;
          }
        }
      }
      const float inv = exponent_float(254 - e);
      for (int i = tid; i < nt * hd / 4; i += kAppendThreads) {
        const float4 x = reinterpret_cast<const float4*>(src)[i];
        reinterpret_cast<uint32_t*>(codes + held * hd)[i] =
            code_of(x.x, inv) | code_of(x.y, inv) << 8 | code_of(x.z, inv) << 16 | code_of(x.w, inv) << 24;
      }
      __syncthreads();  // the old scale has been read
      if (tid == 0) scales[at] = exponent_float(e);
    }
    __syncthreads();
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

__device__ __forceinline__ void store_values(void* out, int bf16, int64_t i4, uint32_t c4, float scale) {
  float v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = (static_cast<float>((c4 >> (8 * j)) & 255u) - 127.5f) * scale;
  if (bf16 != 0) {
    __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    uint2 o;
    memcpy(&o.x, &a, 4);
    memcpy(&o.y, &b, 4);
    static_cast<uint2*>(out)[i4] = o;
  } else {
    static_cast<float4*>(out)[i4] = make_float4(v[0], v[1], v[2], v[3]);
  }
}

constexpr int kReadThreads = 256;

// A CTA per row; thread i four values of K and of V.
__global__ void __launch_bounds__(kReadThreads) paged_read_kernel(const ReadArgs p) {
  pdl_wait();
  pdl_trigger();
  const int r = blockIdx.x, page = p.kv.page, hd = p.kv.hd;
  const int s = seq_of_row(p.rows, r);
  if (s < 0) return;
  const SeqRows sq = seq_rows(p.rows, s, static_cast<int64_t>(p.rows.max_blocks) * page);
  if (sq.n < 0) {
    if (threadIdx.x == 0) paged_error(p.rows);
    return;
  }
  const int pos = sq.p0 + (r - sq.r0);
  const int pg = p.rows.page_table[static_cast<int64_t>(s) * p.rows.max_blocks + (pos >> p.kv.page_log2)];
  const bool ok = pg >= 0 && pg < p.kv.n_pages;
  if (!ok && threadIdx.x == 0) paged_error(p.rows);
  const int n4 = p.kv.n_kv * hd / 4, h4 = hd / 4;
  for (int i = threadIdx.x; i < n4; i += kReadThreads) {
    const int h = i / h4, c = i - h * h4;
    const int64_t at = static_cast<int64_t>(pg) * p.kv.n_kv + h;
    const int64_t off = (at * page + (pos & (page - 1))) * h4 + c, o = static_cast<int64_t>(r) * n4 + i;
    if (p.k_out != nullptr)
      store_values(p.k_out, p.bf16, o, ok ? reinterpret_cast<const uint32_t*>(p.kv.k_codes)[off] : 0u,
                   ok ? p.kv.k_scales[at] : 0.f);
    if (p.v_out != nullptr)
      store_values(p.v_out, p.bf16, o, ok ? reinterpret_cast<const uint32_t*>(p.kv.v_codes)[off] : 0u,
                   ok ? p.kv.v_scales[at] : 0.f);
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
      (q != nullptr && q_stride % 4 != 0))
    return NH_E_ARG;
  if (p.rows.max_rows == 0) return NH_OK;
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.q_norm = q_norm;
  p.k_norm = k_norm;
  p.eps = eps;
  p.n_head = n_head;
  p.rope_len = rope_len;
  p.rope_cs = rope_cs;
  p.qr = qr;
  const int ranks = std::min(8, p.kv.n_kv);
  const int64_t pages = std::min<int64_t>((static_cast<int64_t>(p.rows.max_rows) + p.kv.page - 2) / p.kv.page + 1,
                                          p.rows.max_blocks);
  if (pages > 65535) return NH_E_ARG;
  const size_t smem = sizeof(AppendShared) + 2 * static_cast<size_t>(p.kv.page) * p.kv.hd * sizeof(float);
  static SmemLimit configured;
  if (!ensure_smem(paged_append_kernel, smem, configured)) return NH_E_CUDA;
  return launch_cluster(paged_append_kernel, dim3(ranks, static_cast<unsigned>(pages), p.rows.n_seq),
                        dim3(kAppendThreads), ranks, smem, static_cast<cudaStream_t>(stream), p);
}

extern "C" int nh_paged_read(const NhPagedKv* kv, const NhPagedRows* rows, int32_t out_type, void* k_out, void* v_out,
                             void* stream) {
  ReadArgs p;
  const int rc = paged_args(kv, rows, p.kv, p.rows);
  if (rc != NH_OK) return rc;
  if (out_type != NH_TYPE_F32 && out_type != NH_TYPE_BF16) return NH_E_TYPE;
  if (!paged_aligned(k_out) || !paged_aligned(v_out)) return NH_E_ARG;
  if (p.rows.n_rows == 0 || (k_out == nullptr && v_out == nullptr)) return NH_OK;
  p.bf16 = out_type == NH_TYPE_BF16 ? 1 : 0;
  p.k_out = k_out;
  p.v_out = v_out;
  return launch_pdl(paged_read_kernel, dim3(p.rows.n_rows), dim3(kReadThreads), 0, static_cast<cudaStream_t>(stream),
                    p);
}
