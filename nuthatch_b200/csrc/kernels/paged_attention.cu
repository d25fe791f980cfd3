// Attention over the paged 8-bit K/V cache (nh_paged_attention).
//
// The simplest right form: a warp per (row, head), lanes over the head's
// dimensions, one position after the other with the running maximum and sum of
// the softmax.
#include "common.cuh"
#include "paged.cuh"

namespace nh {

namespace {

struct PagedAttnArgs {
  PagedKv kv;
  PagedRows rows;
  const float* q;
  float* out;
  int n_head, group, window, n_sink;
  float scale;
};

__global__ void __launch_bounds__(32) paged_attention_kernel(const PagedAttnArgs p) {
  pdl_wait();
  pdl_trigger();
  const int r = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, hd = p.kv.hd, per = hd / 32, page = p.kv.page;
  const int s = seq_of_row(p.rows, r);
  if (s < 0) return;
  const SeqRows sq = seq_rows(p.rows, s, static_cast<int64_t>(p.rows.max_blocks) * page);
  if (sq.n < 0) {
    if (lane == 0) paged_error(p.rows);
    return;
  }
  const int pos = sq.p0 + (r - sq.r0), kh = h / p.group;
  const float* q = p.q + (static_cast<int64_t>(r) * p.n_head + h) * hd + lane * per;
  float qv[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  for (int i = 0; i < per; ++i) qv[i] = q[i] * p.scale;
  for (int t = 0; t <= pos; ++t) {
    if (p.window > 0 && t <= pos - p.window && t >= p.n_sink) t = pos - p.window + 1;
    const int pg = p.rows.page_table[static_cast<int64_t>(s) * p.rows.max_blocks + (t >> p.kv.page_log2)];
    if (pg < 0 || pg >= p.kv.n_pages) {
      if (lane == 0) paged_error(p.rows);
      continue;
    }
    const int64_t at = static_cast<int64_t>(pg) * p.kv.n_kv + kh, off = (at * page + (t & (page - 1))) * hd + lane * per;
    const float ks = p.kv.k_scales[at], vs = p.kv.v_scales[at];
    float d = 0.f;
    for (int i = 0; i < per; ++i) d += qv[i] * (static_cast<float>(p.kv.k_codes[off + i]) - 127.5f);
    const float x = warp_sum(d) * ks, mn = fmaxf(m, x), f = expf(m - mn), w = expf(x - mn);
    m = mn;
    l = l * f + w;
    for (int i = 0; i < per; ++i) acc[i] = acc[i] * f + w * vs * (static_cast<float>(p.kv.v_codes[off + i]) - 127.5f);
  }
  float* o = p.out + (static_cast<int64_t>(r) * p.n_head + h) * hd + lane * per;
  for (int i = 0; i < per; ++i) o[i] = l > 0.f ? acc[i] / l : 0.f;
}

}  // namespace

}  // namespace nh

using namespace nh;

extern "C" int nh_paged_attention(const NhPagedKv* kv, const NhPagedRows* rows, const float* qr, int n_head,
                                  float kq_scale, int window, int n_sink, float* out, void* stream) {
  PagedAttnArgs p;
  const int rc = paged_args(kv, rows, p.kv, p.rows);
  if (rc != NH_OK) return rc;
  if (qr == nullptr || out == nullptr || !paged_aligned(qr) || !paged_aligned(out) || n_head <= 0 || n_head > 65535 ||
      n_head % p.kv.n_kv != 0 || window < 0 || n_sink < 0)
    return NH_E_ARG;
  if (p.rows.n_rows == 0) return NH_OK;
  p.q = qr;
  p.out = out;
  p.n_head = n_head;
  p.group = n_head / p.kv.n_kv;
  p.window = window;
  p.n_sink = n_sink;
  p.scale = kq_scale;
  return launch_pdl(paged_attention_kernel, dim3(p.rows.n_rows, n_head), dim3(32), 0,
                    static_cast<cudaStream_t>(stream), p);
}
