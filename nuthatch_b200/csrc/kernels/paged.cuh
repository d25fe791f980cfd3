// What the paged-cache kernels share: the argument blocks' host checks, a
// sequence's rows with their bounds, and the page code.
#pragma once

#include <algorithm>

#include "launch.cuh"
#include "rowdot.cuh"

namespace nh {

struct PagedRows {
  int n_seq, max_rows, n_rows, max_blocks;
  const int32_t* row_off;
  const int32_t* pos0;
  const int32_t* page_table;
  int32_t* err;
};

struct PagedKv {
  uint8_t* k_codes;
  uint8_t* v_codes;
  float* k_scales;
  float* v_scales;
  int n_pages, page, page_log2, n_kv, hd;
};

// The rows [r0, r0 + n) of sequence s at positions p0..; n = -1 when they are
// outside the call's bounds.
struct SeqRows {
  int r0, n, p0;
};

__device__ __forceinline__ void paged_error(const PagedRows& r) {
  if (r.err != nullptr) atomicCAS(r.err, 0, NH_E_ARG);
}

// `limit`: positions that the caller's tables cover.
__device__ __forceinline__ SeqRows seq_rows(const PagedRows& r, int s, int64_t limit) {
  const int a = r.row_off[s], b = r.row_off[s + 1], p0 = r.pos0[s];
  SeqRows q{a, b - a, p0};
  if (a < 0 || b < a || b > r.n_rows || q.n > r.max_rows || p0 < 0 || static_cast<int64_t>(p0) + q.n > limit) q.n = -1;
  return q;
}

inline bool paged_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The host checks of the two argument blocks; fills the kernels' forms.
inline int paged_args(const NhPagedKv* kv, const NhPagedRows* rows, PagedKv& k, PagedRows& r) {
  if (kv == nullptr || rows == nullptr || kv->k_codes == nullptr || kv->v_codes == nullptr ||
      kv->k_scales == nullptr || kv->v_scales == nullptr || rows->row_off == nullptr || rows->pos0 == nullptr ||
      rows->page_table == nullptr)
    return NH_E_ARG;
  if (kv->n_pages <= 0 || kv->n_head_kv <= 0 || kv->n_head_kv > 65535 || kv->head_dim <= 0 ||
      kv->head_dim % 32 != 0 || kv->head_dim > 128 ||
      static_cast<int64_t>(kv->n_head_kv) * kv->page_size * kv->head_dim > (1 << 30) || !paged_aligned(kv->k_codes) ||
      !paged_aligned(kv->v_codes))
    return NH_E_ARG;
  int log2 = 4;
  while (log2 < 7 && (1 << log2) < kv->page_size) ++log2;
  if ((1 << log2) != kv->page_size) return NH_E_ARG;
  // Positions are 32-bit.
  if (rows->n_seq <= 0 || rows->n_seq > 65535 || rows->n_rows < 0 || rows->max_rows < 0 || rows->max_blocks <= 0 ||
      static_cast<int64_t>(rows->max_blocks) * kv->page_size > INT32_MAX - 256)
    return NH_E_ARG;
  k = PagedKv{kv->k_codes, kv->v_codes, kv->k_scales, kv->v_scales, kv->n_pages, kv->page_size, log2,
              kv->n_head_kv, kv->head_dim};
  r = PagedRows{rows->n_seq, std::min(rows->max_rows, rows->n_rows), rows->n_rows, rows->max_blocks, rows->row_off,
                rows->pos0, rows->page_table, rows->err};
  return NH_OK;
}

}  // namespace nh
