// Verification of drafted tokens against the target's probabilities
// (nh_verify_drafts).
//
// A cluster owns one sequence.  Every CTA finds the first refused draft itself
// (a few loads), and with it the one target row that the next token is drawn
// from; the row is cut over the CTAs in id order and over their warps, each
// warp adds up its piece's mass in 64 bits, the CTAs' sums are read through
// distributed shared memory, and the one warp whose piece holds the draw scans
// it again (out of L2) for the id.  The row and, after a refusal, the draft's
// row are the only ones read whole.
#include <cooperative_groups.h>

#include "common.cuh"
#include "launch.cuh"
#include "rowdot.cuh"

namespace cg = cooperative_groups;

namespace nh {

namespace {

constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kChunk = 128;  // ids of one warp step: four consecutive ones a lane

__device__ __forceinline__ double mass(float x) { return x > 0.f ? static_cast<double>(x) : 0.0; }

// The masses of ids [i, i+4) of the drawn distribution: the target row's, less
// the draft row's or the refused id's own (cut >= 0).
struct Source {
  const float* p;
  const float* q;  // or null
  int64_t cut;     // id without mass, or -1
  int64_t n;
  bool vec;        // both rows are 16-byte aligned
};

__device__ __forceinline__ void load4(const float* x, int64_t i, int64_t n, bool vec, float (&o)[4]) {
  if (vec && i + 4 <= n) {
    const float4 f = __ldg(reinterpret_cast<const float4*>(x + i));
    o[0] = f.x;
    o[1] = f.y;
    o[2] = f.z;
    o[3] = f.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = i + j < n ? __ldg(x + i + j) : 0.f;
  }
}

__device__ __forceinline__ void masses4(const Source& s, int64_t i, double (&m)[4]) {
  float p[4], q[4] = {0.f, 0.f, 0.f, 0.f};
  load4(s.p, i, s.n, s.vec, p);
  if (s.q != nullptr) load4(s.q, i, s.n, s.vec, q);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m[j] = i + j == s.cut ? 0.0 : fmax(mass(p[j]) - mass(q[j]), 0.0);
  }
}

__global__ void __launch_bounds__(kVerifyThreads) verify_drafts_kernel(const NhVerifyDrafts d) {
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), nrank = static_cast<int>(cluster.num_blocks());
  const int s = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ double wsum[kVerifyWarps];
  __shared__ double total[2];  // this CTA's mass, for the first and the second pass
  __shared__ int first;
  pdl_wait();
  pdl_trigger();
  const int o = d.draft_off[s], n = d.draft_off[s + 1] - o;
  if (o < 0 || n < 0 || n > d.max_draft || o > d.n_drafts - n) {  // every CTA of the cluster alike
    if (rank == 0 && tid == 0 && d.err != nullptr) atomicCAS(d.err, 0, NH_E_ARG);
    return;
  }
  if (tid == 0) first = n;
  __syncthreads();
  const float* t0 = d.target + static_cast<int64_t>(o + s) * d.target_stride;
  for (int i = tid; i < n; i += kVerifyThreads) {
    const int64_t id = d.draft_ids[o + i];
    bool ok = id >= 0 && id < d.n_vocab;
    if (ok) {
      const double q = d.draft != nullptr ? mass(d.draft[static_cast<int64_t>(o + i) * d.draft_stride + id]) : 1.0;
      ok = static_cast<double>(d.u_accept[o + i]) * q < mass(t0[i * d.target_stride + id]);
    }
    if (!ok) atomicMin(&first, i);
  }
  __syncthreads();
  const int acc = first;
  Source src{t0 + acc * d.target_stride, nullptr, -1, d.n_vocab, false};
  if (acc < n) {
    if (d.draft != nullptr)
      src.q = d.draft + static_cast<int64_t>(o + acc) * d.draft_stride;
    else
      src.cut = d.draft_ids[o + acc];
  }
  src.vec = ((reinterpret_cast<uintptr_t>(src.p) | reinterpret_cast<uintptr_t>(src.q)) & 15) == 0;

  // Pieces of whole chunks, in id order.
  const int64_t chunks = (d.n_vocab + kChunk - 1) / kChunk, parts = static_cast<int64_t>(nrank) * kVerifyWarps;
  const int64_t per = (chunks + parts - 1) / parts;
  const int64_t c0 = min((static_cast<int64_t>(rank) * kVerifyWarps + warp) * per, chunks), c1 = min(c0 + per, chunks);
  double all = 0.0, before = 0.0;
  int pass = 0;
  for (;; ++pass) {
    double sum = 0.0;
    for (int64_t c = c0; c < c1; ++c) {
      double m[4];
      masses4(src, c * kChunk + lane * 4, m);
      sum += (m[0] + m[1]) + (m[2] + m[3]);
    }
    sum = warp_sum_d(sum);
    if (lane == 0) wsum[warp] = sum;
    __syncthreads();
    if (tid == 0) {
      double t = 0.0;
      for (int w = 0; w < kVerifyWarps; ++w) t += wsum[w];
      total[pass] = t;
    }
    cluster.sync();
    all = before = 0.0;
    for (int r = 0; r < nrank; ++r) {
      if (r == rank) before = all;
      all += cluster.map_shared_rank(total, r)[pass];
    }
    if (all > 0.0 || pass == 1 || (src.q == nullptr && src.cut < 0)) break;
    // Nothing is left of the target once the draft is taken off: its own mass.
    src.q = nullptr;
    src.cut = -1;
    src.vec = (reinterpret_cast<uintptr_t>(src.p) & 15) == 0;
    __syncthreads();
  }

  // The piece that holds the draw: the first whose running sum exceeds `goal`,
  // else (rounding, or a draw of 1) the last one with mass.
  const double goal = static_cast<double>(d.u_pick[s]) * all;
  int owner = -1, last = -1;
  double run = 0.0;
  for (int r = 0; r < nrank; ++r) {
    const double v = cluster.map_shared_rank(total, r)[pass];
    run += v;
    if (v > 0.0) last = r;
    if (owner < 0 && v > 0.0 && run > goal) owner = r;
  }
  cluster.sync();  // the last read of the others' shared memory
  if (owner < 0) owner = last;
  int32_t* ids = d.out_ids + static_cast<int64_t>(s) * (d.max_draft + 1);
  if (rank == 0) {
    for (int i = tid; i < acc; i += kVerifyThreads) ids[i] = d.draft_ids[o + i];
    if (tid == 0) {
      d.n_accept[s] = acc;
      if (owner < 0) ids[acc] = -1;
      if (d.err != nullptr) {
        if (owner < 0) atomicCAS(d.err, 0, NH_E_ARG);
        const int64_t id = acc < n ? d.draft_ids[o + acc] : 0;
        if (id < 0 || id >= d.n_vocab) atomicCAS(d.err, 0, NH_E_ARG);
      }
    }
  }
  if (rank != owner) return;
  int mine = -1;
  double at = before, sum_before = before;
  last = -1;
  for (int w = 0; w < kVerifyWarps; ++w) {
    if (wsum[w] > 0.0) {
      last = w;
      sum_before = at;
      if (at + wsum[w] > goal) {
        mine = w;
        break;
      }
    }
    at += wsum[w];
  }
  if (mine < 0) mine = last;
  if (warp != mine) return;
  // Scan of this warp's piece: lane-exclusive running sums in id order.
  double base = sum_before;
  int64_t found = -1, last_id = -1;
  for (int64_t c = c0; c < c1; ++c) {
    double m[4];
    const int64_t i = c * kChunk + lane * 4;
    masses4(src, i, m);
    const double mine4 = (m[0] + m[1]) + (m[2] + m[3]);
    double inc = mine4;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, inc, k);
      if (lane >= k) inc += up;
    }
    double cum = base + (inc - mine4);
    int hit = -1, tail = -1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      cum += m[j];
      if (m[j] > 0.0) {
        tail = j;
        if (hit < 0 && cum > goal) hit = j;
      }
    }
    const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), tails = __ballot_sync(0xffffffffu, tail >= 0);
    if (tails != 0u) {
      const int l = 31 - __clz(tails);
      last_id = c * kChunk + l * 4 + __shfl_sync(0xffffffffu, tail, l);
    }
    if (hits != 0u) {
      const int l = __ffs(hits) - 1;
      found = c * kChunk + l * 4 + __shfl_sync(0xffffffffu, hit, l);
      break;
    }
    base += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) ids[acc] = static_cast<int32_t>(found >= 0 ? found : last_id);
}

}  // namespace

}  // namespace nh

using namespace nh;

extern "C" int nh_verify_drafts(const NhVerifyDrafts* d, void* stream) {
  if (d == nullptr || d->target == nullptr || d->draft_off == nullptr || d->u_pick == nullptr ||
      d->n_accept == nullptr || d->out_ids == nullptr || d->n_seq <= 0 || d->n_seq > 65535 || d->n_drafts < 0 ||
      d->max_draft < 0 || d->max_draft > 1024 || d->n_vocab <= 0 || d->n_vocab > INT32_MAX ||
      d->target_stride < d->n_vocab || (d->draft != nullptr && d->draft_stride < d->n_vocab) ||
      static_cast<int64_t>(d->n_drafts) + d->n_seq > INT32_MAX)
    return NH_E_ARG;
  if (d->n_drafts > 0 && (d->draft_ids == nullptr || d->u_accept == nullptr)) return NH_E_ARG;
  return launch_cluster(verify_drafts_kernel, dim3(8, d->n_seq), dim3(kVerifyThreads), 8, 0,
                        static_cast<cudaStream_t>(stream), *d);
}
