// Verification of drafted tokens against the target's probabilities
// (nh_verify_drafts).
//
// A cluster owns one sequence.  Every CTA finds the first refused draft itself
// (a few loads), and with it the one target row that the next token is drawn
// from; the row is cut over the CTAs in id order and over their warps, each
// warp adds up its piece's mass in 64 bits, and every CTA's sum is written to
// all of them.  The CTA whose part holds the draw finds the warp's piece, then
// all its warps add up that piece's chunks once more (out of L2) for the id.
// The row and, after a refusal, the draft's row are the only ones read whole.
//
// What bounds it: few sequences, the chain of dependent loads (offsets, ids,
// probabilities, row) and the two searches (4 drafts of one sequence over 50,304
// ids: 7.0 us, most of it the launch); many, the rows' bytes (64 sequences of up
// to 5 drafts with their rows 11.3 us, 256 of up to 7 without 16.6 us: 3.1 TB/s).
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
constexpr int kAhead = 4;    // steps whose loads are in flight together
constexpr int kMaxRanks = 8;

// An entry that is not above 0 (a NaN too) has no mass.
__device__ __forceinline__ float mass(float x) { return fmaxf(x, 0.f); }

// The drawn distribution's masses: the target row's, less the draft row's, or
// without the refused id's own (cut >= 0).
struct Source {
  const float* p;
  const float* q;  // or null
  int cut;         // id without mass, or -1
  int n;
  bool vec;        // both rows are 16-byte aligned
};

// A piece of four masses: p less q where that is above 0 (an infinite q leaves nothing).
__device__ __forceinline__ void masses(const float4& p, const float4& q, double (&m)[4]) {
  const float b[4] = {mass(q.x), mass(q.y), mass(q.z), mass(q.w)};
  const float a[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) m[j] = a[j] > b[j] ? static_cast<double>(a[j]) - static_cast<double>(b[j]) : 0.0;
}
__device__ __forceinline__ void masses(const float4& p, double (&m)[4]) {
  m[0] = static_cast<double>(mass(p.x));
  m[1] = static_cast<double>(mass(p.y));
  m[2] = static_cast<double>(mass(p.z));
  m[3] = static_cast<double>(mass(p.w));
}

// Whether chunk c is whole, aligned and without a cut id.
__device__ __forceinline__ bool plain_chunk(const Source& s, int c) {
  return s.vec && c * static_cast<int64_t>(kChunk) + kChunk <= s.n && (s.cut < 0 || s.cut / kChunk != c);
}

__device__ __forceinline__ float4 load4(const float* x, int i, int n) {
  float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
  if (i < n) f.x = __ldg(x + i);
  if (i < n - 1) f.y = __ldg(x + i + 1);
  if (i < n - 2) f.z = __ldg(x + i + 2);
  if (i < n - 3) f.w = __ldg(x + i + 3);
  return f;
}

// Masses of this lane's four ids of any chunk.
__device__ __forceinline__ void chunk_masses(const Source& s, int c, int lane, double (&m)[4]) {
  const int i = c * kChunk + lane * 4;
  if (plain_chunk(s, c)) {
    const float4 p = __ldg(reinterpret_cast<const float4*>(s.p + i));
    if (s.q != nullptr)
      masses(p, __ldg(reinterpret_cast<const float4*>(s.q + i)), m);
    else
      masses(p, m);
    return;
  }
  masses(load4(s.p, i, s.n), s.q != nullptr ? load4(s.q, i, s.n) : make_float4(0.f, 0.f, 0.f, 0.f), m);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (i + j == s.cut) m[j] = 0.0;
}

// The mass of chunks [c0, c1), this lane's share.
template <bool kTwo>
__device__ __forceinline__ double sum_chunks(const Source& s, int c0, int c1, int lane) {
  double sum[kAhead] = {};
  for (int c = c0; c < c1; c += kAhead) {
    if (c + kAhead <= c1 && plain_chunk(s, c + kAhead - 1) && (s.cut < 0 || s.cut / kChunk < c || s.cut / kChunk >= c + kAhead)) {
      float4 p[kAhead], q[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        p[k] = __ldg(reinterpret_cast<const float4*>(s.p + (c + k) * kChunk) + lane);
        if (kTwo) q[k] = __ldg(reinterpret_cast<const float4*>(s.q + (c + k) * kChunk) + lane);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        double m[4];
        if (kTwo)
          masses(p[k], q[k], m);
        else
          masses(p[k], m);
        sum[k] += (m[0] + m[1]) + (m[2] + m[3]);
      }
    } else {
      for (int k = c; k < min(c + kAhead, c1); ++k) {
        double m[4];
        chunk_masses(s, k, lane, m);
        sum[0] += (m[0] + m[1]) + (m[2] + m[3]);
      }
    }
  }
  return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

__device__ __forceinline__ double scan_up(double v, int lane) {
#pragma unroll
  for (int k = 1; k < 32; k <<= 1) {
    const double up = __shfl_up_sync(0xffffffffu, v, k);
    if (lane >= k) v += up;
  }
  return v;
}

// Where a running sum first exceeds `goal` among the n parts v (lane l's is part
// l): the part's index, or the last one with mass (rounding, or a draw of 1),
// or -1; `before` becomes the sum of the parts before it.  Warp-wide.
__device__ __forceinline__ int find_part(double v, int n, double goal, int lane, double& before) {
  v = lane < n ? v : 0.0;
  const double inc = scan_up(v, lane);
  const unsigned mass = __ballot_sync(0xffffffffu, v > 0.0), over = __ballot_sync(0xffffffffu, v > 0.0 && before + inc > goal);
  if (mass == 0u) return -1;
  const int l = over != 0u ? __ffs(over) - 1 : 31 - __clz(mass);
  before += __shfl_sync(0xffffffffu, inc - v, l);
  return l;
}

__global__ void __launch_bounds__(kVerifyThreads) verify_drafts_kernel(const NhVerifyDrafts d) {
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), nrank = static_cast<int>(cluster.num_blocks());
  const int s = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ double wsum[kVerifyWarps];
  __shared__ double total[2][kMaxRanks];  // every CTA's mass, for the first and the second pass
  __shared__ int first;
  pdl_wait();
  pdl_trigger();
  const int o = d.draft_off[s], n = d.draft_off[s + 1] - o;
  const float u_pick = d.u_pick[s];
  if (o < 0 || n < 0 || n > d.max_draft || o > d.n_drafts - n) {  // every CTA of the cluster alike
    if (rank == 0 && tid == 0 && d.err != nullptr) atomicCAS(d.err, 0, NH_E_ARG);
    return;
  }
  if (nrank > 1) cluster.barrier_arrive();  // the others must have started before their shared memory is written
  if (tid == 0) first = n;
  __syncthreads();
  const float* t0 = d.target + static_cast<int64_t>(o + s) * d.target_stride;
  for (int i = tid; i < n; i += kVerifyThreads) {
    const int id = d.draft_ids[o + i];
    const float u = d.u_accept[o + i];
    bool ok = id >= 0 && id < d.n_vocab;
    if (ok) {
      const float q = d.draft != nullptr ? mass(d.draft[static_cast<int64_t>(o + i) * d.draft_stride + id]) : 1.f;
      ok = static_cast<double>(u) * static_cast<double>(q) < static_cast<double>(mass(t0[static_cast<int64_t>(i) * d.target_stride + id]));
    }
    if (!ok) atomicMin(&first, i);
  }
  __syncthreads();
  const int acc = first;
  Source src{t0 + acc * d.target_stride, nullptr, -1, static_cast<int>(d.n_vocab), false};
  if (acc < n) {
    if (d.draft != nullptr)
      src.q = d.draft + static_cast<int64_t>(o + acc) * d.draft_stride;
    else
      src.cut = d.draft_ids[o + acc];
  }
  src.vec = ((reinterpret_cast<uintptr_t>(src.p) | reinterpret_cast<uintptr_t>(src.q)) & 15) == 0;

  // Pieces of whole chunks, in id order.
  const int chunks = (src.n - 1) / kChunk + 1, parts = nrank * kVerifyWarps, per = (chunks + parts - 1) / parts;
  const int c0 = min((rank * kVerifyWarps + warp) * per, chunks), c1 = min(c0 + per, chunks);
  double all = 0.0;
  int pass = 0;
  for (;; ++pass) {
    const double mine = warp_sum_d(src.q != nullptr ? sum_chunks<true>(src, c0, c1, lane) : sum_chunks<false>(src, c0, c1, lane));
    if (lane == 0) wsum[warp] = mine;
    __syncthreads();
    if (warp == 0) {
      const double t = warp_sum_d(lane < kVerifyWarps ? wsum[lane] : 0.0);
      if (nrank > 1 && pass == 0) cluster.barrier_wait();
      if (lane < nrank) cluster.map_shared_rank(&total[pass][0], lane)[rank] = t;
    }
    if (nrank > 1 && pass == 0 && warp != 0) cluster.barrier_wait();
    if (nrank > 1)
      cluster.sync();
    else
      __syncthreads();
    all = warp_sum_d(lane < nrank ? total[pass][lane] : 0.0);
    if (all > 0.0 || pass == 1 || (src.q == nullptr && src.cut < 0)) break;
    // Nothing is left of the target once the draft is taken off: its own mass.
    src.q = nullptr;
    src.cut = -1;
    src.vec = (reinterpret_cast<uintptr_t>(src.p) & 15) == 0;
    __syncthreads();
  }

  const double goal = static_cast<double>(u_pick) * all;
  double before = 0.0;
  int owner = find_part(lane < nrank ? total[pass][lane] : 0.0, nrank, goal, lane, before);
  if (all == INFINITY) owner = -1;  // an infinite entry of the target: no distribution
  int32_t* ids = d.out_ids + static_cast<int64_t>(s) * (d.max_draft + 1);
  if (rank == 0) {
    for (int i = tid; i < acc; i += kVerifyThreads) ids[i] = d.draft_ids[o + i];
    if (tid == 0) {
      d.n_accept[s] = acc;
      if (owner < 0) ids[acc] = -1;
      if (d.err != nullptr) {
        if (owner < 0) atomicCAS(d.err, 0, NH_E_ARG);
        const int id = acc < n ? d.draft_ids[o + acc] : 0;
        if (id < 0 || id >= d.n_vocab) atomicCAS(d.err, 0, NH_E_ARG);
      }
    }
  }
  if (rank != owner) return;
  const int piece = find_part(lane < kVerifyWarps ? wsum[lane] : 0.0, kVerifyWarps, goal, lane, before);
  if (piece < 0) return;  // not reached: the CTA's sum is above 0
  // The piece's chunks, one a warp at a time, until the running sum passes the goal.
  const int b0 = min((rank * kVerifyWarps + piece) * per, chunks), b1 = min(b0 + per, chunks);
  __shared__ double csum[2][kVerifyWarps];
  __shared__ int last;  // the last id with mass so far
  if (tid == 0) last = -1;
  int round = 0;
  for (int c = b0; c < b1; c += kVerifyWarps, round ^= 1) {
    double m[4] = {};
    if (c + warp < b1) chunk_masses(src, c + warp, lane, m);
    const double mine4 = (m[0] + m[1]) + (m[2] + m[3]);
    const double inc = scan_up(mine4, lane);
    if (lane == 31) csum[round][warp] = inc;
    __syncthreads();
    double at = before;
    const double v = lane < kVerifyWarps ? csum[round][lane] : 0.0;
    const int chunk = find_part(v, kVerifyWarps, goal, lane, at);
    const bool over = chunk >= 0 && at + __shfl_sync(0xffffffffu, v, max(chunk, 0)) > goal;
    if (chunk >= 0 && warp == chunk) {
      // The first id whose running sum exceeds the goal, else the chunk's last one with mass.
      double cum = at + (inc - mine4);
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
      const int l = hits != 0u ? __ffs(hits) - 1 : 31 - __clz(tails);
      const int j = __shfl_sync(0xffffffffu, hits != 0u ? hit : tail, l);
      if (lane == 0) last = (c + warp) * kChunk + l * 4 + j;
    }
    if (over) break;  // every warp alike
    before += __shfl_sync(0xffffffffu, scan_up(v, lane), 31);
  }
  __syncthreads();
  if (tid == 0) ids[acc] = last;
}

}  // namespace

}  // namespace nh

using namespace nh;

extern "C" int nh_verify_drafts(const NhVerifyDrafts* d, void* stream) {
  if (d == nullptr || d->target == nullptr || d->draft_off == nullptr || d->u_pick == nullptr ||
      d->n_accept == nullptr || d->out_ids == nullptr || d->n_seq <= 0 || d->n_seq > 65535 || d->n_drafts < 0 ||
      d->max_draft < 0 || d->max_draft > 1024 || d->n_vocab <= 0 || d->n_vocab > (1 << 30) ||
      d->target_stride < d->n_vocab || (d->draft != nullptr && d->draft_stride < d->n_vocab) ||
      static_cast<int64_t>(d->n_drafts) + d->n_seq > INT32_MAX)
    return NH_E_ARG;
  if (d->n_drafts > 0 && (d->draft_ids == nullptr || d->u_accept == nullptr)) return NH_E_ARG;
  // CTAs of a sequence: eight unless the sequences alone fill the machine twice.  (Up to 5 drafts with their rows of 64
  // and of 256 sequences, up to 7 without of 256: 11.9, 26.7 and 17.1 us up to 300 CTAs; 17.6, 32.6 and 23.6 up to 600;
  // 17.6, 42.3 and 36.4 up to 1,200, where the CTAs' searches are the more work.)
  int ranks = kMaxRanks;
  while (ranks > 1 && static_cast<int64_t>(d->n_seq) * ranks > 300) ranks /= 2;
  return launch_cluster(verify_drafts_kernel, dim3(ranks, d->n_seq), dim3(kVerifyThreads), ranks, 0,
                        static_cast<cudaStream_t>(stream), *d);
}
