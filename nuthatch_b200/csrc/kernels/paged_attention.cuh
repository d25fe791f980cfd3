// What the two forms of the paged attention share: arguments, the visible
// range, exact 8-bit codes as f16 operands and the two-part split of f32
// factors.
//
// Arithmetic.  A code u stands for (u - 127.5) * s with s a power of two, and
// (u - 127.5) * 2^-9 is exact in f16.  A query row is scaled by a power of two and
// split into two f16 parts (22 bits of it), likewise a softmax weight; both
// parts' products are exact and the tensor cores add them up in f32.
// A weight carries its page's scale of V over the largest scale that its row
// sees.  Of what that makes the two parts keep 22 bits down to 2^-18 of the
// largest weight (split form; 2^-10 of the maximum in use in the tiled one);
// below, f16's subnormals end, and the error is at most 2^-40 (2^-32): for each
// position that part of the largest magnitude of V that the row sees.
#pragma once

#include "common.cuh"
#include "paged.cuh"

namespace nh {

struct PagedAttnArgs {
  PagedKv kv;
  PagedRows rows;
  const float* q;
  float* out;
  int n_head, group, window, n_sink;
  float scale;
  int few;  // sequences of at most this many queries a KV head (rows x group) go to the split form
};

constexpr float kLog2e = 1.44269504088896340736f;
// A weight in [0, 1] times 2^15 is within f16's range; its second part ends at steps of 2^-24, so that the two keep 22
// bits of weights of 2^-18 and more and are off by at most 2^-25 of the product, 2^-40 of the weight 1, below.
constexpr int kWeightShift = 15;

// Sums of weighted values in their own units pass f32's range where the values are near its end, and their mean does
// not: what is joined over warps and CTAs is smaller by 2^18 (2^18 positions of equal weight and the largest values; the
// least scale, 2^-106, keeps its 24 bits above the subnormals).
constexpr int kRoom = 18;

// 2^e as a float, 0 below the normal range; e <= 127.
__device__ __forceinline__ float pow2i(int e) { return e < -126 ? 0.f : __int_as_float((e + 127) << 23); }
__device__ __forceinline__ int exponent_of(float s) { return ((__float_as_int(s) >> 23) & 255) - 127; }

// Bytes 0, 1 (or 2, 3) of w as (u - 127.5) * 2^-9: the byte alone is the f16
// u * 2^-24, which one fused step scales and moves, exactly.
constexpr int kCodeShift = 9;
__device__ __forceinline__ uint32_t codes_f16(uint32_t w, uint32_t sel) {
  const uint32_t x = __byte_perm(w, 0u, sel);
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x7800)),   // 2^15
                            __half2half2(__ushort_as_half(0xB3F8)));                                       // -127.5 * 2^-9
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) { return codes_f16(w, 0x4140); }
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) { return codes_f16(w, 0x4342); }

// x and y as f16 pairs hi + lo.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 b = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - b.x, y - b.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two f32 operations in one instruction, each rounded as by itself.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
      " fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n"
      " mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

int launch_paged_split(const PagedAttnArgs& p, cudaStream_t s);
int launch_paged_tiles(const PagedAttnArgs& p, cudaStream_t s);

// Tiles of a call at most: no more than whole ones of all rows and a part of one for each sequence, nor than every
// sequence's most.
inline int64_t paged_tiles(const PagedAttnArgs& p) {
  const int64_t most = static_cast<int64_t>(p.rows.max_rows) * p.group;
  return std::min(static_cast<int64_t>(p.rows.n_rows) * p.group / 128 + p.rows.n_seq, p.rows.n_seq * ((most + 127) / 128));
}

}  // namespace nh
