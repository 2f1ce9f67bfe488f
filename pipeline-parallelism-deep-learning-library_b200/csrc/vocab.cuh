// vocab.cuh -- device helpers of the operators over a vocabulary: typed loads, the running softmax of a row, and the
// order of the alternatives.
//
// A softmax over a row is carried as (m, s, t): the largest logit so far, s = sum 2^d and t = sum 2^d d over the row with
// d = (x - m) * scale * log2(e).  All three are f32.  Two parts of a row merge by moving the part with the smaller m to
// the larger one: s' = s 2^u, t' = 2^u (t + u s) with u = (m - m') * scale * log2(e).
//  - A logit of minus infinity has 2^d = 0.  d is held at -1e4 or more wherever it is multiplied, so that a masked place
//    adds -1e4 * 0 and not -inf * 0 = NaN.  2^-1e4 is 0 in f32.
//  - While m is minus infinity (nothing but masked places so far) d is taken against 0, which leaves s = t = 0.
//  - NaN stays: the maximum and the bound on d both pass a NaN on.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "vocab.h"

namespace lcv {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFar = -1e4f;

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

// 2^x, at most 2 units in the last place off; 2^-inf = 0
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// the larger, or NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

template <int DT>
struct Elem;
template <>
struct Elem<LC_F32> {
  using T = float;
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
};
template <>
struct Elem<LC_F16> {
  using T = __half;
  static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<LC_BF16> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
};

// Element offset of row r of an operand.
__device__ __forceinline__ uint64_t row_at(const Rows& g, const RowOperand& o, uint64_t r) {
  if (g.rank == 1) return o.offset + r * o.st[0];
  uint64_t at = o.offset;
  for (int d = g.rank - 1; d >= 0; d--) {
    const uint64_t n = g.shape[d];
    at += (r % n) * o.st[d];
    r /= n;
  }
  return at;
}

struct Soft {
  float m, s, t;
};

// What d is measured from: m, or 0 while there is nothing but masked places.
__device__ __forceinline__ float base_of(float m) { return m == neg_inf() ? 0.0f : m; }

__device__ __forceinline__ Soft merge(const Soft& a, const Soft& b, float c2) {
  Soft r;
  r.m = max_nan(a.m, b.m);
  const float base = base_of(r.m);
  // an empty part (m minus infinity) has s = t = 0: it keeps them, whatever the other part is measured from
  const float ua = a.m == neg_inf() ? 0.0f : max_nan((a.m - base) * c2, kFar);
  const float ub = b.m == neg_inf() ? 0.0f : max_nan((b.m - base) * c2, kFar);
  const float fa = ex2(ua), fb = ex2(ub);
  r.s = a.s * fa + b.s * fb;
  r.t = fa * (a.t + ua * a.s) + fb * (b.t + ub * b.s);
  return r;
}

__device__ __forceinline__ Soft warp_merge(Soft v, float c2) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Soft w{__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o), __shfl_xor_sync(0xffffffffu, v.t, o)};
    // the same operand order on both sides, so that every lane holds the same bits
    v = (threadIdx.x & o) ? merge(w, v, c2) : merge(v, w, c2);
  }
  return v;
}

// The whole block's part of the row, in every thread.  `red`: one entry for each warp.  Ends with a barrier before `red`
// may be written again only if the caller has one.
__device__ __forceinline__ Soft block_merge(Soft v, float c2, Soft* red) {
  v = warp_merge(v, c2);
  const int warps = blockDim.x / 32;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  Soft w = (int)(threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : Soft{neg_inf(), 0.0f, 0.0f};
  return warp_merge(w, c2);
}

// Order of the alternatives: by value, NaN above all, the two zeros equal; equal values by the lower index.  A larger key
// comes first, and no two keys of a row are equal.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if ((b & 0x7fffffffu) == 0u) return 0x80000000u;
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
  return ((uint64_t)order_of(x) << 32) | (uint64_t)(0xffffffffu - index);
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

// scale * (x - m) - log(s): minus infinity for a masked place and for every place of a row that is masked throughout
__device__ __forceinline__ float logprob_of(float x, float m, float total, float scale) {
  return x == neg_inf() && !isnan(m) && !isnan(total) ? neg_inf() : __fsub_rn(__fmul_rn(__fsub_rn(x, m), scale), total);
}

}  // namespace lcv
