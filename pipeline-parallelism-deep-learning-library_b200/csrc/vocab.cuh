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
#include <type_traits>

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

// ---- 16 bytes of a row at a time -------------------------------------------------------------

// two f32 operations in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// 16 bytes of logits as pairs of f32, their largest (NaN if any is), and pairs of f32 rounded back
template <int DT>
struct Vec {  // 16-bit types
  static constexpr int kElems = 8;
  using T2 = typename std::conditional<DT == LC_F16, __half2, __nv_bfloat162>::type;
  static __device__ __forceinline__ T2 word(uint32_t w) { return *reinterpret_cast<const T2*>(&w); }
  static __device__ __forceinline__ float2 up(uint32_t w) {
    if constexpr (DT == LC_F16) return __half22float2(word(w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t down(float2 v) {
    T2 w;
    if constexpr (DT == LC_F16) w = __float22half2_rn(v);
    else w = __float22bfloat162_rn(v);
    return *reinterpret_cast<const uint32_t*>(&w);
  }
  static __device__ __forceinline__ float2 pair(const uint4& q, int i) { return up(i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w); }
  static __device__ __forceinline__ float top(const uint4& q) {
    const T2 m = __hmax2_nan(__hmax2_nan(word(q.x), word(q.y)), __hmax2_nan(word(q.z), word(q.w)));
    const float2 f = up(*reinterpret_cast<const uint32_t*>(&m));
    return max_nan(f.x, f.y);
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&v)[4]) { return make_uint4(down(v[0]), down(v[1]), down(v[2]), down(v[3])); }
  static __device__ __forceinline__ uint4 masked() {
    const uint32_t w = DT == LC_F16 ? 0xfc00fc00u : 0xff80ff80u;
    return make_uint4(w, w, w, w);
  }
};
template <>
struct Vec<LC_F32> {
  static constexpr int kElems = 4;
  static __device__ __forceinline__ float2 pair(const uint4& q, int i) {
    return i == 0 ? make_float2(__uint_as_float(q.x), __uint_as_float(q.y)) : make_float2(__uint_as_float(q.z), __uint_as_float(q.w));
  }
  static __device__ __forceinline__ float top(const uint4& q) {
    return max_nan(max_nan(__uint_as_float(q.x), __uint_as_float(q.y)), max_nan(__uint_as_float(q.z), __uint_as_float(q.w)));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&v)[2]) {
    return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
  }
  static __device__ __forceinline__ uint4 masked() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
};

// 16 bytes that are read once
__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 q;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "l"(p));
  return q;
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
  const int warps = blockDim.x / 32;  // at most 32
  if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  Soft w = (int)(threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : Soft{neg_inf(), 0.0f, 0.0f};
  return warp_merge(w, c2);
}

// The softmax of what one thread has seen, in two lanes of sums.
struct Run {
  float m;
  float2 s, t;
};

// Takes up N vectors whose largest logit is `top`.  SUM_T: with the sum that the entropy needs.
template <int DT, int N, bool SUM_T>
__device__ __forceinline__ void take(Run& r, const uint4 (&q)[N], float top, float c2) {
  const float m = max_nan(r.m, top);
  if (!(m == r.m)) {  // a new largest logit (or a NaN): seldom, after the first vectors of a row
    const float u = r.m == neg_inf() ? 0.0f : max_nan((r.m - base_of(m)) * c2, kFar), f = ex2(u);
    if constexpr (SUM_T) r.t = mul2(both(f), fma2(both(u), r.s, r.t));
    r.s = mul2(both(f), r.s);
    r.m = m;
  }
  const float2 minus = both(-base_of(r.m)), c = both(c2);
#pragma unroll
  for (int n = 0; n < N; n++)
#pragma unroll
    for (int i = 0; i < Vec<DT>::kElems / 2; i++) {
      float2 d = mul2(add2(Vec<DT>::pair(q[n], i), minus), c);
      const float2 e = make_float2(ex2(d.x), ex2(d.y));
      r.s = add2(r.s, e);
      if constexpr (SUM_T) r.t = fma2(e, make_float2(max_nan(d.x, kFar), max_nan(d.y, kFar)), r.t);
    }
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
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o >> 31 ? (o == 0xffffffffu ? 0x7fffffffu : o ^ 0x80000000u) : ~o);
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

// scale * (x - m) - log(s): minus infinity for a masked place and for every place of a row that is masked throughout
__device__ __forceinline__ float logprob_of(float x, float m, float total, float scale) {
  return x == neg_inf() && !isnan(m) && !isnan(total) ? neg_inf() : __fsub_rn(__fmul_rn(__fsub_rn(x, m), scale), total);
}

// ---- a row shared by the blocks of a cluster --------------------------------------------------

// The 16-byte vectors of a row: `head` places before the first aligned one, `vecs` whole ones, `tail` places behind them.
struct Span {
  uint32_t head, vecs, tail;
};
template <int DT>
__device__ __forceinline__ Span span_of(const void* row, uint32_t vocab) {
  constexpr uint32_t kE = Vec<DT>::kElems, kBytes = 16 / kE;
  Span s;
  s.head = min(vocab, (uint32_t)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / kBytes);
  s.vecs = (vocab - s.head) / kE;
  s.tail = vocab - s.head - s.vecs * kE;
  return s;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// The address of this block's shared `p` in block `rank` of the cluster.
__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void store_remote(uint32_t at, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}
__device__ __forceinline__ void store_remote(uint32_t at, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}

}  // namespace lcv
