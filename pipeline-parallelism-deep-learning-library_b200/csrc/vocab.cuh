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
  static __device__ __forceinline__ float2 pair_bounded(const uint4& q, int i) {  // bf16: no place below -1e30
    const uint32_t low = 0xf149f149u;
    const T2 w = __hmax2_nan(word(i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w), word(low));
    return up(*reinterpret_cast<const uint32_t*>(&w));
  }
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

// 16 bytes that start `shift` bytes (0 to 15, a multiple of the element's size) into the 32 of lo and hi.
__device__ __forceinline__ uint4 shifted(const uint4& lo, const uint4& hi, uint32_t shift) {
  const bool two = shift & 8, one = shift & 4;
  const uint32_t a = two ? lo.z : lo.x, b = two ? lo.w : lo.y, c = two ? hi.x : lo.z, d = two ? hi.y : lo.w, e = two ? hi.z : hi.x,
                 f = two ? hi.w : hi.y;
  const uint32_t g = one ? b : a, h = one ? c : b, i = one ? d : c, j = one ? e : d, k = one ? f : e, bits = (shift & 3) * 8;
  return make_uint4(__funnelshift_r(g, h, bits), __funnelshift_r(h, i, bits), __funnelshift_r(i, j, bits), __funnelshift_r(j, k, bits));
}

// 16 bytes that start anywhere, place by place.
template <int DT>
__device__ __forceinline__ uint4 one_by_one(const void* at) {
  if constexpr (DT == LC_F32) {
    const uint32_t* p = static_cast<const uint32_t*>(at);
    return make_uint4(p[0], p[1], p[2], p[3]);
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(at);
    return make_uint4(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16, p[4] | (uint32_t)p[5] << 16, p[6] | (uint32_t)p[7] << 16);
  }
}

// 16 bytes with an L2 policy: kept for a second pass, or let go after it
__device__ __forceinline__ uint64_t keep_in_l2() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_last.b64 %0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint64_t leave_l2() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void bring_to_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
__device__ __forceinline__ uint4 load_with(const void* p, uint64_t policy) {
  uint4 q;
  asm volatile("ld.global.L1::no_allocate.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;"
               : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
               : "l"(p), "l"(policy)
               : "memory");
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

// The larger of a warp's values, or NaN if any is.
__device__ __forceinline__ float warp_top(float v) {
  float y;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(v));
  return y;
}

// A warp's parts, in every lane: moved to the common maximum first, then summed in a tree that is the same for all lanes.
__device__ __forceinline__ Soft warp_merge(Soft v, float c2) {
  const float m = warp_top(v.m);
  const float u = v.m == neg_inf() ? 0.0f : max_nan((v.m - base_of(m)) * c2, kFar), f = ex2(u);
  float s = v.s * f, t = f * (v.t + u * v.s);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    t += __shfl_xor_sync(0xffffffffu, t, o);
  }
  return Soft{m, s, t};
}

// The whole block's part of the row, in every thread.  `red`: one entry for each warp, of at most 32; the caller keeps a
// barrier between two uses.
__device__ __forceinline__ Soft block_merge(Soft v, float c2, Soft* red) {
  v = warp_merge(v, c2);
  const uint32_t warps = blockDim.x / 32, lane = threadIdx.x & 31;
  if (lane == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  return warp_merge(lane < warps ? red[lane] : Soft{neg_inf(), 0.0f, 0.0f}, c2);
}

// The softmax of what one thread has seen, in two lanes of sums.
//
// While m c2 is of an ordinary size, d is one fused multiply-add, x c2 - mc, against mc = m c2 as it rounds: one rounding a
// place, as good as (x - m) c2 with its two.  The sums then stand against mc / c2 and not m; soft_of moves them by the
// difference, off = m c2 - mc.  2^off is a factor of every sum on the way, and off is up to half a step of mc: it stays within
// 2^-5 below kWide, and would overflow the sums from 2^31 on (logits of -1e10, as forbidden tokens are often filled with).
// Rows beyond kWide, and scales far from 1, take (x - m) c2.  What a thread has seen may pass the border either way (its
// first places forbidden, say): the sums then move by the exact distance between what they stood against and what they will.
struct Run {
  float m, mc;
  float2 s, t;
};
constexpr float kWide = 1048576.0f;
__device__ __forceinline__ Run empty_run() { return Run{neg_inf(), 0.0f, make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)}; }
// NaN and the infinities are wide
__device__ __forceinline__ bool is_wide(float m, float c2) { return !(fabsf(m * c2) < kWide) || !(c2 > 1e-3f && c2 < 1e4f); }

// Takes up N vectors whose largest logit is `top`.  SUM_T: with the sum that the entropy needs.
template <int DT, int N, bool SUM_T>
__device__ __forceinline__ void take(Run& r, const uint4 (&q)[N], float top, float c2) {
  const float m = max_nan(r.m, top);
  const bool wide = is_wide(m, c2);
  if (!(m == r.m)) {  // a new largest logit (or a NaN): seldom, after the first vectors of a row
    const float mc = wide ? 0.0f : m * c2;
    const bool was = is_wide(r.m, c2);
    float u = wide ? (was ? (r.m - base_of(m)) * c2 : -__fmaf_rn(m, c2, -r.mc)) : was ? __fmaf_rn(r.m, c2, -mc) : r.mc - mc;
    u = r.m == neg_inf() ? 0.0f : max_nan(u, kFar);
    const float2 f = both(ex2(u));
    if constexpr (SUM_T) r.t = __fmul2_rn(f, __ffma2_rn(both(u), r.s, r.t));
    r.s = __fmul2_rn(f, r.s);
    r.m = m;
    r.mc = mc;
  }
  const float2 c = both(c2);
  if (!wide) {
    const float2 minus = both(-r.mc);
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
      for (int i = 0; i < Vec<DT>::kElems / 2; i++) {
        // a masked place must not give -inf * 0 in the product below: bf16 is bounded before it is widened, two places at a
        // time (-1e30 has weight 0 against an m of ordinary size), the other types behind
        float2 x;
        if constexpr (DT == LC_BF16 && SUM_T) x = Vec<DT>::pair_bounded(q[n], i);
        else x = Vec<DT>::pair(q[n], i);
        float2 d = __ffma2_rn(x, c, minus);
        const float2 e = make_float2(ex2(d.x), ex2(d.y));
        r.s = __fadd2_rn(r.s, e);
        if constexpr (SUM_T) {
          if constexpr (DT != LC_BF16) d = make_float2(max_nan(d.x, kFar), max_nan(d.y, kFar));
          r.t = __ffma2_rn(e, d, r.t);
        }
      }
    return;
  }
  const float2 minus = both(-base_of(r.m));
#pragma unroll
  for (int n = 0; n < N; n++)
#pragma unroll
    for (int i = 0; i < Vec<DT>::kElems / 2; i++) {
      const float2 d = __fmul2_rn(__fadd2_rn(Vec<DT>::pair(q[n], i), minus), c);
      const float2 e = make_float2(ex2(d.x), ex2(d.y));
      r.s = __fadd2_rn(r.s, e);
      if constexpr (SUM_T) r.t = __ffma2_rn(e, make_float2(max_nan(d.x, kFar), max_nan(d.y, kFar)), r.t);
    }
}

__device__ __forceinline__ Soft soft_of(const Run& r, float c2) {
  const float s = r.s.x + r.s.y, t = r.t.x + r.t.y;
  if (is_wide(r.m, c2)) return Soft{r.m, s, t};
  const float off = __fmaf_rn(r.m, c2, -r.mc), f = ex2(-off);  // m c2 - mc
  return Soft{r.m, s * f, f * (t - off * s)};
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
