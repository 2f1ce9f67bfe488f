// token_logprobs.cu -- log probabilities of given tokens under a softmax over the vocabulary, with the entropy of the row
// and its best alternatives, and the gradient of both.
//
// With d_j = scale (x_j - m), m = max x and L = log sum e^d:  log p_j = d_j - L,  H = L - (sum e^d d) / (sum e^d).
// Gradient for g = d(total)/d(log p_t) and h = d(total)/dH:  dx_j = scale (g ([j = t] - p_j) - h p_j (log p_j + H)).
#include <cmath>

#include "vocab.cuh"

namespace {

using namespace lcv;

constexpr int kThreads = 256;
constexpr uint64_t kMaxTop = 128;
constexpr uint64_t kMaxGrid = 1u << 20;  // rows beyond it are looped over

struct ScoreArgs {
  Rows g;
  RowOperand x, targets, logprob, entropy, stats, top_lp, top_id;
  uint32_t vocab, top;
  float scale;
};

// One block a row, every element read where its stride puts it: once for the maximum and the sums, and once more for each
// alternative asked for.
template <int DT>
__global__ void __launch_bounds__(kThreads) token_logprobs_strided(ScoreArgs a) {
  using E = Elem<DT>;
  __shared__ Soft red[kThreads / 32];
  __shared__ uint64_t best[kThreads / 32];
  const float c2 = a.scale * kLog2e;
  for (uint64_t r = blockIdx.x; r < a.g.rows; r += gridDim.x) {
    const typename E::T* x = static_cast<const typename E::T*>(a.x.data) + row_at(a.g, a.x, r);
    Soft part{neg_inf(), 0.0f, 0.0f};
    for (uint32_t j = threadIdx.x; j < a.vocab; j += kThreads) {
      const float v = E::up(x[j * a.x.inner]);
      part = merge(part, Soft{v, v == neg_inf() ? 0.0f : 1.0f, 0.0f}, c2);
    }
    const Soft row = block_merge(part, c2, red);
    const float total = logf(row.s);
    if (threadIdx.x == 0) {
      if (a.logprob.data) {
        const uint32_t t = static_cast<const uint32_t*>(a.targets.data)[row_at(a.g, a.targets, r)];
        static_cast<float*>(a.logprob.data)[row_at(a.g, a.logprob, r)] =
            t < a.vocab ? logprob_of(E::up(x[t * a.x.inner]), row.m, total, a.scale) : 0.0f;
      }
      if (a.entropy.data)
        static_cast<float*>(a.entropy.data)[row_at(a.g, a.entropy, r)] =
            row.m == neg_inf() ? 0.0f : total - kLn2 * (row.t / row.s);
      if (a.stats.data) {
        float* st = static_cast<float*>(a.stats.data) + row_at(a.g, a.stats, r);
        st[0] = row.m;
        st[a.stats.inner] = total;
      }
    }
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < a.top; k++) {
      uint64_t k1 = 0;
      for (uint32_t j = threadIdx.x; j < a.vocab; j += kThreads) {
        const uint64_t key = key_of(E::up(x[j * a.x.inner]), j);
        if ((k == 0 || key < last) && key > k1) k1 = key;
      }
      for (int o = 16; o > 0; o >>= 1) {
        const uint64_t w = __shfl_xor_sync(0xffffffffu, k1, o);
        k1 = w > k1 ? w : k1;
      }
      __syncthreads();
      if ((threadIdx.x & 31) == 0) best[threadIdx.x / 32] = k1;
      __syncthreads();
      for (int w = 0; w < kThreads / 32; w++) k1 = best[w] > k1 ? best[w] : k1;
      last = k1;
      if (threadIdx.x == 0) {
        const uint32_t j = index_of(k1);
        if (a.top_lp.data)
          static_cast<float*>(a.top_lp.data)[row_at(a.g, a.top_lp, r) + k * a.top_lp.inner] =
              logprob_of(E::up(x[j * a.x.inner]), row.m, total, a.scale);
        if (a.top_id.data) static_cast<uint32_t*>(a.top_id.data)[row_at(a.g, a.top_id, r) + k * a.top_id.inner] = j;
      }
    }
    __syncthreads();
  }
}

struct GradArgs {
  Rows g;
  RowOperand x, targets, stats, entropy, d_logprob, d_entropy, dx;
  uint32_t vocab;
  float scale;
};

// What the gradient of a row is made of: dx = 2^d (at + bt d) with d = (x - m) scale log2(e), and the target's own share.
// 1 / sum is taken once a row as e^-L and not within the exponent, where L ~ 10 would cost the last bits of every place.
struct GradRow {
  float base, at, bt, own;
  uint32_t target;
};

__device__ __forceinline__ GradRow grad_row(const GradArgs& a, uint64_t r) {
  GradRow w;
  const float* st = static_cast<const float*>(a.stats.data) + row_at(a.g, a.stats, r);
  const float m = st[0], total = st[a.stats.inner];
  w.base = base_of(m);
  w.target = 0xffffffffu;
  float g = 0.0f, h = 0.0f, ent = 0.0f;
  if (a.d_logprob.data) {
    const uint32_t t = static_cast<const uint32_t*>(a.targets.data)[row_at(a.g, a.targets, r)];
    if (t < a.vocab) {
      w.target = t;
      g = static_cast<const float*>(a.d_logprob.data)[row_at(a.g, a.d_logprob, r)];
    }
  }
  if (a.d_entropy.data) {
    h = static_cast<const float*>(a.d_entropy.data)[row_at(a.g, a.d_entropy, r)];
    ent = static_cast<const float*>(a.entropy.data)[row_at(a.g, a.entropy, r)];
  }
  const float per = a.scale * expf(-total);
  w.own = g * a.scale;
  w.at = -per * (g + h * (ent - total));
  w.bt = -per * h * kLn2;
  if (m == neg_inf()) {  // masked throughout: there is no distribution, and no gradient
    w.at = w.bt = 0.0f;
    w.target = 0xffffffffu;
  }
  return w;
}

__device__ __forceinline__ float grad_of(float x, const GradRow& w, float c2) {
  const float d = max_nan((x - w.base) * c2, kFar);
  return ex2(d) * __fmaf_rn(w.bt, d, w.at);
}

template <int DT>
__global__ void __launch_bounds__(kThreads) token_logprobs_backward_strided(GradArgs a) {
  using E = Elem<DT>;
  const float c2 = a.scale * kLog2e;
  for (uint64_t r = blockIdx.x; r < a.g.rows; r += gridDim.x) {
    const typename E::T* x = static_cast<const typename E::T*>(a.x.data) + row_at(a.g, a.x, r);
    typename E::T* dx = static_cast<typename E::T*>(a.dx.data) + row_at(a.g, a.dx, r);
    const GradRow w = grad_row(a, r);
    for (uint32_t j = threadIdx.x; j < a.vocab; j += kThreads) {
      float v = grad_of(E::up(x[j * a.x.inner]), w, c2);
      if (j == w.target) v += w.own;
      dx[j * a.dx.inner] = E::down(v);
    }
  }
}

lc_status launched(lc_context* ctx, const char* name) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return lc::cuda_fail(e, name);
  lc::record_launch(ctx, name);
  return LC_OK;
}

bool good_scale(float s) { return std::isfinite(s) && s > 0.0f; }

unsigned row_grid(uint64_t rows) { return (unsigned)std::min<uint64_t>(rows, kMaxGrid); }

}  // namespace

using namespace lc;

extern "C" {

lc_status lc_encode_token_logprobs(lc_context* ctx, void* stream, const lc_view* logits, const lc_view* targets, float scale,
                                   const lc_view* logprob, const lc_view* entropy, const lc_view* stats,
                                   const lc_view* top_logprobs, const lc_view* top_ids) {
  Call c("token_logprobs", logits);
  lc_status st = c.start();
  if (st) return st;
  if (!good_scale(scale)) return c.bad("scale must be positive and finite");
  if (!logprob && !entropy && !stats && !top_logprobs && !top_ids) return c.bad("no output asked for");
  if ((targets == nullptr) != (logprob == nullptr)) return c.bad("targets and logprob come together");
  const lc_view* top = top_ids ? top_ids : top_logprobs;
  uint64_t k = 0;
  if (top) {
    if (top->rank != logits->rank) return c.bad("the alternatives must have the logits' leading shape and an axis of their own");
    k = top->shape[top->rank - 1];
    if (k < 1 || k > kMaxTop || k > c.vocab()) return c.bad("the number of alternatives must be 1 to 128 and at most the vocabulary");
  }
  if ((st = c.add(targets, "targets", -1, false)) || (st = c.add(logprob, "logprob", -1, true)) ||
      (st = c.add(entropy, "entropy", -1, true)) || (st = c.add(stats, "stats", 2, true)) ||
      (st = c.add(top_logprobs, "top_logprobs", (int64_t)k, true)) || (st = c.add(top_ids, "top_ids", (int64_t)k, true)))
    return st;
  if (targets && !is_index(targets->dtype)) return c.bad("targets must be i32 or u32");
  if (top_ids && !is_index(top_ids->dtype)) return c.bad("top_ids must be i32 or u32");
  for (const lc_view* v : {logprob, entropy, stats, top_logprobs})
    if (v && v->dtype != LC_F32) return c.bad("logprob, entropy, stats and top_logprobs must be f32");
  if ((st = c.finish(nullptr))) return st;
  if (ctx == nullptr) return c.bad("null context");
  ScoreArgs a{};
  a.g = c.rows();
  if (a.g.rows == 0) return LC_OK;
  a.x = c.operand(logits, a.g.rank);
  a.targets = c.operand(targets, a.g.rank);
  a.logprob = c.operand(logprob, a.g.rank);
  a.entropy = c.operand(entropy, a.g.rank);
  a.stats = c.operand(stats, a.g.rank);
  a.top_lp = c.operand(top_logprobs, a.g.rank);
  a.top_id = c.operand(top_ids, a.g.rank);
  a.vocab = (uint32_t)c.vocab();
  a.top = (uint32_t)k;
  a.scale = scale;
  DeviceGuard on(ctx->device);
  cudaStream_t s = stream_of(ctx, stream);
  const unsigned grid = row_grid(a.g.rows);
  if (logits->dtype == LC_F32) token_logprobs_strided<LC_F32><<<grid, kThreads, 0, s>>>(a);
  else if (logits->dtype == LC_F16) token_logprobs_strided<LC_F16><<<grid, kThreads, 0, s>>>(a);
  else token_logprobs_strided<LC_BF16><<<grid, kThreads, 0, s>>>(a);
  return launched(ctx, "token_logprobs_strided");
}

lc_status lc_encode_token_logprobs_backward(lc_context* ctx, void* stream, const lc_view* logits, const lc_view* targets,
                                            float scale, const lc_view* stats, const lc_view* entropy,
                                            const lc_view* d_logprob, const lc_view* d_entropy, const lc_view* dlogits) {
  Call c("token_logprobs_backward", logits);
  lc_status st = c.start();
  if (st) return st;
  if (!good_scale(scale)) return c.bad("scale must be positive and finite");
  if (!stats || !dlogits) return c.bad("null stats or dlogits");
  if (!d_logprob && !d_entropy) return c.bad("neither d_logprob nor d_entropy given");
  if (d_logprob && !targets) return c.bad("d_logprob needs the targets");
  if (d_entropy && !entropy) return c.bad("d_entropy needs the entropy");
  if ((st = c.add(targets, "targets", -1, false)) || (st = c.add(stats, "stats", 2, false)) ||
      (st = c.add(entropy, "entropy", -1, false)) || (st = c.add(d_logprob, "d_logprob", -1, false)) ||
      (st = c.add(d_entropy, "d_entropy", -1, false)) || (st = c.add(dlogits, "dlogits", (int64_t)c.vocab(), true)))
    return st;
  if (targets && !is_index(targets->dtype)) return c.bad("targets must be i32 or u32");
  for (const lc_view* v : {stats, entropy, d_logprob, d_entropy})
    if (v && v->dtype != LC_F32) return c.bad("stats, entropy, d_logprob and d_entropy must be f32");
  if (dlogits->dtype != logits->dtype) return c.bad("dlogits must have the logits' type");
  if ((st = c.finish(dlogits))) return st;
  if (ctx == nullptr) return c.bad("null context");
  GradArgs a{};
  a.g = c.rows();
  if (a.g.rows == 0) return LC_OK;
  a.x = c.operand(logits, a.g.rank);
  a.targets = c.operand(targets, a.g.rank);
  a.stats = c.operand(stats, a.g.rank);
  a.entropy = c.operand(entropy, a.g.rank);
  a.d_logprob = c.operand(d_logprob, a.g.rank);
  a.d_entropy = c.operand(d_entropy, a.g.rank);
  a.dx = c.operand(dlogits, a.g.rank);
  a.vocab = (uint32_t)c.vocab();
  a.scale = scale;
  DeviceGuard on(ctx->device);
  cudaStream_t s = stream_of(ctx, stream);
  const unsigned grid = row_grid(a.g.rows);
  if (logits->dtype == LC_F32) token_logprobs_backward_strided<LC_F32><<<grid, kThreads, 0, s>>>(a);
  else if (logits->dtype == LC_F16) token_logprobs_backward_strided<LC_F16><<<grid, kThreads, 0, s>>>(a);
  else token_logprobs_backward_strided<LC_BF16><<<grid, kThreads, 0, s>>>(a);
  return launched(ctx, "token_logprobs_backward_strided");
}

}  // extern "C"
