// distill.cu -- distillation from a teacher's best alternatives: the divergence of the student's softmax over the whole
// vocabulary from what the teacher's list says, and its gradient.
//
// A row has the student's logits x over the vocabulary V and the teacher's list of places id_k with values z_k.  Entries
// outside [0, V) are padding; of a place that the list names twice the first entry stands.  q = softmax(scale x), and over
// the entries that stand
//   renormalised:  P = softmax(scale z), r = 0
//   with a tail:   P = e^z (z are log probabilities), r = max(0, 1 - sum P), one bucket for the places outside the list,
//                  to which the student gives Q = sum of q over them; a tail where Q = 0 is left out
//   loss = sum P (log P - log q_id) + r (log r - log Q)
// With c = sum P + r, the gradient with respect to x_j is
//   scale (c q_j - P_k) at the place of entry k,   scale q_j (c - r / Q) outside the list.
// Outside the list everything is measured from the largest logit there (mt, with St = sum e^(scale (x - mt))): the second
// form is e^(scale (x_j - mt)) (c e^(scale (mt - m)) / S - r / St), which stands also where Q underflows.
#include <cmath>

#include "vocab.cuh"

namespace {

using namespace lcv;

constexpr int kThreads = 256;
constexpr uint64_t kMaxList = 256;
constexpr uint64_t kMaxGrid = 1u << 20;
constexpr uint32_t kChunk = 8192;  // places whose list membership is held at once, one bit each

struct DistillArgs {
  Rows g;
  RowOperand x, ids, teacher, d_loss, loss, dx;
  uint32_t vocab, list;
  int teacher_type;
  int tail;
  float scale;
};

struct List {
  uint32_t id[kMaxList];   // a place, or ~0 for an entry that does not stand
  float p[kMaxList];       // the teacher's share
  float logp[kMaxList];
  float x[kMaxList];       // the student's logit there
};

__device__ __forceinline__ float teacher_value(const DistillArgs& a, uint64_t at) {
  if (a.teacher_type == LC_F32) return static_cast<const float*>(a.teacher.data)[at];
  if (a.teacher_type == LC_F16) return __half2float(static_cast<const __half*>(a.teacher.data)[at]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(a.teacher.data)[at]);
}

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0.0;
  for (int w = 0; w < (int)blockDim.x / 32; w++) v += red[w];
  __syncthreads();
  return v;
}

__device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < (int)blockDim.x / 32; w++) v = max_nan(v, red[w]);
  __syncthreads();
  return v;
}

// The teacher's list of row r in shared memory, with sum P in `sum` (64 bits: r = 1 - sum P loses what 32 bits round off).
__device__ __forceinline__ void read_list(const DistillArgs& a, uint64_t r, List& l, float* redf, double* redd, double* sum) {
  const uint32_t* ids = static_cast<const uint32_t*>(a.ids.data) + row_at(a.g, a.ids, r);
  const uint64_t zat = row_at(a.g, a.teacher, r);
  for (uint32_t k = threadIdx.x; k < a.list; k += blockDim.x) l.id[k] = ids[k * a.ids.inner];
  __syncthreads();
  // an entry stands if its place is in the vocabulary and no earlier entry names it; at most one entry a thread
  const uint32_t k = threadIdx.x;
  bool stands = k < a.list && l.id[k] < a.vocab;
  if (stands)
    for (uint32_t i = 0; i < k; i++)
      if (l.id[i] == l.id[k]) {
        stands = false;
        break;
      }
  const float z = stands ? teacher_value(a, zat + k * a.teacher.inner) : neg_inf();
  float top = 0.0f;
  if (!a.tail) {
    top = base_of(block_max(z, redf));
  }
  double e = 0.0, lz = 0.0;
  if (stands) {
    lz = a.tail ? (double)z : (double)a.scale * ((double)z - (double)top);
    e = exp(lz);
  }
  double total = block_sum(e, redd);  // its barriers also order the reads of l.id above before the writes below
  if (k < a.list) {
    if (!stands) l.id[k] = 0xffffffffu;
    double p = e, lp = lz;
    if (!a.tail && stands) {
      p = total > 0.0 || isnan(total) ? e / total : 0.0;
      lp = lz - log(total);
    }
    l.p[k] = (float)p;
    l.logp[k] = (float)lp;
  }
  *sum = a.tail ? total : (total > 0.0 ? 1.0 : (isnan(total) ? total : 0.0));
  __syncthreads();
}

// What a row's loss and gradient are made of once the row and the list are summed up.
struct RowPlan {
  float base, coef;        // outside the list: dx = coef e^(scale (x - base))
  float in_base, in_coef;  // in the list: dx = in_coef e^(scale (x - in_base)) - weight P
  float weight;
};

__device__ __forceinline__ RowPlan plan_row(const DistillArgs& a, const Soft& rest, const Soft& all, double sum, float d_loss,
                                            double* tail_loss) {
  RowPlan w;
  double r = a.tail ? 1.0 - sum : 0.0;
  if (r < 0.0 || rest.s == 0.0f) r = 0.0;
  const double c = sum + r;
  const float lead = (base_of(rest.m) - base_of(all.m)) * a.scale;  // at most 0
  // log Q = log(St) + scale (mt - m) - log(S)
  *tail_loss = r > 0.0 ? r * (log(r) - ((double)logf(rest.s) + (double)lead - (double)logf(all.s))) : r;
  w.weight = d_loss * a.scale;
  w.base = base_of(rest.m);
  w.in_base = base_of(all.m);
  w.coef = rest.s == 0.0f ? 0.0f : (float)(c * (double)expf(lead) / (double)all.s - r / (double)rest.s) * w.weight;
  w.in_coef = all.s == 0.0f ? 0.0f : (float)(c / (double)all.s) * w.weight;
  if (all.m == neg_inf()) w.weight = 0.0f;  // masked throughout: there is no distribution, and no gradient
  return w;
}

// One block a row, every element read where its stride puts it, the list's places told apart by a bitmap of kChunk places
// at a time: once for the sums, once more for the gradient.
template <int DT, bool GRAD>
__global__ void __launch_bounds__(kThreads) distill_strided(DistillArgs a) {
  using E = Elem<DT>;
  __shared__ List l;
  __shared__ uint32_t in_list[kChunk / 32];
  __shared__ Soft red[kThreads / 32];
  __shared__ float redf[kThreads / 32];
  __shared__ double redd[kThreads / 32];
  const float c2 = a.scale * kLog2e;
  for (uint64_t r = blockIdx.x; r < a.g.rows; r += gridDim.x) {
    const typename E::T* x = static_cast<const typename E::T*>(a.x.data) + row_at(a.g, a.x, r);
    double sum;
    read_list(a, r, l, redf, redd, &sum);
    const uint32_t k = threadIdx.x;
    const bool stands = k < a.list && l.id[k] != 0xffffffffu;
    const float xk = stands ? E::up(x[l.id[k] * a.x.inner]) : neg_inf();

    auto chunk = [&](uint32_t from) {  // bits of the places from, from + 1, ...
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < kChunk / 32; i += kThreads) in_list[i] = 0;
      __syncthreads();
      if (stands && l.id[k] >= from && l.id[k] - from < kChunk) atomicOr(&in_list[(l.id[k] - from) / 32], 1u << (l.id[k] - from) % 32);
      __syncthreads();
    };
    auto listed = [&](uint32_t i) { return (in_list[i / 32] >> (i % 32)) & 1u; };

    Soft part{neg_inf(), 0.0f, 0.0f};
    for (uint32_t from = 0; from < a.vocab; from += kChunk) {
      chunk(from);
      const uint32_t n = min(kChunk, a.vocab - from);
      for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        if (listed(i)) continue;
        const float v = E::up(x[(from + i) * a.x.inner]);
        part = merge(part, Soft{v, v == neg_inf() ? 0.0f : 1.0f, 0.0f}, c2);
      }
    }
    const Soft rest = block_merge(part, c2, red);
    __syncthreads();
    const Soft named = block_merge(Soft{xk, xk == neg_inf() ? 0.0f : 1.0f, 0.0f}, c2, red);
    const Soft all = merge(rest, named, c2);
    double tail_loss;
    const float d_loss = a.d_loss.data ? static_cast<const float*>(a.d_loss.data)[row_at(a.g, a.d_loss, r)] : 1.0f;
    const RowPlan w = plan_row(a, rest, all, sum, d_loss, &tail_loss);
    if (a.loss.data) {
      double own = 0.0;
      if (stands && l.p[k] != 0.0f)
        own = (double)l.p[k] * ((double)l.logp[k] - (double)logprob_of(xk, all.m, logf(all.s), a.scale));
      const double total = block_sum(own, redd) + tail_loss;
      if (threadIdx.x == 0) static_cast<float*>(a.loss.data)[row_at(a.g, a.loss, r)] = (float)total;
    }
    if constexpr (GRAD) {
      typename E::T* dx = static_cast<typename E::T*>(a.dx.data) + row_at(a.g, a.dx, r);
      for (uint32_t from = 0; from < a.vocab; from += kChunk) {
        chunk(from);
        const uint32_t n = min(kChunk, a.vocab - from);
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
          if (listed(i)) continue;
          const float v = E::up(x[(from + i) * a.x.inner]);
          dx[(from + i) * a.dx.inner] = E::down(ex2((v - w.base) * c2) * w.coef);
        }
      }
      if (stands) dx[l.id[k] * a.dx.inner] = E::down(ex2((xk - w.in_base) * c2) * w.in_coef - w.weight * l.p[k]);
    }
    __syncthreads();
  }
}

lc_status launched(lc_context* ctx, const char* name) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return lc::cuda_fail(e, name);
  lc::record_launch(ctx, name);
  return LC_OK;
}

template <bool GRAD>
void launch(const DistillArgs& a, int32_t dtype, unsigned grid, cudaStream_t s) {
  if (dtype == LC_F32) distill_strided<LC_F32, GRAD><<<grid, kThreads, 0, s>>>(a);
  else if (dtype == LC_F16) distill_strided<LC_F16, GRAD><<<grid, kThreads, 0, s>>>(a);
  else distill_strided<LC_BF16, GRAD><<<grid, kThreads, 0, s>>>(a);
}

lc_status distill(const char* op, lc_context* ctx, void* stream, const lc_view* logits, const lc_view* ids,
                  const lc_view* teacher, float scale, int32_t tail, const lc_view* d_loss, const lc_view* loss,
                  const lc_view* dlogits) {
  using namespace lc;
  Call c(op, logits);
  lc_status st = c.start();
  if (st) return st;
  if (!std::isfinite(scale) || !(scale > 0.0f)) return c.bad("scale must be positive and finite");
  if (tail != 0 && tail != 1) return c.bad("tail is 0 (renormalised) or 1 (a bucket for the rest)");
  if (!ids || !teacher) return c.bad("null ids or teacher");
  if (ids->rank != logits->rank) return c.bad("ids must have the logits' leading shape and an axis of their own");
  const uint64_t k = ids->shape[ids->rank - 1];
  if (k > kMaxList) return c.bad("the teacher's list holds at most 256 entries a row");
  if ((st = c.add(ids, "ids", (int64_t)k, false)) || (st = c.add(teacher, "teacher", (int64_t)k, false)) ||
      (st = c.add(d_loss, "d_loss", -1, false)) || (st = c.add(loss, "loss", -1, true)) ||
      (st = c.add(dlogits, "dlogits", (int64_t)c.vocab(), true)))
    return st;
  if (!is_index(ids->dtype)) return c.bad("ids must be i32 or u32");
  if (!is_float(teacher->dtype)) return c.bad("teacher must be f32, f16 or bf16");
  for (const lc_view* v : {d_loss, loss})
    if (v && v->dtype != LC_F32) return c.bad("loss and d_loss must be f32");
  if (dlogits && dlogits->dtype != logits->dtype) return c.bad("dlogits must have the logits' type");
  if ((st = c.finish(dlogits))) return st;
  if (ctx == nullptr) return c.bad("null context");
  DistillArgs a{};
  a.g = c.rows();
  if (a.g.rows == 0) return LC_OK;
  a.x = c.operand(logits, a.g.rank);
  a.ids = c.operand(ids, a.g.rank);
  a.teacher = c.operand(teacher, a.g.rank);
  a.d_loss = c.operand(d_loss, a.g.rank);
  a.loss = c.operand(loss, a.g.rank);
  a.dx = c.operand(dlogits, a.g.rank);
  a.vocab = (uint32_t)c.vocab();
  a.list = (uint32_t)k;
  a.teacher_type = teacher->dtype;
  a.tail = tail;
  a.scale = scale;
  DeviceGuard on(ctx->device);
  cudaStream_t s = stream_of(ctx, stream);
  const unsigned grid = (unsigned)std::min<uint64_t>(a.g.rows, kMaxGrid);
  if (dlogits) launch<true>(a, logits->dtype, grid, s);
  else launch<false>(a, logits->dtype, grid, s);
  return launched(ctx, dlogits ? "distill_grad_strided" : "distill_loss_strided");
}

}  // namespace

extern "C" {

lc_status lc_encode_distill_loss(lc_context* ctx, void* stream, const lc_view* logits, const lc_view* ids,
                                 const lc_view* teacher, float scale, int32_t tail, const lc_view* loss) {
  if (loss == nullptr) return lc::fail(LC_ERR_INVALID_ARGUMENT, "distill_loss: null loss");
  return distill("distill_loss", ctx, stream, logits, ids, teacher, scale, tail, nullptr, loss, nullptr);
}

lc_status lc_encode_distill_grad(lc_context* ctx, void* stream, const lc_view* logits, const lc_view* ids,
                                 const lc_view* teacher, float scale, int32_t tail, const lc_view* d_loss,
                                 const lc_view* loss, const lc_view* dlogits) {
  if (dlogits == nullptr) return lc::fail(LC_ERR_INVALID_ARGUMENT, "distill_grad: null dlogits");
  return distill("distill_grad", ctx, stream, logits, ids, teacher, scale, tail, d_loss, loss, dlogits);
}

}  // extern "C"
