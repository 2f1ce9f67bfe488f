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

// ---- the vocabulary as the unit axis -----------------------------------------------------------
//
// One block a row, or a cluster of blocks where there are few rows, each with a slice.  Two passes over the slice: the sums,
// in which a bit for each place tells the list's places, and the gradient.  Between them the blocks of a cluster tell one
// another their sums.  The second pass finds most of the row in L2: the first reads it with a policy that keeps it there,
// the second one that lets it go, and the gradient is stored past the caches.
//
// What bounds it (B200, of the 6465 GB/s of a copy).  The loss alone reads HBM at 6128 GB/s (4096 x 131,072 bf16, 64 entries:
// 176 us).  With the gradient it is 450 us, 4780 GB/s of the bytes that must move: 1.15 times the logits come from HBM
// (some lines are gone before the second pass), and a block's chain from its list over the sums to the gradient leaves the
// memory idle where the other block of its SM cannot fill in.  A fetch of the row's first 128 KB (half of it) into L2 before
// the list took 454 to 446 us (4096 x 32,768 f32: 203 to 192); of the whole row, 509; on short rows and for the loss alone it
// cost time.  Tried and slower: the row in shared memory over a cluster of 8 blocks filled by the copy engine, one pass after
// the other (755 us) or with the next row's sums before this row's gradient (811 us; the fixed work of a block weighs 8
// times); the first 88 KB of a row in shared memory (527 us); lists a row ahead and gradient tiles to whichever warp is free
// (486 us); three or four smaller blocks an SM (505 to 521 us: more rows under way than L2 holds).
// Rows from about 400 KB on are too long for that: 296 of them are more than L2's 126 MB, and most of the second pass comes
// from HBM too (2048 x 131,072 f32: 474 us, floor 332; over 1024 such rows 1.73 times the logits are read).
// Many short rows with long lists are bound by the fixed work of a row, its list above all (8000 x 2001 bf16: 38 us with 16
// entries, 70 with 128, floor 10 and 11; the loss alone with 128: 50).
template <int DT>
constexpr int kUnroll = 32 / Vec<DT>::kElems;  // vectors of a step: 32 places a thread
template <bool GRAD>
constexpr int kRowThreads = GRAD ? 512 : 256;
template <int DT, bool GRAD>
constexpr int kResident = GRAD ? 2 : DT == LC_F32 ? 4 : 6;  // blocks an SM (loss alone, bf16: 178 us with 6, 197 with 4)
constexpr uint32_t kMaxCluster = 8;
constexpr uint64_t kLongSlice = 128 << 10;  // bytes
constexpr uint32_t kAhead = 8192;  // vectors
constexpr uint64_t kMaxBits = 64 << 10;  // bytes of shared memory for a slice's bits

// A thread's entry of the list.
struct Entry {
  uint32_t id;  // ~0 if it does not stand
  double p;     // 64 bits: the loss has sum P scale x beside sum P log P, which cancel to a small part
};

// The teacher's list and the student's logits at its places are worked out by the first `warps` warps, an entry a thread,
// while the others go on with the row.
__device__ __forceinline__ void list_sync(uint32_t warps) {
  if (warps > 1) asm volatile("bar.sync 1, %0;" ::"r"(warps * 32) : "memory");
  else __syncwarp();
}

struct Said {
  double sum, plogp;  // sum P and sum P log P over the entries that stand
  Soft named;         // the student's logits there
};

struct ListWork {  // shared memory of the list's warps
  float top[kMaxList / 32];
  double2 sums[kMaxList / 32];
  Soft named[kMaxList / 32];
};

__device__ __forceinline__ double2 warp_sum(double2 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  return v;
}

// Called by the list's warps: drops this thread's entry if an earlier one names the same place, weighs it, and leaves in
// `said` what the whole list says.  `xk`: the student's logit at the entry's place.
__device__ __forceinline__ void weigh(const DistillArgs& a, const uint32_t* ids, float z, float* xk, Entry* entry, uint32_t warps,
                                      float c2, ListWork* work, Said* said) {
  Entry e = *entry;
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  if (e.id != 0xffffffffu) {
    bool again = false;
    for (uint32_t i = 0; i < threadIdx.x; i++) again |= ids[i] == e.id;
    if (again) e.id = 0xffffffffu;
  }
  if (e.id == 0xffffffffu) z = *xk = neg_inf();
  double lz = z, w = 0.0;
  if (!a.tail) {
    float top = warp_top(z);
    if (warps > 1) {
      if (lane == 0) work->top[warp] = top;
      list_sync(warps);
      top = warp_top(lane < warps ? work->top[lane] : neg_inf());
    }
    lz = (double)a.scale * ((double)z - (double)base_of(top));
  }
  if (e.id != 0xffffffffu) w = exp(lz);
  double2 t = warp_sum(make_double2(w, w > 0.0 || isnan(w) ? w * lz : 0.0));
  Soft named = warp_merge(Soft{*xk, *xk == neg_inf() ? 0.0f : 1.0f, 0.0f}, c2);
  if (warps > 1) {
    if (lane == 0) {
      work->sums[warp] = t;
      work->named[warp] = named;
    }
    list_sync(warps);
    t = warp_sum(lane < warps ? work->sums[lane] : make_double2(0.0, 0.0));
    named = warp_merge(lane < warps ? work->named[lane] : Soft{neg_inf(), 0.0f, 0.0f}, c2);
  }
  e.p = w;
  double sum = t.x, plogp = t.y;
  if (!a.tail) {
    // of the renormalised P = w / total: sum P log P = (sum w lz) / total - log total
    if (t.x > 0.0 || isnan(t.x)) {
      e.p = w / t.x;
      sum = isnan(t.x) ? t.x : 1.0;
      plogp = t.y / t.x - log(t.x);
    } else {  // no entry says anything
      e.p = sum = plogp = 0.0;
    }
  }
  if (threadIdx.x == 0) *said = Said{sum, plogp, named};
  *entry = e;
}

// dx = coef 2^d outside the list, in the same two forms of d as take (vocab.cuh)
struct Tail {
  float minus, coef;
  bool wide;
};

template <int DT>
__device__ __forceinline__ uint4 tail_vec(const uint4& q, const Tail& w, float c2) {
  constexpr int kP = Vec<DT>::kElems / 2;
  float2 y[kP];
  const float2 minus = both(w.minus), c = both(c2), coef = both(w.coef);
  if (!w.wide) {
#pragma unroll
    for (int i = 0; i < kP; i++) y[i] = __ffma2_rn(Vec<DT>::pair(q, i), c, minus);
  } else {
#pragma unroll
    for (int i = 0; i < kP; i++) y[i] = __fmul2_rn(__fadd2_rn(Vec<DT>::pair(q, i), minus), c);
  }
#pragma unroll
  for (int i = 0; i < kP; i++) y[i] = __fmul2_rn(make_float2(ex2(y[i].x), ex2(y[i].y)), coef);
  return Vec<DT>::pack(y);
}

__device__ __forceinline__ float tail_of(float x, const Tail& w, float c2) {
  return ex2(w.wide ? (x + w.minus) * c2 : __fmaf_rn(x, c2, w.minus)) * w.coef;
}

// `bits` say which places of a vector are the list's: they become minus infinity.
template <int DT>
__device__ __forceinline__ void take_out(uint4& q, uint32_t bits) {
  uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (DT == LC_F32) {
      if (bits >> i & 1) w[i] = 0xff800000u;
    } else {
      const uint32_t inf = DT == LC_F16 ? 0xfc00u : 0xff80u;
      if (bits >> (2 * i) & 1) w[i] = (w[i] & 0xffff0000u) | inf;
      if (bits >> (2 * i + 1) & 1) w[i] = (w[i] & 0xffffu) | inf << 16;
    }
  }
  q = make_uint4(w[0], w[1], w[2], w[3]);
}

template <int DT, bool GRAD, bool MOVED>
__global__ void __launch_bounds__(kRowThreads<GRAD>, kResident<DT, GRAD>) distill_rows(DistillArgs a, uint32_t cluster, uint32_t share) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr uint32_t kE = Vec<DT>::kElems;
  constexpr int kU = kUnroll<DT>;
  extern __shared__ __align__(16) uint8_t in_list[];  // [share], a multiple of 16: a byte a vector, a bit a place
  __shared__ uint32_t ids[kMaxList];
  __shared__ Soft red[kRowThreads<GRAD> / 32];
  __shared__ float edges[16];
  __shared__ ListWork work;
  __shared__ Said said;
  __shared__ float2 parts[kMaxCluster];  // (m, s) of the places outside the list, from each block of the cluster
  const uint32_t rank = cluster > 1 ? cluster_rank() : 0, list_warps = max(1u, (a.list + 31) / 32);
  const float c2 = a.scale * kLog2e;
  const uint64_t keep = keep_in_l2(), leave = leave_l2();
  // Cluster barriers alternate: every block's `parts` are free (at first: it has started), and they are filled.
  if (cluster > 1) cluster_arrive();
  for (uint64_t r = blockIdx.x / cluster; r < a.g.rows; r += gridDim.x / cluster) {
    const T* x = static_cast<const T*>(a.x.data) + row_at(a.g, a.x, r);
    const Span span = span_of<DT>(x, a.vocab);
    const uint32_t from = min(span.vecs, rank * share), to = min(span.vecs, from + share);
    const uint4* vec = reinterpret_cast<const uint4*>(x + span.head);
    // the first 128 KB of a long slice come while the list does, a line of 8 vectors at a time
    if (GRAD && blockDim.x == kRowThreads<GRAD>)
      for (uint32_t v = from + threadIdx.x * 8; v < min(to, from + kAhead); v += blockDim.x * 8) bring_to_l2(vec + v);
    Entry entry{0xffffffffu, 0.0};
    float z = neg_inf(), xk = neg_inf();
    if (threadIdx.x < a.list) {
      entry.id = static_cast<const uint32_t*>(a.ids.data)[row_at(a.g, a.ids, r) + threadIdx.x * a.ids.inner];
      z = teacher_value(a, row_at(a.g, a.teacher, r) + threadIdx.x * a.teacher.inner);
      ids[threadIdx.x] = entry.id;
      if (entry.id < a.vocab) xk = E::up(x[entry.id]);
      else entry.id = 0xffffffffu;
    }
    // the places before the vectors (0-7) and behind them (8-15) are block 0's
    uint32_t edge_at = 0xffffffffu;
    if (rank == 0 && threadIdx.x < 16) {
      const uint32_t i = threadIdx.x & 7;
      if (threadIdx.x < 8 ? i < span.head : i < span.tail) {
        edge_at = threadIdx.x < 8 ? i : span.head + span.vecs * kE + i;
        edges[threadIdx.x] = E::up(x[edge_at]);
      }
    }
    for (uint32_t i = threadIdx.x; i < (to - from + 15) / 16; i += blockDim.x) reinterpret_cast<uint4*>(in_list)[i] = make_uint4(0, 0, 0, 0);
    const float d_loss = GRAD && a.d_loss.data ? static_cast<const float*>(a.d_loss.data)[row_at(a.g, a.d_loss, r)] : 1.0f;
    __syncthreads();
    // where the entry's place lies: in the slice's vectors, or among the edges
    bool mine = false;
    if (entry.id != 0xffffffffu) {
      const uint32_t at = entry.id - span.head, v = at / kE;
      if (entry.id >= span.head && at < span.vecs * kE) {
        mine = v >= from && v < to;
        if (mine) atomicOr(reinterpret_cast<uint32_t*>(in_list) + (v - from) / 4, 1u << ((v - from) % 4 * 8 + at % kE));
      } else if (rank == 0) {
        edges[entry.id < span.head ? entry.id : 8 + at - span.vecs * kE] = neg_inf();
        mine = true;
      }
    }
    __syncthreads();
    if (threadIdx.x / 32 < list_warps) weigh(a, ids, z, &xk, &entry, list_warps, c2, &work, &said);
    mine = mine && entry.id != 0xffffffffu;
    Run run = empty_run();
    {
      const uint32_t step = kU * blockDim.x;
      const uint8_t* bits = in_list - from;
      uint32_t v0 = from;
      for (; v0 + step <= to; v0 += step) {
        uint4 q[kU];
        uint32_t m[kU], any = 0;
#pragma unroll
        for (int u = 0; u < kU; u++) q[u] = GRAD ? load_with(vec + v0 + u * blockDim.x + threadIdx.x, keep) : load_once(vec + v0 + u * blockDim.x + threadIdx.x);
#pragma unroll
        for (int u = 0; u < kU; u++) any |= m[u] = bits[v0 + u * blockDim.x + threadIdx.x];
        if (any) {
#pragma unroll
          for (int u = 0; u < kU; u++) take_out<DT>(q[u], m[u]);
        }
        float top = Vec<DT>::top(q[0]);
#pragma unroll
        for (int u = 1; u < kU; u++) top = max_nan(top, Vec<DT>::top(q[u]));
        take<DT, kU, false>(run, q, top, c2);
      }
      if (v0 + threadIdx.x < to) {  // the last step, short of some vectors: masked ones in their place
        uint4 q[kU];
#pragma unroll
        for (int u = 0; u < kU; u++) {
          const uint4* p = vec + v0 + u * blockDim.x + threadIdx.x;
          q[u] = v0 + u * blockDim.x + threadIdx.x >= to ? Vec<DT>::masked() : GRAD ? load_with(p, keep) : load_once(p);
        }
#pragma unroll
        for (int u = 0; u < kU; u++)
          if (v0 + u * blockDim.x + threadIdx.x < to) take_out<DT>(q[u], bits[v0 + u * blockDim.x + threadIdx.x]);
        float top = Vec<DT>::top(q[0]);
#pragma unroll
        for (int u = 1; u < kU; u++) top = max_nan(top, Vec<DT>::top(q[u]));
        take<DT, kU, false>(run, q, top, c2);
      }
    }
    Soft rest = soft_of(run, c2);
    if (edge_at != 0xffffffffu) {
      const float e = edges[threadIdx.x];
      rest = merge(rest, Soft{e, e == neg_inf() ? 0.0f : 1.0f, 0.0f}, c2);
    }
    rest = block_merge(rest, c2, red);  // its barrier is also that of `said`
    const Soft named = said.named;
    if (cluster > 1) {
      cluster_wait();
      if (threadIdx.x < cluster) {
        const uint32_t to_part = remote(&parts[rank], threadIdx.x);
        store_remote(to_part, rest.m);
        store_remote(to_part + 4, rest.s);
      }
      cluster_arrive();
      cluster_wait();
      const uint32_t lane = threadIdx.x & 31;
      rest = warp_merge(lane < cluster ? Soft{parts[lane].x, parts[lane].y, 0.0f} : Soft{neg_inf(), 0.0f, 0.0f}, c2);
      cluster_arrive();
    }
    const Soft all = merge(rest, named, c2);
    double left = a.tail ? 1.0 - said.sum : 0.0;
    if (left < 0.0 || rest.s == 0.0f) left = 0.0;
    const float total = (float)(said.sum + left), tail = (float)left;
    const float lead = (base_of(rest.m) - base_of(all.m)) * a.scale;  // at most 0 where it counts
    if constexpr (GRAD) {
      float weight = d_loss * a.scale;
      // against mc / c2, which is where 2^d is taken from (vocab.cuh)
      Tail w;
      w.wide = is_wide(rest.m, c2);
      w.minus = w.wide ? -base_of(rest.m) : -(rest.m * c2);
      const float off = w.wide ? 0.0f : __fmaf_rn(rest.m, c2, w.minus);
      w.coef = rest.s == 0.0f ? 0.0f : (total * expf(lead) / all.s - tail / rest.s) * weight * ex2(-off);
      const float in_coef = all.s == 0.0f ? 0.0f : total / all.s * weight;
      if (all.m == neg_inf()) weight = 0.0f;  // masked throughout: there is no distribution, and no gradient
      T* dx = static_cast<T*>(a.dx.data) + row_at(a.g, a.dx, r);
      if constexpr (!MOVED) {
        uint4* const dv = reinterpret_cast<uint4*>(dx + span.head);
        const uint32_t step = 4 * blockDim.x;
        uint32_t v0 = from + threadIdx.x;
        for (; v0 + 3 * blockDim.x < to; v0 += step) {
          uint4 q[4];
#pragma unroll
          for (int u = 0; u < 4; u++) q[u] = load_with(vec + v0 + u * blockDim.x, leave);
#pragma unroll
          for (int u = 0; u < 4; u++) __stcs(dv + v0 + u * blockDim.x, tail_vec<DT>(q[u], w, c2));
        }
        if (v0 < to) {
          uint4 q[4];
#pragma unroll
          for (int u = 0; u < 4; u++)
            if (v0 + u * blockDim.x < to) q[u] = load_with(vec + v0 + u * blockDim.x, leave);
#pragma unroll
          for (int u = 0; u < 4; u++)
            if (v0 + u * blockDim.x < to) __stcs(dv + v0 + u * blockDim.x, tail_vec<DT>(q[u], w, c2));
        }
      } else {
        // the slice's places, as whole vectors of dx: each is cut out of two aligned ones of x, of which the second comes
        // from the next lane
        const uint32_t places = (to - from) * kE, lane = threadIdx.x & 31;
        T* const out = dx + span.head + from * kE;
        const Span os = span_of<DT>(out, places);
        const uint32_t shift = os.head * (16 / kE);
        uint4* const dv = reinterpret_cast<uint4*>(out + os.head);
        const uint4* const xa = vec + from;  // vector i of dx is cut out of i and i + 1
        for (uint32_t v0 = (threadIdx.x & ~31u) * 4; v0 < os.vecs; v0 += 4 * blockDim.x) {
          uint4 q[4], last = make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int u = 0; u < 4; u++) {
            const uint32_t v = v0 + u * 32 + lane;
            q[u] = v < to - from ? load_with(xa + v, leave) : make_uint4(0, 0, 0, 0);
          }
          if (lane == 31 && v0 + 128 < to - from) last = load_with(xa + v0 + 128, leave);
#pragma unroll
          for (int u = 0; u < 4; u++) {
            uint4 give = q[u];
            if (u + 1 < 4 && lane == 0) give = q[u + 1 < 4 ? u + 1 : u];
            uint4 next = make_uint4(__shfl_sync(0xffffffffu, give.x, lane + 1), __shfl_sync(0xffffffffu, give.y, lane + 1),
                                    __shfl_sync(0xffffffffu, give.z, lane + 1), __shfl_sync(0xffffffffu, give.w, lane + 1));
            if (u + 1 == 4 && lane == 31) next = last;
            const uint32_t v = v0 + u * 32 + lane;
            if (v < os.vecs) __stcs(dv + v, tail_vec<DT>(shifted(q[u], next, shift), w, c2));
          }
        }
        if (threadIdx.x < 16) {
          const uint32_t i = threadIdx.x & 7;
          if (threadIdx.x < 8 ? i < os.head : i < os.tail) {
            const uint32_t j = threadIdx.x < 8 ? i : os.head + os.vecs * kE + i;
            out[j] = E::down(tail_of(E::up(x[span.head + from * kE + j]), w, c2));
          }
        }
      }
      if (edge_at != 0xffffffffu) dx[edge_at] = E::down(tail_of(edges[threadIdx.x], w, c2));
      __syncthreads();  // the list's places come last
      if (mine) dx[entry.id] = E::down(ex2((xk - base_of(all.m)) * c2) * in_coef - weight * (float)entry.p);
    }
    if (a.loss.data && rank == 0 && threadIdx.x / 32 < list_warps) {
      // sum P (log P - log q) with log q = scale (x - m) - log S; P > 0 at a masked place makes it infinite, P = 0 says nothing
      const bool says = entry.p != 0.0 && entry.id != 0xffffffffu;
      double2 dot = make_double2(says ? entry.p * ((double)a.scale * ((double)xk - (double)base_of(all.m))) : 0.0, 0.0);
      dot = warp_sum(dot);
      if (list_warps > 1) {
        if ((threadIdx.x & 31) == 0) work.sums[threadIdx.x / 32] = dot;
        list_sync(list_warps);
        if (threadIdx.x < 32) dot = warp_sum(threadIdx.x < list_warps ? work.sums[threadIdx.x] : make_double2(0.0, 0.0));
      }
      if (threadIdx.x == 0) {
        double loss = said.plogp - (dot.x - said.sum * (double)logf(all.s));
        if (all.s == 0.0f) loss = said.sum > 0.0 ? (double)__int_as_float(0x7f800000) : said.sum;  // 0, or the teacher's NaN
        if (tail > 0.0f) loss += (double)(tail * (logf(tail) - (logf(rest.s) + lead - logf(all.s))));
        static_cast<float*>(a.loss.data)[row_at(a.g, a.loss, r)] = (float)loss;
      }
    }
    __syncthreads();
  }
  if (cluster > 1) cluster_wait();
}

lc_status launched(lc_context* ctx, const char* name) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return lc::cuda_fail(e, name);
  lc::record_launch(ctx, name);
  return LC_OK;
}

// A cluster for rows that are few, or so long that their bits would not fit in shared memory.
template <int DT, bool GRAD>
cudaError_t launch_rows(const lc_context* ctx, const DistillArgs& a, uint32_t cluster, cudaStream_t stream) {
  constexpr uint64_t kE = Vec<DT>::kElems;
  const uint64_t vecs = a.vocab / kE;
  const uint64_t share = std::max<uint64_t>(16, ((vecs + cluster - 1) / cluster + 15) / 16 * 16);
  const uint64_t busy = std::max<uint64_t>((share + kUnroll<DT> - 1) / kUnroll<DT>, a.list);
  // long slices: two blocks of 512 threads an SM, so that most of the rows under way stay in L2 for their second pass (4096 x
  // 131,072 bf16: 463 us, 505 with four of 256), as far as L2 goes: rows above 400 KB or so do not fit either way; shorter
  // ones: four of 256 (777 x 50,001 bf16: 54.6 us, 59.5 with two of 512)
  const uint64_t most = share * 16 < kLongSlice ? 256 : kRowThreads<GRAD>;
  const uint32_t threads = (uint32_t)std::min<uint64_t>(most, std::max<uint64_t>(32, (busy + 31) / 32 * 32));
  const bool moved = GRAD && apart(a.g, a.x, a.dx, 16 / kE);
  void (*kernel)(DistillArgs, uint32_t, uint32_t) = moved ? distill_rows<DT, GRAD, GRAD> : distill_rows<DT, GRAD, false>;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(std::min<uint64_t>(a.g.rows, kMaxGrid) * cluster));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = share;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  if (cfg.dynamicSmemBytes > (40 << 10)) {
    // the bound belongs to the kernel on its device and not to the call: always the most that any call needs, so that no thread
    // lowers another's between its setting and its launch
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxBits);
    if (e != cudaSuccess) return e;
  }
  return cudaLaunchKernelEx(&cfg, kernel, a, cluster, (uint32_t)share);
}

uint32_t cluster_of(const lc_context* ctx, uint64_t rows, uint64_t vecs) {
  uint32_t cluster = 1;
  while (cluster < kMaxCluster && (vecs > kMaxBits * cluster || (rows * cluster < 2ull * ctx->sm_count && vecs > 1024ull * cluster)))
    cluster *= 2;
  return cluster;
}

// Whether a cluster's shared memory holds the bits of a row of `vocab` places.
bool bits_fit(uint64_t vocab, int32_t dtype) { return vocab / (dtype == LC_F32 ? 4 : 8) <= (kMaxBits - 16) * kMaxCluster; }

// `rows`: by the kernel for rows whose vocabulary is the unit axis and whose bits fit.
template <int DT, bool GRAD>
cudaError_t launch(const lc_context* ctx, const DistillArgs& a, bool rows, cudaStream_t stream) {
  if (rows) return launch_rows<DT, GRAD>(ctx, a, cluster_of(ctx, a.g.rows, a.vocab / Vec<DT>::kElems), stream);
  distill_strided<DT, GRAD><<<(unsigned)std::min<uint64_t>(a.g.rows, kMaxGrid), kThreads, 0, stream>>>(a);
  return cudaSuccess;
}

template <bool GRAD>
cudaError_t launch(const lc_context* ctx, const DistillArgs& a, int32_t dtype, bool rows, cudaStream_t s) {
  if (dtype == LC_F32) return launch<LC_F32, GRAD>(ctx, a, rows, s);
  if (dtype == LC_F16) return launch<LC_F16, GRAD>(ctx, a, rows, s);
  return launch<LC_BF16, GRAD>(ctx, a, rows, s);
}

lc_status distill(const char* op, lc_context* ctx, void* stream, const lc_view* logits, const lc_view* ids,
                  const lc_view* teacher, float scale, int32_t tail, const lc_view* d_loss, const lc_view* loss,
                  const lc_view* dlogits) {
  using namespace lc;
  Call c(op, logits);
  lc_status st = c.start();
  if (st) return st;
  if ((st = c.check_scale(scale))) return st;
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
  const bool unit = a.vocab == 1 || (a.x.inner == 1 && (!dlogits || a.dx.inner == 1));
  const bool rows = unit && bits_fit(a.vocab, logits->dtype);
  const cudaError_t e = dlogits ? launch<true>(ctx, a, logits->dtype, rows, s) : launch<false>(ctx, a, logits->dtype, rows, s);
  if (e != cudaSuccess) return cuda_fail(e, op);
  return launched(ctx, dlogits ? (rows ? "distill_grad_rows" : "distill_grad_strided")
                               : (rows ? "distill_loss_rows" : "distill_loss_strided"));
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
