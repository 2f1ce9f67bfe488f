// token_logprobs.cu -- log probabilities of given tokens under a softmax over the vocabulary, with the entropy of the row
// and its best alternatives, and the gradient of both.
//
// With d_j = scale (x_j - m), m = max x and L = log sum e^d:  log p_j = d_j - L,  H = L - (sum e^d d) / (sum e^d).
// Gradient for g = d(total)/d(log p_t) and h = d(total)/dH:  dx_j = scale (g ([j = t] - p_j) - h p_j (log p_j + H)).
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

// The token of row r, or one outside the vocabulary where none is asked for.
__device__ __forceinline__ uint32_t token_of(const ScoreArgs& a, uint64_t r) {
  return a.logprob.data ? static_cast<const uint32_t*>(a.targets.data)[row_at(a.g, a.targets, r)] : 0xffffffffu;
}

// What a row leaves beside the alternatives.  `xt`: the token's logit, where it is in the vocabulary.
__device__ __forceinline__ void write_row(const ScoreArgs& a, uint64_t r, const Soft& row, float total, uint32_t token, float xt) {
  if (a.logprob.data)
    static_cast<float*>(a.logprob.data)[row_at(a.g, a.logprob, r)] = token < a.vocab ? logprob_of(xt, row.m, total, a.scale) : 0.0f;
  if (a.entropy.data)
    static_cast<float*>(a.entropy.data)[row_at(a.g, a.entropy, r)] = row.m == neg_inf() ? 0.0f : total - kLn2 * (row.t / row.s);
  if (a.stats.data) {
    float* st = static_cast<float*>(a.stats.data) + row_at(a.g, a.stats, r);
    st[0] = row.m;
    st[a.stats.inner] = total;
  }
}

__device__ __forceinline__ void write_best(const ScoreArgs& a, uint64_t r, uint32_t k, uint64_t key, const Soft& row, float total) {
  if (a.top_lp.data)
    static_cast<float*>(a.top_lp.data)[row_at(a.g, a.top_lp, r) + k * a.top_lp.inner] =
        logprob_of(value_of(key), row.m, total, a.scale);
  if (a.top_id.data) static_cast<uint32_t*>(a.top_id.data)[row_at(a.g, a.top_id, r) + k * a.top_id.inner] = index_of(key);
}

// One block a row, every element read where its stride puts it: once for the maximum and the sums, and once more for each
// alternative asked for, so that many of them are dear: 512 x 50,001 bf16 with the vocabulary as the outer axis 108 us, 2.2 ms
// with 20 alternatives, 13.3 ms with 128.
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
      const uint32_t t = token_of(a, r);
      write_row(a, r, row, total, t, t < a.vocab ? E::up(x[t * a.x.inner]) : 0.0f);
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
      if (threadIdx.x == 0) write_best(a, r, k, k1, row, total);
    }
    __syncthreads();
  }
}

// ---- the vocabulary as the unit axis -----------------------------------------------------------
//
// One cluster of blocks a row (one block where there are rows enough): each thread takes up 32 places at a time into its own
// running softmax; threads, blocks and the cluster merge them once at the end, in an order that does not vary.
//
// The alternatives come out of the same pass.  Each thread leaves the order of the largest logit of every step (a slot) in
// shared memory.  A bound that at least K places reach is known without looking at a place again: of the threads' own
// largest, the q-th best of each warp, q = K over the number of warps, and of those the least.  Only slots above the bound
// are read again (some 80 of 4096 for K = 20 of 131,072), and what lies above it is ranked by counting.  Rows whose best
// places crowd together beyond what shared memory holds (a narrow band, a few thousand permitted places side by side) find
// the K-th largest order bit by bit instead: right for every row, and slower.
//
// What bounds it (B200, whole call in a graph, of the 6465 GB/s of a copy): HBM.  2048 x 100,003 f32 with entropy reads at
// 6439 GB/s (127 us), 4096 x 131,072 bf16 at 6436 (167 us); f16 and bf16 have two exponentials for each of f32 and three
// quarters of the exponential unit's rate at that speed.  With K = 20 alternatives the latter takes 208 us (198 without the
// entropy): a block waits for one more read from L2 and some barriers, which the other blocks of its SM cover in part.
// Why small blocks and not a ring of stages that the copy engine fills (3 of 32 KB a block, two blocks of 512 an SM,
// measured: 224 us against 182 with four blocks of 256 and plain loads, 173 with six): a block's end is a chain of barriers,
// and only other blocks can fill it.
// A single row (1 x 131,072 bf16, K = 20) takes 9.7 us over a cluster of 8, nearly all of it latency: 1.4 us to the logits,
// 0.7 to merge, 3.6 for the block's alternatives, the rest for the cluster's.  16 blocks a cluster measured 13.5 us.
constexpr int kMaxThreads = 256;
template <int DT>
constexpr int kUnroll = 32 / Vec<DT>::kElems;  // vectors of a step: 32 places a thread
template <int DT>
constexpr int kResident = DT == LC_F32 ? 4 : 6;  // blocks an SM; 16-bit types: 173 us with 6, 183 with 4 (4096 x 131,072)
constexpr uint32_t kMaxSlots = 4096;
constexpr uint32_t kMaxKeys = 512;
constexpr uint32_t kMaxRead = 256;  // slots that are read again in one go
constexpr uint32_t kMaxCluster = 8;

struct Slice {  // a block's part of a row
  const uint4* vec;    // vector 0 of the row
  uint32_t from, to;   // its vectors
  uint32_t head;       // places before vector 0
  uint32_t per_slot;   // steps of kUnroll * threads vectors that share a slot
};

// Calls f(order, index) for each place of this thread's vectors in slots that reach `least`.
template <int DT, class F>
__device__ __forceinline__ void each_place(const Slice& sl, const uint32_t* slots, uint32_t least, F f) {
  constexpr int kSteps = kUnroll<DT>;
  const uint32_t step = kSteps * blockDim.x;
  uint32_t b = 0;
  for (uint32_t v0 = sl.from; v0 < sl.to; v0 += step, b++) {
    if (slots[(b / sl.per_slot) * blockDim.x + threadIdx.x] < least) continue;
    uint4 q[kSteps];
#pragma unroll
    for (int u = 0; u < kSteps; u++) {
      const uint32_t v = v0 + u * blockDim.x + threadIdx.x;
      q[u] = v < sl.to ? __ldg(sl.vec + v) : Vec<DT>::masked();
    }
#pragma unroll
    for (int u = 0; u < kSteps; u++) {
      const uint32_t v = v0 + u * blockDim.x + threadIdx.x;
      if (v >= sl.to) break;
      if (order_of(Vec<DT>::top(q[u])) < least) continue;
#pragma unroll
      for (int i = 0; i < Vec<DT>::kElems / 2; i++) {
        const float2 x = Vec<DT>::pair(q[u], i);
        const uint32_t j = sl.head + v * Vec<DT>::kElems + 2 * i;
        f(order_of(x.x), j);
        f(order_of(x.y), j + 1);
      }
    }
  }
}

__device__ __forceinline__ uint32_t block_count(uint32_t v, uint32_t* red) {
  v = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  uint32_t n = 0;
  for (uint32_t w = 0; w < blockDim.x / 32; w++) n += red[w];
  return n;
}

// Shared memory of select.
struct Work {
  uint64_t* keys;   // [kMaxKeys]
  uint32_t* read;   // [kMaxRead]
  uint32_t* red;    // one for each warp
  uint32_t* count;  // 2
};

// The `want` best keys of the slice in `best`, best first (fewer if it has fewer; the rest are 0).
// `mine`: the order of the largest logit of this thread's vectors, 0 if it has none.  `edge`, `edge_at`: the order and place
// of the logit before or behind the vectors that this thread holds, 0 if none.  `places`: how many places the slice has.
template <int DT>
__device__ void select(const Slice& sl, const uint32_t* slots, uint32_t mine, uint32_t edge, uint32_t edge_at, uint32_t places,
                       uint32_t want, const Work& w, uint64_t* best) {
  constexpr int kSteps = kUnroll<DT>;
  uint64_t* keys = w.keys;
  uint32_t *red = w.red, *count = w.count;
  const uint32_t warps = blockDim.x / 32, lane = threadIdx.x & 31;
  const uint32_t held = min(warps, (sl.to - sl.from) / 32);  // warps whose every thread has vectors
  const uint32_t q = held ? (want + held - 1) / held : 33;
  for (uint32_t i = threadIdx.x; i < want; i += blockDim.x) best[i] = 0;
  uint32_t bound = 0;
  if (q <= 32) {
    uint32_t left = mine;
    for (uint32_t i = 0; i < q; i++) {
      bound = __reduce_max_sync(0xffffffffu, left);
      if (lane == __ffs(__ballot_sync(0xffffffffu, left == bound)) - 1) left = 0;
    }
  }
  if (lane == 0) red[threadIdx.x / 32] = bound;
  if (threadIdx.x == 0) count[0] = count[1] = 0;
  __syncthreads();
  if (q <= 32) {
    for (uint32_t i = 0; i < held; i++) bound = i == 0 ? red[0] : min(bound, red[i]);
  }
  want = min(want, places);
  // Places above the bound, in any order: their keys are told apart by rank below.
  auto collect = [&](uint32_t o, uint32_t j) {
    if (o > bound) {
      const uint32_t at = atomicAdd(count, 1u);
      if (at < kMaxKeys) keys[at] = ((uint64_t)o << 32) | (0xffffffffu - j);
    }
  };
  // The slots above the bound go to a list first, so that all their vectors are on the way at once.
  const uint32_t step = kSteps * blockDim.x, steps = (sl.to - sl.from + step - 1) / step;
  const uint32_t rows_of_slots = (steps + sl.per_slot - 1) / sl.per_slot;
  for (uint32_t i = 0; i < rows_of_slots; i++)
    if (slots[i * blockDim.x + threadIdx.x] > bound) {
      const uint32_t at = atomicAdd(count + 1, 1u);
      if (at < kMaxRead) w.read[at] = i << 16 | threadIdx.x;
    }
  collect(edge, edge_at);
  __syncthreads();
  const uint32_t reads = count[1], per = sl.per_slot * kSteps;
  if (reads <= kMaxRead) {
    for (uint32_t i = threadIdx.x; i < reads * per; i += blockDim.x) {
      const uint32_t slot = sl.per_slot == 1 ? i / kSteps : i / per, e = w.read[slot], k = i - slot * per;
      const uint32_t v = sl.from + ((e >> 16) * per + k) * blockDim.x + (e & 0xffffu);
      if (v >= sl.to) continue;
      const uint4 q = __ldg(sl.vec + v);
      if (order_of(Vec<DT>::top(q)) <= bound) continue;
#pragma unroll
      for (int i2 = 0; i2 < Vec<DT>::kElems / 2; i2++) {
        const float2 x = Vec<DT>::pair(q, i2);
        const uint32_t j = sl.head + v * Vec<DT>::kElems + 2 * i2;
        collect(order_of(x.x), j);
        collect(order_of(x.y), j + 1);
      }
    }
  } else {
    each_place<DT>(sl, slots, bound + (bound != 0xffffffffu), collect);
  }
  __syncthreads();
  uint32_t n = *count;
  if (n > kMaxKeys) {
    // More than fit (a row whose best places crowd together): find the K-th largest order itself, bit by bit.  Fewer than
    // K places lie above it.
    uint32_t lo = bound, hi = 0xffffffffu;  // at least `want` places reach lo
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      uint32_t c = edge >= mid;
      each_place<DT>(sl, slots, mid, [&](uint32_t o, uint32_t) { c += o >= mid; });
      if (block_count(c, red) >= want) lo = mid;
      else hi = mid - 1;
    }
    bound = lo;
    __syncthreads();
    if (threadIdx.x == 0) *count = 0;
    __syncthreads();
    each_place<DT>(sl, slots, bound + (bound != 0xffffffffu), collect);
    collect(edge, edge_at);
    __syncthreads();
    n = *count;
  }
  if (n < want && bound > 0) {
    // Places equal to the bound, from the lowest index on: the places before the vectors, the vectors in steps of one for
    // each thread, the places behind them.
    uint32_t have = n;
    auto place = [&](uint32_t c, auto put) {  // c: how many this thread has
      uint32_t incl = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= (uint32_t)o) incl += up;
      }
      __syncthreads();
      if (lane == 31) red[threadIdx.x / 32] = incl;
      __syncthreads();
      uint32_t before = have + incl - c, all = have;
      for (uint32_t i = 0; i < warps; i++) {
        if (i < threadIdx.x / 32) before += red[i];
        all += red[i];
      }
      put(before);
      have = all;
    };
    const bool front = edge == bound && edge_at < sl.head;
    place(front, [&](uint32_t at) {
      if (front && at < want) keys[at] = ((uint64_t)edge << 32) | (0xffffffffu - edge_at);
    });
    uint32_t b = 0;
    for (uint32_t v0 = sl.from; v0 < sl.to && have < want; v0 += step, b++) {
      const bool may = slots[(b / sl.per_slot) * blockDim.x + threadIdx.x] >= bound;
      for (int u = 0; u < kSteps && have < want; u++) {
        const uint32_t v = v0 + u * blockDim.x + threadIdx.x;
        uint32_t hits = 0;
        if (may && v < sl.to) {
          const uint4 x = __ldg(sl.vec + v);
#pragma unroll
          for (int i = 0; i < Vec<DT>::kElems / 2; i++) {
            const float2 p = Vec<DT>::pair(x, i);
            hits |= (uint32_t)(order_of(p.x) == bound) << (2 * i) | (uint32_t)(order_of(p.y) == bound) << (2 * i + 1);
          }
        }
        place(__popc(hits), [&](uint32_t at) {
          for (; hits && at < want; hits &= hits - 1, at++)
            keys[at] = ((uint64_t)bound << 32) | (0xffffffffu - (sl.head + v * Vec<DT>::kElems + (__ffs(hits) - 1)));
        });
      }
    }
    if (have < want) {
      const bool back = edge == bound && edge_at >= sl.head;
      place(back, [&](uint32_t at) {
        if (back && at < want) keys[at] = ((uint64_t)edge << 32) | (0xffffffffu - edge_at);
      });
    }
    __syncthreads();
    n = min(have, want);
  }
  for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
    const uint64_t key = keys[i];
    uint32_t rank = 0;
#pragma unroll 8
    for (uint32_t o = 0; o < n; o++) rank += keys[o] > key;
    if (rank < want) best[rank] = key;
  }
  __syncthreads();
}

template <int DT, bool SUM_T, bool TOP>
__global__ void __launch_bounds__(kMaxThreads, kResident<DT>) token_logprobs_rows(ScoreArgs a, uint32_t cluster, uint32_t per_slot) {
  using E = Elem<DT>;
  constexpr uint32_t kE = Vec<DT>::kElems;
  constexpr int kSteps = kUnroll<DT>;
  extern __shared__ uint64_t dyn[];
  __shared__ Soft red[kMaxThreads / 32];
  __shared__ Soft parts[kMaxCluster];
  __shared__ uint32_t read[kMaxRead], red_u[kMaxThreads / 32], count[2];
  const Work work{dyn, read, red_u, count};
  uint64_t* best = dyn + kMaxKeys;                               // [top]
  uint64_t* lists = best + a.top;                                // [cluster][top]: the blocks' best, in block 0
  uint32_t* slots = reinterpret_cast<uint32_t*>(lists + (cluster > 1 ? cluster * a.top : 0));  // [n_slots][threads]
  const uint32_t rank = cluster > 1 ? cluster_rank() : 0;
  const float c2 = a.scale * kLog2e;
  // Cluster barriers alternate: block 0's buffers are free (at first: it has started), and all blocks' parts are in them.
  if (cluster > 1) cluster_arrive();
  for (uint64_t r = blockIdx.x / cluster; r < a.g.rows; r += gridDim.x / cluster) {
    const typename E::T* x = static_cast<const typename E::T*>(a.x.data) + row_at(a.g, a.x, r);
    const Span span = span_of<DT>(x, a.vocab);
    Slice sl;
    sl.vec = reinterpret_cast<const uint4*>(x + span.head);
    sl.head = span.head;
    sl.per_slot = per_slot;
    const uint32_t share = ((span.vecs + cluster - 1) / cluster + 31) / 32 * 32;
    sl.from = min(span.vecs, rank * share);
    sl.to = min(span.vecs, sl.from + share);
    // block 0 has the places before the vectors (threads 0-7) and behind them (8-15), and the token
    float edge = neg_inf(), xt = 0.0f;
    uint32_t edge_at = 0xffffffffu, token = 0xffffffffu;
    if (rank == 0 && threadIdx.x < 16) {
      const uint32_t i = threadIdx.x & 7;
      if (threadIdx.x < 8 ? i < span.head : i < span.tail) {
        edge_at = threadIdx.x < 8 ? i : span.head + span.vecs * kE + i;
        edge = E::up(x[edge_at]);
      }
      if (threadIdx.x == 0) {
        token = token_of(a, r);
        if (token < a.vocab) xt = E::up(x[token]);
      }
    }
    Run run = empty_run();
    uint32_t mine = 0, slot = 0, in_slot = 0;
    uint32_t* next = slots + threadIdx.x;
    const uint32_t step = kSteps * blockDim.x;
    uint32_t v0 = sl.from;
    for (; v0 + step <= sl.to; v0 += step) {
      uint4 q[kSteps];
#pragma unroll
      for (int u = 0; u < kSteps; u++) q[u] = load_once(sl.vec + v0 + u * blockDim.x + threadIdx.x);
      float top = Vec<DT>::top(q[0]);
#pragma unroll
      for (int u = 1; u < kSteps; u++) top = max_nan(top, Vec<DT>::top(q[u]));
      take<DT, kSteps, SUM_T>(run, q, top, c2);
      if constexpr (TOP) {  // the largest of a step's logits goes to its slot
        slot = max(slot, order_of(top));
        if (++in_slot == per_slot || v0 + step >= sl.to) {
          mine = max(mine, slot);
          *next = slot;
          next += blockDim.x;
          slot = in_slot = 0;
        }
      }
    }
    if (v0 < sl.to) {  // the last step, short of some vectors: masked ones in their place
      uint4 q[kSteps];
#pragma unroll
      for (int u = 0; u < kSteps; u++) {
        const uint32_t v = v0 + u * blockDim.x + threadIdx.x;
        q[u] = v < sl.to ? load_once(sl.vec + v) : Vec<DT>::masked();
      }
      const bool any = v0 + threadIdx.x < sl.to;
      float top = Vec<DT>::top(q[0]);
#pragma unroll
      for (int u = 1; u < kSteps; u++) top = max_nan(top, Vec<DT>::top(q[u]));
      if (any) take<DT, kSteps, SUM_T>(run, q, top, c2);
      if constexpr (TOP) {
        if (any) slot = max(slot, order_of(top));
        mine = max(mine, slot);
        *next = slot;
      }
    }
    Soft part = soft_of(run, c2);
    if (edge_at != 0xffffffffu) part = merge(part, Soft{edge, edge == neg_inf() ? 0.0f : 1.0f, 0.0f}, c2);
    Soft row = block_merge(part, c2, red);
    if constexpr (TOP) {
      const uint32_t places = (sl.to - sl.from) * kE + (rank == 0 ? span.head + span.tail : 0);
      select<DT>(sl, slots, mine, edge_at != 0xffffffffu ? order_of(edge) : 0, edge_at, places, a.top, work, best);
    }
    if (cluster > 1) {
      cluster_wait();
      if (threadIdx.x == 0) {
        const uint32_t at = remote(&parts[rank], 0);
        store_remote(at, row.m);
        store_remote(at + 4, row.s);
        store_remote(at + 8, row.t);
      }
      if constexpr (TOP) {
        for (uint32_t i = threadIdx.x; i < a.top; i += blockDim.x) store_remote(remote(lists + rank * a.top + i, 0), best[i]);
      }
      cluster_arrive();
      cluster_wait();
    }
    if (rank == 0) {
      if (cluster > 1) {
        const uint32_t c = threadIdx.x & 31;
        row = warp_merge(c < cluster ? parts[c] : Soft{neg_inf(), 0.0f, 0.0f}, c2);
      }
      const float total = logf(row.s);
      if (threadIdx.x == 0) write_row(a, r, row, total, token, xt);
      if constexpr (TOP) {
        if (cluster == 1) {
          for (uint32_t k = threadIdx.x; k < a.top; k += blockDim.x) write_best(a, r, k, best[k], row, total);
        } else {
          // the K best of the blocks' lists, told apart by rank
          const uint32_t n = cluster * a.top;
          for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
            const uint64_t key = lists[i];
            uint32_t k = key ? 0 : a.top;
#pragma unroll 8
            for (uint32_t o = 0; o < n; o++) k += lists[o] > key;
            if (k < a.top) write_best(a, r, k, key, row, total);
          }
        }
      }
    }
    if (cluster > 1) cluster_arrive();
    __syncthreads();
  }
  if (cluster > 1) cluster_wait();
}

struct GradArgs {
  Rows g;
  RowOperand x, targets, stats, entropy, d_logprob, d_entropy, dx;
  uint32_t vocab;
  float scale;
};

// What the gradient of a row is made of: dx = 2^d (at + bt d), and the target's own share.  d is x c2 - mc, or (x - base) c2
// where the row's largest logit is not of an ordinary size (take in vocab.cuh has the same two forms).  1 / sum is taken
// once a row as e^-L and not within the exponent, where L ~ 10 would cost the last bits of every place.
struct GradRow {
  float minus, at, bt, own;  // minus: -mc, or -base
  bool wide;
  uint32_t target;
};

__device__ __forceinline__ GradRow grad_row(const GradArgs& a, uint64_t r, float c2) {
  GradRow w;
  const float* st = static_cast<const float*>(a.stats.data) + row_at(a.g, a.stats, r);
  const float m = st[0], total = st[a.stats.inner];
  w.wide = is_wide(m, c2);
  w.minus = w.wide ? -base_of(m) : -(m * c2);
  const float off = w.wide ? 0.0f : __fmaf_rn(m, c2, w.minus);  // m c2 - mc
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
  const float per = a.scale * expf(-total) * ex2(-off);
  w.own = g * a.scale;
  w.bt = -per * h * kLn2;
  w.at = -per * (g + h * (ent - total - off * kLn2));
  if (m == neg_inf()) {  // masked throughout: there is no distribution, and no gradient
    w.at = w.bt = 0.0f;
    w.target = 0xffffffffu;
  }
  return w;
}

// ENT: with the entropy's share.  Without it bt is 0 and a masked place needs no bound on d: 2^-inf at = 0.
template <bool ENT>
__device__ __forceinline__ float grad_of(float x, const GradRow& w, float c2) {
  float d = w.wide ? (x + w.minus) * c2 : __fmaf_rn(x, c2, w.minus);
  if constexpr (!ENT) return ex2(d) * w.at;
  d = max_nan(d, kFar);
  return ex2(d) * __fmaf_rn(w.bt, d, w.at);
}

constexpr int kGradThreads = 256;

template <int DT, bool ENT>
__global__ void __launch_bounds__(kGradThreads) token_logprobs_backward_strided(GradArgs a) {
  using E = Elem<DT>;
  const float c2 = a.scale * kLog2e;
  for (uint64_t r = blockIdx.x; r < a.g.rows; r += gridDim.x) {
    const typename E::T* x = static_cast<const typename E::T*>(a.x.data) + row_at(a.g, a.x, r);
    typename E::T* dx = static_cast<typename E::T*>(a.dx.data) + row_at(a.g, a.dx, r);
    const GradRow w = grad_row(a, r, c2);
    for (uint32_t j = threadIdx.x; j < a.vocab; j += kGradThreads) {
      float v = grad_of<ENT>(E::up(x[j * a.x.inner]), w, c2);
      if (j == w.target) v += w.own;
      dx[j * a.dx.inner] = E::down(v);
    }
  }
}

// 16 bytes of dx from 16 bytes of x whose first place is j.
template <int DT, bool ENT>
__device__ __forceinline__ uint4 grad_vec(const uint4& q, uint32_t j, const GradRow& w, float c2) {
  constexpr uint32_t kE = Vec<DT>::kElems;
  float2 y[kE / 2];
  const float2 minus = both(w.minus), c = both(c2), at = both(w.at), bt = both(w.bt);
  if (!w.wide) {
#pragma unroll
    for (uint32_t i = 0; i < kE / 2; i++) y[i] = __ffma2_rn(Vec<DT>::pair(q, i), c, minus);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < kE / 2; i++) y[i] = __fmul2_rn(__fadd2_rn(Vec<DT>::pair(q, i), minus), c);
  }
#pragma unroll
  for (uint32_t i = 0; i < kE / 2; i++) {
    float2 d = y[i];
    if constexpr (ENT) d = make_float2(max_nan(d.x, kFar), max_nan(d.y, kFar));
    y[i] = __fmul2_rn(make_float2(ex2(d.x), ex2(d.y)), ENT ? __ffma2_rn(bt, d, at) : at);
  }
  const uint32_t own = w.target - j;
  if (own < kE) {
#pragma unroll
    for (uint32_t i = 0; i < kE / 2; i++) {
      if (own == 2 * i) y[i].x += w.own;
      if (own == 2 * i + 1) y[i].y += w.own;
    }
  }
  return Vec<DT>::pack(y);
}

// The vocabulary as the unit axis: a block has `steps` steps of kGradUnroll vectors a thread of one row, with all of a
// step's loads on the way before the first is used.  The vectors are those of dx, so that every store is a whole one.
// MOVED: some row of x starts elsewhere within 16 bytes (an odd vocabulary against padded rows).  A vector of it then is cut
// out of two aligned ones, of which the second comes from the next lane (a warp's vectors of a step follow one another), or at
// the end of a warp's vectors from a load of its own.  In steps that reach the row's ends the vectors are read place by place,
// as are the places around them.
// Bound by HBM: 4096 x 131,072 bf16 with the entropy's share 330 us, 6515 GB/s, as fast as a copy; stores that stream past
// the caches and four blocks an SM with registers enough for all loads of a step (434 us with six and spills).  MOVED rows
// (1001 x 50,001 bf16 in padded rows: 43 us, 4650 GB/s; 37 us were the rows alike) pay for the shifts and, more the shorter
// the row, for its first and last step, all of whose vectors are read place by place although only the outermost ones reach
// out of the row (1001 x 131,073: 95 us, 85 alike).  No pipe is full (ALU 42%, issue 50%).  Two loads a vector instead of the
// neighbour's half measured 53 us.
constexpr int kGradUnroll = 4;

template <int DT, bool ENT, bool MOVED>
__global__ void __launch_bounds__(kGradThreads, 4) token_logprobs_backward_rows(GradArgs a, uint32_t tiles, uint32_t steps) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr uint32_t kE = Vec<DT>::kElems;
  constexpr int kU = kGradUnroll;
  const float c2 = a.scale * kLog2e;
  const uint32_t lane = threadIdx.x & 31;
  // vectors of a thread: where the first of a step lies, and how far apart they are
  const uint32_t place = MOVED ? (threadIdx.x & ~31u) * kU + lane : threadIdx.x, apart = MOVED ? 32 : blockDim.x;
  const uint64_t items = a.g.rows * tiles;
  for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const uint64_t r = item / tiles;
    const uint32_t tile = (uint32_t)(item - r * tiles);
    const T* x = static_cast<const T*>(a.x.data) + row_at(a.g, a.x, r);
    T* dx = static_cast<T*>(a.dx.data) + row_at(a.g, a.dx, r);
    const Span span = span_of<DT>(dx, a.vocab);
    const char* xv = reinterpret_cast<const char*>(x + span.head);  // where vector 0 of dx reads
    uint4* dv = reinterpret_cast<uint4*>(dx + span.head);
    const uint32_t shift = reinterpret_cast<uintptr_t>(xv) & 15;
    // the aligned vectors of x that begin and end within the row, where vector v is cut out of v and v + 1
    const uint32_t first = xv - shift < reinterpret_cast<const char*>(x);
    const uint32_t count = (uint32_t)((reinterpret_cast<const char*>(x + a.vocab) - (xv - shift)) / 16);
    const uint32_t step = kU * blockDim.x;
    const uint32_t from = min(span.vecs, tile * steps * step), to = min(span.vecs, from + steps * step);
    bool ready = false;
    GradRow w;
    for (uint32_t v0 = from; v0 < to; v0 += step) {
      uint4 q[kU];
      const uint32_t v = v0 + place;
      if (!MOVED || shift == 0) {
#pragma unroll
        for (int u = 0; u < kU; u++)
          if (v + u * apart < to) q[u] = *reinterpret_cast<const uint4*>(xv + (uint64_t)(v + u * apart) * 16);
      } else if (v0 >= first && v0 + step < count && v0 + step <= to) {
        const uint4* xa = reinterpret_cast<const uint4*>(xv - shift) + v;
#pragma unroll
        for (int u = 0; u < kU; u++) q[u] = __ldg(xa + u * apart);
        uint4 last;
        if (lane == 31) last = __ldg(xa + kU * apart - 31);
#pragma unroll
        for (int u = 0; u < kU; u++) {
          uint4 give = q[u];
          if (u + 1 < kU && lane == 0) give = q[u + 1 < kU ? u + 1 : u];
          uint4 next = make_uint4(__shfl_sync(0xffffffffu, give.x, lane + 1), __shfl_sync(0xffffffffu, give.y, lane + 1),
                                  __shfl_sync(0xffffffffu, give.z, lane + 1), __shfl_sync(0xffffffffu, give.w, lane + 1));
          if (u + 1 == kU && lane == 31) next = last;
          q[u] = shifted(q[u], next, shift);
        }
      } else {
#pragma unroll
        for (int u = 0; u < kU; u++)
          if (v + u * apart < to) q[u] = one_by_one<DT>(xv + (uint64_t)(v + u * apart) * 16);
      }
      if (!ready) w = grad_row(a, r, c2);
      ready = true;
#pragma unroll
      for (int u = 0; u < kU; u++)
        if (v + u * apart < to) __stcs(dv + v + u * apart, grad_vec<DT, ENT>(q[u], span.head + (v + u * apart) * kE, w, c2));
    }
    if (tile == 0 && threadIdx.x < 16) {
      const uint32_t i = threadIdx.x & 7;
      if (threadIdx.x < 8 ? i < span.head : i < span.tail) {
        const uint32_t j = threadIdx.x < 8 ? i : span.head + span.vecs * kE + i;
        if (!ready) w = grad_row(a, r, c2);
        float v = grad_of<ENT>(E::up(x[j]), w, c2);
        if (j == w.target) v += w.own;
        dx[j] = E::down(v);
      }
    }
  }
}

lc_status launched(lc_context* ctx, const char* name) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return lc::cuda_fail(e, name);
  lc::record_launch(ctx, name);
  return LC_OK;
}

// How a row is spread: blocks of `threads` in a cluster of `cluster`, and the slots of its alternatives.
struct Spread {
  uint32_t cluster, threads, n_slots, per_slot;
  size_t shared;
};

// Enough blocks to fill the device, as long as each has a step of 256 threads left to do: one row of 131,072 bf16 over 8
// blocks (37 x 50,001 f32: 9.8 us over 8 blocks a row, 11.2 over 4).  From 2 rows an SM on, one block a row: clusters of 2
// for 2048 rows measured 86 us against 77.  A block has the threads that its vectors keep busy, and 2 for each alternative
// asked for, so that the bound on them (select) comes from several warps.
Spread spread_of(const lc_context* ctx, uint64_t rows, uint64_t vocab, uint32_t elems, uint32_t unroll, uint32_t top) {
  Spread s{};
  const uint64_t vecs = vocab / elems;
  s.cluster = 1;
  while (s.cluster < kMaxCluster && rows * s.cluster < 2ull * ctx->sm_count && vecs / (2 * s.cluster) >= 1ull * unroll * 256)
    s.cluster *= 2;
  const uint64_t share = std::max<uint64_t>(((vecs + s.cluster - 1) / s.cluster + 31) / 32 * 32, 1);
  const uint64_t busy = std::max<uint64_t>((share + unroll - 1) / unroll, 2 * top);
  s.threads = (uint32_t)std::min<uint64_t>(kMaxThreads, (busy + 31) / 32 * 32);
  if (busy > kMaxThreads) {  // several steps: of one length, so that the last one is not nearly empty
    const uint64_t n = (busy + kMaxThreads - 1) / kMaxThreads;
    s.threads = (uint32_t)(((busy + n - 1) / n + 31) / 32 * 32);
  }
  const uint64_t steps = (share + (uint64_t)unroll * s.threads - 1) / ((uint64_t)unroll * s.threads);
  const uint64_t rows_of_slots = std::max<uint64_t>(1, kMaxSlots / s.threads);
  s.per_slot = (uint32_t)((steps + rows_of_slots - 1) / rows_of_slots);
  s.n_slots = (uint32_t)((steps + s.per_slot - 1) / s.per_slot);
  if (top) s.shared = sizeof(uint64_t) * (kMaxKeys + top + (s.cluster > 1 ? s.cluster * top : 0)) + sizeof(uint32_t) * s.n_slots * s.threads;
  return s;
}

template <int DT>
cudaError_t launch_rows(const lc_context* ctx, const ScoreArgs& a, cudaStream_t stream) {
  const Spread s = spread_of(ctx, a.g.rows, a.vocab, Vec<DT>::kElems, kUnroll<DT>, a.top);
  void (*kernel)(ScoreArgs, uint32_t, uint32_t) =
      a.top ? (a.entropy.data ? token_logprobs_rows<DT, true, true> : token_logprobs_rows<DT, false, true>)
            : (a.entropy.data ? token_logprobs_rows<DT, true, false> : token_logprobs_rows<DT, false, false>);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(std::min<uint64_t>(a.g.rows, kMaxGrid) * s.cluster));
  cfg.blockDim = dim3(s.threads);
  cfg.dynamicSmemBytes = s.shared;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = s.cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = s.cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, a, s.cluster, s.per_slot);
}

template <int DT, bool ENT>
void launch_backward(const lc_context* ctx, const GradArgs& a, bool unit, cudaStream_t stream) {
  if (!unit) {
    token_logprobs_backward_strided<DT, ENT><<<(unsigned)std::min<uint64_t>(a.g.rows, kMaxGrid), kGradThreads, 0, stream>>>(a);
    return;
  }
  // short rows take a small block; long ones blocks of up to 4 steps, fewer where that leaves the device idle
  const uint64_t vecs = a.vocab / Vec<DT>::kElems, busy = (vecs + kGradUnroll - 1) / kGradUnroll;
  const uint32_t threads = (uint32_t)std::min<uint64_t>(kGradThreads, std::max<uint64_t>(32, (busy + 31) / 32 * 32));
  const uint64_t step = (uint64_t)kGradUnroll * threads, all = std::max<uint64_t>(1, (vecs + step - 1) / step);
  uint32_t steps = 4;
  while (steps > 1 && a.g.rows * ((all + steps - 1) / steps) < 12ull * ctx->sm_count) steps /= 2;
  const uint32_t tiles = (uint32_t)((all + steps - 1) / steps);
  const unsigned grid = (unsigned)std::min<uint64_t>(a.g.rows * tiles, 0x7fffffffull);
  const bool moved = apart(a.g, a.x, a.dx, 16 / Vec<DT>::kElems);
  auto kernel = moved ? token_logprobs_backward_rows<DT, ENT, true> : token_logprobs_backward_rows<DT, ENT, false>;
  kernel<<<grid, threads, 0, stream>>>(a, tiles, steps);
}

template <int DT>
void launch_backward(const lc_context* ctx, const GradArgs& a, bool unit, cudaStream_t stream) {
  if (a.d_entropy.data) launch_backward<DT, true>(ctx, a, unit, stream);
  else launch_backward<DT, false>(ctx, a, unit, stream);
}

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
  if ((st = c.check_scale(scale))) return st;
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
  if (a.x.inner == 1 || a.vocab == 1) {
    cudaError_t e = logits->dtype == LC_F32 ? launch_rows<LC_F32>(ctx, a, s)
                    : logits->dtype == LC_F16 ? launch_rows<LC_F16>(ctx, a, s) : launch_rows<LC_BF16>(ctx, a, s);
    if (e != cudaSuccess) return cuda_fail(e, "token_logprobs_rows");
    return launched(ctx, "token_logprobs_rows");
  }
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
  if ((st = c.check_scale(scale))) return st;
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
  const bool unit = a.vocab == 1 || (a.x.inner == 1 && a.dx.inner == 1);
  if (logits->dtype == LC_F32) launch_backward<LC_F32>(ctx, a, unit, s);
  else if (logits->dtype == LC_F16) launch_backward<LC_F16>(ctx, a, unit, s);
  else launch_backward<LC_BF16>(ctx, a, unit, s);
  return launched(ctx, unit ? "token_logprobs_backward_rows" : "token_logprobs_backward_strided");
}

}  // extern "C"
