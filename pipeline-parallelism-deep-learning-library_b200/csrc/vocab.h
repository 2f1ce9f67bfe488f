// vocab.h -- host-side checks and row geometry shared by the operators over a vocabulary (token_logprobs.cu,
// distill.cu).
//
// Every operator works on rows: `logits` has shape [..., V], the vocabulary V is the last axis and the leading axes count
// the rows.  Every other operand has the same leading axes, and at most one axis more.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>

#include "internal.h"

namespace lcv {

constexpr int kMaxOperands = 8;       // operands of one call beside the logits
constexpr uint64_t kMaxVocab = 0x7fffffffull;
constexpr float kMaxScale = 0x1p100f;

// The leading axes, merged where every operand steps uniformly over two of them.
struct Rows {
  uint64_t rows;
  int rank;  // at least 1
  uint64_t shape[LC_MAX_RANK];
};

// One operand: element offset of row 0, strides over the merged leading axes, stride of the last axis.
struct RowOperand {
  void* data;
  uint64_t offset;
  uint64_t inner;
  uint64_t st[LC_MAX_RANK];
};

// Whether some row of `a` starts elsewhere within 16 bytes than the same row of `b`, `size` bytes an element.
inline bool apart(const Rows& g, const RowOperand& a, const RowOperand& b, uint64_t size) {
  uint64_t off = (reinterpret_cast<uintptr_t>(a.data) + a.offset * size) ^ (reinterpret_cast<uintptr_t>(b.data) + b.offset * size);
  for (int d = 0; d < g.rank; d++)
    if (g.shape[d] > 1) off |= (a.st[d] - b.st[d]) * size;
  return off % 16 != 0;
}

// Makes the context's device the current one while a call lasts: a caller may be on another device.
class DeviceGuard {
 public:
  explicit DeviceGuard(int device) {
    if (cudaGetDevice(&was_) != cudaSuccess) was_ = device;
    if (was_ != device) cudaSetDevice(device);
    now_ = device;
  }
  ~DeviceGuard() {
    if (was_ != now_) cudaSetDevice(was_);
  }

 private:
  int was_ = 0, now_ = 0;
};

inline bool is_float(int32_t dtype) { return dtype == LC_F32 || dtype == LC_F16 || dtype == LC_BF16; }
inline bool is_index(int32_t dtype) { return dtype == LC_I32 || dtype == LC_U32; }

// Collects the operands of one call, checks them against the logits and lays out their rows.
class Call {
 public:
  // `logits`: [..., V] of f32, f16 or bf16.
  Call(const char* op, const lc_view* logits) : op_(op), x_(logits) {}

  lc_status start() {
    using namespace lc;
    if (x_ == nullptr) return bad("null logits");
    lc_status st = validate(*x_, "logits");
    if (st) return st;
    if (!is_float(x_->dtype)) return bad("logits must be f32, f16 or bf16");
    if (x_->rank < 1) return bad("logits need a vocabulary axis");
    if (vocab() == 0) return bad("the vocabulary is empty");
    if (vocab() > kMaxVocab) return bad("the vocabulary exceeds 2^31 - 1");
    return LC_OK;
  }

  // Far below where scale * log2(e) (2.3e38) or an entropy's gradient times a far place's d (3e34) would leave f32 and make
  // NaN of 0 * infinity.
  lc_status check_scale(float scale) const {
    if (!std::isfinite(scale) || !(scale > 0.0f)) return bad("scale must be positive and finite");
    if (scale > kMaxScale) return bad("scale must be at most 2^100");
    return LC_OK;
  }

  uint64_t vocab() const { return x_->shape[x_->rank - 1]; }
  int lead() const { return x_->rank - 1; }

  // An operand [...] (`extra` < 0) or [..., extra].  `out`: written by the call.  Absent operands (null) are skipped.
  lc_status add(const lc_view* v, const char* name, int64_t extra, bool out) {
    using namespace lc;
    if (v == nullptr) return LC_OK;
    lc_status st = validate(*v, name);
    if (st) return st;
    const int rank = lead() + (extra >= 0 ? 1 : 0);
    if (v->rank != rank || memcmp(v->shape, x_->shape, sizeof(uint64_t) * lead()) != 0 ||
        (extra >= 0 && v->shape[lead()] != (uint64_t)extra))
      return bad(std::string(name) + (extra >= 0 ? " must have the logits' leading shape and a last axis of " + std::to_string(extra)
                                                 : std::string(" must have the logits' leading shape")));
    ops_[n_] = v;
    names_[n_] = name;
    out_[n_] = out;
    n_++;
    return LC_OK;
  }

  // No output may overlap an input or another output; `in_place` names the one that may be the logits themselves.
  lc_status finish(const lc_view* in_place) {
    using namespace lc;
    for (int i = 0; i < n_; i++) {
      if (!out_[i]) continue;
      if (!is_empty(*ops_[i]) && !is_injective(*ops_[i]))
        return bad(std::string(names_[i]) + " is not injective; parallel stores would alias");
      const bool same = ops_[i] == in_place && same_view(*ops_[i], *x_);
      if (!same && may_overlap(*ops_[i], *x_)) return fail(LC_ERR_OVERLAP, std::string(op_) + ": " + names_[i] + " overlaps the logits");
      for (int j = 0; j < n_; j++) {
        if (j == i || (out_[j] && j < i)) continue;
        if (may_overlap(*ops_[i], *ops_[j]))
          return fail(LC_ERR_OVERLAP, std::string(op_) + ": " + names_[i] + " overlaps " + names_[j]);
      }
    }
    return LC_OK;
  }

  Rows rows() {
    Rows r{};
    r.rows = 1;
    for (int d = 0; d < lead(); d++) r.rows *= x_->shape[d];
    int axes[LC_MAX_RANK], n = 0;  // innermost of each merged run
    for (int d = 0; d < lead(); d++) {
      if (x_->shape[d] == 1) continue;
      bool joins = n > 0 && steps(x_, axes[n - 1], d);
      for (int i = 0; i < n_ && joins; i++) joins = steps(ops_[i], axes[n - 1], d);
      if (joins) {
        axes[n - 1] = d;
        r.shape[n - 1] *= x_->shape[d];
      } else {
        axes[n] = d;
        r.shape[n++] = x_->shape[d];
      }
    }
    if (n == 0) {
      axes[0] = -1;
      r.shape[0] = 1;
      n = 1;
    }
    r.rank = n;
    for (int i = 0; i < n; i++) axes_[i] = axes[i];
    return r;
  }

  // After rows(): the operand's place in the merged axes (all zero for an absent one).
  RowOperand operand(const lc_view* v, int rank) const {
    RowOperand o{};
    if (v == nullptr) return o;
    o.data = v->data;
    o.offset = v->offset;
    o.inner = v->rank > lead() ? v->strides[v->rank - 1] : 0;
    for (int i = 0; i < rank; i++) o.st[i] = axes_[i] >= 0 ? v->strides[axes_[i]] : 0;
    return o;
  }

  lc_status bad(const std::string& what) const { return lc::fail(LC_ERR_INVALID_ARGUMENT, std::string(op_) + ": " + what); }

 private:
  // One step over axis `outer` is as long as all of axis `inner`.
  static bool steps(const lc_view* v, int outer, int inner) {
    uint64_t s;
    return !__builtin_mul_overflow(v->strides[inner], v->shape[inner], &s) && v->strides[outer] == s;
  }

  const char* op_;
  const lc_view* x_;
  const lc_view* ops_[kMaxOperands] = {};
  const char* names_[kMaxOperands] = {};
  bool out_[kMaxOperands] = {};
  int n_ = 0;
  int axes_[LC_MAX_RANK] = {};
};

}  // namespace lcv
