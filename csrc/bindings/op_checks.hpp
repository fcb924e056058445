// What the bindings of operators on torch tensors share: checks of arguments,
// of overlap between tensors, and of what autograd has to know.
#pragma once

#include <ATen/ATen.h>
#include <torch/extension.h>

#include <climits>
#include <optional>
#include <stdexcept>
#include <string>

#include "kernels.h"
#include "turbol/common.hpp"

namespace turbol::checks {

inline void chk(bool c, const char* op, const char* m) {
  if (!c) throw std::invalid_argument(std::string(op) + ": " + m);
}
inline void cuda_ok(int e, const char* what) {
  if (e != 0) throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(static_cast<cudaError_t>(e)));
}

inline int type_of(const at::Tensor& t, const char* op) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return TB_BF16;
    case at::kHalf: return TB_F16;
    case at::kFloat: return TB_F32;
    default: throw std::invalid_argument(std::string(op) + ": bf16, fp16 or fp32 values");
  }
}

// Whether t carries a forward-mode tangent.
inline bool is_dual(const at::Tensor& t) { return t._fw_grad(/*level=*/0).defined(); }

// What has no derivative refuses tensors that would want one (forward mode has no
// switch: torch.no_grad() leaves it on).
inline void no_grad(std::initializer_list<const at::Tensor*> ts, const char* op, const char* what = nullptr) {
  const bool on = at::GradMode::is_enabled();
  for (const at::Tensor* t : ts)
    if (is_dual(*t) || (on && t->requires_grad()))
      throw std::invalid_argument(std::string(op) + ": " + (what ? std::string(what) + " " : std::string()) +
                                  (is_dual(*t) ? "has no forward-mode derivative"
                                               : "has no gradient (call it under torch.no_grad)"));
}

// Tells autograd that a kernel writes to `ts`, so that a backward pass that needs
// what was there raises.
inline void written(std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts)
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// Bytes [lo, hi) that a view touches (empty: lo == hi).
struct Range {
  uintptr_t lo, hi;
};
inline Range range_of(const at::Tensor& t) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(t.const_data_ptr());
  const auto sizes = t.sizes(), strides = t.strides();
  int64_t last = 0;
  for (size_t i = 0; i < sizes.size(); ++i) {
    if (sizes[i] == 0) return {p, p};
    last += (sizes[i] - 1) * strides[i];
  }
  return {p, p + static_cast<uintptr_t>(last + 1) * t.element_size()};
}
inline bool apart(const Range& x, const Range& y) { return x.hi <= y.lo || y.hi <= x.lo || x.lo == x.hi || y.lo == y.hi; }
inline bool apart(const at::Tensor& a, const at::Tensor& b) { return apart(range_of(a), range_of(b)); }
// Whether `t` is apart from every one of `others`.
template <size_t N>
bool apart_from_all(const Range& t, const Range (&others)[N]) {
  for (const Range& o : others)
    if (!apart(t, o)) return false;
  return true;
}
inline bool same_view(const at::Tensor& a, const at::Tensor& b) {
  return a.data_ptr() == b.data_ptr() && a.strides() == b.strides() && a.sizes() == b.sizes();
}

inline void index1(const at::Tensor& t, int64_t n, const char* op, const char* m) {
  chk(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous(), op, m);
}

inline int* error_of(const std::optional<at::Tensor>& e, const at::Device& dev, const char* op) {
  if (!e) return nullptr;
  chk(e->scalar_type() == at::kInt && e->numel() >= 1 && e->is_contiguous() && e->device() == dev, op,
      "error is an int32 tensor on the same device");
  return e->data_ptr<int>();
}

using Opt = std::optional<at::Tensor>;

}  // namespace turbol::checks
