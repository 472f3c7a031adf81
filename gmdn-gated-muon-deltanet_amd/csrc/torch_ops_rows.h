// Shared by the operators over (..., d) tensors: their rows, allocations, and
// checks of types and shapes.
#pragma once
#include "torch_ops.h"

#include <ATen/hip/EmptyTensor.h>

namespace gmdn_ops {

using at::ScalarType;

// A contiguous tensor beside x, straight from the allocator: five of them
// through the dispatcher are a sixth of a small call's host time.
inline Tensor fresh(const Tensor& x, at::IntArrayRef sizes, ScalarType dtype) {
  return at::detail::empty_cuda(sizes, dtype, x.device(), std::nullopt);
}
inline Tensor fresh(const Tensor& x, at::IntArrayRef sizes) { return fresh(x, sizes, at::kFloat); }

inline int32_t type_code(ScalarType t, const char* what) {
  TORCH_CHECK(t == at::kBFloat16 || t == at::kFloat, what, " is bfloat16 or float32, got ", t);
  return t == at::kFloat ? GMDN_DTYPE_F32 : GMDN_DTYPE_BF16;
}

// t as `rows` rows of d values.
struct Rows {
  Tensor t;
  int64_t rows, d, stride;
  const void* ptr() const { return t.data_ptr(); }
};
inline Rows rows_of(const Tensor& t, const char* what) {
  TORCH_CHECK(t.dim() >= 1 && t.size(-1) > 0, what, " has rows of at least one value in its last dimension, got shape ",
              t.sizes());
  const int64_t d = t.size(-1), rows = t.numel() / d;
  bool fits = d == 1 || t.stride(-1) == 1;
  int64_t stride = d, extent = -1;  // extent: what the dimension outside has to stride by
  for (int64_t i = t.dim() - 2; fits && i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (extent < 0)
      stride = t.stride(i);
    else
      fits = t.stride(i) == extent;
    extent = t.stride(i) * t.size(i);
  }
  if (rows == 0) return {t, 0, d, d};
  return fits ? Rows{t, rows, d, stride} : Rows{t.contiguous(), rows, d, d};
}

inline std::vector<int64_t> lead(const Tensor& t) { return t.sizes().slice(0, t.dim() - 1).vec(); }
inline std::vector<int64_t> with_last(std::vector<int64_t> s, int64_t n) {
  s.push_back(n);
  return s;
}

inline void check_like(const Tensor& t, const Tensor& x, at::IntArrayRef shape, const char* what) {
  TORCH_CHECK(t.device() == x.device(), what, " is on ", t.device(), ", the operator's input on ", x.device());
  TORCH_CHECK(t.sizes() == shape, what, " has shape ", t.sizes(), " where ", shape, " is expected");
}
// A float32 vector of per-row (or per-group) values, contiguous.
inline Tensor stat(const Tensor& t, const Tensor& x, at::IntArrayRef shape, const char* what) {
  check_like(t, x, shape, what);
  TORCH_CHECK(t.scalar_type() == at::kFloat, what, " is float32, got ", t.scalar_type());
  return t.contiguous();
}
inline OptTensor stat(const OptTensor& t, const Tensor& x, at::IntArrayRef shape, const char* what) {
  if (!t) return t;
  check_like(*t, x, shape, what);
  return t->to(at::kFloat).contiguous();
}
inline const void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }

// Token numbers of the given shape, contiguous int64, beside `like`.
inline Tensor tokens_of(const Tensor& tokens, const Tensor& like, at::IntArrayRef shape) {
  check_like(tokens, like, shape, "tokens");
  TORCH_CHECK(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt, "tokens are int64 or int32, got ",
              tokens.scalar_type());
  return tokens.to(at::kLong).contiguous();
}

}  // namespace gmdn_ops
