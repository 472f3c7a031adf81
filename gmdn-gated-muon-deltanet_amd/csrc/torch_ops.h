// Shared by the files that register torch.ops.gmdn.*: error checks, streams,
// small allocations, and calls of the operators below autograd.
#pragma once
#include "../../include/gmdn_scan.h"

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <optional>
#include <tuple>
#include <type_traits>
#include <vector>

namespace gmdn_ops {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

inline void check(int rc, const char* what) {
  TORCH_CHECK(rc == GMDN_OK, what, " failed with code ", rc, ": ", gmdn_error_string(rc));
}
inline void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
inline float* fp(const Tensor& t) { return t.numel() ? t.data_ptr<float>() : nullptr; }
inline const float* fp(const OptTensor& t) { return t ? t->data_ptr<float>() : nullptr; }
inline Tensor f32_empty(const Tensor& like, at::IntArrayRef size) { return at::empty(size, like.options().dtype(at::kFloat)); }
inline Tensor none_of(const Tensor& like) { return f32_empty(like, {0}); }
inline Tensor bytes_of(const Tensor& like, size_t n) {
  return at::empty({(int64_t)n}, like.options().dtype(at::kByte));
}

inline void check_rank(const Tensor& t, int64_t rank, const char* what) {
  TORCH_CHECK(t.dim() == rank, what, " must have ", rank, " dimensions, got shape ", t.sizes());
}

// Calls through the dispatcher, below autograd.
template <class F>
auto op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
// A kernel's signature with symbolic integers: a traced size reaches the
// schema unspecialised, and only the kernels themselves see plain integers.
template <class F>
struct Symbolic;
template <class R, class... A>
struct Symbolic<R(A...)> {
  using T = R(std::conditional_t<std::is_same_v<A, int64_t>, c10::SymInt, A>...);
};
#define GMDN_OP(fn) \
  ([]() -> const auto& { static const auto h = op<Symbolic<decltype(fn)>::T>("gmdn::" #fn); return h; }())

inline bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// Refuses inputs that carry a forward-mode tangent: calls below autograd would
// return outputs without one, and no error.
inline void refuse_tangents(const char* name, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), "gmdn::", name,
                                " has no forward-mode derivative (jvp)");
}
inline Tensor opt(const OptTensor& t) { return t ? *t : Tensor(); }
inline OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

}  // namespace gmdn_ops
