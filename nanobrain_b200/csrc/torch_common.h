// Shared by the binding's sources.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <torch/extension.h>

#include <optional>

#include "../../include/nb_attn.h"

namespace nbt {

// The device's status word (one pinned int32 that kernels write to when something went wrong).
volatile int32_t* status_ptr(int64_t device);
// Raises what a finished kernel reported. Never synchronises.
void raise_for_status(volatile int32_t* word);
// NB_ATTN_DEBUG=1: synchronise and look at the status word after every call.
void after_launch(volatile int32_t* word);
void check_rc(int rc, const char* what);

void bind_encoder(pybind11::module_& m);
void bind_block(pybind11::module_& m);

// Forward-mode derivatives: does the tensor carry a tangent? (There is one level, 0.) No operator here has them, and a
// call below autograd would drop the tangent, which reads as a derivative of zero.
inline bool has_tangent(const at::Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
inline bool has_tangent(const std::optional<at::Tensor>& t) { return t.has_value() && has_tangent(*t); }
template <typename... T>
void refuse_tangents(const char* op, const T&... tensors) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(tensors) || ...), "nanobrain_b200.", op,
                              ": there are no forward-mode derivatives, but an argument carries a tangent");
}

// ------------------------------------------------------------------------------------------
// Layouts
// ------------------------------------------------------------------------------------------
using at::Tensor;
constexpr int64_t kHeadDim = 64;

// Can the kernels address this tensor in place (head_dim contiguous, 16-byte rows)?
inline bool strides_ok(const Tensor& t) {
  const int64_t n = t.dim();
  if (t.stride(n - 1) != 1 || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) != 0) return false;
  for (int64_t i = 0; i + 1 < n; ++i)
    if (t.size(i) > 1 && (t.stride(i) <= 0 || t.stride(i) % 8 != 0)) return false;
  return true;
}

// Logical [B, H, L, 64]: as it is, or a copy in [B, L, H, 64] memory.
inline Tensor dense_layout(const Tensor& t) {
  return strides_ok(t) ? t : t.transpose(1, 2).contiguous().transpose(1, 2);
}
inline Tensor packed_layout(const Tensor& t) { return strides_ok(t) ? t : t.contiguous(); }

inline nb_attn_tensor dense_desc(const Tensor& t) {
  const int64_t b = t.size(0), h = t.size(1), l = t.size(2);
  return {t.data_ptr(), b > 1 ? t.stride(0) : h * l * kHeadDim, l > 1 ? t.stride(2) : h * kHeadDim,
          h > 1 ? t.stride(1) : kHeadDim};
}
inline nb_attn_tensor packed_desc(const Tensor& t) {
  const int64_t n = t.size(0), h = t.size(1);
  return {t.data_ptr(), 0, n > 1 ? t.stride(0) : h * kHeadDim, h > 1 ? t.stride(1) : kHeadDim};
}

// Uninitialised tensors on the device of `like`, which is current here: from the caching allocator as
// at::empty's, without its two dispatched calls (seven tensors per forward + backward).
inline Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
// Logical [B, H, L, 64] in [B, L, H, 64] memory.
inline Tensor new_dense(const Tensor& like) {
  const int64_t b = like.size(0), h = like.size(1), l = like.size(2);
  return at::detail::empty_strided_cuda({b, h, l, kHeadDim}, {l * h * kHeadDim, kHeadDim, h * kHeadDim, 1},
                                        at::kBFloat16, like.device());
}

}  // namespace nbt
