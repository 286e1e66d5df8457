// What the host paths of all operations share: status codes as exceptions, checks of arguments, and
// whether a call goes through autograd.
#pragma once
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/types.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>

#include "bsp.h"

namespace bsp_host {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---- errors and arguments ----------------------------------------------------------------------
[[noreturn]] inline void raise_status(int rc) {
  const char* msg = bsp_last_error();
  switch (rc) {
    case BSP_ERR_INVALID: TORCH_CHECK_VALUE(false, msg);
    case BSP_ERR_UNSUPPORTED: TORCH_CHECK_NOT_IMPLEMENTED(false, msg);
    default: TORCH_CHECK(false, msg);
  }
  TORCH_CHECK(false, msg);
}
inline void check(int rc) { if (rc != BSP_OK) raise_status(rc); }

inline int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return BSP_F32;
    case at::kHalf: return BSP_F16;
    case at::kBFloat16: return BSP_BF16;
    default: TORCH_CHECK_VALUE(false, "unsupported dtype ", t.scalar_type(), " (float32, float16 and bfloat16 are)");
  }
}

inline void require_cuda(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "torch_blocksparse_b200 runs on CUDA tensors only (got a ", t.device(), " tensor)");
}

// Everything a call reads has to lie on one device, and a pointer has to be of the type it is read as.
inline void require_same(const Tensor& t, const Tensor& ref, const char* what) {
  TORCH_CHECK(t.device() == ref.device(), what, " is on ", t.device(), ", the call runs on ", ref.device());
  TORCH_CHECK_VALUE(t.scalar_type() == ref.scalar_type(), what, " must be ", ref.scalar_type(), " (got ", t.scalar_type(), ")");
}

// Whether a call on these tensors goes through autograd: one of them needs a gradient (a bias or a
// mask too, although it receives none: the result can then be differentiated), or carries a
// forward-mode tangent, which the functions below refuse (passing them by would drop it silently).
inline bool needs_grad(const Tensor& t) { return t.requires_grad(); }
inline bool needs_grad(const OptTensor& t) { return t && t->requires_grad(); }
inline bool has_tangent(const Tensor& t) { return t._fw_grad(0).defined(); }
inline bool has_tangent(const OptTensor& t) { return t && has_tangent(*t); }
template <typename... Ts> bool recorded(const Ts&... t) {
  return (at::GradMode::is_enabled() && (needs_grad(t) || ...)) || (has_tangent(t) || ...);
}
inline void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
inline int64_t vec_of(const Tensor& t) { return 16 / static_cast<int64_t>(t.element_size()); }
inline bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0; }

}  // namespace bsp_host
