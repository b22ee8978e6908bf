// What the operator files share: argument checks, allocation, status of the C ABI.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include "t2fw_b200.h"

namespace t2fw_ops {

#define T2FW_CHECK_INPUT(x)                                             \
  TORCH_CHECK((x).device().is_cuda(), #x " must be a CUDA tensor");     \
  TORCH_CHECK((x).is_contiguous(), #x " must be contiguous")

inline int dtype_code(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kHalf: return T2FW_F16;
    case at::kBFloat16: return T2FW_BF16;
    case at::kFloat: return T2FW_F32;
    case at::kDouble: return T2FW_F64;
    default: TORCH_CHECK(false, "t2fw: unsupported dtype ", t.scalar_type());
  }
  return -1;
}

inline void check_status(int rc, const char *what) {
  TORCH_CHECK(rc == T2FW_OK, what, " failed (status ", rc, "): ", t2fw_last_error());
}

inline void check_same(const at::Tensor &a, const at::Tensor &ref, const char *name) {
  TORCH_CHECK(a.scalar_type() == ref.scalar_type(), name, ": dtype differs from the first tensor's");
  TORCH_CHECK(a.device() == ref.device(), name, ": device differs from the first tensor's");
}

// Uninitialised tensors of `like`'s device straight from the caching allocator: a call makes up to seven
// of them, and each trip through the dispatcher costs about as much host time as a kernel launch.
inline at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor &like) {
  return at::Tensor(at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt));
}
inline at::Tensor new_like(const at::Tensor &t) { return new_tensor(t.sizes(), t.scalar_type(), t); }

// For a tensor of the caller's that a kernel is about to write: what saved it for a backward pass is to notice.  (Inference
// tensors cannot be saved and have no counter.)
inline void mark_changed(const at::Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Scratch of one call: freed when the call returns, which the caching allocator orders on the stream.
inline c10::DataPtr make_scratch(size_t bytes) {
  if (bytes == 0) return c10::DataPtr();
  return c10::cuda::CUDACachingAllocator::get()->allocate(bytes);
}

}  // namespace t2fw_ops
