#pragma once

// Shared helpers of the op layer: the CUDA stream an op runs on and the C-ABI status check.

#include <ATen/core/Tensor.h>
#include <c10/core/TensorImpl.h>
#include <c10/util/Exception.h>

#include "svllm_kernels.h"

namespace svllm::ops::detail {

// Throws c10::Error naming the op when a C-ABI call returns an error status.
inline void check_status(const char* op, int status) {
  TORCH_CHECK(status == SVLLM_OK, op, ": ", svllm_status_string(status), " (status ", status, ")");
}

// A contiguous tensor of `sizes` over `base`'s memory from element `offset` on. Several outputs of
// one call share an allocation this way: a view made by the dispatcher, or another allocation, costs
// its caller about a microsecond, this a tenth of that.
inline at::Tensor carve(const at::Tensor& base, int64_t offset, at::IntArrayRef sizes) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(
      c10::Storage(base.storage()), base.key_set(), base.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(base.storage_offset() + offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

}  // namespace svllm::ops::detail
