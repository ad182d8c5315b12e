#pragma once

// Shared helpers of the op layer: the CUDA stream an op runs on and the C-ABI status check.

#include <ATen/ATen.h>
#include <c10/core/TensorImpl.h>
#include <c10/util/Exception.h>

#include "svllm_kernels.h"

namespace svllm::ops::detail {

// Throws c10::Error naming the op when a C-ABI call returns an error status.
inline void check_status(const char* op, int status) {
  TORCH_CHECK(status == SVLLM_OK, op, ": ", svllm_status_string(status), " (status ", status, ")");
}

// Contiguous output tensors of one call in one allocation, each at a multiple of 16 bytes: another
// allocation, or a view made by the dispatcher, costs its caller about a microsecond, this a tenth.
class Outputs {
 public:
  // `bytes`: the sum of size() over the tensors to come
  Outputs(int64_t bytes, const at::TensorOptions& options)
      : base_(at::empty({bytes}, options.dtype(at::kByte))) {}

  static int64_t size(at::ScalarType dtype, int64_t count) {
    return (count * static_cast<int64_t>(c10::elementSize(dtype)) + 15) / 16 * 16;
  }

  at::Tensor take(at::ScalarType dtype, at::IntArrayRef sizes) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(
        c10::Storage(base_.storage()), base_.key_set(), c10::scalarTypeToTypeMeta(dtype));
    t.unsafeGetTensorImpl()->set_storage_offset(
        used_ / static_cast<int64_t>(c10::elementSize(dtype)));
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    used_ += size(dtype, t.numel());
    return t;
  }

 private:
  at::Tensor base_;
  int64_t used_ = 0;
};

}  // namespace svllm::ops::detail
