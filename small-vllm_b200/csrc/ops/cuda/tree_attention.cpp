// CUDA side of ops::tree_attention: a thin LibTorch -> C ABI shim.
#include <ATen/ATen.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "ops/common.h"
#include "ops/tree_attention_kernels.h"

namespace svllm::ops::cuda_impl {

void tree_attention(const at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache,
                    const at::Tensor& v_cache, const at::Tensor& block_tables,
                    const at::Tensor& seq_lens, const at::Tensor& query_start_loc,
                    const at::Tensor& tree_mask, double scale) {
  const int64_t tokens = q.size(0), heads = q.size(1), dim = q.size(2);
  if (tokens == 0) return;
  const c10::cuda::CUDAGuard device_guard(q.device());
  const auto stream = reinterpret_cast<svllm_stream>(c10::cuda::getCurrentCUDAStream().stream());
  int64_t bytes = 0;
  detail::check_status("tree_attention", svllm_tree_attention_workspace_bytes(dim, &bytes));
  // from the caching allocator per call: calls on other streams, and captured graphs, get their own
  const c10::DataPtr workspace = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);
  detail::check_status(
      "tree_attention",
      svllm_tree_attention_bf16(
          out.mutable_data_ptr(), q.const_data_ptr(), tokens == 1 ? heads * dim : q.stride(0),
          k_cache.const_data_ptr(), v_cache.const_data_ptr(), k_cache.size(0), k_cache.size(1),
          block_tables.const_data_ptr<int32_t>(), block_tables.size(1),
          seq_lens.const_data_ptr<int32_t>(), query_start_loc.const_data_ptr<int32_t>(),
          seq_lens.numel(), tokens, heads, k_cache.size(2), dim,
          tree_mask.defined() ? tree_mask.const_data_ptr<int64_t>() : nullptr,
          tree_mask.defined() ? tree_mask.size(1) : 0, static_cast<float>(scale),
          workspace.get(), bytes, stream));
}

}  // namespace svllm::ops::cuda_impl
