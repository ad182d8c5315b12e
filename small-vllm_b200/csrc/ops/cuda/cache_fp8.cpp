// CUDA side of ops::cache_read_fp8 and ops::decode_attention_fp8: thin LibTorch -> C ABI shims.
#include <ATen/ATen.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "ops/cache_fp8_kernels.h"
#include "ops/common.h"

namespace svllm::ops::cuda_impl {

void cache_read_fp8(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache,
                    const at::Tensor& v_cache, const at::Tensor& k_scale,
                    const at::Tensor& v_scale, const at::Tensor& block_tables,
                    const at::Tensor& seq_lens) {
  if (k.numel() == 0) return;
  const c10::cuda::CUDAGuard device_guard(k.device());
  const auto stream = reinterpret_cast<svllm_stream>(c10::cuda::getCurrentCUDAStream().stream());
  detail::check_status(
      "cache_read_fp8",
      svllm_cache_read_fp8_bf16(
          k.mutable_data_ptr(), v.mutable_data_ptr(), k_cache.const_data_ptr(),
          v_cache.const_data_ptr(), k_scale.const_data_ptr(), v_scale.const_data_ptr(),
          k_cache.size(0), k_cache.size(1), block_tables.const_data_ptr<int32_t>(),
          block_tables.size(1), seq_lens.const_data_ptr<int32_t>(), seq_lens.numel(),
          k_cache.size(2), k_cache.size(3), stream));
}

void decode_attention_fp8(const at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache,
                          const at::Tensor& v_cache, const at::Tensor& k_scale,
                          const at::Tensor& v_scale, const at::Tensor& block_tables,
                          const at::Tensor& seq_lens, double scale) {
  const int64_t requests = q.size(0), heads = q.size(1), dim = q.size(2);
  if (requests == 0) return;
  const c10::cuda::CUDAGuard device_guard(q.device());
  const auto stream = reinterpret_cast<svllm_stream>(c10::cuda::getCurrentCUDAStream().stream());
  int64_t bytes = 0;
  detail::check_status("decode_attention_fp8",
                       svllm_decode_attention_fp8_workspace_bytes(
                           requests, heads, k_cache.size(2), dim, block_tables.size(1),
                           k_cache.size(1), &bytes));
  // from the caching allocator per call: calls on other streams, and captured graphs, get their own
  c10::DataPtr workspace;
  if (bytes > 0) workspace = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);
  detail::check_status(
      "decode_attention_fp8",
      svllm_decode_attention_fp8_bf16(
          out.mutable_data_ptr(), q.const_data_ptr(), requests == 1 ? heads * dim : q.stride(0),
          k_cache.const_data_ptr(), v_cache.const_data_ptr(), k_scale.const_data_ptr(),
          v_scale.const_data_ptr(), k_cache.size(0), k_cache.size(1),
          block_tables.const_data_ptr<int32_t>(), block_tables.size(1),
          seq_lens.const_data_ptr<int32_t>(), requests, heads, k_cache.size(2), dim,
          static_cast<float>(scale), workspace.get(), bytes, stream));
}

}  // namespace svllm::ops::cuda_impl
