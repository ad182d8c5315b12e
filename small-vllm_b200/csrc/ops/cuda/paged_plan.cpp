// CUDA side of ops::paged_plan: a thin LibTorch -> C ABI shim.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "ops/common.h"
#include "ops/paged_plan_kernels.h"

namespace svllm::ops::cuda_impl {

void paged_plan(const PagedPlanTensors& p) {
  const c10::cuda::CUDAGuard device_guard(p.context_lens.device());
  const auto stream = reinterpret_cast<svllm_stream>(c10::cuda::getCurrentCUDAStream().stream());
  const bool tree = p.parents.defined();
  detail::check_status(
      "paged_plan",
      svllm_paged_plan(
          p.context_lens.const_data_ptr<int32_t>(), p.query_lens.const_data_ptr<int32_t>(),
          p.context_lens.numel(), p.block_tables.mutable_data_ptr<int32_t>(),
          p.block_tables.size(1), p.blocks_owned.const_data_ptr<int32_t>(),
          p.free_blocks.mutable_data_ptr<int32_t>(), p.free_blocks.numel(),
          p.free_count.const_data_ptr<int32_t>(), p.block_size,
          tree && p.num_tokens > 0 ? p.parents.const_data_ptr<int32_t>() : nullptr,
          p.max_query_len, p.num_tokens, p.query_start_loc.mutable_data_ptr<int32_t>(),
          p.seq_lens.mutable_data_ptr<int32_t>(), p.slot_mapping.mutable_data_ptr<int64_t>(),
          p.positions.mutable_data_ptr<int64_t>(),
          tree ? p.tree_mask.mutable_data_ptr<int64_t>() : nullptr,
          p.blocks_owned_out.mutable_data_ptr<int32_t>(),
          p.free_count_out.mutable_data_ptr<int32_t>(), stream));
}

}  // namespace svllm::ops::cuda_impl
