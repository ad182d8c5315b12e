#pragma once

// Per-device kernels behind ops::paged_plan. `parents` and `tree_mask` are undefined for chains.

#include <ATen/core/Tensor.h>

#include <cstdint>

namespace svllm::ops {

struct PagedPlanTensors {
  at::Tensor context_lens, query_lens, block_tables, blocks_owned, free_blocks, free_count, parents;
  int64_t num_tokens, block_size, max_query_len;
  at::Tensor query_start_loc, seq_lens, slot_mapping, positions, tree_mask, blocks_owned_out,
      free_count_out;
};

namespace cpu_impl {
void paged_plan(const PagedPlanTensors& p);
}

namespace cuda_impl {
void paged_plan(const PagedPlanTensors& p);
}

}  // namespace svllm::ops
