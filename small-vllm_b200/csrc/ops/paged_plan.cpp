#include "ops/paged_plan.h"

#include <ATen/ATen.h>
#include <c10/util/Exception.h>

#include "ops/common.h"
#include "ops/paged_plan_kernels.h"
#include "svllm_kernels.h"

namespace svllm::ops {

PagedPlan paged_plan(const at::Tensor& context_lens, const at::Tensor& query_lens,
                     const at::Tensor& block_tables, const at::Tensor& blocks_owned,
                     const at::Tensor& free_blocks, const at::Tensor& free_count,
                     int64_t num_tokens, int64_t block_size,
                     const std::optional<at::Tensor>& parents, int64_t max_query_len) {
  const int64_t requests = context_lens.numel();
  const auto check = [&](const at::Tensor& t, const char* name, int64_t dim, int64_t size) {
    TORCH_CHECK(t.scalar_type() == at::kInt && t.is_contiguous(),
                "paged_plan: expected contiguous int32 ", name, ", got ", t.scalar_type());
    TORCH_CHECK(t.dim() == dim && (size < 0 || t.size(0) == size), "paged_plan: ", name,
                " of shape ", t.sizes(), " does not match ", requests, " requests and ",
                num_tokens, " tokens");
    TORCH_CHECK(t.device() == context_lens.device(), "paged_plan: context_lens is on ",
                context_lens.device(), " but ", name, " is on ", t.device());
  };
  TORCH_CHECK(num_tokens >= 0 && block_size > 0, "paged_plan: num_tokens ", num_tokens,
              " must not be negative and block_size ", block_size, " must be positive");
  check(context_lens, "context_lens", 1, requests);
  check(query_lens, "query_lens", 1, requests);
  check(block_tables, "block_tables", 2, requests);
  check(blocks_owned, "blocks_owned", 1, requests);
  check(free_blocks, "free_blocks", 1, -1);
  check(free_count, "free_count", 1, 1);
  TORCH_CHECK(block_tables.size(1) > 0, "paged_plan: block_tables of shape ",
              block_tables.sizes(), " has no room for a block");
  const bool tree = parents.has_value() && parents->defined();
  if (tree) {
    check(*parents, "parents", 1, num_tokens);
    TORCH_CHECK(max_query_len >= 1 && max_query_len <= SVLLM_MAX_TREE_NODES,
                "paged_plan: max_query_len ", max_query_len, " must be in [1, ",
                SVLLM_MAX_TREE_NODES, "] where parents are given");
  }

  PagedPlanTensors p;
  p.context_lens = context_lens;
  p.query_lens = query_lens;
  p.block_tables = block_tables;
  p.blocks_owned = blocks_owned;
  p.free_blocks = free_blocks;
  p.free_count = free_count;
  p.num_tokens = num_tokens;
  p.block_size = block_size;
  p.max_query_len = max_query_len;
  const int64_t words = tree ? (max_query_len + 63) / 64 : 0;
  using detail::Outputs;
  Outputs out(Outputs::size(at::kLong, num_tokens) * 2 +
                  Outputs::size(at::kLong, num_tokens * words) +
                  Outputs::size(at::kInt, requests + 1) + Outputs::size(at::kInt, requests) * 2 +
                  Outputs::size(at::kInt, 1),
              context_lens.options());
  p.slot_mapping = out.take(at::kLong, {num_tokens});
  p.positions = out.take(at::kLong, {num_tokens});
  if (tree) {
    p.parents = *parents;
    p.tree_mask = out.take(at::kLong, {num_tokens, words});
  }
  p.query_start_loc = out.take(at::kInt, {requests + 1});
  p.seq_lens = out.take(at::kInt, {requests});
  p.blocks_owned_out = out.take(at::kInt, {requests});
  p.free_count_out = out.take(at::kInt, {1});
  switch (context_lens.device().type()) {
    case c10::DeviceType::CPU:
      cpu_impl::paged_plan(p);
      break;
    case c10::DeviceType::CUDA:
      cuda_impl::paged_plan(p);
      break;
    default:
      TORCH_CHECK(false, "paged_plan: unsupported device ", context_lens.device());
  }
  return {p.query_start_loc, p.seq_lens, p.slot_mapping, p.positions,
          tree ? std::optional<at::Tensor>(p.tree_mask) : std::nullopt, p.blocks_owned_out,
          p.free_count_out};
}

}  // namespace svllm::ops
