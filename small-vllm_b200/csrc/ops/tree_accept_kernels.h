#pragma once

// Per-device kernels behind ops::tree_accept and ops::tree_commit (`parents` undefined for chains).

#include <ATen/core/Tensor.h>

#include <cstdint>
#include <vector>

namespace svllm::ops {

struct TreeAcceptTensors {
  at::Tensor ids, targets, parents, query_start_loc, seq_lens, context_lens;
  int64_t max_query_len;
  at::Tensor path, tokens, num_accepted, context_lens_out;
};

namespace cpu_impl {
void tree_accept(const TreeAcceptTensors& a);
void tree_commit(const std::vector<at::Tensor>& k_caches, const std::vector<at::Tensor>& v_caches,
                 int64_t num_slots, const at::Tensor& path, const at::Tensor& num_accepted,
                 const at::Tensor& slot_mapping, const at::Tensor& query_start_loc);
}  // namespace cpu_impl

namespace cuda_impl {
void tree_accept(const TreeAcceptTensors& a);
void tree_commit(const std::vector<at::Tensor>& k_caches, const std::vector<at::Tensor>& v_caches,
                 int64_t num_slots, const at::Tensor& path, const at::Tensor& num_accepted,
                 const at::Tensor& slot_mapping, const at::Tensor& query_start_loc);
}  // namespace cuda_impl

}  // namespace svllm::ops
