#pragma once

// Per-device kernels behind ops::tree_attention: out [T, heads, D] contiguous, q [T, heads, D] at
// any token stride, tree_mask undefined for the causal form.

#include <ATen/core/Tensor.h>

namespace svllm::ops {

namespace cpu_impl {
void tree_attention(const at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache,
                    const at::Tensor& v_cache, const at::Tensor& block_tables,
                    const at::Tensor& seq_lens, const at::Tensor& query_start_loc,
                    const at::Tensor& tree_mask, double scale);
}

namespace cuda_impl {
void tree_attention(const at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache,
                    const at::Tensor& v_cache, const at::Tensor& block_tables,
                    const at::Tensor& seq_lens, const at::Tensor& query_start_loc,
                    const at::Tensor& tree_mask, double scale);
}

}  // namespace svllm::ops
