#include "ops/tree_attention.h"

#include <ATen/ATen.h>
#include <c10/util/Exception.h>

#include <cmath>

#include "ops/tree_attention_kernels.h"
#include "svllm_kernels.h"

namespace svllm::ops {

at::Tensor tree_attention(const at::Tensor& q, const at::Tensor& k_cache,
                          const at::Tensor& v_cache, const at::Tensor& block_tables,
                          const at::Tensor& seq_lens, const at::Tensor& query_start_loc,
                          const std::optional<at::Tensor>& tree_mask,
                          const std::optional<double>& scale) {
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || (q.is_cpu() && q.scalar_type() == at::kFloat),
              "tree_attention: expected bf16 q (or fp32 on CPU), got ", q.scalar_type(), " on ",
              q.device());
  TORCH_CHECK(k_cache.scalar_type() == q.scalar_type() && v_cache.scalar_type() == q.scalar_type(),
              "tree_attention: q is ", q.scalar_type(), " but the caches are ",
              k_cache.scalar_type(), " and ", v_cache.scalar_type());
  TORCH_CHECK(q.dim() == 3 && q.size(1) > 0 && q.size(2) > 0,
              "tree_attention: q must be [tokens, heads, head_dim], got shape ", q.sizes());
  const int64_t tokens = q.size(0), heads = q.size(1), dim = q.size(2);
  TORCH_CHECK(tokens == 0 || (q.stride(2) == 1 && (heads == 1 || q.stride(1) == dim) &&
                              (tokens == 1 || q.stride(0) >= heads * dim)),
              "tree_attention: q's heads must be contiguous, got strides ", q.strides());
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.numel() > 0 && k_cache.size(3) == dim &&
                  heads % k_cache.size(2) == 0 && k_cache.is_contiguous() &&
                  v_cache.sizes() == k_cache.sizes() && v_cache.is_contiguous(),
              "tree_attention: caches of shape ", k_cache.sizes(), " and ", v_cache.sizes(),
              " must be contiguous [blocks, block_size, kv_heads, head_dim] for q of shape ",
              q.sizes());
  const int64_t requests = seq_lens.numel();
  const bool lists = block_tables.scalar_type() == at::kInt && block_tables.is_contiguous() &&
                     seq_lens.scalar_type() == at::kInt && seq_lens.is_contiguous() &&
                     query_start_loc.scalar_type() == at::kInt && query_start_loc.is_contiguous();
  TORCH_CHECK(lists,
              "tree_attention: block_tables, seq_lens and query_start_loc must be contiguous int32");
  TORCH_CHECK(seq_lens.dim() == 1 && block_tables.dim() == 2 &&
                  block_tables.size(0) == requests && block_tables.size(1) > 0 &&
                  query_start_loc.dim() == 1 && query_start_loc.size(0) == requests + 1,
              "tree_attention: block_tables ", block_tables.sizes(), ", seq_lens ",
              seq_lens.sizes(), " and query_start_loc ", query_start_loc.sizes(),
              " must be [S, blocks], [S] and [S + 1]");
  const bool tree = tree_mask.has_value() && tree_mask->defined();
  if (tree) {
    TORCH_CHECK(tree_mask->scalar_type() == at::kLong && tree_mask->is_contiguous() &&
                    tree_mask->dim() == 2 && tree_mask->size(0) == tokens &&
                    tree_mask->size(1) > 0 &&
                    tree_mask->size(1) <= SVLLM_MAX_TREE_NODES / 64,
                "tree_attention: tree_mask must be contiguous int64 [tokens, 1 to ",
                SVLLM_MAX_TREE_NODES / 64, " words], got ", tree_mask->scalar_type(), " ",
                tree_mask->sizes(), " for ", tokens, " tokens");
  }
  const bool same_device =
      k_cache.device() == q.device() && v_cache.device() == q.device() &&
      block_tables.device() == q.device() && seq_lens.device() == q.device() &&
      query_start_loc.device() == q.device() && (!tree || tree_mask->device() == q.device());
  TORCH_CHECK(same_device, "tree_attention: q is on ", q.device(),
              " but a cache, the mask or the request lists are elsewhere");
  const double factor = scale.value_or(std::pow(static_cast<double>(dim), -0.5));
  TORCH_CHECK(factor > 0.0 && std::isfinite(static_cast<float>(factor)) &&
                  static_cast<float>(factor) > 0.0f,
              "tree_attention: scale must be positive and finite, got ", factor);

  at::Tensor out = at::empty({tokens, heads, dim}, q.options());
  const at::Tensor mask = tree ? *tree_mask : at::Tensor();
  switch (q.device().type()) {
    case c10::DeviceType::CPU:
      cpu_impl::tree_attention(out, q, k_cache, v_cache, block_tables, seq_lens, query_start_loc,
                               mask, factor);
      break;
    case c10::DeviceType::CUDA:
      cuda_impl::tree_attention(out, q, k_cache, v_cache, block_tables, seq_lens, query_start_loc,
                                mask, factor);
      break;
    default:
      TORCH_CHECK(false, "tree_attention: unsupported device ", q.device());
  }
  return out;
}

}  // namespace svllm::ops
