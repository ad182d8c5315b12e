#include "ops/decode_attention_fp8.h"

#include <ATen/ATen.h>
#include <c10/util/Exception.h>

#include <cmath>

#include "ops/cache_fp8.h"
#include "ops/cache_fp8_kernels.h"

namespace svllm::ops {

at::Tensor decode_attention_fp8(const at::Tensor& q, const at::Tensor& k_cache,
                                const at::Tensor& v_cache, const at::Tensor& k_scale,
                                const at::Tensor& v_scale, const at::Tensor& block_tables,
                                const at::Tensor& seq_lens, const std::optional<double>& scale) {
  constexpr const char* kOp = "decode_attention_fp8";
  TORCH_CHECK(q.scalar_type() == at::kBFloat16, kOp, ": expected bf16 q, got ", q.scalar_type());
  TORCH_CHECK(q.dim() == 3, kOp, ": q must be [requests, heads, head_dim], got shape ", q.sizes());
  detail::check_fp8_cache(kOp, k_cache, v_cache, k_scale, v_scale, q.device());
  detail::check_fp8_pages(kOp, k_cache, block_tables, seq_lens);
  const int64_t requests = q.size(0), heads = q.size(1), dim = q.size(2);
  TORCH_CHECK(dim == k_cache.size(3) && heads > 0 && heads % k_cache.size(2) == 0, kOp,
              ": q of shape ", q.sizes(), " does not match caches of shape ", k_cache.sizes());
  TORCH_CHECK(requests == seq_lens.size(0), kOp, ": ", seq_lens.size(0), " seq_lens for ",
              requests, " requests");
  TORCH_CHECK(requests == 0 || (q.stride(2) == 1 && (heads == 1 || q.stride(1) == dim) &&
                                (requests == 1 || q.stride(0) >= heads * dim)),
              kOp, ": q's heads must be contiguous, got strides ", q.strides());
  const double factor = scale.value_or(std::pow(static_cast<double>(dim), -0.5));
  // also in base 2, which is what the kernel takes
  TORCH_CHECK(factor > 0.0 && std::isfinite(static_cast<float>(factor / std::log(2.0))) &&
                  static_cast<float>(factor) > 0.0f,
              kOp, ": scale must be positive and finite, got ", factor);
  at::Tensor out = at::empty({requests, heads, dim}, q.options());
  switch (q.device().type()) {
    case c10::DeviceType::CPU:
      cpu_impl::decode_attention_fp8(out, q, k_cache, v_cache, k_scale, v_scale, block_tables,
                                     seq_lens, factor);
      break;
    case c10::DeviceType::CUDA:
      cuda_impl::decode_attention_fp8(out, q, k_cache, v_cache, k_scale, v_scale, block_tables,
                                      seq_lens, factor);
      break;
    default:
      TORCH_CHECK(false, kOp, ": unsupported device ", q.device());
  }
  return out;
}

}  // namespace svllm::ops
