#include "ops/cache_fp8.h"

#include <ATen/ATen.h>
#include <c10/util/Exception.h>

#include "ops/cache_fp8_kernels.h"
#include "ops/common.h"

namespace svllm::ops {

namespace detail {

void check_fp8_cache(const char* op, const at::Tensor& k_cache, const at::Tensor& v_cache,
                     const at::Tensor& k_scale, const at::Tensor& v_scale,
                     const at::Device& device) {
  TORCH_CHECK(k_cache.scalar_type() == at::kFloat8_e4m3fn &&
                  v_cache.scalar_type() == at::kFloat8_e4m3fn,
              op, ": expected float8_e4m3fn caches, got ", k_cache.scalar_type(), " and ",
              v_cache.scalar_type());
  TORCH_CHECK(k_scale.scalar_type() == at::kFloat8_e8m0fnu &&
                  v_scale.scalar_type() == at::kFloat8_e8m0fnu,
              op, ": expected float8_e8m0fnu scales, got ", k_scale.scalar_type(), " and ",
              v_scale.scalar_type());
  TORCH_CHECK(k_cache.dim() >= 2 && (k_cache.size(-1) == 64 || k_cache.size(-1) == 128) &&
                  k_cache.size(-2) > 0 && k_cache.is_contiguous() && v_cache.is_contiguous() &&
                  v_cache.sizes() == k_cache.sizes(),
              op, ": caches of shape ", k_cache.sizes(), " and ", v_cache.sizes(),
              " must be contiguous [..., num_kv_heads, 64 or 128]");
  const at::IntArrayRef rows = k_cache.sizes().slice(0, k_cache.dim() - 1);
  TORCH_CHECK(k_scale.sizes() == rows && v_scale.sizes() == rows && k_scale.is_contiguous() &&
                  v_scale.is_contiguous(),
              op, ": scales of shape ", k_scale.sizes(), " and ", v_scale.sizes(),
              " must be contiguous ", rows, ", one for every row of the caches");
  TORCH_CHECK(k_cache.device() == device && v_cache.device() == device &&
                  k_scale.device() == device && v_scale.device() == device,
              op, ": a cache or its scales are not on ", device);
}

void check_fp8_pages(const char* op, const at::Tensor& k_cache, const at::Tensor& block_tables,
                     const at::Tensor& seq_lens) {
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.numel() > 0,
              op, ": caches must be [num_blocks, block_size, num_kv_heads, head_dim], got shape ",
              k_cache.sizes());
  TORCH_CHECK(block_tables.scalar_type() == at::kInt && block_tables.is_contiguous() &&
                  seq_lens.scalar_type() == at::kInt && seq_lens.is_contiguous(),
              op, ": block_tables and seq_lens must be contiguous int32");
  TORCH_CHECK(seq_lens.dim() == 1 && block_tables.dim() == 2 &&
                  block_tables.size(0) == seq_lens.size(0),
              op, ": block_tables ", block_tables.sizes(), " and seq_lens ", seq_lens.sizes(),
              " must be [S, blocks] and [S]");
  TORCH_CHECK(block_tables.device() == k_cache.device() && seq_lens.device() == k_cache.device(),
              op, ": the caches are on ", k_cache.device(), " but block_tables or seq_lens is not");
}

}  // namespace detail

std::tuple<at::Tensor, at::Tensor> cache_read_fp8(const at::Tensor& k_cache,
                                                  const at::Tensor& v_cache,
                                                  const at::Tensor& k_scale,
                                                  const at::Tensor& v_scale,
                                                  const at::Tensor& block_tables,
                                                  const at::Tensor& seq_lens) {
  const at::Device device = k_cache.device();
  detail::check_fp8_cache("cache_read_fp8", k_cache, v_cache, k_scale, v_scale, device);
  detail::check_fp8_pages("cache_read_fp8", k_cache, block_tables, seq_lens);
  TORCH_CHECK(device.is_cpu() || device.is_cuda(), "cache_read_fp8: unsupported device ", device);
  const int64_t shape[] = {seq_lens.size(0), block_tables.size(1) * k_cache.size(1),
                           k_cache.size(2), k_cache.size(3)};
  const int64_t bytes =
      detail::Outputs::size(at::kBFloat16, shape[0] * shape[1] * shape[2] * shape[3]);
  detail::Outputs out(2 * bytes, k_cache.options());
  const at::Tensor k = out.take(at::kBFloat16, shape), v = out.take(at::kBFloat16, shape);
  if (device.is_cuda()) {
    cuda_impl::cache_read_fp8(k, v, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens);
  } else {
    cpu_impl::cache_read_fp8(k, v, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens);
  }
  return {k, v};
}

}  // namespace svllm::ops
