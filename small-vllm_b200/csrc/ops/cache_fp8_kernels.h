#pragma once

// Per-device kernels behind ops::cache_read_fp8 and ops::decode_attention_fp8, which validate the
// inputs, and what their CPU forms share.

#include <ATen/core/Tensor.h>

namespace svllm::ops {

namespace cpu_impl {
// Throws for a request whose length passes its table, whose table names a block outside the cache, or
// with a row whose scale lies outside [2^-60, 2^60].
void check_pages(const char* op, const at::Tensor& k_scale, const at::Tensor& v_scale,
                 const at::Tensor& block_tables, const at::Tensor& seq_lens);
void cache_read_fp8(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache,
                    const at::Tensor& v_cache, const at::Tensor& k_scale,
                    const at::Tensor& v_scale, const at::Tensor& block_tables,
                    const at::Tensor& seq_lens);
void decode_attention_fp8(const at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache,
                          const at::Tensor& v_cache, const at::Tensor& k_scale,
                          const at::Tensor& v_scale, const at::Tensor& block_tables,
                          const at::Tensor& seq_lens, double scale);
}  // namespace cpu_impl

namespace cuda_impl {
void cache_read_fp8(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache,
                    const at::Tensor& v_cache, const at::Tensor& k_scale,
                    const at::Tensor& v_scale, const at::Tensor& block_tables,
                    const at::Tensor& seq_lens);
void decode_attention_fp8(const at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache,
                          const at::Tensor& v_cache, const at::Tensor& k_scale,
                          const at::Tensor& v_scale, const at::Tensor& block_tables,
                          const at::Tensor& seq_lens, double scale);
}  // namespace cuda_impl

}  // namespace svllm::ops
