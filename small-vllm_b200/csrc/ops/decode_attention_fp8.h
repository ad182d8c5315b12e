#pragma once

#include <ATen/core/Tensor.h>

#include <optional>

namespace svllm::ops {

// Definition: Attention of a decode step, one query token per request, over the 8-bit paged KV
//             cache (rope.h: qk_norm_rope_cache_fp8 writes it).
// Formula:    out[s, h] = sum_j softmax_j(scale * q[s, h] . k_j) v_j over the rows j < seq_lens[s]
//             of KV head h / (heads / num_kv_heads), k_j and v_j a row's codes times its scale. A
//             request of length 0, and a head with no score above -infinity, gives zeros.
// Domain:     q [S, heads, head_dim] bf16, heads and head_dim contiguous, requests at any stride of
//             whole 16 bytes (a view of a qkv projection); caches, scales, block_tables and
//             seq_lens as cache_read_fp8 takes them; any number of query heads per KV head; scale
//             positive and finite, head_dim^-0.5 by default; one device.
// Returns:    A new bf16 tensor [S, heads, head_dim]. Softmax and sums are fp32; on CUDA the softmax
//             numerators times V's scales are rounded to f16 for the second product, and those below
//             2^-31 of a head's largest may be lost there; elements of a query below 2^-32 of its head's
//             largest may be off by up to 2^-39 of that.
// Throws:     As cache_read_fp8, and on mismatches of q; on CUDA also for a q off 16 bytes.
at::Tensor decode_attention_fp8(const at::Tensor& q, const at::Tensor& k_cache,
                                const at::Tensor& v_cache, const at::Tensor& k_scale,
                                const at::Tensor& v_scale, const at::Tensor& block_tables,
                                const at::Tensor& seq_lens, const std::optional<double>& scale);

}  // namespace svllm::ops
