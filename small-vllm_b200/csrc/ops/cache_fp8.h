#pragma once

#include <ATen/core/Tensor.h>

#include <tuple>

namespace svllm::ops {

// Definition: The cached rows of whole requests back from the 8-bit cache, in bf16 and in the order
//             of each request: what prefill attention, a verification step or a hand-over to a bf16
//             cache reads.
// Formula:    k[s, j, h] = code * scale of row j of request s, at slot block_tables[s][j /
//             block_size] * block_size + j % block_size, for j < seq_lens[s]; 0 behind it. Exact:
//             a code times its scale is a bf16 value. v likewise.
// Domain:     k_cache and v_cache contiguous float8_e4m3fn [num_blocks, block_size, num_kv_heads,
//             head_dim], head_dim 64 or 128; k_scale and v_scale contiguous float8_e8m0fnu
//             [num_blocks, block_size, num_kv_heads], from 2^-60 to 2^60, which is what the rotary
//             step leaves; block_tables [S, max_blocks] and seq_lens [S] contiguous int32; one device.
// Returns:    k and v, bf16 [S, max_blocks * block_size, num_kv_heads, head_dim]. Seen as
//             [S * max_blocks, block_size, num_kv_heads, head_dim] they are a paged bf16 cache in
//             which page p of request s is block s * max_blocks + p.
// Throws:     c10::Error on dtype, shape, layout or device mismatches, and on CPU for a length past
//             the table, a block outside the cache or a read row's scale out of range. On CUDA those
//             raise a bit of the device error word; the length is cut to the table's, the block read
//             as block 0, the scale taken as the nearest in range.
std::tuple<at::Tensor, at::Tensor> cache_read_fp8(const at::Tensor& k_cache,
                                                  const at::Tensor& v_cache,
                                                  const at::Tensor& k_scale,
                                                  const at::Tensor& v_scale,
                                                  const at::Tensor& block_tables,
                                                  const at::Tensor& seq_lens);

namespace detail {

// The checks that the operators of the 8-bit cache share: dtypes, layouts, shapes that match, one
// device.
void check_fp8_cache(const char* op, const at::Tensor& k_cache, const at::Tensor& v_cache,
                     const at::Tensor& k_scale, const at::Tensor& v_scale,
                     const at::Device& device);

// And of those that read it by block tables.
void check_fp8_pages(const char* op, const at::Tensor& k_cache, const at::Tensor& block_tables,
                     const at::Tensor& seq_lens);

}  // namespace detail

}  // namespace svllm::ops
