#pragma once

#include <ATen/core/Tensor.h>

#include <optional>

namespace svllm::ops {

// Definition: Attention of every token of a step over a paged KV cache that already holds the
//             step's own K and V. A request's tokens are the nodes of a tree of drafted tokens
//             (or a chain): a node sees the request's earlier context, itself and its ancestors.
// Formula:    out[t, h] = sum_j p_j v_j, p = softmax_j(scale * q[t, h] . k_j) over the rows j <
//             context and the nodes j - context whose bit tree_mask[t] has; without a mask the nodes
//             up to t's own (causal). Row j of request b is row block_tables[b][j / block_size] *
//             block_size + j % block_size of the cache, KV head h / (heads / KV heads); context =
//             seq_lens[b] - (query_start_loc[b + 1] - query_start_loc[b]). A token that sees no row, or
//             no score above -infinity, a token of a request with seq_lens 0, and one behind the last request gets zeros.
//             What a token does not see never reaches its output, NaN and infinities included.
// Domain:     q [T, heads, D] with contiguous heads (any token stride: a view of the qkv
//             projection); k_cache, v_cache [blocks, block_size, KV heads, D] contiguous, heads a
//             multiple of KV heads; block_tables [S, B], seq_lens [S], query_start_loc [S + 1]
//             int32 contiguous; tree_mask [T, W] int64 contiguous, W <= 16, bit b of word w standing
//             for node 64 w + b of the same request. scale: positive, by default D^-0.5. bf16, and
//             fp32 on CPU; on CUDA D is 64 or 128 and q's token stride a multiple of 8.
// Returns:    A new [T, heads, D] tensor.
// Throws:     c10::Error on dtype, shape, layout or device mismatches, and on CPU for lengths or
//             blocks out of range; on CUDA those raise the device error word (the request's rows
//             are zero, all rows where query_start_loc does not rise from 0 to at most T; a block
//             outside the cache reads block 0).
at::Tensor tree_attention(const at::Tensor& q, const at::Tensor& k_cache,
                          const at::Tensor& v_cache, const at::Tensor& block_tables,
                          const at::Tensor& seq_lens, const at::Tensor& query_start_loc,
                          const std::optional<at::Tensor>& tree_mask,
                          const std::optional<double>& scale);

}  // namespace svllm::ops
