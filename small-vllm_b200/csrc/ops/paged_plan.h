#pragma once

#include <ATen/core/Tensor.h>

#include <cstdint>
#include <optional>
#include <tuple>

namespace svllm::ops {

// query_start_loc [S + 1] int32, seq_lens [S] int32, slot_mapping [T] int64, positions [T] int64,
// tree_mask [T, W] int64 (none without parents), blocks_owned [S] int32, free_count [1] int32.
using PagedPlan = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor,
                             std::optional<at::Tensor>, at::Tensor, at::Tensor>;

// Definition: The paging of one step, built where the request lengths are: which new KV blocks
//             each request takes from the free list, its block table, and per token its cache slot,
//             its position and, for trees of drafted tokens, the ancestor mask. The outputs are
//             what the rotary + cache-write ops, tree_attention and Model take (the reference's
//             AGENTS.md "Names": slot_mapping, block_tables, seq_lens, query_start_loc).
// Formula:    need = max(0, ceil((context + query) / block_size) - owned); requests are served in
//             order while the free list lasts; block k of the step is free_blocks[free_count - 1 -
//             k]. slot = block * block_size + offset of row context + i, position = context + the
//             node's depth, bit b of word w of a node's mask set where node 64 w + b is the node
//             or its ancestor. A negative query length marks a finished request: its blocks go
//             back on the free list before any is taken. A request the list cannot serve gets
//             seq_lens 0 and slots -1 and keeps what it had; so do tokens behind the last request.
// Domain:     context_lens, query_lens, blocks_owned [S], free_blocks [F], free_count [1], parents
//             [T] int32 contiguous; block_tables [S, B] int32 contiguous, B > 0. num_tokens >= the
//             sum of the query lengths. parents: per node its parent's index within the request,
//             lower than its own, -1 for a root; none = chains (no mask). max_query_len (only used
//             with parents): 1 to 1024, at least every query length; W = ceil(max_query_len / 64).
// Writes:     new entries of block_tables and free_blocks, in place; calling again with the same
//             inputs writes the same.
// Throws:     c10::Error on dtype, shape, layout or device mismatches, and on CPU for lengths out of
//             range; on CUDA those raise the device error word and the request is not served.
PagedPlan paged_plan(const at::Tensor& context_lens, const at::Tensor& query_lens,
                     const at::Tensor& block_tables, const at::Tensor& blocks_owned,
                     const at::Tensor& free_blocks, const at::Tensor& free_count,
                     int64_t num_tokens, int64_t block_size,
                     const std::optional<at::Tensor>& parents, int64_t max_query_len);

}  // namespace svllm::ops
