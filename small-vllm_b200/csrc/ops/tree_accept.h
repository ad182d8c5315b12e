#pragma once

#include <ATen/core/Tensor.h>

#include <cstdint>
#include <optional>
#include <tuple>
#include <vector>

namespace svllm::ops {

// Definition: Greedy acceptance of trees of drafted tokens, after the step that fed them and the
//             argmax over its logits.
// Formula:    Per request, from node 0 (its last accepted token): the walk goes to the first child
//             of the current node whose id is the current node's target, until there is none.
// Domain:     ids [T] int32 or int64, the tokens the step was fed; targets [T] int64, the model's
//             next token after each (ops::argmax, ops::greedy_sample); parents [T] int32 as in
//             paged_plan, none = chains; query_start_loc [S + 1], seq_lens [S] (0: not served),
//             context_lens [S] int32; all contiguous. max_query_len: 1 to 1024, at least every
//             request's number of tokens.
// Returns:    path [S, max_query_len] int32, the nodes walked, -1 behind them; tokens [S,
//             max_query_len] int64, their targets: what the step emits, -1 behind them;
//             num_accepted [S] int32; context_lens + num_accepted [S] int32.
// Throws:     c10::Error on dtype, shape, layout or device mismatches, and on CPU for a
//             query_start_loc out of range; on CUDA that raises the device error word and the
//             request accepts nothing.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> tree_accept(
    const at::Tensor& ids, const at::Tensor& targets, const std::optional<at::Tensor>& parents,
    const at::Tensor& query_start_loc, const at::Tensor& seq_lens, const at::Tensor& context_lens,
    int64_t max_query_len);

// Definition: Moves the accepted nodes' K and V rows to the front of the step's rows, in every
//             layer's cache, so that the next step finds the accepted tokens as its context.
// Formula:    row slot_mapping[start + j] = row slot_mapping[start + path[s][j]] of every cache, 0 <
//             j < num_accepted[s], start = query_start_loc[s]. A negative slot does not move.
// Domain:     k_caches, v_caches: one contiguous [blocks, block_size, KV heads, D] (or [slots, KV
//             heads, D]) tensor per layer, all of one shape and dtype (on CUDA, rows of whole 16
//             bytes); path and num_accepted as tree_accept returns them; slot_mapping [T] int64 and
//             query_start_loc [S + 1] int32 of the step, no slot in it twice. No two caches share memory;
//             the same one twice is refused.
// Throws:     c10::Error on dtype, shape, layout or device mismatches, and on CPU for a path or slot
//             out of range; on CUDA those raise the device error word and the rows do not move.
void tree_commit(const std::vector<at::Tensor>& k_caches, const std::vector<at::Tensor>& v_caches,
                 const at::Tensor& path, const at::Tensor& num_accepted,
                 const at::Tensor& slot_mapping, const at::Tensor& query_start_loc);

}  // namespace svllm::ops
