// CPU kernel of ops::paged_plan: the requests in order, as the CUDA kernel serves them.
#include <ATen/Parallel.h>
#include <c10/util/Exception.h>

#include <algorithm>
#include <cstdint>
#include <vector>

#include "ops/paged_plan_kernels.h"

namespace svllm::ops::cpu_impl {

void paged_plan(const PagedPlanTensors& p) {
  const auto* context = p.context_lens.const_data_ptr<int32_t>();
  const auto* query = p.query_lens.const_data_ptr<int32_t>();
  auto* tables = p.block_tables.mutable_data_ptr<int32_t>();
  const auto* owned = p.blocks_owned.const_data_ptr<int32_t>();
  auto* stack = p.free_blocks.mutable_data_ptr<int32_t>();
  auto* start = p.query_start_loc.mutable_data_ptr<int32_t>();
  auto* seq = p.seq_lens.mutable_data_ptr<int32_t>();
  auto* owned_out = p.blocks_owned_out.mutable_data_ptr<int32_t>();
  const int64_t requests = p.context_lens.numel(), width = p.block_tables.size(1);
  const int64_t bs = p.block_size, capacity = p.free_blocks.numel();
  const bool tree = p.parents.defined();
  int64_t have = p.free_count.const_data_ptr<int32_t>()[0];
  TORCH_CHECK(have >= 0 && have <= capacity, "paged_plan: free_count ", have,
              " outside [0, ", capacity, "]");

  // everything is checked before anything is written
  int64_t tokens = 0, back = 0;
  for (int64_t s = 0; s < requests; ++s) {
    TORCH_CHECK(owned[s] >= 0 && owned[s] <= width, "paged_plan: request ", s, " owns ", owned[s],
                " blocks, its table holds ", width);
    if (query[s] < 0) {
      back += owned[s];
      continue;
    }
    tokens += query[s];
    TORCH_CHECK(context[s] >= 0 && int64_t{context[s]} + query[s] <= width * bs,
                "paged_plan: request ", s, " of ", context[s], " + ", query[s],
                " tokens does not fit a table of ", width, " blocks of ", bs);
    TORCH_CHECK(!tree || query[s] <= p.max_query_len, "paged_plan: request ", s, " has ",
                query[s], " nodes, max_query_len is ", p.max_query_len);
  }
  TORCH_CHECK(tokens <= p.num_tokens, "paged_plan: ", tokens, " tokens, num_tokens is ",
              p.num_tokens);
  TORCH_CHECK(have + back <= capacity, "paged_plan: ", back, " blocks come back to ", have,
              " free ones, free_blocks holds ", capacity);
  const auto* parents = tree ? p.parents.const_data_ptr<int32_t>() : nullptr;
  for (int64_t s = 0, t = 0; tree && s < requests; ++s) {
    for (int32_t i = 0; i < query[s]; ++i, ++t) {
      TORCH_CHECK(parents[t] >= -1 && parents[t] < i, "paged_plan: parent ", parents[t],
                  " of node ", i, " of request ", s, " does not come before it");
    }
  }

  for (int64_t s = 0; s < requests; ++s) {
    for (int32_t i = 0; query[s] < 0 && i < owned[s]; ++i) stack[have++] = tables[s * width + i];
  }
  const int64_t top = have;  // blocks are taken from here down
  int64_t needed = 0;
  start[0] = 0;
  for (int64_t s = 0; s < requests; ++s) {
    const int64_t n = std::max(query[s], 0);
    start[s + 1] = static_cast<int32_t>(start[s] + n);
    if (query[s] < 0) {
      seq[s] = 0;
      owned_out[s] = 0;
      continue;
    }
    const int64_t rows = context[s] + n;
    const int64_t need = n == 0 ? 0 : std::max<int64_t>(0, (rows + bs - 1) / bs - owned[s]);
    const bool served = need == 0 || needed + need <= top;
    if (served) {
      for (int64_t i = 0; i < need; ++i) {
        tables[s * width + owned[s] + i] = stack[top - 1 - needed - i];
      }
      have -= need;
    }
    needed += need;
    seq[s] = served ? static_cast<int32_t>(rows) : 0;
    owned_out[s] = static_cast<int32_t>(owned[s] + (served ? need : 0));
  }
  p.free_count_out.mutable_data_ptr<int32_t>()[0] = static_cast<int32_t>(have);

  auto* slots = p.slot_mapping.mutable_data_ptr<int64_t>();
  auto* positions = p.positions.mutable_data_ptr<int64_t>();
  auto* mask = tree ? p.tree_mask.mutable_data_ptr<int64_t>() : nullptr;
  const int64_t words = tree ? p.tree_mask.size(1) : 0;
  std::fill(slots, slots + p.num_tokens, -1);
  std::fill(positions, positions + p.num_tokens, 0);
  std::fill(mask, mask + p.num_tokens * words, 0);
  for (int64_t s = 0; s < requests; ++s) {
    if (seq[s] == 0) continue;
    std::vector<int64_t> depth(start[s + 1] - start[s]);
    for (int64_t i = 0; i < static_cast<int64_t>(depth.size()); ++i) {
      const int64_t t = start[s] + i, row = context[s] + i;
      slots[t] = tables[s * width + row / bs] * bs + row % bs;
      depth[i] = i;
      if (tree) {
        const int64_t up = parents[t];
        depth[i] = up < 0 ? 0 : depth[up] + 1;
        if (up >= 0) {
          std::copy(mask + (start[s] + up) * words, mask + (start[s] + up + 1) * words,
                    mask + t * words);
        }
        auto& word = reinterpret_cast<uint64_t&>(mask[t * words + i / 64]);
        word |= uint64_t{1} << (i % 64);
      }
      positions[t] = context[s] + depth[i];
    }
  }
}

}  // namespace svllm::ops::cpu_impl
