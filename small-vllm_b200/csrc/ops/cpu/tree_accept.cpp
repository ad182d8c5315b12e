// CPU kernels of ops::tree_accept and ops::tree_commit.
#include <ATen/Parallel.h>
#include <c10/util/Exception.h>

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <functional>
#include <utility>
#include <vector>

#include "ops/tree_accept_kernels.h"

namespace svllm::ops::cpu_impl {
namespace {

void check_starts(const char* op, const int32_t* start, int64_t requests, int64_t tokens) {
  TORCH_CHECK(start[0] >= 0, op, ": query_start_loc starts at ", start[0]);
  for (int64_t s = 0; s < requests; ++s) {
    TORCH_CHECK(start[s + 1] >= start[s] && start[s + 1] <= tokens, op,
                ": query_start_loc falls or ends past ", tokens, " tokens at request ", s);
  }
}

}  // namespace

void tree_accept(const TreeAcceptTensors& a) {
  const auto* start = a.query_start_loc.const_data_ptr<int32_t>();
  const auto* seq = a.seq_lens.const_data_ptr<int32_t>();
  const auto* context = a.context_lens.const_data_ptr<int32_t>();
  const auto* targets = a.targets.const_data_ptr<int64_t>();
  const auto* parents = a.parents.defined() ? a.parents.const_data_ptr<int32_t>() : nullptr;
  const auto* ids32 = a.ids.scalar_type() == at::kInt ? a.ids.const_data_ptr<int32_t>() : nullptr;
  const auto* ids64 = ids32 == nullptr ? a.ids.const_data_ptr<int64_t>() : nullptr;
  const int64_t requests = a.seq_lens.numel(), width = a.max_query_len;
  check_starts("tree_accept", start, requests, a.ids.numel());
  auto* path = a.path.mutable_data_ptr<int32_t>();
  auto* tokens = a.tokens.mutable_data_ptr<int64_t>();
  auto* accepted = a.num_accepted.mutable_data_ptr<int32_t>();
  auto* context_out = a.context_lens_out.mutable_data_ptr<int32_t>();
  std::fill(path, path + requests * width, -1);
  std::fill(tokens, tokens + requests * width, -1);
  for (int64_t s = 0; s < requests; ++s) {
    const int64_t n = seq[s] > 0 ? start[s + 1] - start[s] : 0;
    TORCH_CHECK(n <= width, "tree_accept: request ", s, " has ", n, " nodes, max_query_len is ",
                width);
    int32_t count = 0;
    for (int64_t cur = n > 0 ? 0 : -1; cur >= 0;) {
      const int64_t want = targets[start[s] + cur];
      path[s * width + count] = static_cast<int32_t>(cur);
      tokens[s * width + count] = want;
      ++count;
      int64_t next = -1;
      for (int64_t i = cur + 1; i < n && next < 0; ++i) {
        const int64_t t = start[s] + i;
        const int64_t up = parents != nullptr ? parents[t] : i - 1;
        if (up == cur && (ids32 != nullptr ? ids32[t] : ids64[t]) == want) next = i;
      }
      cur = next;
    }
    accepted[s] = count;
    context_out[s] = context[s] + count;
  }
}

void tree_commit(const std::vector<at::Tensor>& k_caches, const std::vector<at::Tensor>& v_caches,
                 int64_t num_slots, const at::Tensor& path, const at::Tensor& num_accepted,
                 const at::Tensor& slot_mapping, const at::Tensor& query_start_loc) {
  const auto* nodes = path.const_data_ptr<int32_t>();
  const auto* accepted = num_accepted.const_data_ptr<int32_t>();
  const auto* slots = slot_mapping.const_data_ptr<int64_t>();
  const auto* start = query_start_loc.const_data_ptr<int32_t>();
  const int64_t requests = num_accepted.numel(), width = path.size(1);
  check_starts("tree_commit", start, requests, slot_mapping.numel());
  std::vector<const void*> planes;
  for (const auto* caches : {&k_caches, &v_caches}) {
    for (const at::Tensor& c : *caches) planes.push_back(c.const_data_ptr());
  }
  std::sort(planes.begin(), planes.end(), std::less<const void*>());
  TORCH_CHECK(std::adjacent_find(planes.begin(), planes.end()) == planes.end(),
              "tree_commit: invalid argument: a cache is given twice");
  std::vector<std::pair<int64_t, int64_t>> moves;  // source and destination, in order
  for (int64_t s = 0; s < requests; ++s) {
    const int64_t n = start[s + 1] - start[s];
    TORCH_CHECK(accepted[s] >= 0 && accepted[s] <= n && accepted[s] <= width,
                "tree_commit: request ", s, " accepts ", accepted[s], " of ", n, " tokens");
    for (int64_t i = 0; i < accepted[s]; ++i) {
      const int64_t node = nodes[s * width + i];
      TORCH_CHECK(node >= i && node < n && (i == 0 || node > nodes[s * width + i - 1]),
                  "tree_commit: the path of request ", s, " does not rise or leaves its ", n,
                  " nodes at step ", i);
      if (i == 0 || node == i) continue;
      const int64_t src = slots[start[s] + node], dst = slots[start[s] + i];
      TORCH_CHECK(src < num_slots && dst < num_slots, "tree_commit: a slot of request ", s,
                  " lies past the cache's ", num_slots);
      if (src >= 0 && dst >= 0) moves.emplace_back(src, dst);
    }
  }
  const int64_t row = k_caches[0].size(-1) * k_caches[0].size(-2) * k_caches[0].element_size();
  const int64_t layers = static_cast<int64_t>(k_caches.size());
  at::parallel_for(0, 2 * layers, 1, [&](int64_t begin, int64_t end) {
    for (int64_t p = begin; p < end; ++p) {
      const at::Tensor& cache = p < layers ? k_caches[p] : v_caches[p - layers];
      auto* base = static_cast<char*>(cache.mutable_data_ptr());
      for (const auto& [src, dst] : moves) std::memcpy(base + dst * row, base + src * row, row);
    }
  });
}

}  // namespace svllm::ops::cpu_impl
