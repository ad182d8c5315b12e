// CPU kernel of ops::tree_attention: one (token, head) at a time on torch's thread pool, softmax
// and sums in fp32, rounded once.
#include <ATen/Parallel.h>
#include <c10/util/BFloat16.h>
#include <c10/util/Exception.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <limits>
#include <vector>

#include "ops/tree_attention_kernels.h"

namespace svllm::ops::cpu_impl {
namespace {

template <class T>
void attend(const at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache,
            const at::Tensor& v_cache, const at::Tensor& block_tables, const at::Tensor& seq_lens,
            const at::Tensor& query_start_loc, const at::Tensor& tree_mask, float scale) {
  const int64_t tokens = q.size(0), heads = q.size(1), dim = q.size(2);
  const int64_t blocks = k_cache.size(0), bs = k_cache.size(1), kv_heads = k_cache.size(2);
  const int64_t requests = seq_lens.numel(), width = block_tables.size(1);
  const int64_t words = tree_mask.defined() ? tree_mask.size(1) : 0;
  const auto* tables = block_tables.const_data_ptr<int32_t>();
  const auto* seq = seq_lens.const_data_ptr<int32_t>();
  const auto* start = query_start_loc.const_data_ptr<int32_t>();
  const auto* mask = words > 0 ? tree_mask.const_data_ptr<int64_t>() : nullptr;
  TORCH_CHECK(start[0] == 0, "tree_attention: query_start_loc starts at ", start[0]);
  for (int64_t s = 0; s < requests; ++s) {
    const int64_t n = int64_t{start[s + 1]} - start[s];
    TORCH_CHECK(n >= 0 && start[s + 1] <= tokens, "tree_attention: query_start_loc falls or ends "
                "past ", tokens, " tokens at request ", s);
    TORCH_CHECK(seq[s] == 0 || (seq[s] >= n && seq[s] <= width * bs &&
                                (mask == nullptr || n <= 64 * words)),
                "tree_attention: request ", s, " of length ", seq[s], " with ", n,
                " tokens does not fit a table of ", width, " blocks of ", bs, " or the mask");
    for (int64_t j = 0; j * bs < seq[s]; ++j) {
      const int64_t block = tables[s * width + j];
      TORCH_CHECK(block >= 0 && block < blocks, "tree_attention: block ", block, " of request ",
                  s, " outside the cache of ", blocks);
    }
  }
  const T* qp = q.const_data_ptr<T>();
  const T* kp = k_cache.const_data_ptr<T>();
  const T* vp = v_cache.const_data_ptr<T>();
  T* op = out.mutable_data_ptr<T>();
  const int64_t q_stride = q.stride(0);
  at::parallel_for(0, tokens * heads, 1, [&](int64_t begin, int64_t end) {
    std::vector<float> p, sum(dim);
    std::vector<const T*> value;
    for (int64_t u = begin; u < end; ++u) {
      const int64_t t = u / heads, h = u % heads, kh = h / (heads / kv_heads);
      const int64_t s = std::upper_bound(start + 1, start + requests + 1, t) - (start + 1);
      p.clear();
      value.clear();
      std::fill(sum.begin(), sum.end(), 0.0f);
      const int64_t length = s < requests ? seq[s] : 0;
      const int64_t node = s < requests ? t - start[s] : 0;
      const int64_t context = s < requests ? length - (start[s + 1] - start[s]) : 0;
      const T* query = qp + t * q_stride + h * dim;
      float top = -std::numeric_limits<float>::infinity();
      for (int64_t j = 0; j < length; ++j) {
        const int64_t x = j - context;
        if (x >= 0 && (mask == nullptr
                           ? x > node
                           : !((static_cast<uint64_t>(mask[t * words + x / 64]) >> (x % 64)) & 1))) {
          continue;
        }
        const int64_t row = ((tables[s * width + j / bs] * bs + j % bs) * kv_heads + kh) * dim;
        float dot = 0.0f;
        for (int64_t d = 0; d < dim; ++d) {
          dot += static_cast<float>(query[d]) * static_cast<float>(kp[row + d]);
        }
        p.push_back(dot * scale);
        value.push_back(vp + row);
        top = std::max(top, p.back());
      }
      if (std::isinf(top) && top < 0) top = 0.0f;  // every score -inf, or no row at all
      float total = 0.0f;
      for (size_t j = 0; j < p.size(); ++j) {
        const float w = std::exp(p[j] - top);
        total += w;
        for (int64_t d = 0; d < dim; ++d) sum[d] += w * static_cast<float>(value[j][d]);
      }
      for (int64_t d = 0; d < dim; ++d) {
        op[u * dim + d] = static_cast<T>(total == 0.0f ? 0.0f : sum[d] / total);
      }
    }
  });
}

}  // namespace

void tree_attention(const at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache,
                    const at::Tensor& v_cache, const at::Tensor& block_tables,
                    const at::Tensor& seq_lens, const at::Tensor& query_start_loc,
                    const at::Tensor& tree_mask, double scale) {
  if (q.scalar_type() == at::kBFloat16) {
    attend<at::BFloat16>(out, q, k_cache, v_cache, block_tables, seq_lens, query_start_loc,
                         tree_mask, static_cast<float>(scale));
  } else {
    attend<float>(out, q, k_cache, v_cache, block_tables, seq_lens, query_start_loc, tree_mask,
                  static_cast<float>(scale));
  }
}

}  // namespace svllm::ops::cpu_impl
