// CUDA side of ops::tree_accept and ops::tree_commit: thin LibTorch -> C ABI shims.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "ops/common.h"
#include "ops/tree_accept_kernels.h"

namespace svllm::ops::cuda_impl {

void tree_accept(const TreeAcceptTensors& a) {
  const c10::cuda::CUDAGuard device_guard(a.ids.device());
  const auto stream = reinterpret_cast<svllm_stream>(c10::cuda::getCurrentCUDAStream().stream());
  detail::check_status(
      "tree_accept",
      svllm_tree_accept(
          a.ids.const_data_ptr(),
          a.ids.scalar_type() == at::kLong ? SVLLM_INDEX_I64 : SVLLM_INDEX_I32,
          a.targets.const_data_ptr<int64_t>(),
          a.parents.defined() ? a.parents.const_data_ptr<int32_t>() : nullptr,
          a.query_start_loc.const_data_ptr<int32_t>(), a.seq_lens.const_data_ptr<int32_t>(),
          a.context_lens.const_data_ptr<int32_t>(), a.seq_lens.numel(), a.ids.numel(),
          a.max_query_len, a.path.mutable_data_ptr<int32_t>(),
          a.tokens.mutable_data_ptr<int64_t>(), a.num_accepted.mutable_data_ptr<int32_t>(),
          a.context_lens_out.mutable_data_ptr<int32_t>(), stream));
}

void tree_commit(const std::vector<at::Tensor>& k_caches, const std::vector<at::Tensor>& v_caches,
                 int64_t num_slots, const at::Tensor& path, const at::Tensor& num_accepted,
                 const at::Tensor& slot_mapping, const at::Tensor& query_start_loc) {
  const at::Tensor& first = k_caches[0];
  const c10::cuda::CUDAGuard device_guard(first.device());
  const auto stream = reinterpret_cast<svllm_stream>(c10::cuda::getCurrentCUDAStream().stream());
  std::vector<void*> k, v;
  k.reserve(k_caches.size());
  v.reserve(v_caches.size());
  for (const at::Tensor& c : k_caches) k.push_back(c.mutable_data_ptr());
  for (const at::Tensor& c : v_caches) v.push_back(c.mutable_data_ptr());
  detail::check_status(
      "tree_commit",
      svllm_tree_commit(k.data(), v.data(), static_cast<int64_t>(k.size()), num_slots,
                        first.size(-1) * first.size(-2) * first.element_size(),
                        path.const_data_ptr<int32_t>(), num_accepted.const_data_ptr<int32_t>(),
                        slot_mapping.const_data_ptr<int64_t>(),
                        query_start_loc.const_data_ptr<int32_t>(), num_accepted.numel(),
                        slot_mapping.numel(), path.size(1), stream));
}

}  // namespace svllm::ops::cuda_impl
