#include "ops/tree_accept.h"

#include <ATen/ATen.h>
#include <c10/util/Exception.h>

#include <algorithm>
#include <functional>
#include <vector>

#include "ops/common.h"
#include "ops/tree_accept_kernels.h"
#include "svllm_kernels.h"

namespace svllm::ops {
namespace {

void check_list(const char* op, const char* name, const at::Tensor& t, at::ScalarType dtype,
                at::IntArrayRef shape, const at::Device& device) {
  TORCH_CHECK(t.scalar_type() == dtype && t.is_contiguous(), op, ": expected contiguous ", dtype,
              " ", name, ", got ", t.scalar_type());
  TORCH_CHECK(t.sizes() == shape, op, ": ", name, " has shape ", t.sizes(), ", expected ", shape);
  TORCH_CHECK(t.device() == device, op, ": the step is on ", device, " but ", name, " is on ",
              t.device());
}

}  // namespace

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> tree_accept(
    const at::Tensor& ids, const at::Tensor& targets, const std::optional<at::Tensor>& parents,
    const at::Tensor& query_start_loc, const at::Tensor& seq_lens, const at::Tensor& context_lens,
    int64_t max_query_len) {
  TORCH_CHECK(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong,
              "tree_accept: expected int32 or int64 ids, got ", ids.scalar_type());
  TORCH_CHECK(max_query_len >= 1 && max_query_len <= SVLLM_MAX_TREE_NODES,
              "tree_accept: max_query_len ", max_query_len, " must be in [1, ",
              SVLLM_MAX_TREE_NODES, "]");
  const at::Device device = ids.device();
  const int64_t tokens = ids.numel(), requests = seq_lens.numel();
  check_list("tree_accept", "ids", ids, ids.scalar_type(), {tokens}, device);
  check_list("tree_accept", "targets", targets, at::kLong, {tokens}, device);
  check_list("tree_accept", "query_start_loc", query_start_loc, at::kInt, {requests + 1}, device);
  check_list("tree_accept", "seq_lens", seq_lens, at::kInt, {requests}, device);
  check_list("tree_accept", "context_lens", context_lens, at::kInt, {requests}, device);
  TreeAcceptTensors a;
  if (parents.has_value() && parents->defined()) {
    check_list("tree_accept", "parents", *parents, at::kInt, {tokens}, device);
    a.parents = *parents;
  }
  a.ids = ids;
  a.targets = targets;
  a.query_start_loc = query_start_loc;
  a.seq_lens = seq_lens;
  a.context_lens = context_lens;
  a.max_query_len = max_query_len;
  using detail::Outputs;
  Outputs out(Outputs::size(at::kLong, requests * max_query_len) +
                  Outputs::size(at::kInt, requests * max_query_len) +
                  Outputs::size(at::kInt, requests) * 2,
              targets.options());
  a.tokens = out.take(at::kLong, {requests, max_query_len});
  a.path = out.take(at::kInt, {requests, max_query_len});
  a.num_accepted = out.take(at::kInt, {requests});
  a.context_lens_out = out.take(at::kInt, {requests});
  switch (device.type()) {
    case c10::DeviceType::CPU:
      cpu_impl::tree_accept(a);
      break;
    case c10::DeviceType::CUDA:
      cuda_impl::tree_accept(a);
      break;
    default:
      TORCH_CHECK(false, "tree_accept: unsupported device ", device);
  }
  return {a.path, a.tokens, a.num_accepted, a.context_lens_out};
}

void tree_commit(const std::vector<at::Tensor>& k_caches, const std::vector<at::Tensor>& v_caches,
                 const at::Tensor& path, const at::Tensor& num_accepted,
                 const at::Tensor& slot_mapping, const at::Tensor& query_start_loc,
                 const std::vector<at::Tensor>& k_scales,
                 const std::vector<at::Tensor>& v_scales) {
  TORCH_CHECK(!k_caches.empty() && k_caches.size() == v_caches.size(), "tree_commit: ",
              k_caches.size(), " K caches and ", v_caches.size(), " V caches");
  const at::Tensor& first = k_caches[0];
  TORCH_CHECK(first.scalar_type() != at::kFloat8_e8m0fnu,
              "tree_commit: float8_e8m0fnu caches are scales: pass them as k_scales and v_scales");
  TORCH_CHECK(first.dim() >= 3 && first.numel() > 0,
              "tree_commit: caches must be [..., num_kv_heads, head_dim], got shape ",
              first.sizes());
  for (const auto* caches : {&k_caches, &v_caches}) {
    for (const at::Tensor& c : *caches) {
      TORCH_CHECK(c.sizes() == first.sizes() && c.scalar_type() == first.scalar_type() &&
                      c.device() == first.device() && c.is_contiguous(),
                  "tree_commit: caches must be contiguous and of one shape, dtype and device; the "
                  "first K cache is ", first.scalar_type(), " ", first.sizes(), " on ",
                  first.device(), ", another ", c.scalar_type(), " ", c.sizes(), " on ",
                  c.device());
    }
  }
  const bool scaled = !k_scales.empty() || !v_scales.empty();
  const bool codes = first.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(scaled || !codes,
              "tree_commit: float8_e4m3fn caches move with their scales: pass k_scales and v_scales "
              "(a cache without them moves as bytes, uint8)");
  TORCH_CHECK(codes || !scaled, "tree_commit: scales are only of float8_e4m3fn caches, got ",
              first.scalar_type());
  std::vector<at::Tensor> ks, vs;  // as [..., KV heads, 1]
  if (scaled) {
    TORCH_CHECK(k_scales.size() == k_caches.size() && v_scales.size() == v_caches.size(),
                "tree_commit: ", k_scales.size(), " K scales and ", v_scales.size(),
                " V scales for ", k_caches.size(), " layers");
    const at::IntArrayRef rows = first.sizes().slice(0, first.dim() - 1);
    std::vector<const void*> planes;
    for (const auto* scales : {&k_scales, &v_scales}) {
      for (const at::Tensor& c : *scales) {
        TORCH_CHECK(c.sizes() == rows && c.scalar_type() == at::kFloat8_e8m0fnu &&
                        c.device() == first.device() && c.is_contiguous(),
                    "tree_commit: scales must be contiguous float8_e8m0fnu ", rows, " on ",
                    first.device(), ", got ", c.scalar_type(), " ", c.sizes(), " on ", c.device());
        (scales == &k_scales ? ks : vs).push_back(c.unsqueeze(-1));
        planes.push_back(c.const_data_ptr());
      }
    }
    // before any row moves
    std::sort(planes.begin(), planes.end(), std::less<const void*>());
    TORCH_CHECK(std::adjacent_find(planes.begin(), planes.end()) == planes.end(),
                "tree_commit: invalid argument: scales are given twice");
  }
  const at::Device device = first.device();
  const int64_t requests = num_accepted.numel(), tokens = slot_mapping.numel();
  TORCH_CHECK(path.dim() == 2 && path.size(1) >= 1 && path.size(1) <= SVLLM_MAX_TREE_NODES,
              "tree_commit: path must be [requests, 1 to ", SVLLM_MAX_TREE_NODES,
              "], got shape ", path.sizes());
  check_list("tree_commit", "path", path, at::kInt, {requests, path.size(1)}, device);
  check_list("tree_commit", "num_accepted", num_accepted, at::kInt, {requests}, device);
  check_list("tree_commit", "slot_mapping", slot_mapping, at::kLong, {tokens}, device);
  check_list("tree_commit", "query_start_loc", query_start_loc, at::kInt, {requests + 1}, device);
  const int64_t num_slots = first.numel() / (first.size(-1) * first.size(-2));
  switch (device.type()) {
    case c10::DeviceType::CPU:
      cpu_impl::tree_commit(k_caches, v_caches, num_slots, path, num_accepted, slot_mapping,
                            query_start_loc);
      if (scaled) {
        cpu_impl::tree_commit(ks, vs, num_slots, path, num_accepted, slot_mapping,
                              query_start_loc);
      }
      break;
    case c10::DeviceType::CUDA:
      cuda_impl::tree_commit(k_caches, v_caches, num_slots, path, num_accepted, slot_mapping,
                             query_start_loc);
      if (scaled) {
        cuda_impl::tree_commit(ks, vs, num_slots, path, num_accepted, slot_mapping,
                               query_start_loc);
      }
      break;
    default:
      TORCH_CHECK(false, "tree_commit: unsupported device ", device);
  }
}

}  // namespace svllm::ops
