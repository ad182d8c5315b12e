// Greedy acceptance of a tree of drafted tokens, and the move of the accepted nodes' K and V rows.
//
// tree_accept: node 0 of a request is its last accepted token, whose successors were drafted.
// From cur = 0: the model's token after cur is targets[cur]; the walk goes on at the first child
// of cur that holds it, and ends where no child does. The tokens emitted are targets along the
// path, so every request with a node emits at least one. What bounds it is the chain of steps down
// the tree. Measured in a graph: 4 requests of 8 nodes 3.3 us, 1024 of 32 to 64 4.8 (1.8 MB, 0.3 us
// of HBM time); a call costs its host some 6 us.
//
// tree_commit: the step wrote node i of a request to the slot of row context + i; row context +
// j of the sequence, j < accepted, must be node path[j]. Paths rise (a parent comes before its
// child), so path[j] >= j. A copy: 128 requests of 12 to 24 nodes in 28 layers, 143 MB, 23.8 us in
// calls on caches in turn (6.0 TB/s, 0.91 of the copy rate); 20.7 us over and over in a graph, less
// than HBM would take, part of it from L2; one request of 16 nodes 3.8 us in a graph.
#include <cuda_runtime.h>

#include <cstdint>

#include "common.cuh"
#include "host_common.h"

namespace svllm::k {
namespace {

constexpr int kAcceptThreads = 128;

struct AcceptArgs {
  const void* ids;                 // [num_tokens]
  const int64_t* targets;          // [num_tokens]
  const int32_t* parents;          // [num_tokens] or null: chains
  const int32_t* query_start_loc;  // [num_seqs + 1]
  const int32_t* seq_lens;         // [num_seqs]; 0: not served
  const int32_t* context_lens;     // [num_seqs]
  int32_t* path;                   // [num_seqs, max_query_len], -1 behind the last node
  int64_t* tokens;                 // [num_seqs, max_query_len], -1 behind the last token
  int32_t* num_accepted;           // [num_seqs]
  int32_t* context_out;            // [num_seqs]
  int64_t num_tokens;
  int max_query_len;
  int ids_64;
  int* err;
};

// One CTA per request: the nodes are staged in shared memory by all threads (the walk is a
// chain of dependent reads, 30 cycles each there against some 300 from L2), warp 0 walks.
__global__ void __launch_bounds__(kAcceptThreads) tree_accept_kernel(const AcceptArgs a) {
  grid_dependency_sync();
  extern __shared__ int64_t sh[];
  int64_t* sh_target = sh;
  int64_t* sh_id = sh_target + a.max_query_len;
  int32_t* sh_parent = reinterpret_cast<int32_t*>(sh_id + a.max_query_len);
  int32_t* sh_path = sh_parent + a.max_query_len;
  __shared__ int sh_count;

  const int64_t s = blockIdx.x;
  const int tid = threadIdx.x;
  const int64_t start = a.query_start_loc[s], end = a.query_start_loc[s + 1];
  int n = 0;
  if (start < 0 || end < start || end > a.num_tokens || end - start > a.max_query_len) {
    if (tid == 0) raise_error(a.err, kErrBadIndex);
  } else if (a.seq_lens[s] > 0) {
    n = static_cast<int>(end - start);
  }
  for (int i = tid; i < n; i += kAcceptThreads) {
    sh_target[i] = a.targets[start + i];
    sh_id[i] = a.ids_64 ? static_cast<const int64_t*>(a.ids)[start + i]
                        : static_cast<const int32_t*>(a.ids)[start + i];
    sh_parent[i] = a.parents != nullptr ? a.parents[start + i] : i - 1;
  }
  __syncthreads();
  if (tid < kWarpSize) {
    int count = 0;
    int cur = n > 0 ? 0 : -1;
    while (cur >= 0) {
      if (tid == 0) sh_path[count] = cur;
      ++count;
      const int64_t want = sh_target[cur];
      int next = -1;
      for (int base = cur + 1; base < n; base += kWarpSize) {  // children come after cur
        const int i = base + tid;
        const unsigned hit = __ballot_sync(
            0xffffffffu, i < n && sh_parent[i] == cur && sh_id[i] == want);
        if (hit != 0) {
          next = base + __ffs(static_cast<int>(hit)) - 1;
          break;
        }
      }
      cur = next;
    }
    if (tid == 0) {
      sh_count = count;
      a.num_accepted[s] = count;
      a.context_out[s] = a.context_lens[s] + count;
    }
  }
  __syncthreads();
  const int count = sh_count;
  for (int i = tid; i < a.max_query_len; i += kAcceptThreads) {
    const int node = i < count ? sh_path[i] : -1;
    a.path[s * a.max_query_len + i] = node;
    a.tokens[s * a.max_query_len + i] = node >= 0 ? sh_target[node] : -1;
  }
}

constexpr int kCommitThreads = 128;
constexpr int kCommitPlanes = 128;  // K and V planes of one launch, their pointers by value
constexpr int kCommitBatch = 8;     // rows a thread holds between its loads and its stores

struct CommitArgs {
  void* plane[kCommitPlanes];      // [num_slots, row_vecs units] each
  const int32_t* path;             // [num_seqs, max_query_len]
  const int32_t* num_accepted;     // [num_seqs]
  const int64_t* slot_mapping;     // [num_tokens]
  const int32_t* query_start_loc;  // [num_seqs + 1]
  int64_t num_slots;
  int64_t num_tokens;
  int64_t row_vecs;                // units per row: 16-byte vectors, or bytes of scales
  int max_query_len;
  int* err;
};

// One CTA: one request, one plane (K or V of a layer). A thread moves the same 16-byte column
// of every row in order, eight rows loaded before they are stored. That order is enough: row i
// is written after every source path[j], j <= i, has been read, and no later source is row i,
// since path[j] >= j > i. Unit: uint4, or uint8_t for the scales of an 8-bit cache, whose rows are
// a few bytes.
template <class Unit>
__global__ void __launch_bounds__(kCommitThreads) tree_commit_kernel(const CommitArgs a) {
  grid_dependency_sync();
  extern __shared__ int64_t sh[];
  int64_t* sh_src = sh;                       // slots, -1: the row does not move
  int64_t* sh_dst = sh_src + a.max_query_len;
  __shared__ int sh_limit;

  const int64_t s = blockIdx.x;
  const int tid = threadIdx.x;
  const int64_t start = a.query_start_loc[s], end = a.query_start_loc[s + 1];
  int count = a.num_accepted[s];
  if (count <= 1) {
    if (count < 0 && tid == 0) raise_error(a.err, kErrBadIndex);
    return;
  }
  if (start < 0 || end < start || end > a.num_tokens || count > end - start ||
      count > a.max_query_len) {
    if (tid == 0) raise_error(a.err, kErrBadIndex);
    return;
  }
  if (tid == 0) sh_limit = count;
  __syncthreads();
  const int32_t* path = a.path + s * a.max_query_len;
  for (int i = tid; i < count; i += kCommitThreads) {
    const int node = path[i];
    sh_src[i] = -1;
    if (node < i || node >= end - start || (i > 0 && path[i - 1] >= node)) {
      raise_error(a.err, kErrBadIndex);  // not a rising path: no row from here on moves
      atomicMin(&sh_limit, i);
    } else if (node != i) {
      const int64_t src = a.slot_mapping[start + node], dst = a.slot_mapping[start + i];
      if (src >= a.num_slots || dst >= a.num_slots) {
        raise_error(a.err, kErrBadIndex);
      } else if (src >= 0 && dst >= 0) {
        sh_src[i] = src;
        sh_dst[i] = dst;
      }
    }
  }
  __syncthreads();
  count = sh_limit;
  Unit* rows = static_cast<Unit*>(a.plane[blockIdx.y]);
  for (int64_t v = tid; v < a.row_vecs; v += kCommitThreads) {
    for (int base = 1; base < count; base += kCommitBatch) {
      Unit held[kCommitBatch];
#pragma unroll
      for (int e = 0; e < kCommitBatch; ++e) {
        if (base + e < count && sh_src[base + e] >= 0) {
          held[e] = rows[sh_src[base + e] * a.row_vecs + v];
        }
      }
#pragma unroll
      for (int e = 0; e < kCommitBatch; ++e) {
        if (base + e < count && sh_src[base + e] >= 0) {
          rows[sh_dst[base + e] * a.row_vecs + v] = held[e];
        }
      }
    }
  }
}

// Whether two of the planes K and V are the same: a small hash table of those seen, past its room
// each against all before it (a model has a few dozen layers; up to 256 take the table).
bool any_plane_twice(void* const* k, void* const* v, int64_t layers) {
  constexpr int kSlots = 1024;
  const auto plane = [&](int64_t i) { return i < layers ? k[i] : v[i - layers]; };
  const void* seen[kSlots];
  if (4 * layers > kSlots) {
    for (int64_t i = 0; i < 2 * layers; ++i) {
      for (int64_t j = 0; j < i; ++j) {
        if (plane(i) == plane(j)) return true;
      }
    }
    return false;
  }
  int slots = 32;
  while (slots < 4 * layers) slots *= 2;
  for (int i = 0; i < slots; ++i) seen[i] = nullptr;
  for (int64_t i = 0; i < 2 * layers; ++i) {
    const void* p = plane(i);
    // the upper half of a product with an odd constant mixes the page bits down
    int at = static_cast<int>((reinterpret_cast<uint64_t>(p) * 0x9e3779b97f4a7c15u) >> 40) &
             (slots - 1);
    for (; seen[at] != nullptr; at = (at + 1) & (slots - 1)) {
      if (seen[at] == p) return true;
    }
    seen[at] = p;
  }
  return false;
}

}  // namespace
}  // namespace svllm::k

extern "C" int svllm_tree_accept(const void* ids, int id_type, const int64_t* targets,
                                 const int32_t* parents, const int32_t* query_start_loc,
                                 const int32_t* seq_lens, const int32_t* context_lens,
                                 int64_t num_seqs, int64_t num_tokens, int64_t max_query_len,
                                 int32_t* path, int64_t* tokens, int32_t* num_accepted,
                                 int32_t* context_lens_out, svllm_stream stream) {
  using namespace svllm::k;
  if (num_seqs < 0 || num_tokens < 0 || max_query_len <= 0 ||
      (id_type != SVLLM_INDEX_I32 && id_type != SVLLM_INDEX_I64)) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  if (num_seqs == 0) return SVLLM_OK;
  if (query_start_loc == nullptr || seq_lens == nullptr || context_lens == nullptr ||
      path == nullptr || tokens == nullptr || num_accepted == nullptr ||
      context_lens_out == nullptr || (num_tokens > 0 && (ids == nullptr || targets == nullptr))) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  if (max_query_len > SVLLM_MAX_TREE_NODES || num_seqs >= (int64_t{1} << 31) ||
      num_tokens >= (int64_t{1} << 31)) {
    return SVLLM_ERR_TOO_LARGE;
  }
  int device;
  if (current_device(&device) != SVLLM_OK) return SVLLM_ERR_CUDA;
  int* err = library_error_word(device);
  if (err == nullptr) return SVLLM_ERR_CUDA;
  AcceptArgs a{};
  a.ids = ids;
  a.targets = targets;
  a.parents = parents;
  a.query_start_loc = query_start_loc;
  a.seq_lens = seq_lens;
  a.context_lens = context_lens;
  a.path = path;
  a.tokens = tokens;
  a.num_accepted = num_accepted;
  a.context_out = context_lens_out;
  a.num_tokens = num_tokens;
  a.max_query_len = static_cast<int>(max_query_len);
  a.ids_64 = id_type == SVLLM_INDEX_I64;
  a.err = err;
  return launch(tree_accept_kernel, dim3(static_cast<unsigned>(num_seqs)), dim3(kAcceptThreads),
                static_cast<size_t>(max_query_len) * 24, reinterpret_cast<cudaStream_t>(stream),
                1u, a);
}

namespace svllm::k {
namespace {

template <class Unit>
int launch_commit(void* const* k_caches, void* const* v_caches, int64_t num_layers,
                  int64_t num_slots, int64_t row_bytes, const int32_t* path,
                  const int32_t* num_accepted, const int64_t* slot_mapping,
                  const int32_t* query_start_loc, int64_t num_seqs, int64_t num_tokens,
                  int64_t max_query_len, svllm_stream stream) {
  if (num_seqs < 0 || num_tokens < 0 || num_layers < 0 || num_slots < 0 || row_bytes <= 0 ||
      max_query_len <= 0) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  if (num_seqs == 0 || num_layers == 0) return SVLLM_OK;
  if (k_caches == nullptr || v_caches == nullptr || path == nullptr || num_accepted == nullptr ||
      query_start_loc == nullptr || (num_tokens > 0 && slot_mapping == nullptr)) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  for (int64_t l = 0; l < num_layers; ++l) {
    if (k_caches[l] == nullptr || v_caches[l] == nullptr) return SVLLM_ERR_INVALID_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(k_caches[l]) % sizeof(Unit) != 0 ||
        reinterpret_cast<uintptr_t>(v_caches[l]) % sizeof(Unit) != 0) {
      return SVLLM_ERR_UNSUPPORTED;
    }
  }
  if (row_bytes % static_cast<int64_t>(sizeof(Unit)) != 0) return SVLLM_ERR_UNSUPPORTED;
  if (max_query_len > SVLLM_MAX_TREE_NODES || num_seqs >= (int64_t{1} << 31) ||
      num_tokens >= (int64_t{1} << 31)) {
    return SVLLM_ERR_TOO_LARGE;
  }
  if (any_plane_twice(k_caches, v_caches, num_layers)) return SVLLM_ERR_INVALID_ARGUMENT;
  int device;
  if (current_device(&device) != SVLLM_OK) return SVLLM_ERR_CUDA;
  int* err = library_error_word(device);
  if (err == nullptr) return SVLLM_ERR_CUDA;
  CommitArgs a{};
  a.path = path;
  a.num_accepted = num_accepted;
  a.slot_mapping = slot_mapping;
  a.query_start_loc = query_start_loc;
  a.num_slots = num_slots;
  a.num_tokens = num_tokens;
  a.row_vecs = row_bytes / static_cast<int64_t>(sizeof(Unit));
  a.max_query_len = static_cast<int>(max_query_len);
  a.err = err;
  for (int64_t l = 0; l < num_layers; l += kCommitPlanes / 2) {
    unsigned planes = 0;
    for (int64_t m = l; m < num_layers && m < l + kCommitPlanes / 2; ++m) {
      a.plane[planes++] = k_caches[m];
      a.plane[planes++] = v_caches[m];
    }
    const dim3 grid(static_cast<unsigned>(num_seqs), planes);
    const int status = launch(tree_commit_kernel<Unit>, grid, dim3(kCommitThreads),
                              static_cast<size_t>(max_query_len) * 16,
                              reinterpret_cast<cudaStream_t>(stream), 1u, a);
    if (status != SVLLM_OK) return status;
  }
  return SVLLM_OK;
}

}  // namespace
}  // namespace svllm::k

extern "C" int svllm_tree_commit(void* const* k_caches, void* const* v_caches, int64_t num_layers,
                                 int64_t num_slots, int64_t row_bytes, const int32_t* path,
                                 const int32_t* num_accepted, const int64_t* slot_mapping,
                                 const int32_t* query_start_loc, int64_t num_seqs,
                                 int64_t num_tokens, int64_t max_query_len, svllm_stream stream) {
  return svllm::k::launch_commit<uint4>(k_caches, v_caches, num_layers, num_slots, row_bytes, path,
                                        num_accepted, slot_mapping, query_start_loc, num_seqs,
                                        num_tokens, max_query_len, stream);
}

extern "C" int svllm_tree_commit_scales(void* const* k_scales, void* const* v_scales,
                                        int64_t num_layers, int64_t num_slots,
                                        int64_t num_kv_heads, const int32_t* path,
                                        const int32_t* num_accepted, const int64_t* slot_mapping,
                                        const int32_t* query_start_loc, int64_t num_seqs,
                                        int64_t num_tokens, int64_t max_query_len,
                                        svllm_stream stream) {
  return svllm::k::launch_commit<uint8_t>(k_scales, v_scales, num_layers, num_slots, num_kv_heads,
                                          path, num_accepted, slot_mapping, query_start_loc,
                                          num_seqs, num_tokens, max_query_len, stream);
}
