// The paging plan of one step, from request lengths alone: which new KV blocks each request
// takes from the free list (and which a finished one gives back), its block table, and per token
// the cache slot, the position and, for trees of drafted tokens, the ancestor mask.
//
// With context c, query length n and o blocks owned, request s needs max(0, ceil((c + n) / bs) -
// o) blocks. Requests are served in order while the free list lasts: with P the inclusive prefix
// sum of the needs, s is served when P_s is at most the list's length (or its need is 0). Block
// k of the step, counted over all requests, is free_blocks[count - 1 - k].
//
// One CTA does the requests: its scans are a few shuffles for 1024 requests, and no grid-wide
// meeting is needed between giving blocks back and taking them. What bounds it is the chain of
// dependent loads, not bytes. Tokens are independent of one another (a binary search over the
// starts, one table entry, a walk up the parents); few of them follow in the same CTA, many get
// a second kernel over the whole GPU (kFusedTokens).
#include <cuda_runtime.h>

#include <cstdint>

#include "common.cuh"
#include "host_common.h"

namespace svllm::k {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / kWarpSize;
constexpr int kTokenThreads = 256;

// Up to this many tokens are done by the CTA that did the requests; more get a grid of their own.
constexpr int64_t kFusedTokens = 4096;

struct PlanArgs {
  const int32_t* context_lens;   // [num_seqs]
  const int32_t* query_lens;     // [num_seqs]; negative: finished, its blocks come back
  int32_t* block_tables;         // [num_seqs, max_blocks]
  const int32_t* blocks_owned;   // [num_seqs]
  int32_t* free_blocks;          // [free_capacity]
  const int32_t* free_count;     // [1]
  const int32_t* parents;        // [num_tokens] or null: chains
  int32_t* query_start_loc;      // [num_seqs + 1]
  int32_t* seq_lens;             // [num_seqs]; 0 where the request was not served
  int64_t* slot_mapping;         // [num_tokens]
  int64_t* positions;            // [num_tokens]
  int64_t* tree_mask;            // [num_tokens, mask_words]; null without parents
  int32_t* blocks_owned_out;     // [num_seqs]
  int32_t* free_count_out;       // [1]
  int64_t num_seqs;
  int64_t num_tokens;
  int64_t free_capacity;
  int32_t max_blocks;
  int32_t block_size;
  int32_t max_query_len;         // checked where parents are given: the mask's width
  int32_t mask_words;
  int fused;                     // this CTA does the tokens too
  int* err;
};

// Inclusive sum over the CTA's threads; `total` receives the CTA's sum. 64 bits: lengths come
// from the caller unchecked, and their sum must not wrap.
__device__ int64_t block_scan(int64_t v, int64_t* warp_sums, int64_t& total) {
  const int lane = threadIdx.x % kWarpSize, warp = threadIdx.x / kWarpSize;
#pragma unroll
  for (int off = 1; off < kWarpSize; off *= 2) {
    const int64_t up = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += up;
  }
  __syncthreads();  // the previous scan's readers are done
  if (lane == kWarpSize - 1) warp_sums[warp] = v;
  __syncthreads();
  int64_t s = warp_sums[lane];  // kPlanWarps == kWarpSize: every warp sums the sums itself
#pragma unroll
  for (int off = 1; off < kWarpSize; off *= 2) {
    const int64_t up = __shfl_up_sync(0xffffffffu, s, off);
    if (lane >= off) s += up;
  }
  total = __shfl_sync(0xffffffffu, s, kWarpSize - 1);
  const int64_t before = __shfl_sync(0xffffffffu, s, warp > 0 ? warp - 1 : 0);
  return v + (warp > 0 ? before : 0);
}
static_assert(kPlanWarps == kWarpSize, "block_scan sums one value per warp in one warp");

// One token: its request by binary search over the starts, then slot, position and mask. Reads
// what the requests' part wrote, so plain loads (not the read-only path).
__device__ void plan_token(const PlanArgs& a, int64_t t) {
  int64_t lo = 0, hi = a.num_seqs;  // the first request whose end lies beyond t
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (a.query_start_loc[mid + 1] > t) {
      hi = mid;
    } else {
      lo = mid + 1;
    }
  }
  const bool live = lo < a.num_seqs && a.seq_lens[lo] > 0;
  int64_t slot = -1, position = 0;
  int64_t* mask = a.tree_mask == nullptr ? nullptr : a.tree_mask + t * a.mask_words;
  int word = a.mask_words;  // mask words from here on are written
  if (live) {
    const int32_t start = a.query_start_loc[lo];
    const int i = static_cast<int>(t - start);
    const int64_t row = static_cast<int64_t>(a.context_lens[lo]) + i;
    const int64_t page = row / a.block_size;
    slot = static_cast<int64_t>(a.block_tables[lo * a.max_blocks + page]) * a.block_size +
           (row - page * a.block_size);
    int depth = i;
    if (mask != nullptr) {
      // up the tree: parents come before their children, so the words are met in falling order
      depth = -1;
      uint64_t bits = 0;
      int p = i;
      while (p >= 0) {
        for (; word - 1 > p / 64; --word) {
          mask[word - 1] = static_cast<int64_t>(bits);
          bits = 0;
        }
        bits |= uint64_t{1} << (p % 64);
        ++depth;
        int up = a.parents[start + p];
        if (up >= p || up < -1) {  // not a tree: the node counts as a root
          raise_error(a.err, kErrBadIndex);
          up = -1;
        }
        p = up;
      }
      mask[--word] = static_cast<int64_t>(bits);
    }
    position = static_cast<int64_t>(a.context_lens[lo]) + depth;
  }
  if (mask != nullptr) {
    while (word > 0) mask[--word] = 0;
  }
  a.slot_mapping[t] = slot;
  a.positions[t] = position;
}

__global__ void __launch_bounds__(kPlanThreads) plan_requests_kernel(const PlanArgs a) {
  grid_dependency_sync();
  __shared__ int64_t warp_sums[kPlanWarps];
  __shared__ int64_t sh_off[kPlanThreads];  // blocks given back or taken before this request
  __shared__ int32_t sh_count[kPlanThreads];
  __shared__ int32_t sh_owned[kPlanThreads];
  const int tid = threadIdx.x, lane = tid % kWarpSize, warp = tid / kWarpSize;

  int64_t have = a.free_count[0];
  if (have < 0 || have > a.free_capacity) {
    if (tid == 0) raise_error(a.err, kErrBadIndex);
    have = have < 0 ? 0 : a.free_capacity;
  }

  // finished requests: their blocks go on the free list, behind what is there
  int64_t back = 0;
  for (int64_t base = 0; base < a.num_seqs; base += kPlanThreads) {
    const int64_t s = base + tid;
    int64_t give = 0;
    if (s < a.num_seqs && a.query_lens[s] < 0) {
      const int32_t owned = a.blocks_owned[s];
      if (owned < 0 || owned > a.max_blocks) {
        raise_error(a.err, kErrBadIndex);
      } else {
        give = owned;
      }
    }
    int64_t total;
    const int64_t end = block_scan(give, warp_sums, total);
    if (total > 0) {  // the same for every thread
      sh_off[tid] = have + back + end - give;
      sh_count[tid] = static_cast<int32_t>(give);
      __syncthreads();
      for (int k = warp; k < kPlanThreads; k += kPlanWarps) {
        for (int i = lane; i < sh_count[k]; i += kWarpSize) {
          const int64_t to = sh_off[k] + i;
          if (to < a.free_capacity) {
            a.free_blocks[to] = a.block_tables[(base + k) * a.max_blocks + i];
          } else {
            raise_error(a.err, kErrBadIndex);  // no room: the block is dropped
          }
        }
      }
      __syncthreads();  // the next chunk's counts may be written
    }
    back += total;
  }
  have = have + back < a.free_capacity ? have + back : a.free_capacity;
  __syncthreads();  // blocks given back above may be taken below

  int64_t tokens = 0, needed = 0, used = 0;
  for (int64_t base = 0; base < a.num_seqs; base += kPlanThreads) {
    const int64_t s = base + tid;
    const bool is = s < a.num_seqs;
    const int64_t query = is ? a.query_lens[s] : 0;
    const int64_t context = is ? a.context_lens[s] : 0;
    const int64_t owned = is ? a.blocks_owned[s] : 0;
    const int64_t n = query > 0 ? query : 0;
    int64_t total;
    const int64_t tokens_end = tokens + block_scan(n, warp_sums, total);
    tokens += total;
    bool ok = is && query >= 0;
    if (ok && (context < 0 || owned < 0 || owned > a.max_blocks || tokens_end > a.num_tokens ||
               context + n > static_cast<int64_t>(a.max_blocks) * a.block_size ||
               (a.parents != nullptr && n > a.max_query_len))) {
      raise_error(a.err, kErrBadIndex);
      ok = false;
    }
    int64_t need = 0;
    if (ok && n > 0) {
      need = (context + n + a.block_size - 1) / a.block_size - owned;
      if (need < 0) need = 0;
    }
    const int64_t need_end = needed + block_scan(need, warp_sums, total);
    needed += total;
    const bool served = ok && (need == 0 || need_end <= have);
    if (is) {
      a.query_start_loc[s + 1] =
          static_cast<int32_t>(tokens_end < a.num_tokens ? tokens_end : a.num_tokens);
      a.seq_lens[s] = served ? static_cast<int32_t>(context + n) : 0;
      a.blocks_owned_out[s] = query < 0 ? 0 : static_cast<int32_t>(served ? owned + need : owned);
    }
    if (total > 0) {
      // needs are not negative, so the served ones among those with a need come first
      sh_off[tid] = need_end - need;
      sh_count[tid] = served ? static_cast<int32_t>(need) : 0;
      sh_owned[tid] = static_cast<int32_t>(owned);
      __syncthreads();
      for (int k = warp; k < kPlanThreads; k += kPlanWarps) {
        for (int i = lane; i < sh_count[k]; i += kWarpSize) {
          a.block_tables[(base + k) * a.max_blocks + sh_owned[k] + i] =
              a.free_blocks[have - 1 - sh_off[k] - i];
        }
      }
      __syncthreads();
    }
    int64_t took;
    block_scan(served ? need : 0, warp_sums, took);
    used += took;
  }
  if (tid == 0) {
    a.query_start_loc[0] = 0;
    a.free_count_out[0] = static_cast<int32_t>(have - used);
  }
  if (a.fused) {
    __syncthreads();
    for (int64_t t = tid; t < a.num_tokens; t += kPlanThreads) plan_token(a, t);
  }
}

__global__ void __launch_bounds__(kTokenThreads) plan_tokens_kernel(const PlanArgs a) {
  grid_dependency_sync();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kTokenThreads + threadIdx.x;
  if (t < a.num_tokens) plan_token(a, t);
}

}  // namespace
}  // namespace svllm::k

extern "C" int svllm_paged_plan(
    const int32_t* context_lens, const int32_t* query_lens, int64_t num_seqs,
    int32_t* block_tables, int64_t max_blocks, const int32_t* blocks_owned, int32_t* free_blocks,
    int64_t free_capacity, const int32_t* free_count, int64_t block_size, const int32_t* parents,
    int64_t max_query_len, int64_t num_tokens, int32_t* query_start_loc, int32_t* seq_lens,
    int64_t* slot_mapping, int64_t* positions, int64_t* tree_mask, int32_t* blocks_owned_out,
    int32_t* free_count_out, svllm_stream stream) {
  using namespace svllm::k;
  if (num_seqs < 0 || num_tokens < 0 || max_blocks <= 0 || block_size <= 0 || free_capacity < 0 ||
      (parents != nullptr && (max_query_len <= 0 || tree_mask == nullptr))) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  if (free_count == nullptr || query_start_loc == nullptr || free_count_out == nullptr ||
      (free_capacity > 0 && free_blocks == nullptr) ||
      (num_seqs > 0 && (context_lens == nullptr || query_lens == nullptr ||
                        block_tables == nullptr || blocks_owned == nullptr ||
                        seq_lens == nullptr || blocks_owned_out == nullptr)) ||
      (num_tokens > 0 && (slot_mapping == nullptr || positions == nullptr)) ||
      (num_seqs > 0 && blocks_owned == blocks_owned_out) || free_count == free_count_out) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  constexpr int64_t kMax = int64_t{1} << 31;
  if (num_seqs >= kMax / kTokenThreads || num_tokens >= kMax || max_blocks >= kMax ||
      block_size >= kMax || free_capacity >= kMax ||
      (parents != nullptr && max_query_len > SVLLM_MAX_TREE_NODES)) {
    return SVLLM_ERR_TOO_LARGE;
  }
  int device;
  if (current_device(&device) != SVLLM_OK) return SVLLM_ERR_CUDA;
  int* err = library_error_word(device);
  if (err == nullptr) return SVLLM_ERR_CUDA;

  PlanArgs a{};
  a.context_lens = context_lens;
  a.query_lens = query_lens;
  a.block_tables = block_tables;
  a.blocks_owned = blocks_owned;
  a.free_blocks = free_blocks;
  a.free_count = free_count;
  a.parents = parents;
  a.query_start_loc = query_start_loc;
  a.seq_lens = seq_lens;
  a.slot_mapping = slot_mapping;
  a.positions = positions;
  a.tree_mask = parents != nullptr ? tree_mask : nullptr;
  a.blocks_owned_out = blocks_owned_out;
  a.free_count_out = free_count_out;
  a.num_seqs = num_seqs;
  a.num_tokens = num_tokens;
  a.free_capacity = free_capacity;
  a.max_blocks = static_cast<int32_t>(max_blocks);
  a.block_size = static_cast<int32_t>(block_size);
  a.max_query_len = static_cast<int32_t>(max_query_len);
  a.mask_words = parents != nullptr ? static_cast<int32_t>((max_query_len + 63) / 64) : 0;
  a.fused = num_tokens <= kFusedTokens;
  a.err = err;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int status =
      launch(plan_requests_kernel, dim3(1), dim3(kPlanThreads), 0, st, 1u, a);
  if (status != SVLLM_OK || a.fused) return status;
  return launch(plan_tokens_kernel,
                dim3(static_cast<unsigned>((num_tokens + kTokenThreads - 1) / kTokenThreads)),
                dim3(kTokenThreads), 0, st, 1u, a);
}
