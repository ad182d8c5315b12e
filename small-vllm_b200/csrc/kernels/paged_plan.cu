// The paging plan of one step, from request lengths alone: which new KV blocks each request
// takes from the free list (and which a finished one gives back), its block table, and per token
// the cache slot, the position and, for trees of drafted tokens, the ancestor mask.
//
// With context c, query length n and o blocks owned, request s needs max(0, ceil((c + n) / bs) -
// o) blocks. Requests are served in order while the free list lasts: with P the inclusive prefix
// sum of the needs, s is served when P_s is at most the list's length (or its need is 0). Block
// k of the step, counted over all requests, is free_blocks[count - 1 - k].
//
// One CTA does the requests, as many threads as there are requests up to 1024: a scan of (tokens,
// blocks) is a few shuffles, and no grid-wide meeting is needed between giving blocks back and
// taking them. What bounds it is the chain of dependent loads and barriers, not bytes. Tokens are
// independent of one another (a binary search over the starts, one table entry, a walk up the
// parents); few of them follow in the same CTA, the starts and the parents staged in shared memory;
// of many (kFusedTokens) the part that depends on the inputs alone, the walks with the masks and
// positions, is done by more CTAs of the same launch, and a second kernel adds the slots. (It reads
// only what the first wrote: inputs that it read itself before its dependency wait would come from
// kernels of which nothing promises that their writes are visible to it.) Measured in a graph: 4
// requests of 8 nodes 3.2 us, 64 of 16 3.9, 1024 of 64 that take 4 blocks each 7.1 (2.1 MB read and
// written, 0.3 us of HBM time: latency is all there is); a call from the host costs it some 7.5 us,
// 10 with two launches.
#include <cuda_runtime.h>

#include <cstdint>

#include "common.cuh"
#include "host_common.h"

namespace svllm::k {
namespace {

constexpr int kPlanThreads = 1024;  // at most; as many as there are requests, in whole warps
constexpr int kTokenThreads = 256;
constexpr int kStagedStarts = 4096;  // of requests, staged by the CTAs of the walks
constexpr int kOwnBlocks = 8;        // new blocks up to which a request's own lane fetches them

// Up to this many tokens, times the words of a mask, are done by the CTA that did the requests;
// more get CTAs and a second kernel. us in a graph, one kernel against two: 32 tokens 3.2 and 3.5,
// 256 4.0 and 3.8, 512 4.2 and 3.8 (a second launch costs the host some 2 us), 1024 5.3 and 3.8,
// 4096 10.2 and 4.3.
constexpr int64_t kFusedTokens = 512;

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
  int64_t max_rows;              // max_blocks * block_size
  int32_t max_blocks;
  int32_t block_size;
  int32_t max_query_len;         // checked where parents are given: the mask's width
  int32_t mask_words;
  int fused;                     // CTA 0 does the tokens too
  int walks;                     // the CTAs from 1 on do the tokens' walks
  int* err;
};

// Lengths come from the caller unchecked: sums stop at the largest int (which no valid one reaches)
// instead of wrapping.
__device__ __forceinline__ uint32_t add_up(uint32_t a, uint32_t b) {
  return min(a + b, static_cast<uint32_t>(INT32_MAX));
}

// Inclusive sums over the CTA's threads of a pair; `total` receives the CTA's.
__device__ uint2 block_scan(uint2 v, uint2* warp_sums, uint2& total) {
  const int lane = threadIdx.x % kWarpSize, warp = threadIdx.x / kWarpSize;
  const int warps = blockDim.x / kWarpSize;
#pragma unroll
  for (int off = 1; off < kWarpSize; off *= 2) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, v.x, off);
    const uint32_t y = __shfl_up_sync(0xffffffffu, v.y, off);
    if (lane >= off) v = make_uint2(add_up(v.x, x), add_up(v.y, y));
  }
  if (warps == 1) {
    total = make_uint2(__shfl_sync(0xffffffffu, v.x, kWarpSize - 1),
                       __shfl_sync(0xffffffffu, v.y, kWarpSize - 1));
    return v;
  }
  __syncthreads();  // the previous scan's readers are done
  if (lane == kWarpSize - 1) warp_sums[warp] = v;
  __syncthreads();
  uint2 s = lane < warps ? warp_sums[lane] : make_uint2(0, 0);  // every warp sums the sums itself
#pragma unroll
  for (int off = 1; off < kWarpSize; off *= 2) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, s.x, off);
    const uint32_t y = __shfl_up_sync(0xffffffffu, s.y, off);
    if (lane >= off) s = make_uint2(add_up(s.x, x), add_up(s.y, y));
  }
  total = make_uint2(__shfl_sync(0xffffffffu, s.x, kWarpSize - 1),
                     __shfl_sync(0xffffffffu, s.y, kWarpSize - 1));
  if (warp > 0) {
    v.x = add_up(v.x, __shfl_sync(0xffffffffu, s.x, warp - 1));
    v.y = add_up(v.y, __shfl_sync(0xffffffffu, s.y, warp - 1));
  }
  return v;
}
static_assert(kPlanThreads <= kWarpSize * kWarpSize, "one value per warp in one warp");

// A token's request: the first whose end lies beyond it, by binary search over the starts.
__device__ int request_of(const PlanArgs& a, int t, const int32_t* starts) {
  int lo = 0, hi = static_cast<int>(a.num_seqs);
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (starts[mid + 1] > t) {
      hi = mid;
    } else {
      lo = mid + 1;
    }
  }
  return lo;
}

// A token's request and its row there; s < 0: none, or none that its table has room for.
struct TokenRow {
  int s = -1, row = 0;
};

__device__ TokenRow row_of(const PlanArgs& a, int t, int s, int start) {
  TokenRow r;
  if (s < a.num_seqs) {
    const int64_t row = static_cast<int64_t>(a.context_lens[s]) + (t - start);
    if (row >= 0 && row < a.max_rows) {
      r.s = s;
      r.row = static_cast<int>(row);
    }
  }
  return r;
}

// Position and mask of token `t`, node `i` of a request, as if the request were served. `parents`
// (of its first node; null: a chain) may be a staged copy.
__device__ void write_tree(const PlanArgs& a, int t, int i, int row, const int32_t* parents) {
  int depth = i;
  if (parents != nullptr) {
    if (i >= 64 * a.mask_words) return;  // a request wider than the mask: not served
    const int own = parents[i];
    int64_t* mask = a.tree_mask + static_cast<int64_t>(t) * a.mask_words;
    uint64_t bits = 0;
    depth = -1;
    if (a.mask_words == 1) {  // 1024 requests of 64 nodes: 7.1 us, 7.6 by the loop below
      for (int p = i; p >= 0;) {
        bits |= uint64_t{1} << p;
        ++depth;
        const int up = parents[p];
        p = up >= p ? -1 : up;  // not a tree: the node counts as a root
      }
      *mask = static_cast<int64_t>(bits);
    } else {
      // parents come before their children, so the words are met in falling order
      int word = a.mask_words - 1;
      for (int p = i; p >= 0;) {
        for (; word > p >> 6; --word) {
          mask[word] = static_cast<int64_t>(bits);
          bits = 0;
        }
        bits |= uint64_t{1} << (p & 63);
        ++depth;
        const int up = parents[p];
        p = up >= p ? -1 : up;
      }
      for (; word >= 0; --word) {
        mask[word] = static_cast<int64_t>(bits);
        bits = 0;
      }
    }
    if (own >= i || own < -1) raise_error(a.err, kErrBadIndex);
  }
  a.positions[t] = static_cast<int64_t>(row) - i + depth;
}

// A token's slot: what the requests' part wrote, read with plain loads.
struct TokenSlot {
  int64_t slot = 0;
  bool live = false;  // its request is served
};

__device__ TokenSlot find_slot(const PlanArgs& a, const TokenRow& r) {
  TokenSlot x;
  if (r.s >= 0) {
    const int page = r.row / a.block_size;
    const int block = a.block_tables[static_cast<int64_t>(r.s) * a.max_blocks + page];
    x.live = a.seq_lens[r.s] > 0;
    x.slot = static_cast<int64_t>(block) * a.block_size + (r.row - page * a.block_size);
  }
  return x;
}

__device__ void write_slot(const PlanArgs& a, int t, const TokenSlot& x) {
  a.slot_mapping[t] = x.live ? x.slot : -1;
  if (x.live) return;
  a.positions[t] = 0;
  for (int w = 0; w < a.mask_words; ++w) {
    a.tree_mask[static_cast<int64_t>(t) * a.mask_words + w] = 0;
  }
}

// Copies `count` block ids per lane, src[step * k] -> dst[k]: a lane's own when there are up to
// kOwnBlocks, else the warp together, four lanes' at a time. us in a graph, a lane's own against
// together: 64 requests of 1 block 3.4 and 4.8, 1024 of 4 5.8 and 9.3, 1024 of 16 16.4 and 9.5.
__device__ __forceinline__ void copy_blocks(int count, const int32_t* src, int step,
                                            int32_t* dst) {
  const int most = __reduce_max_sync(0xffffffffu, count);
  if (most <= kOwnBlocks) {
    int32_t held[kOwnBlocks];
#pragma unroll
    for (int k = 0; k < kOwnBlocks; ++k) {
      if (k < count) held[k] = src[step * k];
    }
#pragma unroll
    for (int k = 0; k < kOwnBlocks; ++k) {
      if (k < count) dst[k] = held[k];
    }
    return;
  }
  constexpr int kLanes = 4;
#pragma unroll 1
  for (int l = 0; l < kWarpSize; l += kLanes) {
    int n[kLanes], longest = 0;
    const int32_t* from[kLanes];
    int32_t* to[kLanes];
#pragma unroll
    for (int e = 0; e < kLanes; ++e) {
      n[e] = __shfl_sync(0xffffffffu, count, l + e);
      from[e] = reinterpret_cast<const int32_t*>(
          __shfl_sync(0xffffffffu, reinterpret_cast<int64_t>(src), l + e));
      to[e] = reinterpret_cast<int32_t*>(
          __shfl_sync(0xffffffffu, reinterpret_cast<int64_t>(dst), l + e));
      longest = max(longest, n[e]);
    }
#pragma unroll 1
    for (int k = threadIdx.x % kWarpSize; k < longest; k += kWarpSize) {
      int32_t held[kLanes];
#pragma unroll
      for (int e = 0; e < kLanes; ++e) {
        if (k < n[e]) held[e] = from[e][static_cast<int64_t>(step) * k];
      }
#pragma unroll
      for (int e = 0; e < kLanes; ++e) {
        if (k < n[e]) to[e][k] = held[e];
      }
    }
  }
}

// The walks of blockDim tokens, by one of the CTAs beside the requests': position and mask, and in
// slot_mapping, for the kernel that follows, the token's request and row. The starts it needs are
// summed up once more.
__device__ void walk_tokens(const PlanArgs& a, int32_t* starts, uint2* warp_sums) {
  const int n_seqs = static_cast<int>(a.num_seqs), tid = threadIdx.x, threads = blockDim.x;
  uint32_t* ends = reinterpret_cast<uint32_t*>(starts + n_seqs + 1);  // of the threads' requests
  const int each = (n_seqs + threads - 1) / threads;
  const int first = min(n_seqs, tid * each), last = min(n_seqs, first + each);
  uint32_t sum = 0;
  for (int s = first; s < last; ++s) {
    sum = add_up(sum, static_cast<uint32_t>(max(a.query_lens[s], 0)));
    starts[s + 1] = static_cast<int32_t>(sum);
  }
  uint2 total;
  ends[tid] = block_scan(make_uint2(sum, 0), warp_sums, total).x;
  __syncthreads();
  const uint32_t limit = static_cast<uint32_t>(a.num_tokens);
  const uint32_t before = tid == 0 ? 0 : ends[tid - 1];
  for (int s = first; s < last; ++s) {
    starts[s + 1] = static_cast<int32_t>(
        min(add_up(before, static_cast<uint32_t>(starts[s + 1])), limit));
  }
  if (tid == 0) starts[0] = 0;
  __syncthreads();
  const int64_t at = static_cast<int64_t>(blockIdx.x - 1) * threads + tid;
  if (at >= a.num_tokens) return;
  const int t = static_cast<int>(at);
  const int s = request_of(a, t, starts), start = s < n_seqs ? starts[s] : 0;
  const TokenRow r = row_of(a, t, s, start);
  a.slot_mapping[t] = static_cast<int64_t>(r.s) * (int64_t{1} << 32) + r.row;
  if (s < n_seqs) {
    write_tree(a, t, t - start, r.row, a.parents == nullptr ? nullptr : a.parents + start);
  }
}

__global__ void __launch_bounds__(kPlanThreads) plan_requests_kernel(const PlanArgs a) {
  grid_dependency_sync();
  // starts; then parents, for the tokens (fused), or the threads' sums (the CTAs of the walks)
  extern __shared__ int32_t staged[];
  __shared__ uint2 warp_sums[kPlanThreads / kWarpSize];
  __shared__ int used;
  const int tid = threadIdx.x;
  const int threads = blockDim.x, n_seqs = static_cast<int>(a.num_seqs);
  if (blockIdx.x > 0) {
    walk_tokens(a, staged, warp_sums);
    return;
  }
  if (tid == 0) used = 0;
  if (a.fused && a.tree_mask != nullptr) {
    for (int t = tid; t < a.num_tokens; t += threads) staged[n_seqs + 1 + t] = a.parents[t];
  }

  int64_t have = a.free_count[0];
  if (have < 0 || have > a.free_capacity) {
    if (tid == 0) raise_error(a.err, kErrBadIndex);
    have = have < 0 ? 0 : a.free_capacity;
  }

  // finished requests: their blocks go on the free list, behind what is there
  int64_t back = 0;
  int query = 0, context = 0, owned = 0;  // of the last chunk read
  for (int base = 0; base < n_seqs; base += threads) {
    const int s = base + tid;
    query = s < n_seqs ? a.query_lens[s] : 0;
    context = s < n_seqs ? a.context_lens[s] : 0;
    owned = s < n_seqs ? a.blocks_owned[s] : 0;
    if (!__syncthreads_or(query < 0)) continue;
    uint32_t give = 0;
    if (query < 0) {
      if (owned < 0 || owned > a.max_blocks) {
        raise_error(a.err, kErrBadIndex);
      } else {
        give = owned;
      }
    }
    uint2 total;
    const uint2 end = block_scan(make_uint2(give, 0), warp_sums, total);
    const int64_t at = have + back + end.x - give;
    // what finds no room is dropped
    const int64_t room = a.free_capacity - at;
    const int fits = room <= 0 ? 0 : room < give ? static_cast<int>(room) : static_cast<int>(give);
    if (fits < static_cast<int>(give)) raise_error(a.err, kErrBadIndex);
    const int32_t* row = a.block_tables + static_cast<int64_t>(s) * a.max_blocks;
    copy_blocks(fits, row, 1, a.free_blocks + at);
    back += total.x;
  }
  have = have + back < a.free_capacity ? have + back : a.free_capacity;
  __syncthreads();  // blocks given back above may be taken below

  uint32_t tokens = 0, needed = 0;  // of the chunks before
  for (int base = 0; base < n_seqs; base += threads) {
    const int s = base + tid;
    const bool is = s < n_seqs;
    if (n_seqs > threads) {  // else they are in registers
      query = is ? a.query_lens[s] : 0;
      context = is ? a.context_lens[s] : 0;
      owned = is ? a.blocks_owned[s] : 0;
    }
    const int n = query > 0 ? query : 0;
    const int64_t rows = static_cast<int64_t>(context) + n;
    bool ok = is && query >= 0;
    if (ok && (context < 0 || owned < 0 || owned > a.max_blocks || rows > a.max_rows ||
               (a.tree_mask != nullptr && n > a.max_query_len))) {
      raise_error(a.err, kErrBadIndex);
      ok = false;
    }
    int need = 0;
    if (ok && n > 0) {
      need = static_cast<int>((static_cast<uint32_t>(rows) + a.block_size - 1) /
                              static_cast<uint32_t>(a.block_size)) - owned;
      if (need < 0) need = 0;
    }
    uint2 total;
    uint2 end = block_scan(make_uint2(n, need), warp_sums, total);
    end = make_uint2(add_up(end.x, tokens), add_up(end.y, needed));
    if (ok && n > 0 && end.x > a.num_tokens) {
      // past the tokens' room; so is every later request with a token, and their needs, counted
      // in the sums above, come after those of all that are served
      raise_error(a.err, kErrBadIndex);
      ok = false;
    }
    const bool served = ok && (need == 0 || end.y <= have);
    const int32_t start = static_cast<int32_t>(
        end.x < a.num_tokens ? end.x : static_cast<uint32_t>(a.num_tokens));
    if (is) {
      a.query_start_loc[s + 1] = start;
      if (a.fused) staged[s + 1] = start;
      a.seq_lens[s] = served ? static_cast<int32_t>(rows) : 0;
      a.blocks_owned_out[s] = query < 0 ? 0 : served ? owned + need : owned;
    }
    const int take = served ? need : 0;
    if (take > 0) atomicMax(&used, static_cast<int>(end.y));  // the served needs come first
    const int64_t top = have - 1 - (static_cast<int64_t>(end.y) - need);
    int32_t* row = a.block_tables + static_cast<int64_t>(s) * a.max_blocks + owned;
    copy_blocks(take, a.free_blocks + top, -1, row);
    tokens = add_up(tokens, total.x);
    needed = add_up(needed, total.y);
  }
  if (tid == 0) {
    a.query_start_loc[0] = 0;
    if (a.fused) staged[0] = 0;
  }
  __syncthreads();
  if (tid == 0) a.free_count_out[0] = static_cast<int32_t>(have - used);
  if (a.fused) {
    for (int t = tid; t < a.num_tokens; t += threads) {
      const int s = request_of(a, t, staged), start = s < n_seqs ? staged[s] : 0;
      const TokenRow r = row_of(a, t, s, start);
      const TokenSlot x = find_slot(a, r);
      if (s < n_seqs) {
        write_tree(a, t, t - start, r.row,
                   a.parents == nullptr ? nullptr : staged + n_seqs + 1 + start);
      }
      write_slot(a, t, x);
    }
  }
}

// The tokens' slots, after plan_requests_kernel; the walks too where that had too many starts to
// stage.
__global__ void __launch_bounds__(kTokenThreads) plan_tokens_kernel(const PlanArgs a) {
  grid_dependency_sync();
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kTokenThreads + threadIdx.x;
  if (at >= a.num_tokens) return;
  const int t = static_cast<int>(at);
  TokenRow r;
  if (a.walks) {
    const int64_t left = a.slot_mapping[t];
    r.s = static_cast<int>(left >> 32);
    r.row = static_cast<int>(left & 0xffffffff);
  } else {
    const int s = request_of(a, t, a.query_start_loc);
    if (s < a.num_seqs) {
      const int start = a.query_start_loc[s];
      r = row_of(a, t, s, start);
      write_tree(a, t, t - start, r.row, a.parents == nullptr ? nullptr : a.parents + start);
    }
  }
  write_slot(a, t, find_slot(a, r));
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
  if (num_seqs >= kMax / kTokenThreads || num_tokens >= kMax - 1 || max_blocks >= kMax ||
      block_size >= kMax || max_blocks * block_size >= kMax || free_capacity >= kMax ||
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
  a.max_rows = max_blocks * block_size;
  a.max_blocks = static_cast<int32_t>(max_blocks);
  a.block_size = static_cast<int32_t>(block_size);
  a.max_query_len = static_cast<int32_t>(max_query_len);
  a.mask_words = parents != nullptr ? static_cast<int32_t>((max_query_len + 63) / 64) : 0;
  a.fused = num_tokens * (a.mask_words > 1 ? a.mask_words : 1) <= kFusedTokens &&
            num_seqs <= kPlanThreads;
  a.walks = !a.fused && num_seqs <= kStagedStarts;
  a.err = err;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // a thread per request, and per token where those are done here too (512 tokens by 256 threads
  // took 4.7 us instead of 3.9)
  int64_t threads = a.fused && num_tokens > num_seqs ? num_tokens : num_seqs;
  if (threads < (a.walks ? kTokenThreads : 1)) threads = a.walks ? kTokenThreads : 1;
  threads = threads > kPlanThreads ? kPlanThreads : round_up(threads, kWarpSize);
  const int64_t beside = a.walks ? (num_tokens + threads - 1) / threads : 0;
  int64_t staged = 0;  // ints
  if (a.fused) staged = num_seqs + 1 + (parents != nullptr ? num_tokens : 0);
  if (a.walks) staged = num_seqs + 1 + threads;
  const int status = launch(plan_requests_kernel, dim3(static_cast<unsigned>(1 + beside)),
                            dim3(static_cast<unsigned>(threads)), static_cast<size_t>(staged) * 4,
                            st, 1u, a);
  if (status != SVLLM_OK || a.fused || num_tokens == 0) return status;
  return launch(plan_tokens_kernel,
                dim3(static_cast<unsigned>((num_tokens + kTokenThreads - 1) / kTokenThreads)),
                dim3(kTokenThreads), 0, st, 1u, a);
}
