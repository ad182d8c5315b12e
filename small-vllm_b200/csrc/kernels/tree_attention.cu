// Attention of a step's tokens over a paged KV cache that holds the step's own rows too: the
// nodes of a tree of drafted tokens see the request's context and their ancestors.
//
//   o[t, h] = sum_j p_j v_j,  p = softmax_j(scale * q[t, h] . k_j),
//   j < context, or j = context + node with the node's bit in tree_mask[t]
//
// One warp per (token, head): each lane scores one of 32 cache rows, then every row's value is
// added by all lanes, 16 bytes or less of it each.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "common.cuh"
#include "host_common.h"

namespace svllm::k {
namespace {

struct TreeAttnArgs {
  void* out;                       // [num_tokens, num_heads, head_dim] bf16, contiguous
  const void* q;                   // [num_tokens, num_heads, head_dim] bf16, token stride q_stride
  const void* k_cache;             // [num_blocks, block_size, num_kv_heads, head_dim] bf16
  const void* v_cache;
  const int32_t* block_tables;     // [num_seqs, max_blocks]
  const int32_t* seq_lens;         // [num_seqs]
  const int32_t* query_start_loc;  // [num_seqs + 1]
  const int64_t* tree_mask;        // [num_tokens, mask_words] or null: causal
  int64_t q_stride;
  int64_t num_blocks;
  int64_t num_tokens;
  int64_t num_seqs;
  int max_blocks;
  int block_size;
  int num_heads;
  int num_kv_heads;
  int mask_words;
  float scale_log2;
  int* err;
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int D>
__global__ void __launch_bounds__(128) tree_attention_simple_kernel(const TreeAttnArgs a) {
  grid_dependency_sync();
  constexpr int kPer = D / kWarpSize;  // output elements per lane
  const int lane = threadIdx.x % kWarpSize;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWarpSize;
  const int64_t t = unit / a.num_heads;
  const int h = static_cast<int>(unit % a.num_heads);
  if (t >= a.num_tokens) return;
  const int kh = h / (a.num_heads / a.num_kv_heads);

  int64_t b = 0;  // the request: the first whose end lies beyond t
  while (b < a.num_seqs && a.query_start_loc[b + 1] <= t) ++b;
  int64_t context = 0, seq = 0, node = 0;
  if (b < a.num_seqs) {
    const int64_t start = a.query_start_loc[b];
    const int64_t n = a.query_start_loc[b + 1] - start;
    seq = a.seq_lens[b];
    context = seq - n;
    node = t - start;
    if (seq != 0 && (context < 0 || seq > static_cast<int64_t>(a.max_blocks) * a.block_size ||
                     (a.tree_mask != nullptr && n > 64 * a.mask_words))) {
      raise_error(a.err, kErrBadIndex);
      seq = 0;
    }
  }
  float q[D];
  const __nv_bfloat16* qp =
      static_cast<const __nv_bfloat16*>(a.q) + t * a.q_stride + static_cast<int64_t>(h) * D;
  for (int d = 0; d < D; ++d) q[d] = __bfloat162float(qp[d]);
  float m = -__builtin_huge_valf(), l = 0.0f, acc[kPer] = {};
  const int32_t* table = a.block_tables + b * a.max_blocks;
  for (int64_t j0 = 0; j0 < seq; j0 += kWarpSize) {
    const int64_t j = j0 + lane;
    bool sees = j < context;
    if (!sees && j < seq) {
      const int64_t x = j - context;
      sees = a.tree_mask == nullptr
                 ? x <= node
                 : (static_cast<uint64_t>(a.tree_mask[t * a.mask_words + x / 64]) >> (x % 64)) & 1;
    }
    int64_t row = 0;
    float s = -__builtin_huge_valf();
    if (sees) {
      int64_t blk = table[j / a.block_size];
      if (blk < 0 || blk >= a.num_blocks) {
        raise_error(a.err, kErrBadIndex);
        blk = 0;
      }
      row = ((blk * a.block_size + j % a.block_size) * a.num_kv_heads + kh) * D;
      const __nv_bfloat16* kp = static_cast<const __nv_bfloat16*>(a.k_cache) + row;
      s = 0.0f;
      for (int d = 0; d < D; ++d) s = fmaf(q[d], __bfloat162float(kp[d]), s);
      s *= a.scale_log2;
    }
    float mx = s;
    for (int off = 16; off > 0; off /= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    mx = fmaxf(m, mx);
    const float base = mx == -__builtin_huge_valf() ? 0.0f : mx;
    const float al = exp2_approx(m - base);
    const float p = sees ? exp2_approx(s - base) : 0.0f;
    l = l * al + p;
    for (int e = 0; e < kPer; ++e) acc[e] *= al;
    m = mx;
    unsigned live = __ballot_sync(0xffffffffu, sees);
    while (live != 0) {
      const int src = __ffs(static_cast<int>(live)) - 1;
      live &= live - 1;
      const float pj = __shfl_sync(0xffffffffu, p, src);
      const int64_t rj = __shfl_sync(0xffffffffu, row, src);
      const __nv_bfloat16* vp = static_cast<const __nv_bfloat16*>(a.v_cache) + rj + lane * kPer;
      for (int e = 0; e < kPer; ++e) acc[e] = fmaf(pj, __bfloat162float(vp[e]), acc[e]);
    }
  }
  for (int off = 16; off > 0; off /= 2) l += __shfl_xor_sync(0xffffffffu, l, off);
  __nv_bfloat16* out =
      static_cast<__nv_bfloat16*>(a.out) + (t * a.num_heads + h) * D + lane * kPer;
  // a sum of zero: the token saw no row (a NaN sum stays NaN)
  for (int e = 0; e < kPer; ++e) out[e] = __float2bfloat16_rn(l == 0.0f ? 0.0f : acc[e] / l);
}

}  // namespace
}  // namespace svllm::k

extern "C" int svllm_tree_attention_workspace_bytes(int64_t head_dim, int64_t* bytes) {
  if (bytes == nullptr || head_dim <= 0) return SVLLM_ERR_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 128) return SVLLM_ERR_UNSUPPORTED;
  *bytes = 0;
  return SVLLM_OK;
}

extern "C" int svllm_tree_attention_bf16(
    void* out, const void* q, int64_t q_token_stride, const void* k_cache, const void* v_cache,
    int64_t num_blocks, int64_t block_size, const int32_t* block_tables, int64_t max_blocks,
    const int32_t* seq_lens, const int32_t* query_start_loc, int64_t num_seqs, int64_t num_tokens,
    int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, const int64_t* tree_mask,
    int64_t mask_words, float scale, void* workspace, int64_t workspace_bytes,
    svllm_stream stream) {
  using namespace svllm::k;
  if (num_seqs < 0 || num_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads % num_kv_heads != 0 || head_dim <= 0 || block_size <= 0 || max_blocks <= 0 ||
      num_blocks <= 0 || q_token_stride < num_heads * head_dim || !(scale > 0.0f) ||
      !std::isfinite(scale) || (tree_mask != nullptr && mask_words <= 0)) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  if (num_tokens == 0) return SVLLM_OK;
  if (out == nullptr || q == nullptr || k_cache == nullptr || v_cache == nullptr ||
      query_start_loc == nullptr ||
      (num_seqs > 0 && (block_tables == nullptr || seq_lens == nullptr))) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  if ((head_dim != 64 && head_dim != 128) || !aligned16(out) || !aligned16(q) ||
      !aligned16(k_cache) || !aligned16(v_cache) || (q_token_stride * 2) % 16 != 0) {
    return SVLLM_ERR_UNSUPPORTED;
  }
  constexpr int64_t kMax = int64_t{1} << 31;
  if (num_seqs >= kMax || num_tokens * num_heads >= kMax || max_blocks >= kMax ||
      block_size >= (int64_t{1} << 20) || max_blocks * block_size >= kMax ||
      (tree_mask != nullptr && mask_words > SVLLM_MAX_TREE_NODES / 64)) {
    return SVLLM_ERR_TOO_LARGE;
  }
  (void)workspace;
  (void)workspace_bytes;
  int device;
  if (current_device(&device) != SVLLM_OK) return SVLLM_ERR_CUDA;
  int* err = library_error_word(device);
  if (err == nullptr) return SVLLM_ERR_CUDA;
  TreeAttnArgs a{};
  a.out = out;
  a.q = q;
  a.k_cache = k_cache;
  a.v_cache = v_cache;
  a.block_tables = block_tables;
  a.seq_lens = seq_lens;
  a.query_start_loc = query_start_loc;
  a.tree_mask = tree_mask;
  a.q_stride = q_token_stride;
  a.num_blocks = num_blocks;
  a.num_tokens = num_tokens;
  a.num_seqs = num_seqs;
  a.max_blocks = static_cast<int>(max_blocks);
  a.block_size = static_cast<int>(block_size);
  a.num_heads = static_cast<int>(num_heads);
  a.num_kv_heads = static_cast<int>(num_kv_heads);
  a.mask_words = static_cast<int>(mask_words);
  a.scale_log2 = static_cast<float>(static_cast<double>(scale) / std::log(2.0));
  a.err = err;
  const dim3 grid(static_cast<unsigned>((num_tokens * num_heads + 3) / 4));
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return head_dim == 128 ? launch(tree_attention_simple_kernel<128>, grid, dim3(128), 0, s, 1u, a)
                         : launch(tree_attention_simple_kernel<64>, grid, dim3(128), 0, s, 1u, a);
}
