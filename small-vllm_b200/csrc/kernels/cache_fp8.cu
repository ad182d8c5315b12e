// Writing and reading the 8-bit KV cache (its format: fp8.cuh).
//
// svllm_qk_norm_rope_cache_fp8_bf16 / svllm_rope_cache_fp8_bf16: a decoder layer's rotary step
// with the quantised cache write in the same pass. Per token and head of dimension D, in fp32:
//   x'_i = x_i * rsqrt(mean_j x_j^2 + eps) * w_i                      (the kind with norms only)
//   y_i = x'_i cos a_i - x'_{i+D/2} sin a_i,  y_{i+D/2} = x'_{i+D/2} cos a_i + x'_i sin a_i
// with a_i = position * inv_freq[i]; q <- bf16(y) in place; y of k and the unchanged v are
// quantised into the token's slot. Every value is rounded once, where it is stored (the bf16
// rotary ops round after each step, as Hugging Face's modules do; a code is rounded far more
// coarsely than that, and this way nothing is rounded twice). k itself stays as it was, which
// saves its write. The angle is formed in half turns in fp64 and reduced there, so far positions
// keep all of fp32's precision and sincospif never takes its slow path.
//
// The bound is memory: per token 4 Hq D + 4 Hk D bytes of bf16 and 2 Hk (D + 1) of cache.
//
// svllm_cache_read_fp8_bf16: the rows of whole requests back in bf16 (exact), as pages in the
// order of the request: [num_seqs, max_blocks * block_size, Hk, D], zeros behind a request's end.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "common.cuh"
#include "fp8.cuh"
#include "host_common.h"

namespace svllm::k {
namespace {

constexpr int kMaxHalf = 64;  // head_dim 64 or 128
constexpr int kThreads = 256;

struct CacheWriteArgs {
  void* q;        // [num_tokens, num_heads, D] bf16 at q_stride elements a token
  const void* k;  // [num_tokens, num_kv_heads, D]
  const void* v;
  const void* q_weight;  // [D], null without norms
  const void* k_weight;
  const void* positions;
  const int64_t* slots;
  uint8_t* k_cache;  // [num_slots, num_kv_heads, D]
  uint8_t* v_cache;
  uint8_t* k_scale;  // [num_slots, num_kv_heads]
  uint8_t* v_scale;
  int64_t num_tokens;
  int64_t q_stride, k_stride, v_stride;
  int64_t num_slots;
  int num_heads, num_kv_heads;
  int parts;  // units a token is cut into
  int pos_is_i64;
  int early_dependents;
  float eps;
  int* err;
  float inv_freq[kMaxHalf];
};

// Eight bf16 values: one 16-byte vector, or, where rows are not aligned to 16 bytes, eight loads.
// Not the read-only path: q is written by the same thread later.
template <bool kAligned>
__device__ __forceinline__ uint4 load8(const uint8_t* p) {
  if constexpr (kAligned) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p));
    return r;
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = h[2 * i] | (static_cast<uint32_t>(h[2 * i + 1]) << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <bool kAligned>
__device__ __forceinline__ void store8(uint8_t* p, const uint4& v) {
  if constexpr (kAligned) {
    st_global_v4(p, v);
  } else {
    uint16_t* h = reinterpret_cast<uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[2 * i] = static_cast<uint16_t>(word(v, i));
      h[2 * i + 1] = static_cast<uint16_t>(word(v, i) >> 16);
    }
  }
}

template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
  for (int offset = G / 2; offset > 0; offset /= 2) {
    v = max(v, __shfl_xor_sync(0xffffffffu, v, offset));
  }
  return v;
}

// The heads of a token in order, q then k then v, are dealt to passes of 32 / G heads, G = D / 16
// lanes a head; lane j of a head holds elements [8j, 8j + 8) and the matching ones of the second
// half, so that every rotation pair is in one lane. A unit is kPasses passes of a token, and a
// warp's: all its loads are issued before the first is used.
template <int D, bool kNorm, bool kAligned, int kPasses>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(
    const __grid_constant__ CacheWriteArgs a) {
  grid_dependency_wait();
  if (a.early_dependents) allow_dependents();
  constexpr int G = D / 16;
  constexpr int kHeads = kWarpSize / G;  // heads a pass
  constexpr int kHalf = D / 2;
  __shared__ __align__(16) float trig[kThreads / kWarpSize][2][kHalf];

  const int warp = threadIdx.x / kWarpSize;
  const int lane = threadIdx.x % kWarpSize;
  const int sub = lane % G;
  const int rotated = a.num_heads + a.num_kv_heads;
  const int total = rotated + a.num_kv_heads;

  // half turns per position of the pairs this lane works out
  double turns[kHalf / kWarpSize];
#pragma unroll
  for (int i = 0; i < kHalf / kWarpSize; ++i) {
    turns[i] = static_cast<double>(a.inv_freq[lane + i * kWarpSize]) * 0.31830988618379067154;
  }
  uint4 weight[4] = {};  // q and k, first and second half
  if constexpr (kNorm) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const void* w = i < 2 ? a.q_weight : a.k_weight;
      weight[i] = load8<kAligned>(static_cast<const uint8_t*>(w) + (i % 2 * kHalf + 8 * sub) * 2);
    }
  }

  const int64_t units = a.num_tokens * a.parts;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / kWarpSize);
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (kThreads / kWarpSize) + warp; u < units;
       u += step) {
    const int64_t t = u / a.parts;
    const int first = static_cast<int>(u % a.parts) * kPasses * kHeads;
    int64_t slot = __ldg(reinterpret_cast<const long long*>(a.slots) + t);
    if (slot >= a.num_slots) {
      if (lane == 0) raise_error(a.err, kErrBadIndex);
      slot = -1;
    }
    // a padding token's k and v are not read
    const int last = slot < 0 ? a.num_heads : total;
    uint4 lo[kPasses], hi[kPasses];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int h = first + p * kHeads + lane / G;
      if (h < last) {
        const uint8_t* row =
            h < a.num_heads
                ? static_cast<const uint8_t*>(a.q) + (t * a.q_stride + int64_t{h} * D) * 2
            : h < rotated
                ? static_cast<const uint8_t*>(a.k) +
                      (t * a.k_stride + int64_t{h - a.num_heads} * D) * 2
                : static_cast<const uint8_t*>(a.v) + (t * a.v_stride + int64_t{h - rotated} * D) * 2;
        lo[p] = load8<kAligned>(row + 16 * sub);
        hi[p] = load8<kAligned>(row + 2 * kHalf + 16 * sub);
      } else {
        lo[p] = hi[p] = make_uint4(0, 0, 0, 0);
      }
    }
    float c[8] = {}, s[8] = {};
    if (first < rotated) {
      const double pos =
          a.pos_is_i64
              ? static_cast<double>(__ldg(static_cast<const long long*>(a.positions) + t))
              : static_cast<double>(__ldg(static_cast<const int*>(a.positions) + t));
      __syncwarp();  // the unit before has been read
#pragma unroll
      for (int i = 0; i < kHalf / kWarpSize; ++i) {
        const double x = pos * turns[i];
        const float r = static_cast<float>(fma(-2.0, rint(0.5 * x), x));  // in [-1, 1]
        sincospif(r, &trig[warp][1][lane + i * kWarpSize], &trig[warp][0][lane + i * kWarpSize]);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 c4 = reinterpret_cast<const float4*>(&trig[warp][0][8 * sub])[i];
        const float4 s4 = reinterpret_cast<const float4*>(&trig[warp][1][8 * sub])[i];
        c[4 * i] = c4.x, c[4 * i + 1] = c4.y, c[4 * i + 2] = c4.z, c[4 * i + 3] = c4.w;
        s[4 * i] = s4.x, s[4 * i + 1] = s4.y, s[4 * i + 2] = s4.z, s[4 * i + 3] = s4.w;
      }
    }
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int pass = first + p * kHeads;
      if (pass >= last) break;
      const int h = pass + lane / G;
      float x[8], y[8];
      unpack<Bf16>(lo[p], x);
      unpack<Bf16>(hi[p], y);
      if (pass < rotated) {  // not a pass of v alone
        float xr[8], yr[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) xr[e] = x[e], yr[e] = y[e];
        if constexpr (kNorm) {
          float sum = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], fmaf(y[e], y[e], sum));
          const float inv = rsqrtf(group_sum<G>(sum) * (1.0f / D) + a.eps);
          float wl[8], wh[8];
          unpack<Bf16>(h < a.num_heads ? weight[0] : weight[2], wl);
          unpack<Bf16>(h < a.num_heads ? weight[1] : weight[3], wh);
#pragma unroll
          for (int e = 0; e < 8; ++e) xr[e] = x[e] * inv * wl[e], yr[e] = y[e] * inv * wh[e];
        }
        if (h < rotated) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] = fmaf(xr[e], c[e], -(yr[e] * s[e]));
            y[e] = fmaf(yr[e], c[e], xr[e] * s[e]);
          }
        }
      }
      if (h < a.num_heads) {
        uint8_t* row = static_cast<uint8_t*>(a.q) + (t * a.q_stride + int64_t{h} * D) * 2;
        store8<kAligned>(row + 16 * sub, pack<Bf16>(x));
        store8<kAligned>(row + 2 * kHalf + 16 * sub, pack<Bf16>(y));
      }
      if (pass + kHeads <= a.num_heads) continue;  // a pass of q alone
      uint32_t amax = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        amax = max(amax, max(__float_as_uint(x[e]) & 0x7fffffffu,
                             __float_as_uint(y[e]) & 0x7fffffffu));
      }
      amax = group_max<G>(amax);
      if (__any_sync(0xffffffffu, amax >= 0x7f800000u)) {
        // infinities and NaN become the NaN code and do not count for the scale
        amax = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (isfinite(x[e])) amax = max(amax, __float_as_uint(x[e]) & 0x7fffffffu);
          else x[e] = __int_as_float(0x7fffffff);
          if (isfinite(y[e])) amax = max(amax, __float_as_uint(y[e]) & 0x7fffffffu);
          else y[e] = __int_as_float(0x7fffffff);
        }
        amax = group_max<G>(amax);
      }
      const int exponent = scale_exponent(amax);
      if (h >= a.num_heads && h < last) {
        const float f = exp2_int(-exponent);
        uint32_t cl[2], ch[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          cl[i] = pack_e4m3x2(x[4 * i] * f, x[4 * i + 1] * f) |
                  (pack_e4m3x2(x[4 * i + 2] * f, x[4 * i + 3] * f) << 16);
          ch[i] = pack_e4m3x2(y[4 * i] * f, y[4 * i + 1] * f) |
                  (pack_e4m3x2(y[4 * i + 2] * f, y[4 * i + 3] * f) << 16);
        }
        const bool is_k = h < rotated;
        const int64_t row = slot * a.num_kv_heads + (is_k ? h - a.num_heads : h - rotated);
        uint8_t* codes = (is_k ? a.k_cache : a.v_cache) + row * D;
        *reinterpret_cast<uint2*>(codes + 8 * sub) = make_uint2(cl[0], cl[1]);
        *reinterpret_cast<uint2*>(codes + kHalf + 8 * sub) = make_uint2(ch[0], ch[1]);
        if (sub == 0) {
          (is_k ? a.k_scale : a.v_scale)[row] = static_cast<uint8_t>(exponent + kScaleBias);
        }
      }
    }
  }
}

using WriteKernel = void (*)(CacheWriteArgs);

template <int D, bool kNorm>
WriteKernel pick_write(bool aligned, bool one_pass) {
  if (aligned) {
    return one_pass ? cache_write_kernel<D, kNorm, true, 1> : cache_write_kernel<D, kNorm, true, 4>;
  }
  return cache_write_kernel<D, kNorm, false, 1>;
}

int launch_cache_write(CacheWriteArgs a, bool norm, int pos_type, int64_t num_heads,
                       int64_t num_kv_heads, int64_t head_dim, const float* inv_freq,
                       cudaStream_t stream) {
  if (a.num_tokens < 0 || num_heads < 0 || num_kv_heads <= 0 || head_dim <= 0 || a.num_slots < 0 ||
      (pos_type != SVLLM_INDEX_I32 && pos_type != SVLLM_INDEX_I64) || inv_freq == nullptr ||
      (num_heads > 0 && a.q_stride < num_heads * head_dim) ||
      a.k_stride < num_kv_heads * head_dim || a.v_stride < num_kv_heads * head_dim) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  if (a.num_tokens == 0) return SVLLM_OK;
  if ((num_heads > 0 && a.q == nullptr) || a.k == nullptr || a.v == nullptr ||
      a.positions == nullptr || a.slots == nullptr || a.k_cache == nullptr ||
      a.v_cache == nullptr || a.k_scale == nullptr || a.v_scale == nullptr ||
      (norm && (a.q_weight == nullptr || a.k_weight == nullptr)) ||
      (reinterpret_cast<uintptr_t>(a.slots) & 7u) != 0) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  if (num_heads > (1 << 16) || num_kv_heads > (1 << 16)) return SVLLM_ERR_TOO_LARGE;
  if ((head_dim != 64 && head_dim != 128) || !aligned16(a.k_cache) || !aligned16(a.v_cache)) {
    return SVLLM_ERR_UNSUPPORTED;
  }
  int device;
  if (current_device(&device) != SVLLM_OK) return SVLLM_ERR_CUDA;
  a.err = library_error_word(device);
  if (a.err == nullptr) return SVLLM_ERR_CUDA;
  a.num_heads = static_cast<int>(num_heads);
  a.num_kv_heads = static_cast<int>(num_kv_heads);
  a.pos_is_i64 = pos_type == SVLLM_INDEX_I64;
  std::memcpy(a.inv_freq, inv_freq, sizeof(float) * (head_dim / 2));
  const bool aligned = aligned16(a.q) && aligned16(a.k) && aligned16(a.v) &&
                       (!norm || (aligned16(a.q_weight) && aligned16(a.k_weight))) &&
                       a.q_stride % 8 == 0 && a.k_stride % 8 == 0 && a.v_stride % 8 == 0;
  const int heads_a_pass = kWarpSize / static_cast<int>(head_dim / 16);
  const int64_t passes =
      (num_heads + 2 * num_kv_heads + heads_a_pass - 1) / heads_a_pass;
  // few tokens: a pass a warp, so that their chains run side by side
  const bool one_pass = !aligned || a.num_tokens * passes <= int64_t{64} * sm_count(device);
  a.parts = static_cast<int>(one_pass ? passes : (passes + 3) / 4);
  const WriteKernel kernel = head_dim == 128
                                 ? (norm ? pick_write<128, true>(aligned, one_pass)
                                         : pick_write<128, false>(aligned, one_pass))
                                 : (norm ? pick_write<64, true>(aligned, one_pass)
                                         : pick_write<64, false>(aligned, one_pass));
  const int per_sm = blocks_per_sm(reinterpret_cast<const void*>(kernel), kThreads, 0, device);
  constexpr int kWarps = kThreads / kWarpSize;
  const int64_t grid =
      persistent_grid((a.num_tokens * a.parts + kWarps - 1) / kWarps, device, per_sm);
  a.early_dependents = early_dependents(
      a.num_tokens * head_dim * (4 * num_heads + 6 * num_kv_heads));
  return launch(kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, stream, 1u, a);
}

struct CacheReadArgs {
  uint8_t* out[2];          // K and V: [num_seqs, max_blocks * block_size, Hk, D] bf16
  const uint8_t* cache[2];  // [num_blocks, block_size, Hk, D]
  const uint8_t* scale[2];  // [num_blocks, block_size, Hk]
  const int32_t* block_tables;
  const int32_t* seq_lens;
  int64_t num_blocks;
  int64_t max_rows;  // max_blocks * block_size
  int64_t row_vecs;  // 16-byte vectors of codes in a cached row: Hk * D / 16
  int max_blocks;
  int block_size;
  int num_kv_heads;
  int head_vecs;  // D / 16
  int early_dependents;
  int* err;
};

// Four codes of a word times a power of two, as four bf16 values (exact).
__device__ __forceinline__ uint2 dequantise4(uint32_t w, float f) {
  const uint32_t l = e4m3_to_f16x2_lo(w), h = e4m3_to_f16x2_hi(w);
  float x[4];
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}"
      : "=f"(x[0]), "=f"(x[1])
      : "r"(l));
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}"
      : "=f"(x[2]), "=f"(x[3])
      : "r"(h));
  return make_uint2(pack_bf16x2(x[0] * f, x[1] * f), pack_bf16x2(x[2] * f, x[3] * f));
}

// A block takes one page of one request, K or V (blockIdx.y); a thread one 16-byte vector of codes
// at a time. Bound by memory: 1 byte and a scale's share read, 2 written per element.
__global__ void __launch_bounds__(kThreads) cache_read_kernel(
    const __grid_constant__ CacheReadArgs a) {
  grid_dependency_wait();
  if (a.early_dependents) allow_dependents();
  const int64_t page = blockIdx.x;
  const int64_t seq = page / a.max_blocks;
  const int64_t row0 = (page % a.max_blocks) * a.block_size;
  int64_t len = a.seq_lens[seq];
  if (len < 0 || len > a.max_rows) {
    if (threadIdx.x == 0) raise_error(a.err, kErrBadIndex);
    len = len < 0 ? 0 : a.max_rows;
  }
  const int64_t rows = min(static_cast<int64_t>(a.block_size), max(int64_t{0}, len - row0));
  int64_t blk = 0;
  if (rows > 0) {
    blk = a.block_tables[page];
    if (blk < 0 || blk >= a.num_blocks) {
      if (threadIdx.x == 0) raise_error(a.err, kErrBadIndex);
      blk = 0;
    }
  }
  const uint8_t* codes = a.cache[blockIdx.y] + blk * a.block_size * a.row_vecs * 16;
  const uint8_t* scale = a.scale[blockIdx.y] + blk * a.block_size * a.num_kv_heads;
  uint8_t* out = a.out[blockIdx.y] + page * a.block_size * a.row_vecs * 32;
  const int64_t live = rows * a.row_vecs, all = a.block_size * a.row_vecs;
  for (int64_t i = threadIdx.x; i < all; i += kThreads) {
    uint4 x0 = make_uint4(0, 0, 0, 0), x1 = x0;
    if (i < live) {
      const uint4 w = ld_global_nc_v4(codes + i * 16);
      const float f = scale_value(__ldg(scale + i / a.head_vecs));
      const uint2 d0 = dequantise4(w.x, f), d1 = dequantise4(w.y, f);
      const uint2 d2 = dequantise4(w.z, f), d3 = dequantise4(w.w, f);
      x0 = make_uint4(d0.x, d0.y, d1.x, d1.y);
      x1 = make_uint4(d2.x, d2.y, d3.x, d3.y);
    }
    st_global_v4(out + i * 32, x0);
    st_global_v4(out + i * 32 + 16, x1);
  }
}

}  // namespace
}  // namespace svllm::k

extern "C" int svllm_qk_norm_rope_cache_fp8_bf16(
    void* q, const void* k, const void* v, const void* q_weight, const void* k_weight,
    const void* positions, int pos_type, const int64_t* slot_mapping, void* k_cache, void* v_cache,
    void* k_scale, void* v_scale, int64_t num_slots, int64_t num_tokens, int64_t num_heads,
    int64_t num_kv_heads, int64_t head_dim, int64_t q_row_stride, int64_t k_row_stride,
    int64_t v_row_stride, float eps, const float* inv_freq, svllm_stream stream) {
  svllm::k::CacheWriteArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.positions = positions;
  a.slots = slot_mapping;
  a.k_cache = static_cast<uint8_t*>(k_cache);
  a.v_cache = static_cast<uint8_t*>(v_cache);
  a.k_scale = static_cast<uint8_t*>(k_scale);
  a.v_scale = static_cast<uint8_t*>(v_scale);
  a.num_tokens = num_tokens;
  a.q_stride = q_row_stride;
  a.k_stride = k_row_stride;
  a.v_stride = v_row_stride;
  a.num_slots = num_slots;
  a.eps = eps;
  return svllm::k::launch_cache_write(a, true, pos_type, num_heads, num_kv_heads, head_dim,
                                      inv_freq, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int svllm_rope_cache_fp8_bf16(
    void* q, const void* k, const void* v, const void* positions, int pos_type,
    const int64_t* slot_mapping, void* k_cache, void* v_cache, void* k_scale, void* v_scale,
    int64_t num_slots, int64_t num_tokens, int64_t num_heads, int64_t num_kv_heads,
    int64_t head_dim, int64_t q_row_stride, int64_t k_row_stride, int64_t v_row_stride,
    const float* inv_freq, svllm_stream stream) {
  svllm::k::CacheWriteArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.positions = positions;
  a.slots = slot_mapping;
  a.k_cache = static_cast<uint8_t*>(k_cache);
  a.v_cache = static_cast<uint8_t*>(v_cache);
  a.k_scale = static_cast<uint8_t*>(k_scale);
  a.v_scale = static_cast<uint8_t*>(v_scale);
  a.num_tokens = num_tokens;
  a.q_stride = q_row_stride;
  a.k_stride = k_row_stride;
  a.v_stride = v_row_stride;
  a.num_slots = num_slots;
  return svllm::k::launch_cache_write(a, false, pos_type, num_heads, num_kv_heads, head_dim,
                                      inv_freq, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int svllm_cache_read_fp8_bf16(void* k_out, void* v_out, const void* k_cache,
                                         const void* v_cache, const void* k_scale,
                                         const void* v_scale, int64_t num_blocks,
                                         int64_t block_size, const int32_t* block_tables,
                                         int64_t max_blocks, const int32_t* seq_lens,
                                         int64_t num_seqs, int64_t num_kv_heads, int64_t head_dim,
                                         svllm_stream stream) {
  using namespace svllm::k;
  if (num_seqs < 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || max_blocks < 0 ||
      num_blocks <= 0) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  if (num_seqs == 0 || max_blocks == 0) return SVLLM_OK;
  if (k_out == nullptr || v_out == nullptr || k_cache == nullptr || v_cache == nullptr ||
      k_scale == nullptr || v_scale == nullptr || block_tables == nullptr || seq_lens == nullptr) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  constexpr int64_t kInt = int64_t{1} << 31;
  if (num_kv_heads > (1 << 16) || block_size >= (int64_t{1} << 20) || max_blocks >= kInt ||
      num_seqs >= kInt || num_seqs * max_blocks >= kInt) {
    return SVLLM_ERR_TOO_LARGE;
  }
  if ((head_dim != 64 && head_dim != 128) || !aligned16(k_out) || !aligned16(v_out) ||
      !aligned16(k_cache) || !aligned16(v_cache)) {
    return SVLLM_ERR_UNSUPPORTED;
  }
  int device;
  if (current_device(&device) != SVLLM_OK) return SVLLM_ERR_CUDA;
  CacheReadArgs a{};
  a.err = library_error_word(device);
  if (a.err == nullptr) return SVLLM_ERR_CUDA;
  a.out[0] = static_cast<uint8_t*>(k_out);
  a.out[1] = static_cast<uint8_t*>(v_out);
  a.cache[0] = static_cast<const uint8_t*>(k_cache);
  a.cache[1] = static_cast<const uint8_t*>(v_cache);
  a.scale[0] = static_cast<const uint8_t*>(k_scale);
  a.scale[1] = static_cast<const uint8_t*>(v_scale);
  a.block_tables = block_tables;
  a.seq_lens = seq_lens;
  a.num_blocks = num_blocks;
  a.max_blocks = static_cast<int>(max_blocks);
  a.block_size = static_cast<int>(block_size);
  a.max_rows = max_blocks * block_size;
  a.num_kv_heads = static_cast<int>(num_kv_heads);
  a.head_vecs = static_cast<int>(head_dim / 16);
  a.row_vecs = num_kv_heads * a.head_vecs;
  a.early_dependents = early_dependents(num_seqs * a.max_rows * a.row_vecs * 96);
  return launch(cache_read_kernel, dim3(static_cast<unsigned>(num_seqs * max_blocks), 2),
                dim3(kThreads), 0, reinterpret_cast<cudaStream_t>(stream), 1u, a);
}
