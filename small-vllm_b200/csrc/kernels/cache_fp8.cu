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
// The bound is memory: per token 4 Hq D + 4 Hk D bytes of bf16 and 2 Hk (D + 1) of cache. Measured on
// a B200 (us in a graph; in brackets the bytes at the copy rate): 16/8 heads of 128, 1 token 2.3, 256
// tokens 3.5 (0.6), 65536 tokens 146-151 (146); 24/8 heads of 64, 5003 tokens 8.9 (7.2). Small batches
// are a launch and three trips to memory. 65536 tokens took 197 with loads to registers and 209 with
// the first ring of bulk copies; since then positions and slots are loaded a token ahead, no head has
// a branch (a token with a value that is not finite is done again at its end), the norm's weights are
// folded into the rotation once a token, and fp32 values are worked on in pairs.
//
// svllm_cache_read_fp8_bf16: the rows of whole requests back in bf16 (exact), as pages in the
// order of the request: [num_seqs, max_blocks * block_size, Hk, D], zeros behind a request's end. 32
// requests of 4183 to 8192 rows 225 us (230 at the copy rate); one page a block took 272.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>
#include <type_traits>

#include "common.cuh"
#include "fp8.cuh"
#include "host_common.h"

namespace svllm::k {
namespace {

constexpr int kMaxHalf = 64;  // head_dim 64 or 128
constexpr int kThreads = 256;
constexpr int kBulkWarps = 12, kBulkMinWarps = 4;
// A third stage takes from middling batches what it gives large ones (us with two and three, 16/8 heads
// of 128: 5003 tokens 18.0, 19.6; 65536 151.4, 147.1).
constexpr int kBulkStages = 2;
// More passes than so many per SM take the bulk kernel (us direct and bulk, 16/8 heads of 128: 256
// tokens 3.6, 4.5; 400 5.4, 4.5; 1184 9.1, 5.0; 24/8 of 64: 400 2.6, 3.3; 600 3.6, 3.4; 1184 4.5, 3.5).
constexpr int kDirectPassesPerSm = 16;
constexpr int64_t kBulkSmem = 210 * 1024;
constexpr int kReadVecs = 4;  // 16-code vectors a thread of the read-back takes

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

// 256 bits, which is what 16 codes become.
__device__ __forceinline__ void st_global_v8(void* p, const uint4& x, const uint4& y) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(x.x),
               "r"(x.y), "r"(x.z), "r"(x.w), "r"(y.x), "r"(y.y), "r"(y.z), "r"(y.w)
               : "memory");
}

template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
  for (int offset = G / 2; offset > 0; offset /= 2) {
    v = max(v, __shfl_xor_sync(0xffffffffu, v, offset));
  }
  return v;
}

// The larger magnitude's bits; a NaN is larger than any number.
__device__ __forceinline__ float max_abs_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(fabsf(a)), "f"(fabsf(b)));
  return d;
}

// A lane's 8 + 8 elements of a head as packed fp32 pairs: word i of each half.
struct Pairs {
  uint64_t lo[4], hi[4];
  __device__ __forceinline__ void unpack(const uint4& l, const uint4& h) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t wl = word(l, i), wh = word(h, i);
      lo[i] = f32x2(__uint_as_float(wl << 16), __uint_as_float(wl & 0xffff0000u));
      hi[i] = f32x2(__uint_as_float(wh << 16), __uint_as_float(wh & 0xffff0000u));
    }
  }
};

// What turns a lane's elements of a head, the norm's weights included:
//   y_lo = inv (x_lo a + x_hi b),  y_hi = inv (x_hi c + x_lo d)
// with a = w_lo cos, b = -w_hi sin, c = w_hi cos, d = w_lo sin. Worked out once for all heads of a
// token that share the weights.
struct Turn {
  uint64_t a[4], b[4], c[4], d[4];

  // cs, sn: the token's cosines and sines of this lane's eight pairs, in shared memory
  template <bool kNorm>
  __device__ __forceinline__ void set(const float* cs, const float* sn, const uint4& w_lo,
                                      const uint4& w_hi) {
    Pairs w;
    if constexpr (kNorm) w.unpack(w_lo, w_hi);
    const uint64_t minus = f32x2(-1.0f, -1.0f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 c4 = reinterpret_cast<const float4*>(cs)[i];
      const float4 s4 = reinterpret_cast<const float4*>(sn)[i];
      const uint64_t cc[2] = {f32x2(c4.x, c4.y), f32x2(c4.z, c4.w)};
      const uint64_t ss[2] = {f32x2(s4.x, s4.y), f32x2(s4.z, s4.w)};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int n = 2 * i + e;
        const uint64_t neg = f32x2_mul(ss[e], minus);
        if constexpr (kNorm) {
          a[n] = f32x2_mul(w.lo[n], cc[e]);
          b[n] = f32x2_mul(w.hi[n], neg);
          c[n] = f32x2_mul(w.hi[n], cc[e]);
          d[n] = f32x2_mul(w.lo[n], ss[e]);
        } else {
          a[n] = c[n] = cc[e];
          b[n] = neg;
          d[n] = ss[e];
        }
      }
    }
  }

  // x turned in place; returns inv (1 without norms), which is left to the caller: it goes with
  // what follows.
  template <int D, bool kNorm>
  __device__ __forceinline__ float apply(Pairs& x, float eps) const {
    float inv = 1.0f;
    if constexpr (kNorm) {
      uint64_t sum = f32x2_mul(x.lo[0], x.lo[0]);
      sum = f32x2_fma(x.hi[0], x.hi[0], sum);
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        sum = f32x2_fma(x.lo[i], x.lo[i], sum);
        sum = f32x2_fma(x.hi[i], x.hi[i], sum);
      }
      float s0, s1;
      f32x2_split(sum, s0, s1);
      inv = rsqrtf(group_sum<D / 16>(s0 + s1) * (1.0f / D) + eps);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t lo = f32x2_fma(x.lo[i], a[i], f32x2_mul(x.hi[i], b[i]));
      x.hi[i] = f32x2_fma(x.hi[i], c[i], f32x2_mul(x.lo[i], d[i]));
      x.lo[i] = lo;
    }
    return inv;
  }
};

// inv times a lane's turned elements as bf16.
__device__ __forceinline__ uint4 round_half(const uint64_t (&x)[4], float inv) {
  const uint64_t inv2 = f32x2(inv, inv);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    f32x2_split(f32x2_mul(x[i], inv2), a, b);
    w[i] = pack_bf16x2(a, b);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// f times a lane's elements as codes.
__device__ __forceinline__ uint2 code_half(const uint64_t (&x)[4], float f) {
  const uint64_t f2 = f32x2(f, f);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    f32x2_split(f32x2_mul(x[i], f2), a, b);
    w[i] = pack_e4m3x2(a, b);
  }
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// Infinities and NaN of a head become NaN, which turns into the NaN code, and do not count for the
// maximum: that of the lane's others.
__device__ __forceinline__ uint32_t drop_non_finite(uint64_t (&x)[4]) {
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[2];
    f32x2_split(x[i], v[0], v[1]);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (isfinite(v[e])) amax = max(amax, __float_as_uint(v[e]) & 0x7fffffffu);
      else v[e] = __int_as_float(0x7fffffff);
    }
    x[i] = f32x2(v[0], v[1]);
  }
  return amax;
}

// inv times a head's elements x into the cache row `row` (slot * heads + head): codes and scale.
// amax_bits: the largest magnitude of inv x in this lane, in fp32 bits. Every lane of the warp
// calls; `write` where the head exists. kCareful: the head may hold values that are not finite;
// without it such a head's row is wrong, and the return value tells.
template <int D, bool kCareful>
__device__ __forceinline__ bool quantise(Pairs& x, float inv, uint32_t amax_bits, bool write,
                                         int64_t row, uint8_t* cache, uint8_t* scales, int sub) {
  amax_bits = group_max<D / 16>(amax_bits);
  const bool odd = amax_bits >= 0x7f800000u;
  if constexpr (kCareful) {
    const uint64_t inv2 = f32x2(inv, inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x.lo[i] = f32x2_mul(x.lo[i], inv2);
      x.hi[i] = f32x2_mul(x.hi[i], inv2);
    }
    inv = 1.0f;
    amax_bits = max(drop_non_finite(x.lo), drop_non_finite(x.hi));
    amax_bits = group_max<D / 16>(amax_bits);
  }
  const int e = scale_exponent(amax_bits);
  const float f = inv * exp2_int(-e);
  const uint2 lo = code_half(x.lo, f), hi = code_half(x.hi, f);
  if (write) {
    uint8_t* codes = cache + row * D;
    *reinterpret_cast<uint2*>(codes + 8 * sub) = lo;
    *reinterpret_cast<uint2*>(codes + D / 2 + 8 * sub) = hi;
    if (sub == 0) scales[row] = static_cast<uint8_t>(e + kScaleBias);
  }
  return odd && write;
}

// The three kinds of heads; hl, hh: a lane's two vectors of the head.
template <int D, bool kNorm, bool kAligned>
__device__ __forceinline__ void write_q(const CacheWriteArgs& a, const Turn& turn, const uint4& hl,
                                        const uint4& hh, int64_t t, int h, int sub) {
  Pairs x;
  x.unpack(hl, hh);
  const float inv = turn.apply<D, kNorm>(x, a.eps);
  if (h >= a.num_heads) return;
  uint8_t* row = static_cast<uint8_t*>(a.q) + (t * a.q_stride + int64_t{h} * D) * 2;
  store8<kAligned>(row + 16 * sub, round_half(x.lo, inv));
  store8<kAligned>(row + D + 16 * sub, round_half(x.hi, inv));
}

template <int D, bool kNorm, bool kCareful>
__device__ __forceinline__ bool write_k(const CacheWriteArgs& a, const Turn& turn, const uint4& hl,
                                        const uint4& hh, int64_t slot, int h, int sub) {
  Pairs x;
  x.unpack(hl, hh);
  const float inv = turn.apply<D, kNorm>(x, a.eps);
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float l0, l1, h0, h1;
    f32x2_split(x.lo[i], l0, l1);
    f32x2_split(x.hi[i], h0, h1);
    amax = max_abs_nan(amax, max_abs_nan(max_abs_nan(l0, l1), max_abs_nan(h0, h1)));
  }
  // rounding is monotone, so inv times the largest is the largest of the products
  return quantise<D, kCareful>(x, inv, __float_as_uint(amax * inv) & 0x7fffffffu,
                               h < a.num_kv_heads, slot * a.num_kv_heads + h, a.k_cache, a.k_scale,
                               sub);
}

template <int D, bool kCareful>
__device__ __forceinline__ bool write_v(const CacheWriteArgs& a, const uint4& hl, const uint4& hh,
                                        int64_t slot, int h, int sub) {
  uint32_t amax = 0;  // two at a time: magnitudes of bf16 are ordered as whole numbers
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    amax = __vmaxu2(amax, __vmaxu2(word(hl, i) & 0x7fff7fffu, word(hh, i) & 0x7fff7fffu));
  }
  Pairs x;
  x.unpack(hl, hh);
  return quantise<D, kCareful>(x, 1.0f, max(amax << 16, amax & 0xffff0000u), h < a.num_kv_heads,
                               slot * a.num_kv_heads + h, a.v_cache, a.v_scale, sub);
}

// The (cos, sin) of a token's D / 2 pairs into a warp's shared memory: `turns` half turns per
// position of the pairs lane, lane + 32, ..., reduced in fp64 to [-1, 1].
template <int D>
__device__ __forceinline__ void trig_of(int64_t position, const double (&turns)[D / 64], float* cs,
                                        float* sn) {
  const int lane = threadIdx.x % kWarpSize;
  const double pos = static_cast<double>(position);
  __syncwarp();  // the token before has been read
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const double x = pos * turns[i];
    sincospif(static_cast<float>(fma(-2.0, rint(0.5 * x), x)), sn + lane + i * kWarpSize,
              cs + lane + i * kWarpSize);
  }
  __syncwarp();
}

template <int D>
__device__ __forceinline__ void half_turns(const CacheWriteArgs& a, double (&turns)[D / 64]) {
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    turns[i] = static_cast<double>(a.inv_freq[threadIdx.x % kWarpSize + i * kWarpSize]) *
               0.31830988618379067154;  // 1 / pi
  }
}

// This lane's block of each half of q's and k's norm weights.
template <int D, bool kNorm, bool kAligned>
__device__ __forceinline__ void load_weights(const CacheWriteArgs& a, int sub, uint4 (&w)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = make_uint4(0, 0, 0, 0);
    if constexpr (kNorm) {
      const void* p = i < 2 ? a.q_weight : a.k_weight;
      w[i] = load8<kAligned>(static_cast<const uint8_t*>(p) + (i % 2 * (D / 2) + 8 * sub) * 2);
    }
  }
}

__device__ __forceinline__ int64_t position_of(const CacheWriteArgs& a, int64_t t) {
  return a.pos_is_i64 ? __ldg(static_cast<const long long*>(a.positions) + t)
                      : __ldg(static_cast<const int*>(a.positions) + t);
}

__device__ __forceinline__ int64_t slot_of(const CacheWriteArgs& a, int64_t t) {
  return __ldg(reinterpret_cast<const long long*>(a.slots) + t);
}

// A token's slot, negative for "write no cache"; one past the cache raises the error word.
__device__ __forceinline__ int64_t checked_slot(const CacheWriteArgs& a, int64_t slot) {
  if (slot >= a.num_slots) {
    if (threadIdx.x % kWarpSize == 0) raise_error(a.err, kErrBadIndex);
    slot = -1;
  }
  return slot;
}

// Both kernels deal heads to passes of 32 / G, G = D / 16 lanes a head; lane j of a head holds
// elements [8j, 8j + 8) and the matching ones of the second half, so that every rotation pair is in
// one lane. The passes of q come first, then those of k, then of v.

// Few tokens, and rows off 16 bytes: a warp takes a pass, straight from global memory, so that a
// token's chains run side by side.
template <int D, bool kNorm, bool kAligned>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(
    const __grid_constant__ CacheWriteArgs a) {
  grid_dependency_wait();
  if (a.early_dependents) allow_dependents();
  constexpr int G = D / 16;
  constexpr int kHeads = kWarpSize / G;
  __shared__ __align__(16) float trig[kThreads / kWarpSize][2][D / 2];
  const int warp = threadIdx.x / kWarpSize, lane = threadIdx.x % kWarpSize;
  const int sub = lane % G;
  const int q_passes = (a.num_heads + kHeads - 1) / kHeads;
  const int k_passes = (a.num_kv_heads + kHeads - 1) / kHeads;
  const int passes = q_passes + 2 * k_passes;
  double turns[D / 64];
  half_turns<D>(a, turns);
  uint4 weight[4];
  load_weights<D, kNorm, kAligned>(a, sub, weight);

  const int64_t units = a.num_tokens * passes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / kWarpSize);
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (kThreads / kWarpSize) + warp; u < units;
       u += step) {
    const int64_t t = u / passes;
    const int pass = static_cast<int>(u - t * passes);
    const int kind = pass < q_passes ? 0 : pass < q_passes + k_passes ? 1 : 2;
    const int64_t slot = kind == 0 ? 0 : checked_slot(a, slot_of(a, t));
    if (slot < 0) continue;
    const int h = (pass - (kind == 0 ? 0 : q_passes + (kind - 1) * k_passes)) * kHeads + lane / G;
    const uint8_t* row = static_cast<const uint8_t*>(kind == 0 ? a.q : kind == 1 ? a.k : a.v) +
                         (t * (kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride) +
                          int64_t{h} * D) * 2;
    uint4 hl = make_uint4(0, 0, 0, 0), hh = hl;
    if (h < (kind == 0 ? a.num_heads : a.num_kv_heads)) {
      hl = load8<kAligned>(row + 16 * sub);
      hh = load8<kAligned>(row + D + 16 * sub);
    }
    if (kind == 2) {
      if (__any_sync(0xffffffffu, write_v<D, false>(a, hl, hh, slot, h, sub))) {
        write_v<D, true>(a, hl, hh, slot, h, sub);
      }
      continue;
    }
    trig_of<D>(position_of(a, t), turns, trig[warp][0], trig[warp][1]);
    Turn turn;
    turn.set<kNorm>(&trig[warp][0][8 * sub], &trig[warp][1][8 * sub],
                    kind == 0 ? weight[0] : weight[2], kind == 0 ? weight[1] : weight[3]);
    if (kind == 0) {
      write_q<D, kNorm, kAligned>(a, turn, hl, hh, t, h, sub);
    } else if (__any_sync(0xffffffffu, write_k<D, kNorm, false>(a, turn, hl, hh, slot, h, sub))) {
      write_k<D, kNorm, true>(a, turn, hl, hh, slot, h, sub);
    }
  }
}

// Many tokens: a warp takes whole tokens, whose q, k and v rows bulk copies bring into a ring of
// stages that the warp owns (a token ahead, without registers held for it). cos and sin and what
// becomes of them with the weights (Turn) are worked out once a token.
template <int D, bool kNorm>
__global__ void __launch_bounds__(kBulkWarps * kWarpSize, 1) cache_write_bulk_kernel(
    const __grid_constant__ CacheWriteArgs a) {
  grid_dependency_wait();
  if (a.early_dependents) allow_dependents();
  constexpr int G = D / 16;
  constexpr int kHeads = kWarpSize / G;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(16) float trig[kBulkWarps][2][D / 2];
  __shared__ uint64_t bars[kBulkWarps][kBulkStages];
  const int warps = blockDim.x / kWarpSize;
  const int warp = threadIdx.x / kWarpSize, lane = threadIdx.x % kWarpSize;
  const int sub = lane % G;
  const uint32_t q_bytes = static_cast<uint32_t>(a.num_heads) * D * 2;
  const uint32_t k_bytes = static_cast<uint32_t>(a.num_kv_heads) * D * 2;
  const uint32_t stage_bytes = q_bytes + 2 * k_bytes;
  uint8_t* ring = smem + static_cast<size_t>(warp) * kBulkStages * stage_bytes;
  if (lane == 0) {
    for (int s = 0; s < kBulkStages; ++s) mbar_init(&bars[warp][s], 1);
    fence_mbar_init();
  }
  double turns[D / 64];
  half_turns<D>(a, turns);
  uint4 weight[4];
  load_weights<D, kNorm, true>(a, sub, weight);
  __syncwarp();

  const WarpUnits wu =
      warp_units(a.num_tokens, static_cast<int64_t>(gridDim.x) * warps,
                 static_cast<int64_t>(blockIdx.x) * warps + warp, true);
  const auto issue = [&](int64_t j) {
    const int s = static_cast<int>(j % kBulkStages);
    uint8_t* st = ring + s * stage_bytes;
    const int64_t t = wu.at(j);
    mbar_arrive_expect_tx(&bars[warp][s], stage_bytes);
    if (q_bytes) {
      bulk_load(st, static_cast<const uint8_t*>(a.q) + t * a.q_stride * 2, q_bytes, &bars[warp][s]);
    }
    bulk_load(st + q_bytes, static_cast<const uint8_t*>(a.k) + t * a.k_stride * 2, k_bytes,
              &bars[warp][s]);
    bulk_load(st + q_bytes + k_bytes, static_cast<const uint8_t*>(a.v) + t * a.v_stride * 2,
              k_bytes, &bars[warp][s]);
  };
  if (lane == 0) {
    for (int64_t j = 0; j < min(static_cast<int64_t>(kBulkStages), wu.count); ++j) issue(j);
  }
  // a token's position and slot are loaded while the one before it is worked on
  int64_t position = 0, slot = -1;
  if (wu.count > 0) {
    position = position_of(a, wu.at(0));
    slot = slot_of(a, wu.at(0));
  }
  int64_t j = 0;
  for (; j < wu.count; ++j) {
    const int64_t t = wu.at(j);
    const int64_t this_slot = checked_slot(a, slot), this_position = position;
    if (j + 1 < wu.count) {
      position = position_of(a, wu.at(j + 1));
      slot = slot_of(a, wu.at(j + 1));
    }
    trig_of<D>(this_position, turns, trig[warp][0], trig[warp][1]);
    const int s = static_cast<int>(j % kBulkStages);
    const uint32_t parity = static_cast<uint32_t>((j / kBulkStages) & 1);
    if (!__all_sync(0xffffffffu, mbar_wait_bounded(&bars[warp][s], parity))) break;
    const uint8_t* st = ring + s * stage_bytes + (lane / G) * (D * 2) + 16 * sub;
    Turn turn;
    turn.set<kNorm>(&trig[warp][0][8 * sub], &trig[warp][1][8 * sub], weight[0], weight[1]);
    // (a pass that reads past the last head stays within the token's rows, or within the ring:
    // the launch leaves a pass's room behind it)
#pragma unroll 4
    for (int h0 = 0; h0 < a.num_heads; h0 += kHeads) {
      const uint8_t* p = st + h0 * (D * 2);
      write_q<D, kNorm, true>(a, turn, ld_shared_v4(p), ld_shared_v4(p + D), t, h0 + lane / G, sub);
    }
    if (this_slot >= 0) {
      if constexpr (kNorm) {
        turn.set<kNorm>(&trig[warp][0][8 * sub], &trig[warp][1][8 * sub], weight[2], weight[3]);
      }
      const auto write_kv = [&](auto careful) {
        constexpr bool kCareful = decltype(careful)::value;
        bool odd = false;
#pragma unroll 2
        for (int h0 = 0; h0 < a.num_kv_heads; h0 += kHeads) {
          const uint8_t* p = st + q_bytes + h0 * (D * 2);
          const uint8_t* pv = p + k_bytes;
          odd |= write_k<D, kNorm, kCareful>(a, turn, ld_shared_v4(p), ld_shared_v4(p + D),
                                             this_slot, h0 + lane / G, sub);
          odd |= write_v<D, kCareful>(a, ld_shared_v4(pv), ld_shared_v4(pv + D), this_slot,
                                      h0 + lane / G, sub);
        }
        return odd;
      };
      if (__any_sync(0xffffffffu, write_kv(std::false_type{}))) write_kv(std::true_type{});
    }
    __syncwarp();
    if (lane == 0 && j + kBulkStages < wu.count) {
      fence_proxy_async_smem();
      issue(j + kBulkStages);
    }
  }
  if (j < wu.count) {  // a copy did not land: wait for the others in flight, within the limit
    if (lane == 0) {
      raise_error(a.err, kErrWaitTimeout);
      for (int64_t m = j; m < min(j + kBulkStages, wu.count); ++m) {
        mbar_wait_bounded(&bars[warp][m % kBulkStages],
                          static_cast<uint32_t>((m / kBulkStages) & 1));
      }
    }
    __syncwarp();
  }
}

// The bulk kernel's warps: eight or twelve, as far as their rings fit. An SM takes its tokens in rounds
// of one a warp, and a round lasts as long as its bytes or as a warp's chain over a token, which is
// counted in the bytes that pass meanwhile (a pass of k and v costs three of q: maxima and codes; the
// norms cost a third). The form with the smaller sum is taken. Past kFewTokens an SM the rings stream,
// which twelve warps do 12-17% slower, so their sum has to be smaller by as much. us with eight and with
// twelve warps, by the tokens an SM:
//   6/2 heads of 64, norms:    9: 4.1, 3.1   16: 4.2, 4.6    36: 8.1, 6.1     443: 84.6, 65.4
//   24/8 of 64:                9: 4.7, 3.8   16: 5.0, 5.7    36: 11.1, 9.5    443: 95.5, 108.0
//   8/8 of 128, norms:         9: 6.5, 5.3   16: 7.0, 8.2    40: 16.1, 16.7   443: 130.8, 106.0
//   8/8 of 128:               11: 5.9, 4.8   15: 5.9, 7.2    45: 16.0, 15.5   443: 108.7, 123.9
//   16/8 of 128, norms:        9: 7.2, 6.0   16: 7.6, 9.3    40: 18.3, 19.9   443: 151.7, 172.1
//   32/4 of 128, norms (ten):  9: 7.7, 5.7   16: 8.5, 10.3   20: 12.8, 11.9   443: 224.5, 230.8
// Over 587 such pairs of 26 layouts, 136 of them timed after the rule was set, the choice costs at most
// 8% against the better of the two.
int bulk_warps(int64_t per_sm, int64_t bytes, int64_t q_passes, int64_t kv_passes, bool norm,
               int64_t fit) {
  if (fit <= 8) return static_cast<int>(fit);
  constexpr int64_t kChainStart = 40 * 1024, kFewTokens = 64;
  const int64_t chain = kChainStart + (norm ? 8 : 6) * 1024 * (q_passes + 3 * kv_passes);
  const auto sum = [&](int64_t warps) {
    return (per_sm + warps - 1) / warps * (warps * bytes > chain ? warps * bytes : chain);
  };
  const int64_t many = fit < kBulkWarps ? fit : kBulkWarps;
  const bool better =
      per_sm <= kFewTokens ? sum(many) < sum(8) : 23 * sum(many) < 20 * sum(8);
  return static_cast<int>(better ? many : 8);
}

using WriteKernel = void (*)(CacheWriteArgs);

template <int D, bool kNorm>
int launch_write(const CacheWriteArgs& a, bool aligned, int device, cudaStream_t stream) {
  constexpr int kHeads = kWarpSize / (D / 16);
  const int64_t token_bytes = (a.num_heads + 2 * int64_t{a.num_kv_heads}) * D * 2;
  const int64_t passes = (a.num_heads + kHeads - 1) / kHeads +
                         2 * ((a.num_kv_heads + kHeads - 1) / kHeads);
  const WriteKernel bulk = cache_write_bulk_kernel<D, kNorm>;
  // as many warps as their rings fit (a pass of the last stage may read a pass's bytes past it)
  constexpr int64_t kPassBytes = kHeads * D * 2;
  const int64_t fit = (kBulkSmem - kPassBytes) / (kBulkStages * token_bytes);
  const int64_t kv_passes = (a.num_kv_heads + kHeads - 1) / kHeads;
  const int warps = bulk_warps((a.num_tokens + sm_count(device) - 1) / sm_count(device),
                               (4 * int64_t{a.num_heads} + 6 * int64_t{a.num_kv_heads}) * D,
                               passes - 2 * kv_passes, kv_passes, kNorm, fit);
  if (aligned && a.num_tokens * passes > int64_t{kDirectPassesPerSm} * sm_count(device) &&
      warps >= kBulkMinWarps) {
    const size_t smem = static_cast<size_t>(warps * kBulkStages * token_bytes + kPassBytes);
    const int ctas = blocks_per_sm(reinterpret_cast<const void*>(bulk), warps * kWarpSize, smem,
                                   device);
    if (ctas <= 0) return SVLLM_ERR_CUDA;
    const int64_t grid = persistent_grid((a.num_tokens + warps - 1) / warps, device, ctas);
    return launch(bulk, dim3(static_cast<unsigned>(grid)), dim3(warps * kWarpSize), smem, stream,
                  1u, a);
  }
  const WriteKernel kernel =
      aligned ? cache_write_kernel<D, kNorm, true> : cache_write_kernel<D, kNorm, false>;
  const int ctas = blocks_per_sm(reinterpret_cast<const void*>(kernel), kThreads, 0, device);
  if (ctas <= 0) return SVLLM_ERR_CUDA;
  constexpr int kWarps = kThreads / kWarpSize;
  const int64_t grid =
      persistent_grid((a.num_tokens * passes + kWarps - 1) / kWarps, device, ctas);
  return launch(kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, stream, 1u, a);
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
  a.early_dependents = early_dependents(
      a.num_tokens * head_dim * (4 * num_heads + 6 * num_kv_heads));
  return head_dim == 128 ? (norm ? launch_write<128, true>(a, aligned, device, stream)
                                 : launch_write<128, false>(a, aligned, device, stream))
                         : (norm ? launch_write<64, true>(a, aligned, device, stream)
                                 : launch_write<64, false>(a, aligned, device, stream));
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
  int head_shift;  // of a vector's index to its head's: log2(D / 16)
  int runs;        // blocks of a request
  Divider page;    // by the block size
  Divider by_row;  // by the vectors of a row
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

// A block takes a run of rows of a request, K or V (blockIdx.y); a thread 16 codes of a row at a
// time, kReadVecs of them in flight: the length, the table's entries and the codes are each loaded
// for all before the first is used. Bound by memory: 1 byte and a scale's share read, 2 written per
// element.
__global__ void __launch_bounds__(kThreads) cache_read_kernel(
    const __grid_constant__ CacheReadArgs a) {
  grid_dependency_wait();
  if (a.early_dependents) allow_dependents();
  const int64_t seq = blockIdx.x / a.runs;
  const int64_t run = blockIdx.x - seq * a.runs;
  const int64_t first = run * (kThreads * kReadVecs);  // vector of the request
  const int64_t all = a.max_rows * a.row_vecs;
  int64_t len = __ldg(a.seq_lens + seq);
  const int32_t* table = a.block_tables + seq * a.max_blocks;
  const uint8_t* cache = a.cache[blockIdx.y];
  const uint8_t* scales = a.scale[blockIdx.y];
  uint8_t* out = a.out[blockIdx.y] + seq * all * 32;
  int64_t blk[kReadVecs];
  int row[kReadVecs], vec[kReadVecs], in_page[kReadVecs];
#pragma unroll
  for (int i = 0; i < kReadVecs; ++i) {
    const int64_t v = first + i * kThreads + threadIdx.x;
    row[i] = vec[i] = in_page[i] = 0;
    blk[i] = 0;
    if (v < all) {
      row[i] = static_cast<int>(a.by_row.divide(static_cast<int>(v)));
      vec[i] = static_cast<int>(v) - row[i] * static_cast<int>(a.row_vecs);
      const int page = a.page.divide(row[i]);
      in_page[i] = row[i] - page * a.block_size;
      blk[i] = __ldg(table + page);
    }
  }
  if (len < 0 || len > a.max_rows) {
    if (threadIdx.x == 0 && run == 0) raise_error(a.err, kErrBadIndex);
    len = len < 0 ? 0 : a.max_rows;
  }
  uint4 codes[kReadVecs];
  uint32_t scale[kReadVecs];
#pragma unroll
  for (int i = 0; i < kReadVecs; ++i) {
    codes[i] = make_uint4(0, 0, 0, 0);
    scale[i] = kScaleBias;
    const int64_t v = first + i * kThreads + threadIdx.x;
    if (v < all && row[i] < len) {
      if (blk[i] < 0 || blk[i] >= a.num_blocks) {
        raise_error(a.err, kErrBadIndex);  // an entry outside the cache: read block 0
        blk[i] = 0;
      }
      const int64_t slot = blk[i] * a.block_size + in_page[i];
      codes[i] = ld_global_nc_v4(cache + (slot * a.row_vecs + vec[i]) * 16);
      scale[i] = __ldg(scales + slot * a.num_kv_heads + (vec[i] >> a.head_shift));
    }
  }
#pragma unroll
  for (int i = 0; i < kReadVecs; ++i) {
    const int64_t v = first + i * kThreads + threadIdx.x;
    if (v >= all) break;
    const uint32_t used = scale_in_range(scale[i]);
    if (used != scale[i]) raise_error(a.err, kErrBadIndex);
    const float f = scale_value(used);
    const uint2 d0 = dequantise4(codes[i].x, f), d1 = dequantise4(codes[i].y, f);
    const uint2 d2 = dequantise4(codes[i].z, f), d3 = dequantise4(codes[i].w, f);
    st_global_v8(out + v * 32, make_uint4(d0.x, d0.y, d1.x, d1.y),
                 make_uint4(d2.x, d2.y, d3.x, d3.y));
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
  const auto aligned32 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; };
  if ((head_dim != 64 && head_dim != 128) || !aligned32(k_out) || !aligned32(v_out) ||
      !aligned16(k_cache) || !aligned16(v_cache)) {
    return SVLLM_ERR_UNSUPPORTED;
  }
  const int64_t head_vecs = head_dim / 16;
  if (num_kv_heads > (1 << 16) || block_size >= (int64_t{1} << 20) || max_blocks >= kInt ||
      num_seqs >= kInt || max_blocks * block_size >= kInt ||
      max_blocks * block_size * num_kv_heads * head_vecs >= kInt ||
      // blocks of the launch
      num_seqs * (max_blocks * block_size * num_kv_heads * head_vecs / (kThreads * kReadVecs) + 1) >=
          kInt) {
    return SVLLM_ERR_TOO_LARGE;
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
  a.head_shift = head_dim == 128 ? 3 : 2;
  a.row_vecs = num_kv_heads * head_vecs;
  a.page = make_divider(block_size);
  a.by_row = make_divider(a.row_vecs);
  constexpr int64_t kRun = kThreads * kReadVecs;
  const int64_t runs = (a.max_rows * a.row_vecs + kRun - 1) / kRun;
  a.runs = static_cast<int>(runs);
  a.early_dependents = early_dependents(num_seqs * a.max_rows * a.row_vecs * 96);
  return launch(cache_read_kernel, dim3(static_cast<unsigned>(num_seqs * runs), 2),
                dim3(kThreads), 0, reinterpret_cast<cudaStream_t>(stream), 1u, a);
}
