// Decode attention over the 8-bit paged KV cache (its format: fp8.cuh): one query token per request,
// up to eight query heads of a KV head served by one pass over that head's cached rows.
//
//   o[b, h] = sum_j p_j 2^ev_j vc_j / sum_j p_j,  p_j = exp(scale * 2^ek_j * q[b, h] . kc_j)
//
// over j < seq_lens[b], with kc_j, vc_j the codes and ek_j, ev_j the scales' exponents of the row
// at slot block_tables[b][j / block_size] * block_size + j % block_size.
//
// The products run on the tensor cores in f16 (mma.sync m16n8k16, fp32 accumulators): every e4m3
// code is an f16 number, so converting costs one instruction for two codes and nothing in
// precision. The other operands are made to fit f16's range by powers of two: q of each head is
// scaled so that its largest magnitude lies in [2^14, 2^15) (exact for all elements down to 2^-32
// of it), and the weights are w_j = 2^(y_j - m + 14) with y_j = x_j + ev_j, x_j the score in base
// 2 and m the running maximum of y_j, so w_j <= 2^14 and the smallest f16 stands for 2^-38 of the
// largest weight. The rows' scales thus never touch the codes: 2^ek multiplies a score, ev adds to
// it (in the one rounding of an fma), and the denominator is l = sum_j w_j 2^-ev_j, in fp32. (The
// weights are taken from y and p from them, not the other way round: at scores so large that x + ev
// rounds, both then carry the same error, and no weight passes 2^14.) The weights are rounded to
// f16 (2^-11 of each, an eighth of a bf16 rounding) because the product takes no wider operand.
//
// Layout. A warp takes steps of 32 cached rows, lane = 4 g + t:
//   S^T[16 rows x 8 heads] = K[16 x D] . Q^T[D x 8]: lane loads rows g, g + 8 of K, 16 bytes at
//     64 c + 16 t of piece c; a 4-byte word of it is one k-step (the same permutation of the
//     head dimension on both sides);
//   O^T[D x 8] += V^T[D x 16 rows] . P^T[16 x 8]: lane loads rows 2t, 2t + 1, 2t + 8, 2t + 9 of V,
//     D / 8 bytes at g * D / 8. V's transpose is two byte permutations of a word of two rows, which
//     pair their codes before the conversion; P^T comes from S^T by movmatrix.
// A CTA takes one (request, KV head, group of up to eight query heads) and a split of the rows;
// its warps share the split. The splits of one such item form a thread-block cluster that merges
// its (max, sum, partial output) through distributed shared memory.
#include <cuda_runtime.h>

#include <cfloat>
#include <cmath>
#include <cstdint>

#include "common.cuh"
#include "fp8.cuh"
#include "host_common.h"

namespace svllm::k {
namespace {

constexpr int kMaxSplits = 8;    // the portable cluster size
constexpr int kStepRows = 32;    // cached rows a warp takes at a time
constexpr int kGroup = 8;        // query heads of a CTA: the N of the products
constexpr float kWeightBits = 14.0f;  // weights reach 2^14, so that f16 keeps small ones

struct AttnArgs {
  void* out;      // [num_seqs, num_heads, D] bf16, contiguous
  const void* q;  // [num_seqs, num_heads, D] bf16, token stride q_stride
  const uint8_t* k_cache;  // [num_blocks, block_size, num_kv_heads, D]
  const uint8_t* v_cache;
  const uint8_t* k_scale;  // [num_blocks, block_size, num_kv_heads]
  const uint8_t* v_scale;
  const int32_t* block_tables;  // [num_seqs, max_blocks]
  const int32_t* seq_lens;      // [num_seqs]
  int64_t q_stride;
  int64_t num_blocks;
  int max_blocks;
  int max_rows;  // max_blocks * block_size
  int block_size;
  Divider page;  // by the block size
  int num_heads;
  int num_kv_heads;
  int group;   // query heads per KV head
  int groups;  // CTAs they are dealt to
  int splits;
  float scale_log2;
  int* err;
};

__device__ __forceinline__ uint32_t transpose8x8_b16(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// This lane's bytes of a V row: 16 at D = 128, 8 at D = 64.
template <int D>
struct VPart {
  uint32_t w[D / 32];
  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (D == 128) {
      const uint4 x = ld_global_nc_v4(p);
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else {
      asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];"
                   : "=r"(w[0]), "=r"(w[1])
                   : "l"(p));
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) w[i] = 0;
  }
};

template <int D, int kWarps>
__global__ void __launch_bounds__(kWarps * kWarpSize) decode_attention_fp8_kernel(
    const __grid_constant__ AttnArgs a) {
  grid_dependency_sync();
  constexpr int kThreads = kWarps * kWarpSize;
  constexpr int kPieces = D / 64;  // 16-byte pieces per lane of a K row
  constexpr int kTiles = D / 16;   // m-tiles of O^T
  extern __shared__ __align__(16) float shared[];  // warp_acc [kWarps][heads][D], part [heads][D]
  __shared__ float warp_m[kWarps][kGroup], warp_l[kWarps][kGroup];
  __shared__ float m_sm[kGroup], l_sm[kGroup];

  const int split = static_cast<int>(blockIdx.x % a.splits);
  const int64_t item = blockIdx.x / a.splits;
  const int hg = static_cast<int>(item % a.groups);
  const int kh = static_cast<int>(item / a.groups % a.num_kv_heads);
  const int64_t b = item / a.groups / a.num_kv_heads;
  const int heads = min(kGroup, a.group - hg * kGroup);  // this CTA's
  const int head0 = kh * a.group + hg * kGroup;
  const int warp = threadIdx.x / kWarpSize;
  const int lane = threadIdx.x % kWarpSize;
  const int g = lane >> 2;
  const int t = lane & 3;
  float* part = shared + kWarps * heads * D;

  int seq_len = a.seq_lens[b];
  if (seq_len < 0 || seq_len > a.max_rows) {
    if (threadIdx.x == 0) raise_error(a.err, kErrBadIndex);
    seq_len = seq_len < 0 ? 0 : a.max_rows;
  }
  // this CTA's split of the rows, then this warp's share of it, both in whole steps
  const int steps = (seq_len + kStepRows - 1) / kStepRows;
  const int split_steps = (steps + a.splits - 1) / a.splits;
  const int warp_steps = (split_steps + kWarps - 1) / kWarps;
  const int step0 = min(steps, split * split_steps + warp * warp_steps);
  const int step1 = min(steps, min((split + 1) * split_steps, step0 + warp_steps));
  const int w_begin = step0 * kStepRows;
  const int w_end = min(seq_len, step1 * kStepRows);
  const int32_t* table = a.block_tables + b * a.max_blocks;

  // Q^T's B fragments in f16: head g, this lane's dims. Scaled by a power of two per head.
  uint32_t qf[kPieces][8];
  float x_scale[2];  // of the scores of heads 2t and 2t + 1
  {
    uint32_t raw[kPieces][8];
    uint32_t amax = 0;
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
#pragma unroll
      for (int i = 0; i < 8; ++i) raw[c][i] = 0;
      if (g < heads) {
        const uint8_t* qp = static_cast<const uint8_t*>(a.q) +
                            (b * a.q_stride + static_cast<int64_t>(head0 + g) * D + 64 * c + 16 * t) * 2;
        const uint4 q0 = ld_global_nc_v4(qp), q1 = ld_global_nc_v4(qp + 16);
        raw[c][0] = q0.x, raw[c][1] = q0.y, raw[c][2] = q0.z, raw[c][3] = q0.w;
        raw[c][4] = q1.x, raw[c][5] = q1.y, raw[c][6] = q1.z, raw[c][7] = q1.w;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        amax = max(amax, max(raw[c][i] & 0x7fffu, (raw[c][i] >> 16) & 0x7fffu));
      }
    }
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // the largest magnitude's exponent; the shift to 14 as two factors, either inside fp32
    const int shift = 14 - (static_cast<int>(amax >> 7) - 127);  // [-114, 141]
    const int s0 = shift / 2, s1 = shift - s0;
    const float f0 = exp2_int(s0), f1 = exp2_int(s1);
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        qf[c][i] = pack_f16x2(__uint_as_float(raw[c][i] << 16) * f0 * f1,
                              __uint_as_float(raw[c][i] & 0xffff0000u) * f0 * f1);
      }
    }
    const float back = a.scale_log2 * exp2_int(-s0) * exp2_int(-s1);
    x_scale[0] = __shfl_sync(0xffffffffu, back, 8 * t);      // lane of head 2t
    x_scale[1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);  // of head 2t + 1
  }

  float acc[kTiles][4];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0.0f;
  }
  // the running maximum of y of heads 2t, 2t + 1; finite, so that no difference with a score
  // of -infinity is NaN
  float m[2] = {-FLT_MAX, -FLT_MAX};
  float l[2] = {0.0f, 0.0f};  // this lane's rows only, summed over the warp at the end

  const int64_t row_bytes = static_cast<int64_t>(a.num_kv_heads) * D;
  const uint8_t* kc = a.k_cache + static_cast<int64_t>(kh) * D + 16 * t;
  const uint8_t* vc = a.v_cache + static_cast<int64_t>(kh) * D + g * (D / 8);

  // lane r's row of a step: its slot and its two scale bytes (1 past the end, and unused)
  uint32_t slot = 0, scales = 0;
  const auto look_up = [&](int r0) {
    const int j = r0 + lane;
    slot = 0;
    scales = (kScaleBias << 8) | kScaleBias;
    if (j < w_end) {
      const int page = a.page.divide(j);
      int blk = __ldg(table + page);
      if (static_cast<uint64_t>(blk) >= static_cast<uint64_t>(a.num_blocks)) {
        raise_error(a.err, kErrBadIndex);  // an entry outside the cache: read block 0
        blk = 0;
      }
      slot = static_cast<uint32_t>(blk) * static_cast<uint32_t>(a.block_size) +
             static_cast<uint32_t>(j - page * a.block_size);
      const int64_t at = static_cast<int64_t>(slot) * a.num_kv_heads + kh;
      scales = __ldg(a.k_scale + at) | (static_cast<uint32_t>(__ldg(a.v_scale + at)) << 8);
    }
  };

  if (w_begin < w_end) look_up(w_begin);
  for (int r0 = w_begin; r0 < w_end; r0 += kStepRows) {
    uint4 k[2][2][kPieces];  // tile, row g or g + 8, piece
    VPart<D> v[2][4];        // tile, rows 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 16 * i + 8 * e + g;
        const uint8_t* p = kc + __shfl_sync(0xffffffffu, slot, r) * row_bytes;
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
          k[i][e][c] = r0 + r < w_end ? ld_global_nc_v4(p + 64 * c) : make_uint4(0, 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 16 * i + 8 * (e >> 1) + 2 * t + (e & 1);
        const uint8_t* p = vc + __shfl_sync(0xffffffffu, slot, r) * row_bytes;
        if (r0 + r < w_end) v[i][e].load(p);
        else v[i][e].clear();  // codes of rows past the end are zeros: 0 * w, never NaN
      }
    }
    const uint32_t step_scales = scales;
    if (r0 + kStepRows < w_end) look_up(r0 + kStepRows);

    // S^T: lane holds rows g, g + 8 of both tiles x heads 2t, 2t + 1
    float y[2][4];
    float unscale[2][2];  // 2^-ev
    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t w0 = word(k[i][0][c], w), w1 = word(k[i][1][c], w);
          mma_16816_f16(s, e4m3_to_f16x2_lo(w0), e4m3_to_f16x2_lo(w1), e4m3_to_f16x2_hi(w0),
                        e4m3_to_f16x2_hi(w1), qf[c][2 * w], qf[c][2 * w + 1]);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 16 * i + 8 * e + g;
        const uint32_t sc = __shfl_sync(0xffffffffu, step_scales, r);
        const float ks = scale_value(sc & 0xffu);
        const float ev = static_cast<float>(static_cast<int>(sc >> 8) - kScaleBias);
        unscale[i][e] = scale_value(2 * kScaleBias - (sc >> 8));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float v = fmaf(s[2 * e + h], x_scale[h] * ks, ev);
          y[i][2 * e + h] = r0 + r < w_end ? v : -__builtin_huge_valf();
          top[h] = fmaxf(top[h], y[i][2 * e + h]);
        }
      }
    }
#pragma unroll
    for (int off = 4; off < kWarpSize; off *= 2) {
      top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], off));
      top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], off));
    }
    if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {  // the maximum moved
      const float al[2] = {exp2_approx(m[0] - top[0]), exp2_approx(m[1] - top[1])};
      l[0] *= al[0];
      l[1] *= al[1];
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] *= al[e & 1];
      }
      m[0] = top[0];
      m[1] = top[1];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] = exp2_approx(y[i][e] - m[e & 1] + kWeightBits);
        l[e & 1] = fmaf(p[e], unscale[i][e >> 1], l[e & 1]);
      }
      const uint32_t b0 = transpose8x8_b16(pack_f16x2(p[0], p[1]));  // rows 2t, 2t + 1 of head g
      const uint32_t b1 = transpose8x8_b16(pack_f16x2(p[2], p[3]));  // and + 8
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        const uint32_t lo0 = __byte_perm(v[i][0].w[w], v[i][1].w[w], 0x5140);
        const uint32_t hi0 = __byte_perm(v[i][0].w[w], v[i][1].w[w], 0x7362);
        const uint32_t lo1 = __byte_perm(v[i][2].w[w], v[i][3].w[w], 0x5140);
        const uint32_t hi1 = __byte_perm(v[i][2].w[w], v[i][3].w[w], 0x7362);
        mma_16816_f16(acc[2 * w], e4m3_to_f16x2_lo(lo0), e4m3_to_f16x2_hi(lo0),
                      e4m3_to_f16x2_lo(lo1), e4m3_to_f16x2_hi(lo1), b0, b1);
        mma_16816_f16(acc[2 * w + 1], e4m3_to_f16x2_lo(hi0), e4m3_to_f16x2_hi(hi0),
                      e4m3_to_f16x2_lo(hi1), e4m3_to_f16x2_hi(hi1), b0, b1);
      }
    }
  }
#pragma unroll
  for (int off = 4; off < kWarpSize; off *= 2) {
    l[0] += __shfl_xor_sync(0xffffffffu, l[0], off);
    l[1] += __shfl_xor_sync(0xffffffffu, l[1], off);
  }
  // O^T element (dim, head): m-tile i holds dims g * D / 8 + 2 i (elements 0, 1: heads 2t, 2t + 1)
  // and + 1 (elements 2, 3)
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (2 * t + h < heads) {
      if (g == 0) {
        warp_m[warp][2 * t + h] = m[h];
        warp_l[warp][2 * t + h] = l[h];
      }
      float* dst = shared + (warp * heads + 2 * t + h) * D + g * (D / 8);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        *reinterpret_cast<float2*>(dst + 2 * i) = make_float2(acc[i][h], acc[i][2 + h]);
      }
    }
  }
  __syncthreads();
  // the warps' (max, sum, partial) merged into the CTA's
  if (threadIdx.x < heads) {
    const int h = threadIdx.x;
    float mx = warp_m[0][h];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, warp_m[w][h]);
    float ls = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) ls += warp_l[w][h] * exp2_approx(warp_m[w][h] - mx);
    m_sm[h] = mx;
    l_sm[h] = ls;
  }
  for (int idx = threadIdx.x; idx < heads * D; idx += kThreads) {
    const int h = idx / D;
    float mx = warp_m[0][h];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, warp_m[w][h]);
    float o = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) o += shared[w * heads * D + idx] * exp2_approx(warp_m[w][h] - mx);
    part[idx] = o;
  }
  __syncthreads();

  __nv_bfloat16* out =
      static_cast<__nv_bfloat16*>(a.out) + (b * a.num_heads + head0) * static_cast<int64_t>(D);
  if (a.splits == 1) {
    for (int idx = threadIdx.x; idx < heads * D; idx += kThreads) {
      const float ls = l_sm[idx / D];
      out[idx] = __float2bfloat16_rn(ls == 0.0f ? 0.0f : part[idx] / ls);
    }
    return;
  }
  // CTA r of the cluster combines and writes output elements [r * per, (r + 1) * per)
  cluster_sync_all();
  const int per = heads * D / a.splits;
  const int first = static_cast<int>(cluster_rank()) * per;
  for (int idx = first + threadIdx.x; idx < first + per; idx += kThreads) {
    const int h = idx / D;
    float mr[kMaxSplits], lr[kMaxSplits], pr[kMaxSplits];
#pragma unroll
    for (int r = 0; r < kMaxSplits; ++r) {
      if (r < a.splits) {
        mr[r] = ld_remote_f32(&m_sm[h], r);
        lr[r] = ld_remote_f32(&l_sm[h], r);
        pr[r] = ld_remote_f32(&part[idx], r);
      }
    }
    float mx = mr[0];
#pragma unroll
    for (int r = 1; r < kMaxSplits; ++r) {
      if (r < a.splits) mx = fmaxf(mx, mr[r]);
    }
    float o = 0.0f, ls = 0.0f;
#pragma unroll
    for (int r = 0; r < kMaxSplits; ++r) {
      if (r < a.splits) {
        const float w = exp2_approx(mr[r] - mx);
        o += w * pr[r];
        ls += w * lr[r];
      }
    }
    out[idx] = __float2bfloat16_rn(ls == 0.0f ? 0.0f : o / ls);
  }
  cluster_sync_all();  // every CTA's shared memory stays valid until the others have read it
}

template <int D, int kWarps>
int launch_attention(const AttnArgs& a, int64_t blocks, int device, cudaStream_t stream) {
  const int heads = a.group < kGroup ? a.group : kGroup;
  const size_t smem = static_cast<size_t>(kWarps + 1) * heads * D * 4;
  const auto kernel = decode_attention_fp8_kernel<D, kWarps>;
  if (blocks_per_sm(reinterpret_cast<const void*>(kernel), kWarps * kWarpSize, smem, device) <= 0) {
    return SVLLM_ERR_CUDA;
  }
  return launch_serialized(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kWarps * kWarpSize),
                           smem, stream, static_cast<unsigned>(a.splits), a);
}

template <int D>
int dispatch(const AttnArgs& a, int64_t blocks, int64_t split_steps, int device,
             cudaStream_t stream) {
  const int64_t sms = sm_count(device);
  if (blocks <= sms && split_steps >= 8) return launch_attention<D, 8>(a, blocks, device, stream);
  return launch_attention<D, 4>(a, blocks, device, stream);
}

}  // namespace
}  // namespace svllm::k

extern "C" int svllm_decode_attention_fp8_bf16(
    void* out, const void* q, int64_t q_token_stride, const void* k_cache, const void* v_cache,
    const void* k_scale, const void* v_scale, int64_t num_blocks, int64_t block_size,
    const int32_t* block_tables, int64_t max_blocks, const int32_t* seq_lens, int64_t num_seqs,
    int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, float scale, svllm_stream stream) {
  using namespace svllm::k;
  if (num_seqs < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      block_size <= 0 || max_blocks < 0 || num_blocks <= 0 || head_dim <= 0 ||
      q_token_stride < num_heads * head_dim || !(scale > 0.0f) || !std::isfinite(scale)) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  if (num_seqs == 0) return SVLLM_OK;
  if (out == nullptr || q == nullptr || k_cache == nullptr || v_cache == nullptr ||
      k_scale == nullptr || v_scale == nullptr || (max_blocks > 0 && block_tables == nullptr) ||
      seq_lens == nullptr) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  constexpr int64_t kInt = int64_t{1} << 31;
  const int64_t group = num_heads / num_kv_heads;
  const int64_t groups = (group + kGroup - 1) / kGroup;
  if (num_heads > (1 << 16) || block_size >= (1 << 20) || max_blocks >= kInt ||
      max_blocks * block_size >= kInt - kStepRows || num_blocks >= kInt ||
      num_blocks * block_size >= kInt || num_seqs >= kInt ||
      num_seqs * num_kv_heads * groups * kMaxSplits >= kInt) {
    return SVLLM_ERR_TOO_LARGE;
  }
  if ((head_dim != 64 && head_dim != 128) || !aligned16(q) || !aligned16(k_cache) ||
      !aligned16(v_cache) || q_token_stride % 8 != 0) {
    return SVLLM_ERR_UNSUPPORTED;
  }
  int device;
  if (current_device(&device) != SVLLM_OK) return SVLLM_ERR_CUDA;
  AttnArgs a{};
  a.err = library_error_word(device);
  if (a.err == nullptr) return SVLLM_ERR_CUDA;
  a.out = out;
  a.q = q;
  a.k_cache = static_cast<const uint8_t*>(k_cache);
  a.v_cache = static_cast<const uint8_t*>(v_cache);
  a.k_scale = static_cast<const uint8_t*>(k_scale);
  a.v_scale = static_cast<const uint8_t*>(v_scale);
  a.block_tables = block_tables;
  a.seq_lens = seq_lens;
  a.q_stride = q_token_stride;
  a.num_blocks = num_blocks;
  a.max_blocks = static_cast<int>(max_blocks);
  a.max_rows = static_cast<int>(max_blocks * block_size);
  a.block_size = static_cast<int>(block_size);
  a.page = make_divider(block_size);
  a.num_heads = static_cast<int>(num_heads);
  a.num_kv_heads = static_cast<int>(num_kv_heads);
  a.group = static_cast<int>(group);
  a.groups = static_cast<int>(groups);
  a.scale_log2 = static_cast<float>(static_cast<double>(scale) / std::log(2.0));
  // Split the rows until there are about two CTAs per SM, never below 64 rows per split.
  const int64_t items = num_seqs * num_kv_heads * groups;
  int64_t splits = (2 * sm_count(device) + items - 1) / items;
  const int64_t by_length = (a.max_rows + 63) / 64;
  splits = splits < by_length ? splits : by_length;
  int pow2 = 1;
  while (pow2 * 2 <= splits && pow2 * 2 <= kMaxSplits) pow2 *= 2;
  a.splits = pow2;
  const int64_t split_steps = ((a.max_rows + kStepRows - 1) / kStepRows + pow2 - 1) / pow2;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return head_dim == 128 ? dispatch<128>(a, items * pow2, split_steps, device, s)
                         : dispatch<64>(a, items * pow2, split_steps, device, s);
}
