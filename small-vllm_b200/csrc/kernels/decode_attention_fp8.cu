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
// of it, the others off by up to 2^-39 of it), and the weights are w_j = 2^(y_j - m + 6) with y_j =
// x_j + ev_j, x_j the score in base 2 and m a maximum of the y_j that is moved only when one passes it
// by 8: w_j <= 2^14, the largest is 2^6 at least, and f16's smallest number, 2^-24, stands for 2^-30 of
// it or less (a weight below half of that is lost). The rows' scales thus never touch the codes: 2^ek
// multiplies a score, ev adds to it (in the one rounding of an fma). The weights are rounded to f16
// (2^-11 of each, an eighth of a bf16 rounding) because the product takes no wider operand.
//
// The denominator is l = sum_j 2^(d_j - ev_j) with d_j = y_j - m + 6, in fp32. Its terms have an
// exponential of their own: w_j 2^-ev_j would lose a row whose w_j is below 2^-126, and with scales
// 120 binades apart such a row may be most of the sum. m lies within 60 of the largest x (and 8 of
// slack), so the largest term is between 2^-54 and 2^74, and one below 2^-126 less than 2^-72 of it.
// For the same reason l is moved to another maximum in two steps (half_factor). (x is taken from y,
// not y from x: at scores so large that x + ev rounds, weight and term then carry the same error.)
//
// Layout. A warp takes steps of 32 cached rows, lane = 4 g + t:
//   S^T[16 rows x 8 heads] = K[16 x D] . Q^T[D x 8]: lane holds rows g, g + 8 of K, 16 bytes at
//     64 c + 16 t of piece c; a 4-byte word of it is one k-step (the same permutation of the
//     head dimension on both sides);
//   O^T[D x 8] += V^T[D x 16 rows] . P^T[16 x 8]: lane holds rows 2t, 2t + 1, 2t + 8, 2t + 9 of V,
//     D / 8 bytes at g * D / 8. V's transpose is two byte permutations of a word of two rows, which
//     pair their codes before the conversion; P^T comes from S^T by movmatrix.
//
// Work. An item is one (request, KV head, group of up to eight query heads). Rows travel by cp.async,
// 16 bytes a lane, into a ring of two stages that each warp owns. Two kernels:
//   * By lines (long tables, or many items): the steps of all items form one line, in that order,
//     of which each warp takes an equal share, found from the device-side lengths. A warp runs on
//     from item to item without waiting for another; the parts of items that are cut go to a
//     workspace, and a third kernel joins them in a fixed order. Head_dim 64: two KV heads an item,
//     so that a row's copy fills a 128-byte line (the L2's requests bound the kernel otherwise).
//   * By items (short tables and few items): a CTA takes an item, its warps deal the steps among
//     them and merge through shared memory; up to eight CTAs share an item as a thread-block cluster,
//     which merges through distributed shared memory. One launch.
//
// What bounds it, measured on a B200 (16/8 heads of 128, us in a graph): 64 requests of 2064 to 4096
// rows, 407 MB, 76.5-76.9. The warps stream at 6.6 TB/s once they run, 62 us; 4 us go by until the first
// rows are there (lengths 0.8, the share 0.5, table and rows, each a trip to memory after the other),
// the last warps end 4 behind the mean, and the join takes 3. One request of 32760 rows: 18.1, of
// which 10.5 are the stream. A step of 32 rows takes 577 warp instructions; 39 % of the issue slots are
// used. More loads in flight gave nothing (three stages 79.1, twelve warps 77.1-78.9, fourteen 81.5, the
// next load after the products 80.7); a CTA per share whose warps merge at every item's end took 98,
// rows loaded to registers instead of shared memory 168.
#include <cuda_runtime.h>

#include <cfloat>
#include <cmath>
#include <cstdint>

#include "common.cuh"
#include "fp8.cuh"
#include "host_common.h"

namespace svllm::k {
namespace {

constexpr int kStepRows = 32;    // cached rows a warp takes at a time
constexpr int kGroup = 8;        // query heads of an item: the N of the products
constexpr int kStages = 2;       // of a warp's ring
constexpr int kLineWarps = 8;    // of a CTA by lines, one per SM
constexpr int kItemWarps = 8;    // of a CTA by items
constexpr int kMinShare = 2;     // steps of a warp's share at least
// KV heads of an item by lines at head_dim 64, so that a row fills a 128-byte line, and from how many
// steps a warp on, were every request as long as its table (us, one and two, 32/8 heads of 64: 64
// requests of 2048-4096 rows, 110 steps, 61.4, 43.9; 16 of 2048-4096, 14 steps, 19.8, 19.7; 13 of
// 140-2500, 24/8 heads, 7 steps, 10.0, 11.8).
constexpr int kPair = 2, kPairSteps = 14;
constexpr int kMaxSplits = 8;    // CTAs of an item: the portable cluster size
constexpr int kItemSteps = 4;    // by items up to this many steps of a warp
constexpr int kJoinThreads = 256;
// The join of items whose number of parts (of one of middling length) is up to kJoinFewParts takes a
// thread for four outputs, with kJoinFew parts in flight; with more parts lanes and warps share them.
// Few parts are bound by the instructions of so many warps, many by the trips to memory. us with the
// form for few and for many, requests of 2048-4096 rows (or 1-4096 where marked), by their parts:
//   heads of 128, 16/8:  5: 53.0, 54.0   7: 37.6, 38.5   8: 31.6, 32.0   9: 29.9, 30.2   10: 27.0, 26.1
//   32/4:                6: 32.3, 33.0*  7: 36.1, 36.8   8: 27.8, 27.9*  9: 25.1, 24.9*  10: 23.2, 22.8*
//   heads of 64, 32/8:   4: 49.8, 53.1   5: 45.2, 45.5*  6: 31.4, 32.1   6: 38.8, 37.7*   7: 37.9, 36.9
//   24/4:                5: 40.5, 41.8*  6: 49.9, 51.8   6: 35.4, 35.7*  7: 32.4, 32.1*  10: 31.5, 30.0
//   8/8 and 9/3:         4: 48.5, 49.1   5: 42.1, 42.0*  6: 36.7, 34.8*  6: 33.4, 32.4*   7: 36.6, 35.4
constexpr int kJoinFew = 8;
template <int D>
constexpr int kJoinFewParts = D == 128 ? 7 : 5;
// Parts a lane has in flight there. At head_dim 128 five are what fits beside a CTA by lines (64
// registers), so that the join's CTAs wait where they will run (us, five and eight: one request of
// 32760 rows 18.2, 19.4; 48 of 88-4096, 32/4 heads, 27.9, 28.6; but 24, 28/4 heads, 21.4, 21.2). At 64
// six do (32 of 2048-4096, 32/8 heads, five, six and eight: 27.8, 27.4, 27.7).
template <int D>
constexpr int kJoinMany = D == 128 ? 5 : 6;
// The running maximum is moved only when a score passes it by kSlack, so that most steps need one
// vote instead of a maximum over the warp. Weights reach 2^(kWeightBits + kSlack).
constexpr float kWeightBits = 6.0f, kSlack = 8.0f;

// Where an item's parts are: the first share that holds one, and how many (1: the item is whole, and
// its output written).
struct JoinEntry {
  int share;
  int parts;
};

struct AttnArgs {
  void* out;      // [num_seqs, num_heads, D] bf16, contiguous
  const void* q;  // [num_seqs, num_heads, D] bf16, token stride q_stride
  const uint8_t* k_cache;  // [num_blocks, block_size, num_kv_heads, D]
  const uint8_t* v_cache;
  const uint8_t* k_scale;  // [num_blocks, block_size, num_kv_heads]
  const uint8_t* v_scale;
  const int32_t* block_tables;  // [num_seqs, max_blocks]
  const int32_t* seq_lens;      // [num_seqs]
  // What the warps by lines leave of cut items, for the join: [shares][2][heads of an item], of the
  // item that a share continues and of one that it begins.
  JoinEntry* table;  // [items]
  float2* part_ml;   // maximum and sum
  float* part_acc;   // [D] each
  int64_t q_stride;
  int64_t num_blocks;
  int num_seqs;
  int max_blocks;
  int max_rows;  // max_blocks * block_size
  int block_size;
  Divider page;  // by the block size
  int num_heads;
  int num_kv_heads;
  int group;   // query heads per KV head
  int groups;  // items they are dealt to
  int subs;    // items of a request
  int shares;  // warps by lines
  int splits;  // CTAs of an item, by items
  float scale_log2;
  int* err;
};

// Half of what moves sums from the maximum m to another: they are multiplied by it twice, so that a
// denominator, whose terms lie up to 2^60 above and below its numerator's, loses nothing that counts
// where the whole factor is below fp32's smallest.
__device__ __forceinline__ float half_factor(float m, float to) {
  return exp2_approx(0.5f * (m - to));
}

__device__ __forceinline__ uint32_t transpose8x8_b16(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// 16 bytes to shared memory, zeros where !valid.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(valid ? 16 : 0)
               : "memory");
}

__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}

template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "r"(a)
               : "memory");
  return r;
}

__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a) : "memory");
  return r;
}

// Where 16-byte chunk c of row r lies in a tile of 32 rows of `kWidth` bytes: permuted so that both
// products' reads (a quarter of a warp: two rows times four chunks of K, four even or odd rows times
// two chunks of V) touch every bank once.
template <int kWidth>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  if constexpr (kWidth == 128) {
    return static_cast<uint32_t>(r * 128 + ((c ^ (r & 6) ^ ((r & 1) << 2)) << 4));
  } else {
    return static_cast<uint32_t>((r >> 1) * 128 + (((r ^ (r >> 2)) & 1) << 6) +
                                 ((c ^ (((r >> 1) & 1) << 1)) << 4));
  }
}

// The scale bytes of a row's K and V in one word, as they are used.
__device__ __forceinline__ uint32_t scales_of(const AttnArgs& a, uint32_t k, uint32_t v) {
  const uint32_t ks = scale_in_range(k), vs = scale_in_range(v);
  if (ks != k || vs != v) raise_error(a.err, kErrBadIndex);
  return ks | (vs << 8);
}

// A request's length, and the steps of its items: one at least, so that a request without rows
// gets its zeros.
__device__ __forceinline__ int clamp_len(const AttnArgs& a, int n) {
  return max(0, min(n, a.max_rows));
}

__device__ __forceinline__ int item_steps(int len) {
  return max(1, (len + kStepRows - 1) / kStepRows);
}

// An item's heads: kHeads neighbouring KV heads (the last item of an odd number of them has one
// less) and, of each, the same up to eight query heads.
template <int kHeads>
struct Heads {
  int kv, live;      // the first KV head, and how many there are
  int first, count;  // of the first KV head: its first query head, and how many
  __device__ __forceinline__ Heads(const AttnArgs& a, int sub) {
    const int run = a.groups == 1 ? sub : sub / a.groups;
    const int hg = sub - run * a.groups;
    kv = run * kHeads;
    live = min(kHeads, a.num_kv_heads - kv);
    first = kv * a.group + hg * kGroup;
    count = min(kGroup, a.group - hg * kGroup);
  }
};

// One step's copies: 32 rows of K, then of V, of kHeads KV heads side by side.
template <int D, int kHeads>
struct Loader {
  static constexpr int kWidth = D * kHeads;
  static constexpr int kChunks = kWidth / 16;  // 16-byte chunks of a row
  static constexpr int kTileBytes = kStepRows * kWidth;
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kLoads = kStepRows * kChunks / kWarpSize;  // a lane, K and V each
  static constexpr int kRowsALoad = kWarpSize / kChunks;

  // The table entry of lane r's row of a step; any where the row does not exist.
  static __device__ __forceinline__ int block_of(const AttnArgs& a, int b, int step, int len) {
    const int j = step * kStepRows + static_cast<int>(threadIdx.x) % kWarpSize;
    if (j >= len) return 0;
    return __ldg(a.block_tables + static_cast<int64_t>(b) * a.max_blocks + a.page.divide(j));
  }

  // Copies the step's rows to `dst` and loads lane r's row's scale bytes (the first KV head's lowest),
  // which nothing waits for here.
  static __device__ __forceinline__ void issue(const AttnArgs& a, uint32_t dst, int block,
                                               const Heads<kHeads>& heads, int step, int len,
                                               uint32_t (&k_scale)[kHeads],
                                               uint32_t (&v_scale)[kHeads]) {
    const int lane = static_cast<int>(threadIdx.x) % kWarpSize;
    const int r0 = step * kStepRows, j = r0 + lane;
    uint32_t slot = 0;
#pragma unroll
    for (int i = 0; i < kHeads; ++i) k_scale[i] = v_scale[i] = kScaleBias;
    if (j < len) {
      if (static_cast<uint64_t>(block) >= static_cast<uint64_t>(a.num_blocks)) {
        raise_error(a.err, kErrBadIndex);  // an entry outside the cache: read block 0
        block = 0;
      }
      slot = static_cast<uint32_t>(block) * static_cast<uint32_t>(a.block_size) +
             static_cast<uint32_t>(j - a.page.divide(j) * a.block_size);
      const int64_t at = static_cast<int64_t>(slot) * a.num_kv_heads + heads.kv;
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        if (i < heads.live) {
          k_scale[i] = __ldg(a.k_scale + at + i);
          v_scale[i] = __ldg(a.v_scale + at + i);
        }
      }
    }
    const int c = lane % kChunks;
    const bool live = kHeads == 1 || c * 16 < heads.live * D;
    const int64_t row_bytes = static_cast<int64_t>(a.num_kv_heads) * D;
    // (a chunk of a KV head that does not exist copies nothing; its address is the first head's)
    const uint8_t* k = a.k_cache + static_cast<int64_t>(heads.kv) * D + (live ? c * 16 : 0);
    const int64_t v = a.v_cache - a.k_cache;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = i * kRowsALoad + lane / kChunks;
      const uint8_t* p = k + __shfl_sync(0xffffffffu, slot, r) * row_bytes;
      const bool valid = r0 + r < len && live;  // zeros past the end: 0 * w, never NaN
      cp_async16(dst + tile_at<kWidth>(r, c), p, valid);
      cp_async16(dst + kTileBytes + tile_at<kWidth>(r, c), p + v, valid);
    }
  }
};

// Q^T's B fragments in f16: head g, this lane's dims, scaled by a power of two per head.
template <int D>
struct Queries {
  static constexpr int kPieces = D / 64;  // 16-byte pieces per lane of a K row
  uint32_t f[kPieces][8];
  float x_scale[2];  // of the scores of heads 2t and 2t + 1

  // chunk(i): 16-byte chunk i of query head g; zeros for a head that does not exist.
  template <class Chunk>
  __device__ __forceinline__ void set(float scale_log2, const Chunk& chunk) {
    const int t = static_cast<int>(threadIdx.x) & 3;
    uint32_t raw[kPieces][8];
    uint32_t amax = 0;
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      const uint4 q0 = chunk(8 * c + 2 * t), q1 = chunk(8 * c + 2 * t + 1);
      raw[c][0] = q0.x, raw[c][1] = q0.y, raw[c][2] = q0.z, raw[c][3] = q0.w;
      raw[c][4] = q1.x, raw[c][5] = q1.y, raw[c][6] = q1.z, raw[c][7] = q1.w;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        amax = max(amax, max(raw[c][i] & 0x7fffu, (raw[c][i] >> 16) & 0x7fffu));
      }
    }
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // the largest magnitude's exponent to 14, as two factors, either inside fp32
    const int shift = 14 - (static_cast<int>(amax >> 7) - 127);  // [-114, 141]
    const int s0 = shift / 2, s1 = shift - s0;
    const float f0 = exp2_int(s0), f1 = exp2_int(s1);
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[c][i] = pack_f16x2(__uint_as_float(raw[c][i] << 16) * f0 * f1,
                             __uint_as_float(raw[c][i] & 0xffff0000u) * f0 * f1);
      }
    }
    const float back = scale_log2 * exp2_int(-s0) * exp2_int(-s1);
    x_scale[0] = __shfl_sync(0xffffffffu, back, 8 * t);      // lane of head 2t
    x_scale[1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);  // of head 2t + 1
  }
};

// A warp's running sums over an item's rows, for one of its KV heads. kWidth: of a row of the tiles.
template <int D, int kWidth>
struct Sums {
  static constexpr int kTiles = D / 16;  // m-tiles of O^T
  // O^T element (dim, head): m-tile i holds dims g * D / 8 + 2 i (elements 0, 1: heads 2t, 2t + 1)
  // and + 1 (elements 2, 3)
  float acc[kTiles][4];
  // the running maximum of y of heads 2t, 2t + 1; finite, so that no difference with a score of
  // -infinity is NaN
  float m[2];
  float l[2];  // this lane's rows only, until reduce()

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = 0.0f;
    }
    m[0] = m[1] = -FLT_MAX;
    l[0] = l[1] = 0.0f;
  }

  // Adds a step: the tile in shared memory and the KV head's place in its rows, lane r's row's scale
  // bytes, how many rows exist.
  __device__ __forceinline__ void step(uint32_t tile, int place, uint32_t scales, int live,
                                       const Queries<D>& q) {
    const int chunk = place * (D / 16);
    const int lane = static_cast<int>(threadIdx.x) % kWarpSize;
    const int g = lane >> 2, t = lane & 3;
    // S^T: lane holds rows g, g + 8 of both tiles x heads 2t, 2t + 1
    float y[2][4];
    float v_exp[2][2];  // ev
    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < Queries<D>::kPieces; ++c) {
        const uint4 k0 = lds128(tile + tile_at<kWidth>(16 * i + g, chunk + 4 * c + t));
        const uint4 k1 = lds128(tile + tile_at<kWidth>(16 * i + 8 + g, chunk + 4 * c + t));
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t w0 = word(k0, w), w1 = word(k1, w);
          mma_16816_f16(s, e4m3_to_f16x2_lo(w0), e4m3_to_f16x2_lo(w1), e4m3_to_f16x2_hi(w0),
                        e4m3_to_f16x2_hi(w1), q.f[c][2 * w], q.f[c][2 * w + 1]);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 16 * i + 8 * e + g;
        const uint32_t sc = __shfl_sync(0xffffffffu, scales, r);
        const float ks = scale_value(sc & 0xffu);
        const float ev = static_cast<float>(static_cast<int>(sc >> 8) - kScaleBias);
        v_exp[i][e] = ev;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // (s * ks is exact; the two factors' product may leave fp32 where s is 0)
          const float v = fmaf(s[2 * e + h] * ks, q.x_scale[h], ev);
          y[i][2 * e + h] = r < live ? v : -__builtin_huge_valf();
          top[h] = fmaxf(top[h], y[i][2 * e + h]);
        }
      }
    }
    // (differences, as the weights take them: fp32 may round m + kSlack up to the next score)
    if (__any_sync(0xffffffffu, top[0] - m[0] > kSlack || top[1] - m[1] > kSlack)) {
#pragma unroll
      for (int off = 4; off < kWarpSize; off *= 2) {
        top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], off));
        top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], off));
      }
      const float half[2] = {half_factor(m[0], top[0]), half_factor(m[1], top[1])};
      const float al[2] = {half[0] * half[0], half[1] * half[1]};
      l[0] = l[0] * half[0] * half[0];
      l[1] = l[1] * half[1] * half[1];
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
        const float d = y[i][e] - m[e & 1] + kWeightBits;
        p[e] = exp2_approx(d);
        l[e & 1] += exp2_approx(d - v_exp[i][e >> 1]);
      }
      const uint32_t b0 = transpose8x8_b16(pack_f16x2(p[0], p[1]));  // rows 2t, 2t + 1 of head g
      const uint32_t b1 = transpose8x8_b16(pack_f16x2(p[2], p[3]));  // and + 8
      uint32_t v[4][D / 32];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 16 * i + 8 * (e >> 1) + 2 * t + (e & 1);
        const uint32_t at = tile + kStepRows * kWidth;
        if constexpr (D == 128) {
          const uint4 x = lds128(at + tile_at<kWidth>(r, chunk + g));
          v[e][0] = x.x, v[e][1] = x.y, v[e][2] = x.z, v[e][3] = x.w;
        } else {
          const uint2 x = lds64(at + tile_at<kWidth>(r, chunk + (g >> 1)) + 8 * (g & 1));
          v[e][0] = x.x, v[e][1] = x.y;
        }
      }
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        const uint32_t lo0 = __byte_perm(v[0][w], v[1][w], 0x5140);
        const uint32_t hi0 = __byte_perm(v[0][w], v[1][w], 0x7362);
        const uint32_t lo1 = __byte_perm(v[2][w], v[3][w], 0x5140);
        const uint32_t hi1 = __byte_perm(v[2][w], v[3][w], 0x7362);
        mma_16816_f16(acc[2 * w], e4m3_to_f16x2_lo(lo0), e4m3_to_f16x2_hi(lo0),
                      e4m3_to_f16x2_lo(lo1), e4m3_to_f16x2_hi(lo1), b0, b1);
        mma_16816_f16(acc[2 * w + 1], e4m3_to_f16x2_lo(hi0), e4m3_to_f16x2_hi(hi0),
                      e4m3_to_f16x2_lo(hi1), e4m3_to_f16x2_hi(hi1), b0, b1);
      }
    }
  }

  // l of the whole warp.
  __device__ __forceinline__ void reduce() {
#pragma unroll
    for (int off = 4; off < kWarpSize; off *= 2) {
      l[0] += __shfl_xor_sync(0xffffffffu, l[0], off);
      l[1] += __shfl_xor_sync(0xffffffffu, l[1], off);
    }
  }
};

// ------------------------------------------------------------------------------------- by lines

// A run of steps of one item.
struct Segment {
  int b;
  int sub;    // KV head (or pair) * groups + group of query heads
  int first;  // its first step in the item
  int n;      // its steps
  int steps;  // the item's
  int len;
  int left;   // steps of the share from this segment on
};

// The line as every warp sees it.
struct Line {
  int total;   // steps
  int shares;  // no more than steps, so that none is empty
  int base, extra;  // steps of a share, and how many shares have one more
  int b0;      // the share's first request; lane i holds the length of request b0 + i
  int len;

  __device__ __forceinline__ int begin(int c) const { return c * base + min(c, extra); }
  // The first share that begins at step `at` or behind it.
  __device__ __forceinline__ int first_from(int at) const {
    const int wide = extra * (base + 1);
    return at <= wide ? (at + base) / (base + 1) : extra + (at - wide + base - 1) / base;
  }
};

__device__ __forceinline__ int length_of(const AttnArgs& a, const Line& line, int b) {
  const int held = __shfl_sync(0xffffffffu, line.len, (b - line.b0) & (kWarpSize - 1));
  return b - line.b0 < kWarpSize ? held : clamp_len(a, __ldg(a.seq_lens + b));
}

// The segment after s; s.left tells whether there is one. Every lane of a warp.
__device__ __forceinline__ void next_segment(const AttnArgs& a, const Line& line, Segment& s) {
  s.left -= s.n;
  s.first = 0;
  if (++s.sub == a.subs) {
    s.sub = 0;
    ++s.b;
    if (s.left > 0) {
      s.len = length_of(a, line, s.b);
      s.steps = item_steps(s.len);
    }
  }
  s.n = min(s.steps, s.left);
}

// Share c of the line: its first segment. A lane takes a run of requests.
__device__ __forceinline__ Segment first_segment(const AttnArgs& a, int c, Line& line) {
  const int lane = static_cast<int>(threadIdx.x) % kWarpSize;
  const int subs = a.subs;
  const int per = (a.num_seqs + kWarpSize - 1) / kWarpSize;
  const int begin = min(a.num_seqs, lane * per), end = min(a.num_seqs, begin + per);
  int sum = 0, len = 0;
  bool bad = false;
#pragma unroll 4
  for (int b = begin; b < end; ++b) {
    const int n = __ldg(a.seq_lens + b);
    bad |= n < 0 || n > a.max_rows;
    len = clamp_len(a, n);
    sum += item_steps(len) * subs;
  }
  if (bad && c == 0) raise_error(a.err, kErrBadIndex);
  int scan = sum;
#pragma unroll
  for (int off = 1; off < kWarpSize; off *= 2) {
    const int up = __shfl_up_sync(0xffffffffu, scan, off);
    if (lane >= off) scan += up;
  }
  line.total = __shfl_sync(0xffffffffu, scan, kWarpSize - 1);
  line.shares = min(a.shares, (line.total + kMinShare - 1) / kMinShare);
  line.base = line.total / line.shares;
  line.extra = line.total - line.base * line.shares;
  Segment s{};
  if (c >= line.shares) return s;
  const int lo = line.begin(c);
  // the lane whose requests hold the share's first step walks them
  int found = begin, off = lo - (scan - sum);
  const bool mine = off >= 0 && off < sum;
  if (mine && per > 1) {
    for (;; ++found) {
      const int n = item_steps(clamp_len(a, __ldg(a.seq_lens + found))) * subs;
      if (off < n) break;
      off -= n;
    }
  }
  const int owner = __ffs(static_cast<int>(__ballot_sync(0xffffffffu, mine))) - 1;
  s.b = __shfl_sync(0xffffffffu, found, owner);
  off = __shfl_sync(0xffffffffu, off, owner);
  if (per == 1) {  // a lane holds a request's length already
    line.b0 = 0;
    line.len = len;
  } else {
    line.b0 = s.b;
    line.len = s.b + lane < a.num_seqs ? clamp_len(a, __ldg(a.seq_lens + s.b + lane)) : 0;
  }
  s.len = length_of(a, line, s.b);
  s.steps = item_steps(s.len);
  s.sub = off / s.steps;
  s.first = off - s.sub * s.steps;
  s.left = line.begin(c + 1) - lo;
  s.n = min(s.steps - s.first, s.left);
  return s;
}

template <int D, int kHeads>
__global__ void __launch_bounds__(kLineWarps * kWarpSize, 1) decode_attention_fp8_lines(
    const __grid_constant__ AttnArgs a) {
  grid_dependency_sync();
  using Load = Loader<D, kHeads>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x / kWarpSize;
  const int lane = threadIdx.x % kWarpSize;
  const int g = lane >> 2;
  const int t = lane & 3;
  const int held_heads = min(a.group, kGroup);
  const uint32_t ring = smem_addr(smem) + warp * kStages * Load::kStageBytes;

  // neighbouring shares on different SMs, so that few shares find many SMs
  const int share = warp * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x);
  Line line;
  Segment seg = first_segment(a, share, line);
  if (seg.left <= 0) return;

  // ---- loads: `ahead` walks the share in front of the products
  Segment ahead = seg;
  int ahead_step = 0;
  int block = Load::block_of(a, ahead.b, ahead.first, ahead.len);
  uint32_t k_scales[kStages - 1][kHeads], v_scales[kStages - 1][kHeads];  // of the stages in flight
  const auto load = [&](int stage, uint32_t (&k_scale)[kHeads], uint32_t (&v_scale)[kHeads]) {
    if (ahead.left > 0) {
      Load::issue(a, ring + stage * Load::kStageBytes, block, Heads<kHeads>(a, ahead.sub),
                  ahead.first + ahead_step, ahead.len, k_scale, v_scale);
      if (++ahead_step == ahead.n) {
        next_segment(a, line, ahead);
        ahead_step = 0;
      }
      if (ahead.left > 0) block = Load::block_of(a, ahead.b, ahead.first + ahead_step, ahead.len);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load(i, k_scales[i], v_scales[i]);

  Queries<D> q[kHeads];
  Sums<D, Load::kWidth> sums[kHeads];
  int stage = 0, at = 0;  // `at`: the step of the segment
  while (true) {
    const Heads<kHeads> heads(a, seg.sub);
    if (at == 0) {  // rows are on their way meanwhile
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        const uint8_t* src =
            static_cast<const uint8_t*>(a.q) +
            (seg.b * a.q_stride + static_cast<int64_t>(heads.first + i * a.group + g) * D) * 2;
        const bool real = i < heads.live && g < heads.count;
        q[i].set(a.scale_log2, [&](int n) {
          return real ? ld_global_nc_v4(src + n * 16) : make_uint4(0, 0, 0, 0);
        });
        sums[i].clear();
      }
    }
    cp_async_wait<kStages - 2>();
    __syncwarp();  // every lane's copies have landed, and every lane is done with the stage before
    uint32_t scales[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      scales[i] = scales_of(a, k_scales[0][i], v_scales[0][i]);
#pragma unroll
      for (int n = 0; n + 1 < kStages - 1; ++n) {
        k_scales[n][i] = k_scales[n + 1][i];
        v_scales[n][i] = v_scales[n + 1][i];
      }
    }
    load(stage == 0 ? kStages - 1 : stage - 1, k_scales[kStages - 2], v_scales[kStages - 2]);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      sums[i].step(ring + stage * Load::kStageBytes, i, scales[i],
                   seg.len - (seg.first + at) * kStepRows, q[i]);
    }
    stage = stage + 1 == kStages ? 0 : stage + 1;
    if (++at < seg.n) continue;

    // ---- the segment's end: the item's output, or a part
    const bool cut = seg.n < seg.steps;
    if (seg.first == 0 && lane == 0) {
      // the item ends behind this share by the steps that it lacks
      const int end = line.begin(share + 1) + seg.steps - seg.n;
      a.table[static_cast<int64_t>(seg.b) * a.subs + seg.sub] = {
          share, cut ? line.first_from(end) - share : 1};
    }
    const int64_t part =
        (2 * static_cast<int64_t>(share) + (seg.first == 0 ? 1 : 0)) * (kHeads * held_heads);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      sums[i].reduce();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int head = 2 * t + h;
        if (i >= heads.live || head >= heads.count) continue;
        if (cut) {
          const int64_t at_head = part + i * held_heads + head;
          if (g == 0) a.part_ml[at_head] = make_float2(sums[i].m[h], sums[i].l[h]);
          float4* dst = reinterpret_cast<float4*>(a.part_acc + at_head * D + g * (D / 8));
#pragma unroll
          for (int n = 0; n < D / 16; n += 2) {
            dst[n / 2] = make_float4(sums[i].acc[n][h], sums[i].acc[n][2 + h],
                                     sums[i].acc[n + 1][h], sums[i].acc[n + 1][2 + h]);
          }
        } else {
          const float f = sums[i].l[h] == 0.0f ? 0.0f : 1.0f / sums[i].l[h];
          uint32_t w[D / 16];
#pragma unroll
          for (int n = 0; n < D / 16; ++n) {
            w[n] = pack_bf16x2(sums[i].acc[n][h] * f, sums[i].acc[n][2 + h] * f);
          }
          const int64_t out =
              (static_cast<int64_t>(seg.b) * a.num_heads + heads.first + i * a.group + head) * D;
          uint8_t* dst = static_cast<uint8_t*>(a.out) + (out + g * (D / 8)) * 2;
#pragma unroll
          for (int n = 0; n < D / 16; n += 4) {
            st_global_v4(dst + n * 4, make_uint4(w[n], w[n + 1], w[n + 2], w[n + 3]));
          }
        }
      }
    }
    next_segment(a, line, seg);
    at = 0;
    if (seg.left <= 0) break;
  }
}

// Joins the parts of the items that were cut: blockIdx.x the item, `spread` warps for each 32 of its
// outputs. A lane takes four dims of every 4 spread-th part, kJoinMany of them in flight; its
// fellows' sums come by shuffles, the other warps' through shared memory. The order is fixed by the
// sizes, so results repeat.
template <int D, int kHeads>
__global__ void __launch_bounds__(kJoinThreads) decode_attention_fp8_join(
    const __grid_constant__ AttnArgs a, int spread) {
  grid_dependency_sync();
  constexpr int kWarps = kJoinThreads / kWarpSize;
  constexpr int kRuns = D / 32;  // of 32 dims in a head
  __shared__ float4 others[kWarps][8];
  __shared__ float2 others_ml[kWarps];
  const JoinEntry entry = a.table[blockIdx.x];
  if (entry.parts <= 1) return;
  const int b = static_cast<int>(blockIdx.x) / a.subs;
  const Heads<kHeads> heads(a, static_cast<int>(blockIdx.x) - b * a.subs);
  const int held_heads = min(a.group, kGroup);
  const int warp = threadIdx.x / kWarpSize, lane = threadIdx.x % kWarpSize;
  const int mate = warp % spread;  // this warp's place among those of its run
  const int run = (static_cast<int>(blockIdx.y) * kWarps + warp) / spread;
  const int kv = run / (kRuns * heads.count);  // of the item's KV heads
  const int head = run / kRuns - kv * heads.count;
  const bool real = kv < heads.live;
  const int d = run % kRuns * 32 + lane % 8 * 4;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float m = -FLT_MAX, l = 0.0f;
  const int step = 4 * spread;
  for (int p0 = lane / 8 * spread + mate; real && p0 < entry.parts; p0 += step * kJoinMany<D>) {
    float2 ml[kJoinMany<D>];
    float4 x[kJoinMany<D>];
#pragma unroll
    for (int i = 0; i < kJoinMany<D>; ++i) {
      const int p = p0 + i * step;
      ml[i] = make_float2(-FLT_MAX, 0.0f);
      x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (p < entry.parts) {
        // the first part is the one that begins the item; the others continue it
        const int64_t at =
            (2 * static_cast<int64_t>(entry.share + p) + (p == 0 ? 1 : 0)) * (kHeads * held_heads) +
            kv * held_heads + head;
        ml[i] = a.part_ml[at];
        x[i] = *reinterpret_cast<const float4*>(a.part_acc + at * D + d);
      }
    }
    float mx = m;
#pragma unroll
    for (int i = 0; i < kJoinMany<D>; ++i) mx = fmaxf(mx, ml[i].x);
    const float f0 = half_factor(m, mx), f = f0 * f0;
    l = l * f0 * f0;
    acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
#pragma unroll
    for (int i = 0; i < kJoinMany<D>; ++i) {
      const float w0 = half_factor(ml[i].x, mx), w = w0 * w0;
      l = fmaf(ml[i].y * w0, w0, l);
      acc = make_float4(fmaf(x[i].x, w, acc.x), fmaf(x[i].y, w, acc.y), fmaf(x[i].z, w, acc.z),
                        fmaf(x[i].w, w, acc.w));
    }
    m = mx;
  }
#pragma unroll
  for (int off = 8; off < kWarpSize; off *= 2) {
    const float mx = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    const float f0 = half_factor(m, mx), f = f0 * f0;
    m = mx;
    l = l * f0 * f0;
    acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
    l += __shfl_xor_sync(0xffffffffu, l, off);
    acc.x += __shfl_xor_sync(0xffffffffu, acc.x, off);
    acc.y += __shfl_xor_sync(0xffffffffu, acc.y, off);
    acc.z += __shfl_xor_sync(0xffffffffu, acc.z, off);
    acc.w += __shfl_xor_sync(0xffffffffu, acc.w, off);
  }
  if (spread > 1) {
    if (lane < 8) {
      others[warp][lane] = acc;
      if (lane == 0) others_ml[warp] = make_float2(m, l);
    }
    __syncthreads();
    if (mate != 0) return;
    for (int w = warp + 1; w < warp + spread; ++w) {
      const float2 ml = others_ml[w];
      const float4 x = others[w][lane % 8];
      const float mx = fmaxf(m, ml.x);
      const float h0 = half_factor(m, mx), h1 = half_factor(ml.x, mx);
      const float f0 = h0 * h0, f1 = h1 * h1;
      m = mx;
      l = l * h0 * h0 + ml.y * h1 * h1;
      acc = make_float4(acc.x * f0 + x.x * f1, acc.y * f0 + x.y * f1, acc.z * f0 + x.z * f1,
                        acc.w * f0 + x.w * f1);
    }
  }
  if (lane < 8 && real) {
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    uint8_t* dst = static_cast<uint8_t*>(a.out) +
                   ((static_cast<int64_t>(b) * a.num_heads + heads.first + kv * a.group + head) *
                        D + d) * 2;
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(pack_bf16x2(acc.x * r, acc.y * r), pack_bf16x2(acc.z * r, acc.w * r));
  }
}

// The same where items have few parts: a thread joins four outputs, kJoinFew parts in flight; a CTA
// takes as many items as fit it, `per_item` threads each.
template <int D, int kHeads>
__global__ void __launch_bounds__(kJoinThreads) decode_attention_fp8_join_few(
    const __grid_constant__ AttnArgs a, int items, int per_item) {
  grid_dependency_sync();
  const int in_cta = static_cast<int>(threadIdx.x) / per_item;
  const int64_t item =
      static_cast<int64_t>(blockIdx.x) * (static_cast<int>(blockDim.x) / per_item) + in_cta;
  if (item >= items) return;
  const JoinEntry entry = a.table[item];
  if (entry.parts <= 1) return;
  const int held_heads = min(a.group, kGroup);
  const int b = static_cast<int>(item) / a.subs;
  const Heads<kHeads> heads(a, static_cast<int>(item) - b * a.subs);
  const int within = static_cast<int>(threadIdx.x) - in_cta * per_item;
  const int row = within / (D / 4), d = within % (D / 4) * 4;
  const int kv = kHeads == 1 ? 0 : row / held_heads;
  const int head = row - kv * held_heads;
  if (kv >= heads.live || head >= heads.count) return;
  // the first part is the one that begins the item; the others continue it
  const int begins = kHeads * held_heads, stride = 2 * begins;
  const int64_t at = static_cast<int64_t>(entry.share) * stride + row;
  const float2* part_ml = a.part_ml + at;
  const float* part_acc = a.part_acc + at * D + d;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float m = -FLT_MAX, l = 0.0f;
  for (int p0 = 0; p0 < entry.parts; p0 += kJoinFew) {
    float2 ml[kJoinFew];
    float4 x[kJoinFew];
#pragma unroll
    for (int i = 0; i < kJoinFew; ++i) {
      const int p = min(p0 + i, entry.parts - 1);
      const int off = p == 0 ? begins : p * stride;
      ml[i] = part_ml[off];
      x[i] = *reinterpret_cast<const float4*>(part_acc + static_cast<int64_t>(off) * D);
    }
#pragma unroll
    for (int i = 0; i < kJoinFew; ++i) {  // the last part again: a weight of 0
      if (p0 + i >= entry.parts) ml[i] = make_float2(-__builtin_huge_valf(), 0.0f);
    }
    float mx = m;
#pragma unroll
    for (int i = 0; i < kJoinFew; ++i) mx = fmaxf(mx, ml[i].x);
    const float f0 = half_factor(m, mx), f = f0 * f0;
    m = mx;
    l = l * f0 * f0;
    acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
#pragma unroll
    for (int i = 0; i < kJoinFew; ++i) {
      const float w0 = half_factor(ml[i].x, mx), w = w0 * w0;
      l = fmaf(ml[i].y * w0, w0, l);
      acc = make_float4(fmaf(x[i].x, w, acc.x), fmaf(x[i].y, w, acc.y), fmaf(x[i].z, w, acc.z),
                        fmaf(x[i].w, w, acc.w));
    }
  }
  const float r = l == 0.0f ? 0.0f : 1.0f / l;
  uint8_t* dst = static_cast<uint8_t*>(a.out) +
                 ((static_cast<int64_t>(b) * a.num_heads + heads.first + kv * a.group + head) * D +
                  d) * 2;
  *reinterpret_cast<uint2*>(dst) =
      make_uint2(pack_bf16x2(acc.x * r, acc.y * r), pack_bf16x2(acc.z * r, acc.w * r));
}

// ------------------------------------------------------------------------------------- by items

template <int D>
__global__ void __launch_bounds__(kItemWarps * kWarpSize, D == 128 ? 1 : 2) decode_attention_fp8_items(
    const __grid_constant__ AttnArgs a) {
  grid_dependency_sync();
  constexpr int kThreads = kItemWarps * kWarpSize;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float warp_m[kItemWarps][kGroup], warp_l[kItemWarps][kGroup];
  __shared__ float split_m[kGroup], split_l[kGroup];
  const int warp = threadIdx.x / kWarpSize;
  const int lane = threadIdx.x % kWarpSize;
  const int g = lane >> 2;
  const int t = lane & 3;
  using Load = Loader<D, 1>;
  const int item = static_cast<int>(blockIdx.x) / a.splits;
  const int split = static_cast<int>(blockIdx.x) - item * a.splits;
  const int b = item / a.subs, sub = item - b * a.subs;
  const Heads<1> heads(a, sub);
  const uint32_t ring = smem_addr(smem) + warp * kStages * Load::kStageBytes;

  const int n = __ldg(a.seq_lens + b);
  if (threadIdx.x == 0 && (n < 0 || n > a.max_rows)) raise_error(a.err, kErrBadIndex);
  const int len = clamp_len(a, n);
  // this split's steps, which the warps deal among them
  const int of_split = (item_steps(len) + a.splits - 1) / a.splits;
  const int steps = min(item_steps(len), (split + 1) * of_split);
  const int begin = split * of_split + warp;

  int block = Load::block_of(a, b, begin, len);
  uint32_t k_scales[kStages][1], v_scales[kStages][1];
  const auto load = [&](int stage, int step, uint32_t (&k_scale)[1], uint32_t (&v_scale)[1]) {
    if (step < steps) {
      Load::issue(a, ring + stage * Load::kStageBytes, block, heads, step, len, k_scale, v_scale);
      block = Load::block_of(a, b, step + kItemWarps, len);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages; ++i) {
    load(i, begin + i * kItemWarps, k_scales[i], v_scales[i]);
  }
  Queries<D> q;
  const uint8_t* src = static_cast<const uint8_t*>(a.q) +
                       (b * a.q_stride + static_cast<int64_t>(heads.first + g) * D) * 2;
  q.set(a.scale_log2, [&](int i) {
    return g < heads.count ? ld_global_nc_v4(src + i * 16) : make_uint4(0, 0, 0, 0);
  });
  Sums<D, D> sums;
  sums.clear();
  int stage = 0;
  for (int step = begin; step < steps; step += kItemWarps) {
    cp_async_wait<kStages - 1>();
    __syncwarp();
    sums.step(ring + stage * Load::kStageBytes, 0, scales_of(a, k_scales[0][0], v_scales[0][0]),
              len - step * kStepRows, q);
#pragma unroll
    for (int i = 0; i + 1 < kStages; ++i) {
      k_scales[i][0] = k_scales[i + 1][0];
      v_scales[i][0] = v_scales[i + 1][0];
    }
    __syncwarp();  // every lane is done with the stage
    load(stage, step + kStages * kItemWarps, k_scales[kStages - 1], v_scales[kStages - 1]);
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  sums.reduce();
  cp_async_wait<0>();
  __syncthreads();  // the rings are free
  float* accs = reinterpret_cast<float*>(smem);  // [warps][heads][D]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int head = 2 * t + h;
    if (head >= heads.count) continue;
    if (g == 0) {
      warp_m[warp][head] = sums.m[h];
      warp_l[warp][head] = sums.l[h];
    }
    float4* dst = reinterpret_cast<float4*>(accs + (warp * heads.count + head) * D + g * (D / 8));
#pragma unroll
    for (int i = 0; i < D / 16; i += 2) {
      dst[i / 2] = make_float4(sums.acc[i][h], sums.acc[i][2 + h], sums.acc[i + 1][h],
                               sums.acc[i + 1][2 + h]);
    }
  }
  __syncthreads();
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) +
                       (static_cast<int64_t>(b) * a.num_heads + heads.first) * D;
  float* part = accs + kItemWarps * heads.count * D;  // [heads][D], of the split
  for (int idx = threadIdx.x; idx < heads.count * D; idx += kThreads) {
    const int h = idx / D;
    float mx = warp_m[0][h];
#pragma unroll
    for (int w = 1; w < kItemWarps; ++w) mx = fmaxf(mx, warp_m[w][h]);
    float o = 0.0f, ls = 0.0f;
#pragma unroll
    for (int w = 0; w < kItemWarps; ++w) {
      const float f = half_factor(warp_m[w][h], mx);
      o = fmaf(accs[w * heads.count * D + idx], f * f, o);
      ls = fmaf(warp_l[w][h] * f, f, ls);
    }
    if (a.splits == 1) {
      out[idx] = __float2bfloat16_rn(ls == 0.0f ? 0.0f : o / ls);
    } else {
      part[idx] = o;
      if (idx % D == 0) {
        split_m[h] = mx;
        split_l[h] = ls;
      }
    }
  }
  if (a.splits == 1) return;
  // The splits of an item are a thread-block cluster: each joins and writes a slice of the outputs
  // from all of them, through distributed shared memory.
  cluster_sync_all();
  const int per = heads.count * D / a.splits;
  for (int idx = split * per + threadIdx.x; idx < (split + 1) * per; idx += kThreads) {
    const int h = idx / D;
    float m[kMaxSplits], l[kMaxSplits], x[kMaxSplits];
#pragma unroll
    for (int r = 0; r < kMaxSplits; ++r) {
      m[r] = -FLT_MAX;
      l[r] = x[r] = 0.0f;
      if (r < a.splits) {
        m[r] = ld_remote_f32(&split_m[h], r);
        l[r] = ld_remote_f32(&split_l[h], r);
        x[r] = ld_remote_f32(&part[idx], r);
      }
    }
    float mx = m[0];
#pragma unroll
    for (int r = 1; r < kMaxSplits; ++r) mx = fmaxf(mx, m[r]);
    float o = 0.0f, ls = 0.0f;
#pragma unroll
    for (int r = 0; r < kMaxSplits; ++r) {
      const float f = half_factor(m[r], mx);
      o = fmaf(x[r], f * f, o);
      ls = fmaf(l[r] * f, f, ls);
    }
    out[idx] = __float2bfloat16_rn(ls == 0.0f ? 0.0f : o / ls);
  }
  cluster_sync_all();  // every CTA's shared memory stays valid until the others have read it
}

int64_t line_shares(int device) { return static_cast<int64_t>(sm_count(device)) * kLineWarps; }

template <int D>
int launch_items(const AttnArgs& a, int64_t items, int device, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(kItemWarps) * kStages * Loader<D, 1>::kStageBytes;
  static_assert(kItemWarps * kStages * Loader<D, 1>::kStageBytes >= (kItemWarps + 1) * kGroup * D * 4,
                "the merge takes the rings");
  const auto kernel = decode_attention_fp8_items<D>;
  if (blocks_per_sm(reinterpret_cast<const void*>(kernel), kItemWarps * kWarpSize, smem, device) <=
      0) {
    return SVLLM_ERR_CUDA;
  }
  return launch(kernel, dim3(static_cast<unsigned>(items * a.splits)),
                dim3(kItemWarps * kWarpSize), smem, stream, static_cast<unsigned>(a.splits), a);
}

template <int D, int kHeads>
int launch_lines(const AttnArgs& a, int64_t items, int device, cudaStream_t stream) {
  const int heads = a.group < kGroup ? a.group : kGroup;
  const size_t smem = static_cast<size_t>(kLineWarps) * kStages * Loader<D, kHeads>::kStageBytes;
  const auto kernel = decode_attention_fp8_lines<D, kHeads>;
  if (blocks_per_sm(reinterpret_cast<const void*>(kernel), kLineWarps * kWarpSize, smem, device) <=
      0) {
    return SVLLM_ERR_CUDA;
  }
  const unsigned sms = static_cast<unsigned>(sm_count(device));
  const int status =
      launch(kernel, dim3(sms), dim3(kLineWarps * kWarpSize), smem, stream, 1u, a);
  if (status != SVLLM_OK) return status;
  const int64_t parts = line_shares(device) / items + 2;  // of an item of middling length
  if (parts <= kJoinFewParts<D>) {
    const int per_item = kHeads * heads * (D / 4);
    const int a_cta = kJoinThreads / per_item;
    return launch(decode_attention_fp8_join_few<D, kHeads>,
                  dim3(static_cast<unsigned>((items + a_cta - 1) / a_cta)),
                  dim3(static_cast<unsigned>(a_cta * per_item)), 0, stream, 1u, a,
                  static_cast<int>(items), per_item);
  }
  // up to four parts a lane, as far as the warps of a CTA go
  int spread = 1;
  while (spread < kJoinThreads / kWarpSize && parts > 16 * spread) spread *= 2;
  const int runs = kHeads * heads * (D / 32) * spread;
  const unsigned slices = static_cast<unsigned>((runs * kWarpSize + kJoinThreads - 1) / kJoinThreads);
  return launch(decode_attention_fp8_join<D, kHeads>, dim3(static_cast<unsigned>(items), slices),
                dim3(kJoinThreads), 0, stream, 1u, a, spread);
}

// CTAs of an item, by items; 0: by lines. `wave`: how many such CTAs run at a time. Measured, by
// lines and by items (us in a graph, 16/8 heads of 128): 1 request of 100 rows 7.2, 3.6; 1 of 2000
// 8.7, 5.6; 8 of 2000 11.7, 9.9; 16 of 500 9.5, 6.1; 32 of 500, two waves, 11.5, 10.8; but 32 of 1000,
// two waves of four steps, 17.6, 19.1, and 64 of 100, four waves, 10.2, 11.8.
int item_splits(int64_t max_rows, int64_t items, int64_t wave) {
  int splits = 1;
  while (2 * splits <= kMaxSplits && 2 * splits * items <= wave &&
         splits * kItemWarps * kStepRows < max_rows) {
    splits *= 2;
  }
  const int64_t rows = int64_t{splits} * kItemWarps * kStepRows;  // of a step of all warps
  const int64_t steps = max_rows > rows ? (max_rows + rows - 1) / rows : 1;
  const int64_t waves = (items * splits + wave - 1) / wave;
  return waves <= 2 && waves * steps <= kItemSteps ? splits : 0;
}

constexpr int64_t kInt = int64_t{1} << 31;
constexpr int64_t kMaxSeqs = 1 << 20, kMaxHeads = 1 << 16, kMaxBlockSize = 1 << 20;
constexpr int64_t kMaxRows = kInt - kStepRows;

// How a call is dealt to CTAs, and its workspace: none by items.
struct Workspace {
  int64_t side_by_side;  // KV heads of an item
  int64_t subs;          // items of a request
  int64_t items, splits, ml, acc, bytes;
  Workspace(int64_t num_seqs, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
            int64_t max_rows, int device) {
    const int64_t group = num_heads / num_kv_heads;
    const int64_t groups = (group + kGroup - 1) / kGroup;
    const int64_t held = group < kGroup ? group : kGroup;
    ml = acc = bytes = 0;
    side_by_side = 1;
    // shared memory leaves room for one CTA by items on an SM at head_dim 128, registers for two at 64
    subs = num_kv_heads * groups;
    items = num_seqs * subs;
    splits = item_splits(max_rows, items, sm_count(device) * (head_dim == 128 ? 1 : 2));
    if (splits > 0) return;
    const int64_t steps = items * ((max_rows + kStepRows - 1) / kStepRows) / line_shares(device);
    side_by_side = head_dim == 64 && steps >= kPairSteps ? kPair : 1;
    subs = (num_kv_heads + side_by_side - 1) / side_by_side * groups;
    items = num_seqs * subs;
    const int64_t parts = 2 * line_shares(device) * side_by_side * held;
    ml = round_up(items * static_cast<int64_t>(sizeof(JoinEntry)), 256);
    acc = ml + round_up(parts * static_cast<int64_t>(sizeof(float2)), 256);
    bytes = acc + parts * head_dim * static_cast<int64_t>(sizeof(float));
  }
};

}  // namespace
}  // namespace svllm::k

extern "C" int svllm_decode_attention_fp8_workspace_bytes(int64_t num_seqs, int64_t num_heads,
                                                          int64_t num_kv_heads, int64_t head_dim,
                                                          int64_t max_blocks, int64_t block_size,
                                                          int64_t* bytes) {
  using namespace svllm::k;
  if (bytes == nullptr || num_seqs < 0 || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads % num_kv_heads != 0 || max_blocks < 0 || block_size <= 0) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  if (head_dim != 64 && head_dim != 128) return SVLLM_ERR_UNSUPPORTED;
  if (num_seqs >= kMaxSeqs || num_heads > kMaxHeads || max_blocks >= kInt ||
      block_size >= kMaxBlockSize || max_blocks * block_size >= kMaxRows) {
    return SVLLM_ERR_TOO_LARGE;
  }
  int device;
  if (current_device(&device) != SVLLM_OK) return SVLLM_ERR_CUDA;
  *bytes = Workspace(num_seqs, num_heads, num_kv_heads, head_dim, max_blocks * block_size, device)
               .bytes;
  return SVLLM_OK;
}

extern "C" int svllm_decode_attention_fp8_bf16(
    void* out, const void* q, int64_t q_token_stride, const void* k_cache, const void* v_cache,
    const void* k_scale, const void* v_scale, int64_t num_blocks, int64_t block_size,
    const int32_t* block_tables, int64_t max_blocks, const int32_t* seq_lens, int64_t num_seqs,
    int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, float scale, void* workspace,
    int64_t workspace_bytes, svllm_stream stream) {
  using namespace svllm::k;
  if (num_seqs < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      block_size <= 0 || max_blocks < 0 || num_blocks <= 0 || head_dim <= 0 ||
      q_token_stride < num_heads * head_dim || !(scale > 0.0f) ||
      !std::isfinite(static_cast<float>(static_cast<double>(scale) / std::log(2.0)))) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  if (num_seqs == 0) return SVLLM_OK;
  if (out == nullptr || q == nullptr || k_cache == nullptr || v_cache == nullptr ||
      k_scale == nullptr || v_scale == nullptr || (max_blocks > 0 && block_tables == nullptr) ||
      seq_lens == nullptr) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  const int64_t group = num_heads / num_kv_heads;
  const int64_t groups = (group + kGroup - 1) / kGroup;
  if (num_heads > kMaxHeads || block_size >= kMaxBlockSize || max_blocks >= kInt ||
      max_blocks * block_size >= kMaxRows || num_blocks >= kInt ||
      num_blocks * block_size >= kInt || num_seqs >= kMaxSeqs ||
      // the line's steps, were every request as long as its table
      num_seqs * num_kv_heads * groups * (max_blocks * block_size / kStepRows + 1) >= kInt) {
    return SVLLM_ERR_TOO_LARGE;
  }
  if ((head_dim != 64 && head_dim != 128) || !aligned16(out) || !aligned16(q) || !aligned16(k_cache) ||
      !aligned16(v_cache) || q_token_stride % 8 != 0) {
    return SVLLM_ERR_UNSUPPORTED;
  }
  int device;
  if (current_device(&device) != SVLLM_OK) return SVLLM_ERR_CUDA;
  const Workspace w(num_seqs, num_heads, num_kv_heads, head_dim, max_blocks * block_size, device);
  if (w.bytes > 0 && (workspace == nullptr || workspace_bytes < w.bytes || !aligned16(workspace))) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
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
  a.subs = static_cast<int>(w.subs);
  a.scale_log2 = static_cast<float>(static_cast<double>(scale) / std::log(2.0));
  a.num_seqs = static_cast<int>(num_seqs);
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (w.splits > 0) {
    a.splits = static_cast<int>(w.splits);
    return head_dim == 128 ? launch_items<128>(a, w.items, device, s)
                           : launch_items<64>(a, w.items, device, s);
  }
  a.shares = static_cast<int>(line_shares(device));
  uint8_t* base = static_cast<uint8_t*>(workspace);
  a.table = reinterpret_cast<JoinEntry*>(base);
  a.part_ml = reinterpret_cast<float2*>(base + w.ml);
  a.part_acc = reinterpret_cast<float*>(base + w.acc);
  if (head_dim == 128) return launch_lines<128, 1>(a, w.items, device, s);
  return w.side_by_side == kPair ? launch_lines<64, kPair>(a, w.items, device, s)
                                 : launch_lines<64, 1>(a, w.items, device, s);
}
