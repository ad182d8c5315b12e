// Attention of a step's tokens over a paged KV cache that holds the step's own rows too: the
// nodes of a tree of drafted tokens see the request's context and their ancestors.
//
//   o[t, h] = sum_j p_j v_j,  p = softmax_j(scale * q[t, h] . k_j),
//   j < context, or j = context + node with the node's bit in tree_mask[t]
//
// The query heads of a KV head share its cached rows, so a request's n tokens make n * G query
// rows per KV head (G = heads / KV heads), and the cache is read once per 128 or 256 of them. At
// R rows a cached row of D elements costs 4 R D operations and 4 D bytes: up to the R of a few
// hundred where the tensor pipe becomes the bound (1616 TFLOP/s against 6.55 TB/s: 247), the
// stream over K and V is what bounds this kernel.
//
// Work: rows come in M tiles of 128 (row = node * G + head), cached rows in tiles of 128. An item
// is either two M tiles of one (request, KV head), which share every K and V tile, or, for a last
// odd M tile, that tile of two neighbouring KV heads. Items times their key tiles form one line of
// steps; each CTA (one per SM) computes the line's length from the request lengths and takes an
// equal share, so ragged batches and single long requests fill the GPU alike and the host needs no
// lengths. An item cut by a share's border leaves unnormalised partial sums in the workspace, which
// a second small kernel joins.
//
// In a CTA: two or four warps bring K and V rows through the block table with TMA into
// 128-byte-swizzled tiles (any block size: a page may end anywhere in a tile); one thread issues
// tcgen05.mma: S = Q K^T into TMEM, then O += P V with P read from TMEM and V as the N-major
// operand, alternating between two accumulators so that the tensor pipe works on one M tile while
// the other's softmax runs; two groups of 4 warps do the softmax, one thread per row, and write P
// (bf16, as the second product takes it) over S. The running maximum is a reference that moves only
// when a row exceeds it by 2^8, so O in TMEM is seldom rescaled; the sums are fp32 and the result
// does not depend on the reference. Masked scores are replaced after the product. Four or two
// helper warps bring the query rows and, since 0 * NaN would reach rows that do not see it, zero
// the values of V that are not finite in the tiles that hold tree nodes; they are added again, for
// the rows that see them, at the end. One warp lists the CTA's segments for all others.
//
// Measured in a graph, inputs past L2, head_dim 128: 64 requests of 48 to 64 nodes over 2048 to
// 4096 rows, 16 heads on 8 KV heads, 203 us (1.08 GB, 5.3 TB/s: 0.82 of the copy rate; 219 to 237
// under a load that runs into the power limit). The main kernel takes 185 of them, in steady state
// at the copy rate, a tenth of it start and ends of segments; the join takes the rest. 8 requests
// of 100 to 128 nodes over 1024 to 4096, 32 heads on 4 KV heads, 86 us (0.75 PFLOP/s), main kernel
// 73: a KV head's rows go to four items, 5.6 TB/s through L2, and a step takes 3500 cycles where
// its products take 2048: per accumulator those and the softmax (1580 cycles, 1260 of them the
// exponentials) wait for each other. Parts of 64 cached rows with their scores a part ahead took
// 119: products of N = 64 take as long as those of 128. 32 nodes over 32768 rows 41 us, 20 of them
// the stream, 10 the join of some 37 segments per item. 8 nodes over 128 rows 8.2 us: one tile's
// chain of dependent steps, most of it the first fetch of the roles' code; 10.2 where the table is
// wider, since a join is launched then (whole_items). Without a mask a prompt of 4096 tokens, 16
// heads on 8 KV heads, takes 161 us: every item goes over all rows of its request, although those
// past its last node are masked, up to half of them.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstring>

#include "common.cuh"
#include "host_common.h"
#include "umma.cuh"

namespace svllm::k {
namespace {

constexpr int kTile = 128;            // query rows per M tile, cached rows per key tile
constexpr int kSoftmaxWarps = 8;      // two groups of 4: accumulators 0 and 1
constexpr int kSideWarps = 6;         // helpers (query rows, check of V), then loaders (K, V)
constexpr int kMmaWarp = kSoftmaxWarps + kSideWarps;
constexpr int kPlanWarp = kMmaWarp + 1;  // lists the CTA's segments, zeroes rows without an item
constexpr int kThreads = (kPlanWarp + 1) * kWarpSize;
constexpr int kWarps = kThreads / kWarpSize;
// Registers per thread after the split of the launch's 512 x 128: the softmax warps hold a row of
// scores each, 8 x 32 x 192 + 8 x 32 x 64 = 65536.
constexpr int kSoftmaxRegisters = 192, kOtherRegisters = 64;
constexpr int kHalfBytes = kTile * 128;  // 128 rows of one 128-byte swizzle atom
constexpr uint32_t kTmemColumns = 512;
constexpr uint32_t kScores = 0;       // TMEM columns: S (and P) of accumulator w at 128 w,
constexpr uint32_t kOutput = 256;     // O at 256 + 128 w
constexpr float kRescaleAbove = 8.0f;  // in powers of two
constexpr int kJoinThreads = 2;       // of a join block, per element of head_dim
// Boxes of fewer rows than this take four loaders and two helpers, others two and four. us with two
// and four loaders: 12-row pages (boxes of 4), the 64 requests above 268 and 213, 32 chains of 5
// nodes 65 and 50, 13 short requests 22.7 and 23.4; 8-row pages 214 and 207, 50 and 44, but 1
// request of 8 nodes 8.7 and 9.3, 8 of up to 128 86 and 90; 16-row pages no gain.
constexpr int kSmallBox = 8;
constexpr int kMaxCtas = 256;         // one per SM; the join lists their borders

template <int D>
struct Shape {
  static constexpr int kHalves = D / 64;
  static constexpr int kTileBytes = kHalves * kHalfBytes;
  static constexpr int kStages = D == 128 ? 5 : 10;
  static constexpr size_t kSmem = 1024 + static_cast<size_t>(kTileBytes) * (2 + kStages);
  // partial sums of one accumulator: O as [D / 4][128 rows][4], then the rows' maxima and sums
  static constexpr int kPartFloats = (D + 2) * kTile;
};

// A segment whose item is cut, for the join: what one word says of it (0: nothing to join; else
// kCut, the ends that are cut, and the rows of each accumulator), and where its rows go.
struct Cut {
  int token0;                      // the request's first token
  int kv_head[2], row0[2];         // per accumulator
};
constexpr int kCut = 1, kCutFront = 2, kCutBack = 4, kCutRows = 3, kCutRowBits = 8;

__device__ __forceinline__ int cut_rows(int mark, int w) {
  return (mark >> (kCutRows + kCutRowBits * w)) & ((1 << kCutRowBits) - 1);
}

struct TreeAttnArgs {
  void* out;                       // [num_tokens, num_heads, head_dim] bf16, contiguous
  const void* q;                   // [num_tokens, num_heads, head_dim] bf16, token stride q_stride
  const void* k_cache;             // [num_blocks, block_size, num_kv_heads, head_dim] bf16
  const void* v_cache;
  const int32_t* block_tables;     // [num_seqs, max_blocks]
  const int32_t* seq_lens;         // [num_seqs]
  const int32_t* query_start_loc;  // [num_seqs + 1]
  const int64_t* tree_mask;        // [num_tokens, mask_words] or null: causal
  float* parts;                    // [CTAs][2][2] partial sums
  int* marks;                      // [CTAs][2]: a CTA's first and last segment
  Cut* cuts;                       // [CTAs][2]
  int64_t q_stride;
  int64_t num_blocks;
  int num_tokens;
  int num_seqs;
  int max_blocks;
  int max_length;                  // rows that a block table holds
  int max_nodes;                   // nodes that the mask's words hold
  int whole;                       // 1: items are not cut
  int block_size;
  Divider page;                    // by the block size
  int group;                       // query heads per KV head
  Divider by_group;
  int num_kv_heads;
  int cache_slots;
  int box_rows;                    // rows of a TMA box; 1: four rows gathered per instruction
  int mask_words;
  float scale_log2;                // scale * log2(e): scores are kept in powers of two
  int* err;
};

// One request's share of the line. Valid lengths only: anything else has no items.
struct Request {
  int start, nodes, context, length;  // first token, tokens, earlier rows, all rows
  int steps;                          // key tiles
  int pairs;                          // items of two M tiles per KV head
  int odd;                            // 1: a last single M tile, in items of two KV heads
  bool bad;                           // starts or lengths out of range
  bool astray;                        // starts that fall or lie outside the tokens
};

__device__ __forceinline__ Request load_request(const TreeAttnArgs& a, int s) {
  Request r{};
  const int begin = a.query_start_loc[s], end = a.query_start_loc[s + 1];
  const int length = a.seq_lens[s];
  if (begin < 0 || end < begin || end > a.num_tokens) {
    r.bad = r.astray = true;
    return r;
  }
  r.start = begin;
  r.nodes = end - begin;
  if (length == 0) return r;
  if (length < r.nodes || length > a.max_length || r.nodes > a.max_nodes) {
    r.bad = true;
    return r;
  }
  r.length = length;
  r.context = length - r.nodes;
  if (r.nodes > 0) {
    const int tiles = (r.nodes * a.group + kTile - 1) / kTile;
    r.steps = (length + kTile - 1) / kTile;
    r.pairs = tiles / 2;
    r.odd = tiles & 1;
  }
  return r;
}

// Steps of the line, weighted: a step over two KV heads loads twice what the others load.
__device__ __forceinline__ int request_cost(const TreeAttnArgs& a, const Request& r) {
  return a.num_kv_heads * r.steps * (r.pairs + r.odd);
}

// Costs of requests whose starts rise from 0 add up to an int (checked on the host from the sizes).
// Of others, of which nothing is done, the sum stops at the largest int instead of wrapping.
__device__ __forceinline__ int add_costs(int a, int b) {
  return static_cast<int>(min(static_cast<unsigned>(a) + static_cast<unsigned>(b),
                              static_cast<unsigned>(INT32_MAX)));
}

// A place on the line: request, item of the request, step of the item.
struct Place {
  int s, item, step;
};

__device__ __forceinline__ Place locate(const TreeAttnArgs& a, int s, const Request& r, int at) {
  // items of two M tiles first, of steps that weigh 1; then two KV heads' last tiles, steps of 2
  const int shared = a.num_kv_heads * r.pairs * r.steps;
  const int weight = at < shared ? 1 : 2;
  if (weight == 2) at -= shared;
  const unsigned length = weight * r.steps;
  Place p{s, static_cast<int>(at / length), 0};
  const int rest = at - p.item * static_cast<int>(length);
  if (weight == 2) {
    // a last odd KV head is alone in its item, whose steps weigh 1
    p.step = 2 * p.item + 1 < a.num_kv_heads ? (rest + 1) / 2 : rest;
    p.item += a.num_kv_heads * r.pairs;
    if (p.step == r.steps) {  // rounded up to the item's end
      ++p.item;
      p.step = 0;
    }
  } else {
    p.step = rest;
  }
  return p;
}

// A run of steps of one item. The plan warp lists a CTA's segments in a ring; the other warps copy
// one at a time.
struct Segment {
  int s, start, nodes, context, length;  // the request
  int shared;                    // both accumulators take the same K and V
  int active;                    // accumulators in use, 1 or 2; 0: the end of the list
  int kv_head[2], row0[2], rows[2];
  int lane0;                     // where accumulator 1's rows begin in its tile
  int step0, step1;
  int front, back;               // cut there
};

// Barriers and flags of one CTA. A V tile with tree nodes lands on its own barrier, for the
// helpers, which signal when it is checked; kFull stands for all other tiles. (A slot's parity
// counts the uses of one barrier, so every waiter of a barrier has to see all of them.)
constexpr int kMaxStages = 10;
constexpr int kSegments = 4;    // of the list's ring
constexpr int kFull = 0, kLanded = kFull + kMaxStages;
constexpr int kChecked = kLanded + kMaxStages, kFullQ = kChecked + kMaxStages;
constexpr int kEmpty = kFullQ + 1, kEmptyQ = kEmpty + kMaxStages;
constexpr int kScoresDone = kEmptyQ + 1, kWeightsDone = kScoresDone + 2;
constexpr int kOutputDone = kWeightsDone + 2, kDrain = kOutputDone + 2;
constexpr int kListed = kDrain + 1, kRead = kListed + kSegments, kBarriers = kRead + kSegments;

__device__ __forceinline__ int arrivals(int bar, int helpers) {
  if (bar < kChecked) return kSideWarps - helpers;
  if (bar < kEmpty) return helpers * kWarpSize;
  if (bar >= kRead) return kPlanWarp;  // every other warp
  return bar == kWeightsDone || bar == kWeightsDone + 1 ? 4 * kWarpSize : 1;
}

struct Sync {
  uint64_t bar[kBarriers];
  uint32_t tmem_base;
  int abort;
  // per helper warp, accumulator and segment modulo 8: V held something not finite. A warp clears
  // its own word when it begins a segment; no warp is more than kSegments behind another then, so
  // nobody still reads the one that the segment 8 before left there.
  int odd_values[kSideWarps][2][2 * kSegments];
  int costs[kWarps];     // of the warps' shares of the requests
  Segment list[kSegments];
};

// The warp waits for a phase together: true for all lanes, or false for all once the pipeline is
// aborting. The roles' loops are long straight code, bound by instruction fetch, so the common case
// is a few instructions: a short loop of bounded tries; only then the abort flag and the clock.
__device__ __forceinline__ bool warp_wait(Sync& sy, int bar, uint32_t parity, int* err) {
  const uint32_t at = smem_addr(&sy.bar[0]) + bar * 8;
  uint64_t start = 0;
  while (true) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\t"
        "mov.u32 n, 64;\n\t"
        "TRY:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "@p bra DONE;\n\t"
        "sub.u32 n, n, 1;\n\t"
        "setp.ne.u32 q, n, 0;\n\t"
        "@q bra TRY;\n\t"
        "DONE:\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(at), "r"(parity)
        : "memory");
    if (__all_sync(0xffffffffu, done != 0)) return true;
    const uint64_t now = global_timer_ns();
    if (start == 0) start = now;
    if (now - start > kWaitLimitNs) {
      sy.abort = 1;
      raise_error(err, kErrWaitTimeout);
    }
    if (__any_sync(0xffffffffu, *static_cast<volatile int*>(&sy.abort) != 0)) return false;
  }
}

// Inclusive sum of costs over the warp's lanes.
__device__ __forceinline__ int sum_up_to_lane(int v, int lane) {
#pragma unroll
  for (int off = 1; off < kWarpSize; off *= 2) {
    const int up = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v = add_costs(v, up);
  }
  return v;
}

// The borders of this CTA's share of the line. `own`: lane i holds the cost of the i-th `chunk` of
// requests; with a chunk of 1, `r` is the lane's request. `astray`: the starts do not rise from 0
// to at most the number of tokens, so no request has items.
__device__ __forceinline__ void find_share(const TreeAttnArgs& a, Request r, int own, int chunk,
                                           bool astray, int lane, Place (&places)[2]) {
  const int upto = sum_up_to_lane(own, lane);
  const int total = astray ? 0 : __shfl_sync(0xffffffffu, upto, kWarpSize - 1);
  // at least two steps each: a shorter share costs more in the join than it saves (1 request of 8
  // nodes over 128 rows: 12.7 us with 2, 16.4 with 4; 13 requests of up to 37 nodes 27 and 38)
  const int share = max(2, static_cast<int>((total + gridDim.x - 1u) / gridDim.x));
#pragma unroll 1
  for (int e = 0; e < 2; ++e) {
    const int64_t border = static_cast<int64_t>(blockIdx.x + e) * share;
    Place p{a.num_seqs, 0, 0};
    if (border < total) {
      // the lane whose chunk of requests holds it, then the request
      int owner = __ffs(static_cast<int>(__ballot_sync(0xffffffffu, border < upto))) - 1;
      int before = __shfl_sync(0xffffffffu, upto - own, owner);
      int s = owner, cost = own;
      if (chunk > 1) {
        const int end = min(a.num_seqs, (owner + 1) * chunk);
#pragma unroll 1
        for (int s0 = owner * chunk;; s0 += kWarpSize) {
          s = s0 + lane;
          r = Request{};
          if (s < end) r = load_request(a, s);
          cost = request_cost(a, r);
          const int sum = add_costs(before, sum_up_to_lane(cost, lane));
          const unsigned past = __ballot_sync(0xffffffffu, border < sum);
          if (past != 0) {
            owner = __ffs(static_cast<int>(past)) - 1;
            s = s0 + owner;
            before = __shfl_sync(0xffffffffu, sum - cost, owner);
            break;
          }
          before = __shfl_sync(0xffffffffu, sum, kWarpSize - 1);
        }
      }
      if (lane == owner) p = locate(a, s, r, static_cast<int>(border) - before);
      if (a.whole && p.step > 0) {  // on to the next item
        ++p.item;
        p.step = 0;
      }
      p.s = __shfl_sync(0xffffffffu, p.s, owner);
      p.item = __shfl_sync(0xffffffffu, p.item, owner);
      p.step = __shfl_sync(0xffffffffu, p.step, owner);
    }
    if (e == 0) places[0] = p;
    places[1] = p;
  }
}

// The plan warp: lists the segments of [at, end).
__device__ __forceinline__ void plan(const TreeAttnArgs& a, Sync& sy, Place at, const Place end,
                                     int lane) {
  Request r{};
  int loaded = -1;
  const auto list = [&](int index, const Segment& g) {
    const int slot = index % kSegments;
    if (!warp_wait(sy, kRead + slot, (index / kSegments & 1) ^ 1, a.err)) return false;
    if (lane == 0) {
      sy.list[slot] = g;
      mbar_arrive(&sy.bar[kListed + slot]);
    }
    return true;
  };
  int index = 0;
#pragma unroll 1
  while (at.s < a.num_seqs &&
         (at.s < end.s || (at.s == end.s && (at.item < end.item ||
                                             (at.item == end.item && at.step < end.step))))) {
    if (at.s != loaded) {
      r = load_request(a, at.s);
      loaded = at.s;
    }
    const int shared_items = a.num_kv_heads * r.pairs;
    const int items = r.steps == 0 ? 0 : shared_items + r.odd * ((a.num_kv_heads + 1) / 2);
    if (at.item >= items) {
      at = Place{at.s + 1, 0, 0};
      continue;
    }
    Segment g;
    g.s = at.s;
    g.start = r.start;
    g.nodes = r.nodes;
    g.context = r.context;
    g.length = r.length;
    g.shared = at.item < shared_items;
    const int all_rows = r.nodes * a.group;
    if (g.shared) {
      g.active = 2;
      g.kv_head[0] = g.kv_head[1] = at.item / r.pairs;
      g.row0[0] = (at.item - g.kv_head[0] * r.pairs) * 2 * kTile;
      g.row0[1] = g.row0[0] + kTile;
      g.rows[0] = kTile;
      g.rows[1] = min(kTile, all_rows - g.row0[1]);
    } else {
      g.kv_head[0] = 2 * (at.item - shared_items);
      g.kv_head[1] = g.kv_head[0] + 1;
      g.active = g.kv_head[1] < a.num_kv_heads ? 2 : 1;
      g.row0[0] = g.row0[1] = r.pairs * 2 * kTile;
      g.rows[0] = all_rows - g.row0[0];
      g.rows[1] = g.active == 2 ? g.rows[0] : 0;
    }
    // one warp of each group works on up to 32 rows: not two that share a scheduler
    g.lane0 = g.rows[1] <= kTile / 2 ? kTile / 2 : 0;
    g.step0 = at.step;
    g.step1 = at.s == end.s && at.item == end.item ? end.step : r.steps;
    g.front = g.step0 > 0;
    g.back = g.step1 < r.steps;
    if (!list(index, g)) return;
    ++index;
    at = Place{at.s, at.item + 1, 0};
  }
  Segment none{};
  list(index, none);
}

// One of a pair, without an address: the array stays in registers.
__device__ __forceinline__ int pick(const int (&pair)[2], int w) {
  return w == 0 ? pair[0] : pair[1];
}

// The list's segment `index`, for a warp that reads them all in order; false at its end.
__device__ __forceinline__ bool next_segment(const TreeAttnArgs& a, Sync& sy, int index,
                                             Segment& g) {
  const int slot = index % kSegments;
  if (!warp_wait(sy, kListed + slot, index / kSegments & 1, a.err)) return false;
  // broadcast from one lane, so that the compiler knows the warp agrees on them
  constexpr int kWords = sizeof(Segment) / sizeof(int);
  const int* from = reinterpret_cast<const int*>(&sy.list[slot]);
  int words[kWords];
#pragma unroll
  for (int i = 0; i < kWords; ++i) words[i] = __shfl_sync(0xffffffffu, from[i], 0);
  memcpy(&g, words, sizeof(Segment));
  if (threadIdx.x % kWarpSize == 0) mbar_arrive(&sy.bar[kRead + slot]);
  return g.active > 0;
}

// A ring of tiles: the slot in use and the parity of its current round.
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void advance(int stages) {
    if (++slot == stages) {
      slot = 0;
      phase ^= 1;
    }
  }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src)
               : "memory");
}

// Arrives on `bar` (one of its counted arrivals) once this thread's copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar))
               : "memory");
}

__device__ __forceinline__ void cp_async_wait_all() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Zeroes the non-finite halves of a word of two bf16; true if there were any.
__device__ __forceinline__ bool drop_odd(uint32_t& w) {
  const bool lo = (w & 0x7f80u) == 0x7f80u, hi = (w & 0x7f800000u) == 0x7f800000u;
  if (lo) w &= 0xffff0000u;
  if (hi) w &= 0x0000ffffu;
  return lo || hi;
}

// The V tiles of these steps hold tree nodes.
__device__ __forceinline__ bool has_nodes(const Segment& g, int step) {
  return (step + 1) * kTile > g.context;
}

// One of the warps that bring K and V, tile after tile in the order in which the tensor cores take
// them: every kLoaderWarps-th TMA instruction of each tile (one costs its issuer some 60 cycles, a
// tile of 16-row pages has 16). Where the block size allows, a TMA box is a run of 4 to 128 rows
// that no page border can fall into, gcd(block_size, 128); otherwise an instruction gathers 4 rows.
// With 12-row pages and two loaders the 64 requests above took 268 us in boxes of 4 rows and 329
// gathered; with pages of one row the gather takes 254 with four loaders. Copies of 16 bytes per
// thread (cp.async) took 290 there and more than the gather in every smaller case. Issued by all
// lanes at once, each its own rows, the gather took 603.
template <int D, int kLoaderWarps>
struct Loader {
  using S = Shape<D>;
  const TreeAttnArgs& a;
  Sync& sy;
  const CUtensorMap& map_k;
  const CUtensorMap& map_v;
  uint8_t* ring;
  int part, lane;        // part 0 .. kLoaderWarps - 1 of every tile
  Ring at{};
  uint64_t used = 0, parity = 0;  // barriers signalled so far, and the parity of their next use

  // The cache slot of row j of the request; past its end a slot past the cache, which reads as
  // zeros.
  __device__ __forceinline__ int cache_slot(const Segment& g, int j) const {
    if (j >= g.length) return a.cache_slots;
    const int page = a.page.divide(j);
    int block = a.block_tables[static_cast<int64_t>(g.s) * a.max_blocks + page];
    if (static_cast<uint64_t>(block) >= static_cast<uint64_t>(a.num_blocks)) {
      raise_error(a.err, kErrBadIndex);  // outside the cache: block 0 is read
      block = 0;
    }
    return block * a.block_size + (j - page * a.block_size);
  }

  // This lane's rows of key tile `step`: the first of box `lane`, or four rows from 4 * lane on.
  __device__ __forceinline__ void find_rows(const Segment& g, int step, int (&rows)[4]) const {
    if (step >= g.step1) return;
    if (a.box_rows > 1) {
      const int j = lane * a.box_rows;
      if (j < kTile) rows[0] = cache_slot(g, step * kTile + j);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) rows[i] = cache_slot(g, step * kTile + 4 * lane + i);
    }
  }

  // This warp's part of one tile into the ring's next slot.
  __device__ __forceinline__ bool load(const CUtensorMap* map, int full, const int (&rows)[4],
                                       int kv_head) {
    if (!warp_wait(sy, kEmpty + at.slot, at.phase ^ 1, a.err)) return false;
    // boxes (or groups of 4 rows) part, part + kLoaderWarps, ..., both halves of a row together
    const int rows_each = a.box_rows > 1 ? a.box_rows : 4;
    const int count = kTile / rows_each;
    const int mine = (count - part + kLoaderWarps - 1) / kLoaderWarps;
    uint64_t* bar = &sy.bar[full + at.slot];
    const uint32_t dst = smem_addr(ring + at.slot * S::kTileBytes);
    const int column = kv_head * D;
    if (elect_one()) mbar_arrive_expect_tx(bar, mine * rows_each * 128 * S::kHalves);
    __syncwarp();
    if (a.box_rows > 1) {
#pragma unroll 1
      for (int i = part; i < count; i += kLoaderWarps) {
        const int row = __shfl_sync(0xffffffffu, rows[0], i);
        if (elect_one()) {
#pragma unroll
          for (int h = 0; h < S::kHalves; ++h) {
            tma_load_2d(dst + h * kHalfBytes + i * rows_each * 128, map,
                        column + h * kTmaBoxCols, row, bar);
          }
        }
      }
    } else {
#pragma unroll 1
      for (int i = part; i < kTile / 4; i += kLoaderWarps) {
        int32_t y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = __shfl_sync(0xffffffffu, rows[e], i);
        if (elect_one()) {
#pragma unroll
          for (int h = 0; h < S::kHalves; ++h) {
            tma_gather4(dst + h * kHalfBytes + i * 512, map, column + h * kTmaBoxCols, y, bar);
          }
        }
      }
    }
    used |= uint64_t{1} << (full + at.slot);
    parity ^= uint64_t{1} << (full + at.slot);
    at.advance(S::kStages);
    return true;
  }

  __device__ __forceinline__ void run() {
    Segment g;
    bool ok = true;
#pragma unroll 1
    for (int index = 0; ok && next_segment(a, sy, index, g); ++index) {
      const int heads = g.shared ? 1 : g.active;
      int before[4] = {}, now[4] = {}, next[4] = {};
#pragma unroll 1
      for (int step = g.step0 - 1; ok && step <= g.step1; ++step) {
        find_rows(g, step + 1, next);
        // V of the step before, then K, head by head
#pragma unroll 1
        for (int i = 0; ok && step >= g.step0 && i < 2 * heads; ++i) {
          const bool values = i % 2 == 0;
          if (values ? step == g.step0 : step == g.step1) continue;
          int rows[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) rows[e] = values ? before[e] : now[e];
          ok = load(values ? &map_v : &map_k,
                    values && has_nodes(g, step - 1) ? kLanded : kFull, rows,
                    i < 2 ? g.kv_head[0] : g.kv_head[1]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          before[e] = now[e];
          now[e] = next[e];
        }
      }
    }
    // every copy has landed before the CTA exits: the last use of each barrier
#pragma unroll 1
    for (int bar = 0; bar < kChecked; ++bar) {
      if ((used >> bar) & 1) mbar_wait_bounded(&sy.bar[bar], ((parity >> bar) & 1) ^ 1);
    }
  }
};
static_assert(kChecked <= 64, "one bit per barrier that a copy may signal");

// The helper warps: the query rows of each segment, and the V tiles that hold tree nodes,
// whose values that are not finite are zeroed before the tensor cores see them.
template <int D, int kHelperWarps>
__device__ __forceinline__ void help(const TreeAttnArgs& a, Sync& sy, uint8_t* q_tiles,
                                     uint8_t* ring, int warp, int lane) {
  using S = Shape<D>;
  constexpr int kLanes = D / 8;  // lanes per query row: 16 bytes each
  constexpr int kRowsAtOnce = kWarpSize / kLanes;
  const auto wait = [&](int bar, uint32_t parity) {
    return warp_wait(sy, bar, parity, a.err);
  };
  Ring ring_at;
  uint32_t landed = 0;  // parity of the next use of each slot's barrier
  Segment g;
  bool ok = true;
#pragma unroll 1
  for (int index = 0; ok && next_segment(a, sy, index, g); ++index) {
    ok = wait(kEmptyQ, (index & 1) ^ 1);
    if (!ok) break;
    if (lane < 2) sy.odd_values[warp][lane][index % (2 * kSegments)] = 0;
    __syncwarp();
#pragma unroll 1
    for (int w = 0; w < g.active; ++w) {
      // row = node * group + head of the KV head; what lies outside the request's rows of the tile
      // stays as it was: nothing reads the products of those
      const int rows = pick(g.rows, w), lane0 = w == 0 ? 0 : g.lane0, c = lane % kLanes;
      const uint32_t base = smem_addr(q_tiles + w * S::kTileBytes) + (c / 8) * kHalfBytes;
      const auto* src = static_cast<const __nv_bfloat16*>(a.q) + c * 8;
      // the warps share the rows, up to 32 at a time, whose places a lane each works out
      const int share = (rows + kHelperWarps - 1) / kHelperWarps;
      const int block =
          min(kWarpSize, (share + kRowsAtOnce - 1) / kRowsAtOnce * kRowsAtOnce);
#pragma unroll 1
      for (int r0 = warp * block; r0 < rows; r0 += kHelperWarps * block) {
        const int row = pick(g.row0, w) + min(r0 + lane, rows - 1);
        const int node = a.by_group.divide(row);
        const int64_t offset =
            (g.start + node) * a.q_stride +
            (static_cast<int64_t>(pick(g.kv_head, w) - node) * a.group + row) * D;
        const int count = min(block, rows - r0);
#pragma unroll 4
        for (int i = 0; i < count; i += kRowsAtOnce) {
          const int r = i + lane / kLanes, x = lane0 + r0 + r;
          const int64_t from = __shfl_sync(0xffffffffu, offset, r);
          if (r < count) cp_async16(base + x * 128 + (((c % 8) ^ (x & 7)) << 4), src + from);
        }
      }
    }
    cp_async_arrive(&sy.bar[kFullQ]);
#pragma unroll 1
    for (int step = g.step0; ok && step <= g.step1; ++step) {
#pragma unroll 1
      for (int w = 0; ok && w < (g.shared ? 1 : g.active); ++w) {
        if (step > g.step0) {
          if (has_nodes(g, step - 1)) {
            ok = wait(kLanded + ring_at.slot, (landed >> ring_at.slot) & 1);
            if (!ok) break;
            landed ^= 1u << ring_at.slot;
            auto* tile = reinterpret_cast<uint4*>(ring + ring_at.slot * S::kTileBytes);
            // rows of the tile that are nodes, and behind them whatever the pages hold
            const int first_row = max(0, g.context - (step - 1) * kTile);
            const int end_row = g.length - (step - 1) * kTile;
            bool odd = false;
#pragma unroll 1
            for (int h = 0; h < S::kHalves; ++h) {
#pragma unroll 4
              for (int i = first_row * 8 + warp * kWarpSize + lane; i < kHalfBytes / 16;
                   i += kHelperWarps * kWarpSize) {
                uint4& at = tile[h * (kHalfBytes / 16) + i];
                uint4 x = at;
                if (i / 8 >= end_row) {
                  at = make_uint4(0, 0, 0, 0);
                } else if (drop_odd(x.x) | drop_odd(x.y) | drop_odd(x.z) | drop_odd(x.w)) {
                  at = x;
                  odd = true;
                }
              }
            }
            if (odd) {
              sy.odd_values[warp][w][index % (2 * kSegments)] = 1;
              if (g.shared) sy.odd_values[warp][1][index % (2 * kSegments)] = 1;
            }
            fence_proxy_async_smem();
            mbar_arrive(&sy.bar[kChecked + ring_at.slot]);
          }
          ring_at.advance(S::kStages);
        }
        if (step < g.step1) ring_at.advance(S::kStages);  // a K tile
      }
    }
  }
  cp_async_wait_all();  // also after an abort: no copy is in flight when the CTA exits
}

// The warp that issues the matrix products, one lane of it each of them.
template <int D>
__device__ __forceinline__ void issue_products(const TreeAttnArgs& a, Sync& sy,
                                               const uint8_t* q_tiles, const uint8_t* ring) {
  using S = Shape<D>;
  constexpr uint32_t kIdescS = idesc_bf16(kTile, kTile);
  constexpr uint32_t kIdescO = idesc_bf16(kTile, D) | kIdescBMajorN;
  // descriptors of the first tile of each kind; a tile further on, the start address moves
  constexpr uint64_t kTileStep = S::kTileBytes >> 4;
  const uint64_t q_desc = smem_desc_k_sw128(q_tiles), k_desc = smem_desc_k_sw128(ring);
  const uint64_t v_desc = smem_desc_mn_sw128(ring, kHalfBytes);
  const uint32_t tmem = __shfl_sync(0xffffffffu, sy.tmem_base, 0);
  Ring ring_at;
  int k_slot = 0, v_slot = 0;           // the tiles in use
  uint32_t full = 0, checked = 0;       // parity of the next use of each slot's barriers
  uint32_t weights_phase = 0;           // one bit per accumulator
  bool ok = true;
  const auto wait = [&](int bar, uint32_t parity) {
    ok = warp_wait(sy, bar, parity, a.err);
    return ok;
  };
  // the ring's next tile, and its slot
  const auto take = [&](bool nodes) {
    const int slot = ring_at.slot;
    const uint32_t bit = 1u << slot;
    wait((nodes ? kChecked : kFull) + slot, ((nodes ? checked : full) & bit) != 0);
    checked ^= nodes ? bit : 0;
    full ^= nodes ? 0 : bit;
    ring_at.advance(S::kStages);
    return slot;
  };
  Segment g;
#pragma unroll 1
  for (int index = 0; ok && next_segment(a, sy, index, g); ++index) {
    if (!wait(kFullQ, index & 1)) break;
    fence_proxy_async_smem();  // the helpers' copies, before the tensor cores' reads
#pragma unroll 1
    for (int step = g.step0 - 1; ok && step < g.step1; ++step) {
#pragma unroll 1
      for (int w = 0; ok && w < g.active; ++w) {
        const bool first_use = !g.shared || w == 0, last_use = !g.shared || w == 1;
        if (step >= g.step0) {
          if (first_use) v_slot = take(has_nodes(g, step));
          if (!ok || !wait(kWeightsDone + w, (weights_phase >> w) & 1)) break;
          weights_phase ^= 1u << w;
          tc_fence_after();  // the weights are in TMEM; the tiles need no such fence
          if (elect_one()) {
            const uint64_t vd = v_desc + v_slot * kTileStep;
            const uint32_t first = step > g.step0;
#pragma unroll
            for (int kk = 0; kk < kTile / 16; ++kk) {
              umma_bf16_ts(tmem + kOutput + w * kTile, tmem + kScores + w * kTile + kk * 8,
                           vd + ((kk * 2048) >> 4), kIdescO, kk != 0 ? 1u : first);
            }
            if (last_use) umma_commit(&sy.bar[kEmpty + v_slot]);
            if (step + 1 == g.step1) umma_commit(&sy.bar[kOutputDone + w]);
          }
        }
        if (step + 1 < g.step1) {
          // the next step's scores; they may overwrite these weights: products complete in order
          if (first_use) k_slot = take(false);
          if (!ok) break;
          if (elect_one()) {
            const uint64_t qd = q_desc + w * kTileStep;
            const uint64_t kd = k_desc + k_slot * kTileStep;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint64_t step_k = ((kk / 4) * kHalfBytes + (kk % 4) * 32) >> 4;
              umma_bf16(tmem + kScores + w * kTile, qd + step_k, kd + step_k, kIdescS, kk != 0);
            }
            umma_commit(&sy.bar[kScoresDone + w]);
            if (last_use) umma_commit(&sy.bar[kEmpty + k_slot]);
            if (step + 2 == g.step1 && w == g.active - 1) umma_commit(&sy.bar[kEmptyQ]);
          }
        }
      }
    }
  }
  // every product this thread issued has completed before the TMEM is freed
  if (elect_one()) umma_commit(&sy.bar[kDrain]);
  mbar_wait_bounded(&sy.bar[kDrain], 0);
}

// Whether a node sees its request's row j.
__device__ __forceinline__ bool sees(const Segment& g, const int64_t* mask, int node, int j) {
  const int rel = j - g.context;
  if (rel < 0 || mask == nullptr) return rel <= node;
  return (static_cast<uint64_t>(mask[rel >> 6]) >> (rel & 63)) & 1;
}

// Which of the 128 cached rows from j on a node sees, as bits.
__device__ __forceinline__ void visible(const TreeAttnArgs& a, const Segment& g,
                                        const int64_t* mask, int node, int j,
                                        uint64_t (&bits)[2]) {
  const int rel = j - g.context;  // node index of row j
  const int limit = mask == nullptr ? min(g.nodes, node + 1) : g.nodes;
  bits[0] = bits[1] = ~uint64_t{0};
  if (rel + kTile > 0 && mask != nullptr) {
    // 128 bits of the mask from bit `rel` on, ones for the context before it
    const int lo = rel >> 6, sh = rel & 63;
    uint64_t w[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      w[i] = lo + i < 0                ? ~uint64_t{0}
             : lo + i < a.mask_words ? static_cast<uint64_t>(mask[lo + i])
                                     : 0;
    }
    bits[0] = sh == 0 ? w[0] : (w[0] >> sh) | (w[1] << (64 - sh));
    bits[1] = sh == 0 ? w[1] : (w[1] >> sh) | (w[2] << (64 - sh));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int left = limit - rel - 64 * i;  // rows before the end
    if (left < 64) bits[i] = left <= 0 ? 0 : bits[i] & ((uint64_t{1} << left) - 1);
  }
}

// Softmax and epilogue of accumulator w; this thread owns row `row` of the tile.
template <int D, int kHelperWarps>
__device__ __forceinline__ void softmax(const TreeAttnArgs& a, Sync& sy, int w) {
  using S = Shape<D>;
  const int quarter = (threadIdx.x / kWarpSize) % 4;
  const uint32_t lanes = static_cast<uint32_t>(quarter * kWarpSize) << 16;
  const uint32_t scores = sy.tmem_base + kScores + w * kTile + lanes;
  const uint32_t output = sy.tmem_base + kOutput + w * kTile + lanes;
  const float kInf = __builtin_huge_valf();
  uint32_t scores_phase = 0, output_phase = 0;
  Segment g;
#pragma unroll 1
  for (int index = 0; next_segment(a, sy, index, g); ++index) {
    if (w >= g.active) continue;
    const int lane0 = w == 0 ? 0 : g.lane0;
    const int row = quarter * kWarpSize + threadIdx.x % kWarpSize - lane0;
    const bool valid = row >= 0 && row < pick(g.rows, w);
    const bool any = __any_sync(0xffffffffu, valid);  // the warp holds rows of the request
    const int at_row = pick(g.row0, w) + (valid ? row : 0);
    const int node = a.by_group.divide(at_row);
    const int64_t token = g.start + node;
    const int64_t* mask =
        a.tree_mask == nullptr ? nullptr : a.tree_mask + token * a.mask_words;
    float ref = -kInf, sum = 0.0f;
#pragma unroll 1
    for (int step = g.step0; step < g.step1; ++step) {
      // the mask's words are fetched while the scores are on their way
      const bool masked = any && (step + 1) * kTile > g.context;
      uint64_t bits[2] = {};
      if (masked) visible(a, g, mask, node, step * kTile, bits);
      // the warp leaves together: the TMEM loads below are collective
      if (!warp_wait(sy, kScoresDone + w, scores_phase, a.err)) return;
      scores_phase ^= 1;
      tc_fence_after();
      if (any) {
        uint32_t x[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_load32(scores + 32 * c, x[c]);
        tmem_wait_load();
        if (masked) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const auto see = static_cast<uint32_t>(bits[c / 2] >> (32 * (c % 2)));
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (!((see >> i) & 1)) x[c][i] = __float_as_uint(-kInf);
            }
          }
        }
        float tops[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tops[c] = __uint_as_float(x[c][0]);
#pragma unroll
          for (int i = 1; i + 1 < 32; i += 2) {  // one three-operand maximum each
            tops[c] = fmaxf(fmaxf(tops[c], __uint_as_float(x[c][i])),
                            __uint_as_float(x[c][i + 1]));
          }
          tops[c] = fmaxf(tops[c], __uint_as_float(x[c][31]));
        }
        // the reference moves when it is the first or is exceeded by 2^8
        float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * a.scale_log2;
        if (ref != -kInf && !(top > ref + kRescaleAbove)) top = ref;
        const bool moved = valid && top != ref;
        if (step > g.step0 && __any_sync(0xffffffffu, moved)) {
          const float f = moved ? exp2_approx(ref - top) : 1.0f;
          sum *= f;
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_load16(output + c, o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_store16(output + c, o);
          }
        }
        ref = top;
        const float base = ref == -kInf ? 0.0f : ref;
        const uint64_t scale2 = f32x2(a.scale_log2, a.scale_log2), base2 = f32x2(-base, -base);
        uint64_t sum2[2] = {f32x2(sum, 0.0f), f32x2(0.0f, 0.0f)};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t p[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float lo, hi;
            f32x2_split(f32x2_fma(f32x2(__uint_as_float(x[c][2 * i]),
                                        __uint_as_float(x[c][2 * i + 1])),
                                  scale2, base2),
                        lo, hi);
            lo = exp2_approx(lo);
            hi = exp2_approx(hi);
            sum2[i % 2] = f32x2_add(sum2[i % 2], f32x2(lo, hi));
            p[i] = pack_bf16x2(lo, hi);
          }
          tmem_store16(scores + 16 * c, p);  // over the scores, which have all been read
        }
        float s0, s1, s2, s3;
        f32x2_split(sum2[0], s0, s1);
        f32x2_split(sum2[1], s2, s3);
        sum = (s0 + s1) + (s2 + s3);
        tmem_wait_store();
      }
      tc_fence_before();
      mbar_arrive(&sy.bar[kWeightsDone + w]);
    }

    if (!warp_wait(sy, kOutputDone + w, output_phase, a.err)) return;
    output_phase ^= 1;
    tc_fence_after();
    const bool cut = g.front || g.back;
    // a CTA has at most two cut segments: its first and its last
    const int slot = index == 0 ? 0 : 1;
    float* part = a.parts + ((static_cast<int64_t>(blockIdx.x) * 2 + slot) * 2 + w) *
                                S::kPartFloats;
    if (cut && threadIdx.x % (4 * kWarpSize) == 0 && w == 0) {
      a.marks[blockIdx.x * 2 + slot] = kCut | (g.front ? kCutFront : 0) |
                                       (g.back ? kCutBack : 0) | g.rows[0] << kCutRows |
                                       g.rows[1] << (kCutRows + kCutRowBits);
      Cut& c = a.cuts[blockIdx.x * 2 + slot];
      c.token0 = g.start;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        c.kv_head[x] = g.kv_head[x];
        c.row0[x] = g.row0[x];
      }
    }
    if (any) {
      int odd = 0;
#pragma unroll
      for (int h = 0; h < kHelperWarps; ++h) {
        odd |= *static_cast<volatile int*>(&sy.odd_values[h][w][index % (2 * kSegments)]);
      }
      const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
      __nv_bfloat16* out =
          static_cast<__nv_bfloat16*>(a.out) +
          ((token * a.num_kv_heads + pick(g.kv_head, w) - node) * a.group + at_row) * D;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t x[32];
        tmem_load32(output + c, x);
        tmem_wait_load();
        float o[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(x[i]);
        if (odd && valid) {
          // V values that are not finite, of the rows this node sees: the weights are positive
          const int first = max(g.step0 * kTile, g.context);
          const int last = min(g.step1 * kTile, g.length);
#pragma unroll 1
          for (int j = first; j < last; ++j) {
            if (!sees(g, mask, node, j)) continue;
            const int page = a.page.divide(j);
            int64_t block = a.block_tables[static_cast<int64_t>(g.s) * a.max_blocks + page];
            if (block < 0 || block >= a.num_blocks) block = 0;
            const auto* v = static_cast<const uint16_t*>(a.v_cache) +
                            ((block * a.block_size + (j - page * a.block_size)) *
                                 a.num_kv_heads + pick(g.kv_head, w)) * D + c;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const uint32_t bits = static_cast<uint32_t>(v[i]) << 16;
              if ((bits & 0x7f800000u) == 0x7f800000u) o[i] += __uint_as_float(bits);
            }
          }
        }
        if (cut && valid) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            *reinterpret_cast<float4*>(part + (((c + i) / 4) * kTile + row) * 4) =
                make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        } else if (valid) {
          // a sum of zero: the node saw no row
          float f[8];
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = sum == 0.0f ? 0.0f : o[i + e] * inverse;
            st_global_v4(out + c + i, pack<Bf16>(f));
          }
        }
      }
      if (cut && valid) {
        part[D * kTile + row] = ref;
        part[(D + 1) * kTile + row] = sum;
      }
    }
  }
}

// Rows that no item covers are zero: those of requests that were not served, and what lies behind
// the last; all of them where the starts lead astray. One warp per CTA, every gridDim-th request or
// row.
__device__ __forceinline__ void fill_rest(const TreeAttnArgs& a, bool astray, int64_t row_vecs,
                                          int lane) {
  uint4* out = static_cast<uint4*>(a.out);
  if (astray && lane == 0) raise_error(a.err, kErrBadIndex);
  for (int s = blockIdx.x; !astray && s < a.num_seqs; s += gridDim.x) {
    const Request r = load_request(a, s);
    if (r.bad && lane == 0) raise_error(a.err, kErrBadIndex);
    if (r.steps > 0) continue;
    for (int64_t i = lane; i < static_cast<int64_t>(r.nodes) * row_vecs; i += kWarpSize) {
      st_global_v4(out + r.start * row_vecs + i, make_uint4(0, 0, 0, 0));
    }
  }
  const int64_t tail = astray ? 0 : a.query_start_loc[a.num_seqs];
  for (int64_t t = tail + blockIdx.x; t < a.num_tokens; t += gridDim.x) {
    for (int64_t i = lane; i < row_vecs; i += kWarpSize) {
      st_global_v4(out + t * row_vecs + i, make_uint4(0, 0, 0, 0));
    }
  }
}

template <int D, int kHelperWarps>
__global__ void __launch_bounds__(kThreads, 1)
    tree_attention_kernel(const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v, const TreeAttnArgs a) {
  using S = Shape<D>;
  constexpr int kLoadWarp = kSoftmaxWarps + kHelperWarps;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Sync sy;
  uint8_t* q_tiles = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  uint8_t* ring = q_tiles + 2 * S::kTileBytes;
  const int tid = threadIdx.x;
  const int warp = __shfl_sync(0xffffffffu, tid / kWarpSize, 0), lane = tid % kWarpSize;

  if (tid < kBarriers) {
    mbar_init(&sy.bar[tid], arrivals(tid, kHelperWarps));
    fence_mbar_init();
  }
  if (tid == 0) sy.abort = 0;

  grid_dependency_sync();
  // not before: no CTA holds TMEM while it waits for another grid
  if (warp == kMmaWarp) tmem_alloc(&sy.tmem_base, kTmemColumns);
  if (tid == 0) {
    a.marks[blockIdx.x * 2] = 0;
    a.marks[blockIdx.x * 2 + 1] = 0;
  }
  // this CTA's share of the line: a batch of up to 32 requests is planned by one warp while the
  // others set up; of a larger one every warp adds up a part first, which for small batches too
  // took 12.7 us instead of 12.2 (1 request), 27.8 instead of 24.9 (13), 93.7 instead of 90.5 (8)
  const bool few = a.num_seqs <= kWarpSize;
  const int chunk = few ? 1 : (a.num_seqs + kWarps - 1) / kWarps;
  static_assert(kWarpSize > kWarps, "a chunk of 1 request is one that its lane has loaded");
  bool astray = false;
  if (!few) {
    int cost = 0;
#pragma unroll 1
    for (int s = warp * chunk + lane; s < min(a.num_seqs, (warp + 1) * chunk); s += kWarpSize) {
      const Request r = load_request(a, s);
      cost = add_costs(cost, request_cost(a, r));
      astray |= r.astray;
    }
#pragma unroll
    for (int off = 16; off > 0; off /= 2) {
      cost = add_costs(cost, __shfl_xor_sync(0xffffffffu, cost, off));
    }
    if (lane == 0) sy.costs[warp] = cost;
    astray = __syncthreads_or(astray);
  }
  Place places[2]{};
  if (warp == kPlanWarp) {
    Request r{};
    int cost = 0;
    if (!few) {
      if (lane < kWarps) cost = sy.costs[lane];
    } else if (lane < a.num_seqs) {
      r = load_request(a, lane);
      cost = request_cost(a, r);
    }
    astray = __any_sync(0xffffffffu, astray | r.astray | (a.query_start_loc[0] != 0));
    find_share(a, r, cost, chunk, astray, lane, places);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  if (warp < kSoftmaxWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegisters));
    softmax<D, kHelperWarps>(a, sy, warp / 4);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
    if (warp < kLoadWarp) {
      help<D, kHelperWarps>(a, sy, q_tiles, ring, warp - kSoftmaxWarps, lane);
    } else if (warp < kMmaWarp) {
      Loader<D, kSideWarps - kHelperWarps> l{a, sy, map_k, map_v, ring, warp - kLoadWarp, lane};
      l.run();
    } else if (warp == kMmaWarp) {
      issue_products<D>(a, sy, q_tiles, ring);
    } else {
      plan(a, sy, places[0], places[1], lane);
      fill_rest(a, astray, static_cast<int64_t>(a.num_kv_heads) * a.group * D / 8, lane);
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(sy.tmem_base, kTmemColumns);
}

__device__ __forceinline__ float ld_global_f32(const float* p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}

__device__ __forceinline__ float4 ld_global_f32x4(const float* p) {
  float4 v;
  asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "l"(p));
  return v;
}

// A cut item, as the join's blocks list them.
struct JoinItem {
  int first, border, segments;   // cut `first`, then the first cuts of the CTAs from `border` on
  int mark;                      // of the first cut
};

// Joins units of kRows rows of one accumulator of an item: every gridDim-th of them, counted row
// group by row group over all items, so that those with rows lie together and spread over the
// blocks. A thread does kPieces times 16 bytes of a row, kBatch segments at a time, all their loads
// before any use. With m and l the maxima and sums of the segments, M the largest m:
//   o = sum 2^(m - M) O / sum 2^(m - M) l.
template <int D, int kRows, int kBatch>
__device__ __forceinline__ void join_units(const TreeAttnArgs& a, const JoinItem* items,
                                           const Cut* cuts, int count) {
  using S = Shape<D>;
  constexpr int kApart = kJoinThreads * D / kRows;  // between a thread's pieces
  constexpr int kPieces = D / 4 / kApart;
  const float kInf = __builtin_huge_valf();
  const int piece = threadIdx.x / kRows;
  const int total = count * 2 * (kTile / kRows);
#pragma unroll 1
  for (int unit = blockIdx.x; unit < total; unit += gridDim.x) {
    const int group = unit / (2 * count), rest = unit - group * 2 * count, w = rest & 1;
    const JoinItem& it = items[rest >> 1];
    const int row = group * kRows + threadIdx.x % kRows, rows = cut_rows(it.mark, w);
    if (group * kRows >= rows) continue;
    float top = -kInf, sum = 0.0f;
    float4 o[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float* const parts =
        a.parts + w * S::kPartFloats + (piece * kTile + row) * 4;
    const int to_stats = D * kTile - piece * kTile * 4 - row * 3;
    constexpr int64_t kSlotFloats = 2 * S::kPartFloats;
#pragma unroll 1
    for (int e0 = 0; e0 < it.segments; e0 += kBatch) {
      float m[kBatch], l[kBatch];
      float4 x[kBatch][kPieces];
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        m[e] = -kInf;
        l[e] = 0.0f;
        if (e0 + e < it.segments) {
          const int slot = e0 + e == 0 ? it.first : (it.border - 1 + e0 + e) * 2;
          const float* p = parts + slot * kSlotFloats;
          m[e] = ld_global_f32(p + to_stats);
          l[e] = ld_global_f32(p + to_stats + kTile);
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            x[e][i] = ld_global_f32x4(p + i * kApart * kTile * 4);
          }
        }
      }
      float up = top;
#pragma unroll
      for (int e = 0; e < kBatch; ++e) up = fmaxf(up, m[e]);
      const float base = up == -kInf ? 0.0f : up;
      const float f0 = exp2_approx(top - base);
      top = up;
      sum *= f0;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        o[i] = make_float4(o[i].x * f0, o[i].y * f0, o[i].z * f0, o[i].w * f0);
      }
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        if (l[e] != 0.0f) {  // a segment of which the node sees nothing has no part
          const float f = exp2_approx(m[e] - base);
          sum = fmaf(f, l[e], sum);
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            o[i].x = fmaf(f, x[e][i].x, o[i].x);
            o[i].y = fmaf(f, x[e][i].y, o[i].y);
            o[i].z = fmaf(f, x[e][i].z, o[i].z);
            o[i].w = fmaf(f, x[e][i].w, o[i].w);
          }
        }
      }
    }
    if (row >= rows) continue;
    const Cut& c = cuts[it.first];
    const int at_row = pick(c.row0, w) + row;
    const int node = a.by_group.divide(at_row);
    auto* out = static_cast<__nv_bfloat16*>(a.out) +
                ((static_cast<int64_t>(c.token0 + node) * a.num_kv_heads + pick(c.kv_head, w) -
                  node) * a.group + at_row) * D + piece * 4;
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;  // zero: the node saw no row
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (sum == 0.0f) o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      *reinterpret_cast<uint2*>(out + i * kApart * 4) =
          make_uint2(pack_bf16x2(o[i].x * inverse, o[i].y * inverse),
                     pack_bf16x2(o[i].z * inverse, o[i].w * inverse));
    }
  }
}

// Joins the segments of each cut item. A border between two CTAs' shares that lies inside an item
// is the item's if it is the first of those; each block lists these items (one thread per border)
// and takes every gridDim-th unit of them: of 16 rows, whose segments are mostly two or three (each
// row's factors are then worked out by half as many threads), or where that leaves blocks without
// work, with long items of many segments, of 8. With 8 rows everywhere 8 requests of up to 128
// nodes took 93 us instead of 86, with 16 everywhere one of 32 nodes over 32768 51 instead of 41.
// The join moves up to 39 MB through L2 once more: 6 us for small batches, 13 to 15 for the
// largest.
template <int D>
__global__ void __launch_bounds__(kJoinThreads * D, 256 / D) tree_attention_join_kernel(
    const TreeAttnArgs a, int ctas) {
  grid_dependency_sync();
  constexpr int kBlock = kJoinThreads * D;
  __shared__ JoinItem items[kMaxCtas];
  __shared__ int marks[2 * kMaxCtas];
  __shared__ Cut cuts[2 * kMaxCtas];
  __shared__ int warp_counts[kBlock / kWarpSize];
  __shared__ uint8_t inside[kMaxCtas + 1];  // the border lies inside an item; 2: as its first
  const int tid = threadIdx.x, lane = tid % kWarpSize;
  for (int i = tid; i < 2 * ctas; i += kBlock) {
    marks[i] = a.marks[i];
    cuts[i] = a.cuts[i];  // anything where the mark is 0
  }
  __syncthreads();
  for (int b = tid; b <= ctas; b += kBlock) {
    uint8_t kind = 0;
    // the segment before the border: the previous CTA's second cut one, else its first
    if (b > 0 && b < ctas && (marks[b * 2] & kCutFront)) {
      kind = marks[b * 2 - 1] != 0 || !(marks[b * 2 - 2] & kCutFront) ? 2 : 1;
    }
    inside[b] = kind;
  }
  __syncthreads();
  int count = 0;
  for (int b0 = 0; b0 < ctas; b0 += kBlock) {
    const int b = b0 + tid;
    const bool own = b < ctas && inside[b] == 2;
    const unsigned owners = __ballot_sync(0xffffffffu, own);
    if (lane == 0) warp_counts[tid / kWarpSize] = __popc(owners);
    __syncthreads();
    int at = count + __popc(owners & ((1u << lane) - 1));
    for (int i = 0; i < kBlock / kWarpSize; ++i) {
      if (i < tid / kWarpSize) at += warp_counts[i];
      count += warp_counts[i];
    }
    if (own) {
      JoinItem it;
      it.border = b;
      it.first = b * 2 - (marks[b * 2 - 1] != 0 ? 1 : 2);
      it.segments = 2;
      while (inside[b + it.segments - 1] == 1) ++it.segments;
      it.mark = marks[it.first];
      items[at] = it;
    }
    __syncthreads();
  }

  if (count * 2 * (kTile / 16) >= static_cast<int>(gridDim.x)) {
    join_units<D, 16, 3>(a, items, cuts, count);
  } else {
    join_units<D, 8, 8>(a, items, cuts, count);
  }
}

inline int attention_ctas(int device) {
  const int sms = sm_count(device);
  return sms < kMaxCtas ? sms : kMaxCtas;
}

// Workspace: the partial sums of every CTA, then its cuts.
template <int D>
int64_t workspace_bytes(int ctas) {
  return static_cast<int64_t>(ctas) *
         (4 * Shape<D>::kPartFloats * 4 + 2 * static_cast<int64_t>(sizeof(Cut) + sizeof(int)));
}

// Whether items stay whole, so that there is nothing to join. A join costs 4 us and more with the
// rows, a longer share of one item some 1.3 us a tile: whole items where no table holds more than
// two tiles, and up to four where there is work for every CTA all the same. us cut and whole, 16
// heads on 8 KV heads of 128, rows of a table: 208, 1 request of 8 nodes 12.0 and 10.9; 240, 64 of
// 40 34.4 and 24.8; 416, 1 of 8 12.3 and 15.4, 4 of 8 13.4 and 15.5, 16 of 8 19.1 and 16.2; 448, 64
// of 40 42.6 and 36.1; 912, 64 of 8 45.3 and 53.2. The host knows the tables' width, not the
// lengths: short requests over wide tables (of a captured step, say) are cut and joined. 1 request
// of 8 nodes over 128 rows takes 8.2 us with a table of 128 rows and 10.2 with one of 4096, 64 of
// 40 over 240 rows 23.9 and 34.1, 8 of 16 over 416 14.6 with both.
inline bool whole_items(const TreeAttnArgs& a, int ctas) {
  const int64_t steps = (a.max_length + kTile - 1) / kTile;
  if (steps <= 2) return true;
  if (steps > 4 || a.num_seqs == 0) return false;
  const int64_t nodes = (a.num_tokens + a.num_seqs - 1) / a.num_seqs;  // of a request, on average
  const int64_t tiles = (nodes * a.group + kTile - 1) / kTile;
  return a.num_seqs * a.num_kv_heads * steps * ((tiles + 1) / 2) >= 2 * ctas;
}

template <int D>
int launch_tree_attention(TreeAttnArgs& a, void* workspace, int device, cudaStream_t stream) {
  const int ctas = attention_ctas(device);
  a.parts = static_cast<float*>(workspace);
  a.marks = reinterpret_cast<int*>(a.parts + static_cast<int64_t>(ctas) * 4 *
                                                 Shape<D>::kPartFloats);
  a.cuts = reinterpret_cast<Cut*>(a.marks + 2 * ctas);
  a.whole = whole_items(a, ctas);
  CUtensorMap map_k, map_v;
  const int64_t cols = static_cast<int64_t>(a.num_kv_heads) * D;
  if (!make_map(&map_k, a.k_cache, a.cache_slots, cols, cols, a.box_rows) ||
      !make_map(&map_v, a.v_cache, a.cache_slots, cols, cols, a.box_rows)) {
    return SVLLM_ERR_CUDA;
  }
  // raises the kernel's shared-memory limit on its first use
  const auto kernel =
      a.box_rows < kSmallBox ? tree_attention_kernel<D, 2> : tree_attention_kernel<D, 4>;
  if (blocks_per_sm(reinterpret_cast<const void*>(kernel), kThreads, Shape<D>::kSmem, device) <
      1) {
    return SVLLM_ERR_CUDA;
  }
  const int status = launch(kernel, dim3(ctas), dim3(kThreads), Shape<D>::kSmem, stream, 1u,
                            map_k, map_v, a);
  if (status != SVLLM_OK || ctas < 2 || a.whole) return status;
  // as many blocks as are resident at once
  return launch(tree_attention_join_kernel<D>, dim3(256 / D * ctas), dim3(kJoinThreads * D), 0,
                stream, 1u, a, ctas);
}

}  // namespace
}  // namespace svllm::k

extern "C" int svllm_tree_attention_workspace_bytes(int64_t head_dim, int64_t* bytes) {
  using namespace svllm::k;
  if (bytes == nullptr || head_dim <= 0) return SVLLM_ERR_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 128) return SVLLM_ERR_UNSUPPORTED;
  int device;
  if (current_device(&device) != SVLLM_OK) return SVLLM_ERR_CUDA;
  const int ctas = attention_ctas(device);
  *bytes = head_dim == 128 ? workspace_bytes<128>(ctas) : workspace_bytes<64>(ctas);
  return SVLLM_OK;
}

extern "C" int svllm_tree_attention_bf16(
    void* out, const void* q, int64_t q_token_stride, const void* k_cache, const void* v_cache,
    int64_t num_blocks, int64_t block_size, const int32_t* block_tables, int64_t max_blocks,
    const int32_t* seq_lens, const int32_t* query_start_loc, int64_t num_seqs, int64_t num_tokens,
    int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, const int64_t* tree_mask,
    int64_t mask_words, float scale, void* workspace, int64_t workspace_size,
    svllm_stream stream) {
  using namespace svllm::k;
  if (num_seqs < 0 || num_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads % num_kv_heads != 0 || head_dim <= 0 || block_size <= 0 || max_blocks <= 0 ||
      num_blocks <= 0 || !(scale > 0.0f) || !std::isfinite(scale * 2.0f) ||
      (tree_mask != nullptr && mask_words <= 0)) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  if (head_dim != 64 && head_dim != 128) return SVLLM_ERR_UNSUPPORTED;
  constexpr int64_t kMax = int64_t{1} << 31;
  if (num_seqs >= kMax || num_tokens >= kMax || num_heads >= (int64_t{1} << 20) ||
      num_tokens * num_heads >= kMax || max_blocks >= kMax || num_blocks >= kMax ||
      block_size >= (int64_t{1} << 20) || max_blocks * block_size >= kMax ||
      num_blocks * block_size >= kMax ||
      (tree_mask != nullptr && mask_words > SVLLM_MAX_TREE_NODES / 64)) {
    return SVLLM_ERR_TOO_LARGE;
  }
  if (q_token_stride < num_heads * head_dim) return SVLLM_ERR_INVALID_ARGUMENT;
  if (num_tokens == 0) return SVLLM_OK;
  if (out == nullptr || q == nullptr || k_cache == nullptr || v_cache == nullptr ||
      query_start_loc == nullptr ||
      (num_seqs > 0 && (block_tables == nullptr || seq_lens == nullptr))) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
  if (!aligned16(out) || !aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) ||
      (q_token_stride * 2) % 16 != 0) {
    return SVLLM_ERR_UNSUPPORTED;
  }
  // the line of steps is counted in 32 bits: its length is at most most * tiles
  const int64_t most = (max_blocks * block_size / 128 + 1) * num_kv_heads;
  const int64_t tiles = num_tokens * (num_heads / num_kv_heads) / 128 + num_seqs;
  if (most >= kMax || tiles >= kMax / most) return SVLLM_ERR_TOO_LARGE;
  int64_t needed = 0;
  const int sized = svllm_tree_attention_workspace_bytes(head_dim, &needed);
  if (sized != SVLLM_OK) return sized;
  if (workspace == nullptr || workspace_size < needed || !aligned16(workspace)) {
    return SVLLM_ERR_INVALID_ARGUMENT;
  }
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
  a.num_tokens = static_cast<int>(num_tokens);
  a.num_seqs = static_cast<int>(num_seqs);
  a.max_blocks = static_cast<int>(max_blocks);
  a.block_size = static_cast<int>(block_size);
  a.page = make_divider(block_size);
  a.group = static_cast<int>(num_heads / num_kv_heads);
  a.max_length = static_cast<int>(max_blocks * block_size);
  a.max_nodes = tree_mask != nullptr ? static_cast<int>(64 * mask_words) : INT32_MAX;
  a.by_group = make_divider(a.group);
  a.num_kv_heads = static_cast<int>(num_kv_heads);
  a.cache_slots = static_cast<int>(num_blocks * block_size);
  a.box_rows = 128;
  while (block_size % a.box_rows != 0) a.box_rows /= 2;
  if (a.box_rows < 4) a.box_rows = 1;
  a.mask_words = static_cast<int>(mask_words);
  a.scale_log2 = static_cast<float>(static_cast<double>(scale) / std::log(2.0));
  a.err = err;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return head_dim == 128 ? launch_tree_attention<128>(a, workspace, device, s)
                         : launch_tree_attention<64>(a, workspace, device, s);
}
