// Device-side building blocks shared by the sm_100a layer-op kernels.
//
// Everything here is memory plumbing for token-row-parallel streaming ops: bf16 <-> fp32
// conversion with the rounding the Hugging Face composites use, 16-byte vectors, mbarrier and
// bulk-copy (TMA, non-tensor, never multicast) wrappers, bounded waits, and the device error
// word that kernels raise instead of trapping.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace svllm::k {

constexpr int kWarpSize = 32;

// Device error word bits. A kernel never traps: it records the condition here and carries on
// (bad ids) or stops its own work (a wait that ran out), so the CUDA context stays usable.
constexpr int kErrBadIndex = 1;     // an embedding id outside [0, vocab)
constexpr int kErrWaitTimeout = 2;  // a bulk copy did not land within the wait limit

// A wait on an mbarrier gives up after this many nanoseconds of %globaltimer.
constexpr uint64_t kWaitLimitNs = 2000000000ull;

// ---------------------------------------------------------------------------------------------
// Element types. The kernels are written once over Elem and instantiated for bf16 and fp32.

struct Bf16 {
  using Storage = __nv_bfloat16;
  static constexpr int kPerVec = 8;  // elements per 16-byte vector
  __device__ static __forceinline__ float to_float(Storage v) { return __bfloat162float(v); }
  __device__ static __forceinline__ Storage from_float(float v) { return __float2bfloat16_rn(v); }
  // Round an fp32 intermediate to the storage type and back, as a bf16 torch op does.
  __device__ static __forceinline__ float round(float v) {
    return __bfloat162float(__float2bfloat16_rn(v));
  }
};

struct F32 {
  using Storage = float;
  static constexpr int kPerVec = 4;
  __device__ static __forceinline__ float to_float(Storage v) { return v; }
  __device__ static __forceinline__ Storage from_float(float v) { return v; }
  __device__ static __forceinline__ float round(float v) { return v; }
};

// Unpack a 16-byte vector into kPerVec floats, and pack kPerVec floats (rounded) back.
template <class E>
__device__ __forceinline__ void unpack(const uint4& raw, float (&f)[E::kPerVec]);

template <>
__device__ __forceinline__ void unpack<Bf16>(const uint4& raw, float (&f)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // bf16 -> fp32 is exact: the bf16 bits are the high half of the fp32 bits
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

template <>
__device__ __forceinline__ void unpack<F32>(const uint4& raw, float (&f)[4]) {
  f[0] = __uint_as_float(raw.x);
  f[1] = __uint_as_float(raw.y);
  f[2] = __uint_as_float(raw.z);
  f[3] = __uint_as_float(raw.w);
}

template <class E>
__device__ __forceinline__ uint4 pack(const float (&f)[E::kPerVec]);

template <>
__device__ __forceinline__ uint4 pack<Bf16>(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // cvt.rn.bf16x2.f32 rounds both halves to nearest even, like __float2bfloat16_rn
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <>
__device__ __forceinline__ uint4 pack<F32>(const float (&f)[4]) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                    __float_as_uint(f[3]));
}

// ---------------------------------------------------------------------------------------------
// Packed bf16 arithmetic. For bf16 operands these give exactly the result of the fp32 operation
// followed by one round-to-nearest-even to bf16 (the sequence a bf16 torch op performs):
//   * the product of two bf16 values has a 16-bit significand, so it is exact in fp32 and the
//     fp32 rounding step is the identity;
//   * a sum or difference is exact in fp32 unless the exponents differ by 16 or more, and then
//     the smaller operand is below 2^-8 of the larger's last bf16 place, so both routes round to
//     the larger operand.
// (Both arguments assume normal numbers; bf16 subnormals, below 1.2e-38, never occur in these
// ops' activations.) One instruction handles two elements.

__device__ __forceinline__ uint32_t bf16x2_mul(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

__device__ __forceinline__ uint32_t bf16x2_add(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

__device__ __forceinline__ uint32_t bf16x2_sub(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Two fp32 values rounded to nearest even into one bf16x2 word (lo in the low half).
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// Packed fp32 pairs (sm_100's .f32x2 instructions): one instruction performs the fp32 operation,
// each with its own round-to-nearest-even, on both halves, so results equal two scalar ops.
__device__ __forceinline__ uint64_t f32x2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}

__device__ __forceinline__ void f32x2_split(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}

__device__ __forceinline__ uint64_t f32x2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

__device__ __forceinline__ uint64_t f32x2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __forceinline__ uint64_t f32x2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// 2^x (the ex2 instruction; 2^-inf = 0).
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// j / d for 0 <= j < 2^31 by a precomputed reciprocal and a shift (Granlund and Montgomery,
// "Division by invariant integers using multiplication", 1994): shift = ceil(log2 d), magic =
// floor(2^32 (2^shift - d) / d) + 1.
struct Divider {
  uint32_t magic;
  int shift;
  __device__ __forceinline__ int divide(int j) const {
    return static_cast<int>((__umulhi(static_cast<uint32_t>(j), magic) +
                             static_cast<uint32_t>(j)) >> shift);
  }
};

inline Divider make_divider(int64_t d) {
  Divider r{};
  while ((int64_t{1} << r.shift) < d) ++r.shift;
  r.magic = static_cast<uint32_t>(
      ((uint64_t{1} << 32) * ((uint64_t{1} << r.shift) - static_cast<uint64_t>(d))) /
          static_cast<uint64_t>(d) + 1);
  return r;
}

__device__ __forceinline__ uint32_t word(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// ---------------------------------------------------------------------------------------------
// Per-vector steps shared by the norm kernels.

// residual' = round(x + residual) for one 16-byte vector.
template <class E>
__device__ __forceinline__ uint4 add_vec(const uint4& x, const uint4& r);

template <>
__device__ __forceinline__ uint4 add_vec<Bf16>(const uint4& x, const uint4& r) {
  return make_uint4(bf16x2_add(x.x, r.x), bf16x2_add(x.y, r.y), bf16x2_add(x.z, r.z),
                    bf16x2_add(x.w, r.w));
}

template <>
__device__ __forceinline__ uint4 add_vec<F32>(const uint4& x, const uint4& r) {
  return make_uint4(__float_as_uint(__fadd_rn(__uint_as_float(x.x), __uint_as_float(r.x))),
                    __float_as_uint(__fadd_rn(__uint_as_float(x.y), __uint_as_float(r.y))),
                    __float_as_uint(__fadd_rn(__uint_as_float(x.z), __uint_as_float(r.z))),
                    __float_as_uint(__fadd_rn(__uint_as_float(x.w), __uint_as_float(r.w))));
}

// out = round(round(h * inv_rms) * w) for one 16-byte vector of h and of the weight.
template <class E>
__device__ __forceinline__ uint4 normalize_vec(const uint4& h, float inv_rms, const uint4& w);

template <>
__device__ __forceinline__ uint4 normalize_vec<Bf16>(const uint4& h, float inv_rms,
                                                     const uint4& w) {
  float f[8];
  unpack<Bf16>(h, f);
  uint32_t n[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    n[i] = pack_bf16x2(__fmul_rn(f[2 * i], inv_rms), __fmul_rn(f[2 * i + 1], inv_rms));
  }
  return make_uint4(bf16x2_mul(n[0], w.x), bf16x2_mul(n[1], w.y), bf16x2_mul(n[2], w.z),
                    bf16x2_mul(n[3], w.w));
}

// normalize_vec<Bf16> with the scaling by inv_rms as four packed fp32 multiplies (same results).
__device__ __forceinline__ uint4 normalize_vec_packed(const uint4& h, float inv_rms,
                                                      const uint4& w) {
  float f[8];
  unpack<Bf16>(h, f);
  uint32_t n[4];
  const uint64_t inv2 = f32x2(inv_rms, inv_rms);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    f32x2_split(f32x2_mul(f32x2(f[2 * i], f[2 * i + 1]), inv2), a, b);
    n[i] = pack_bf16x2(a, b);
  }
  return make_uint4(bf16x2_mul(n[0], w.x), bf16x2_mul(n[1], w.y), bf16x2_mul(n[2], w.z),
                    bf16x2_mul(n[3], w.w));
}

template <>
__device__ __forceinline__ uint4 normalize_vec<F32>(const uint4& h, float inv_rms,
                                                    const uint4& w) {
  float f[4], wf[4];
  unpack<F32>(h, f);
  unpack<F32>(w, wf);
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = __fmul_rn(__fmul_rn(f[e], inv_rms), wf[e]);
  return pack<F32>(f);
}

// ---------------------------------------------------------------------------------------------
// Global memory access with streaming hints.

__device__ __forceinline__ uint4 ld_global_nc_v4(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

__device__ __forceinline__ void st_global_v4(void* p, const uint4& v) {
  asm volatile("st.global.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

__device__ __forceinline__ uint4 ld_shared_v4(const void* p) {
  uint4 r;
  const uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p));
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "r"(a));
  return r;
}

// ---------------------------------------------------------------------------------------------
// mbarrier + bulk copy (cp.async.bulk, the non-tensor TMA path). No copy in this library is
// broadcast to other CTAs of a cluster: every copy moves this GPU's own memory into its own CTA.

// Programmatic dependent launch, in two halves. grid_dependency_wait: wait until the kernel
// before this one in the stream has completed and its memory is visible (a no-op when launched
// without the attribute); every kernel runs it first, before any memory access.
// allow_dependents: let the next kernel in the stream be scheduled now, while this one runs; a
// kernel that never calls it lets the next one be scheduled as its CTAs exit.
__device__ __forceinline__ void grid_dependency_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ void allow_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Both, for kernels that always let the next one be scheduled at their start.
__device__ __forceinline__ void grid_dependency_sync() {
  grid_dependency_wait();
  allow_dependents();
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// d += a * b on the tensor cores: A 16x16 bf16 (row), B 16x8 bf16 (col), fp32 accumulators.
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// This CTA's rank in its thread-block cluster.
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// Every thread of every CTA of the cluster: shared-memory writes before it are visible to the
// cluster's reads after it.
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;"
               ::: "memory");
}

// A float of cluster CTA `rank`'s shared memory at the address of `p` in this CTA's. Not
// volatile: the loads of a merge are independent and may be in flight together (a cluster
// barrier before them orders them after the writes).
__device__ __forceinline__ float ld_remote_f32(const float* p, uint32_t rank) {
  uint32_t addr;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_addr(p)), "r"(rank));
  float v;
  asm("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count)
               : "memory");
}

// Makes initialised mbarriers visible to the async proxy before the first bulk copy uses them.
__device__ __forceinline__ void fence_mbar_init() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

// Orders this thread's earlier generic-proxy shared-memory accesses before later async-proxy
// ones (a bulk copy overwriting a stage the warp has just read, or a bulk store of a stage the
// warp has just written).
__device__ __forceinline__ void fence_proxy_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ void mbar_arrive_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)),
               "r"(bytes)
               : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// One bounded try: the thread may sleep (without issuing) until the phase completes or the
// suspend-time hint (ns) passes, so a warp waiting on HBM costs almost no issue slots.
constexpr uint32_t kTryWaitSuspendNs = 1000000;

__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_addr(bar)), "r"(parity), "n"(kTryWaitSuspendNs)
      : "memory");
  return done != 0;
}

__device__ __forceinline__ uint64_t global_timer_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

// Waits for the phase with the given parity to complete. Returns false if it has not after
// kWaitLimitNs; the caller then raises kErrWaitTimeout and stops.
__device__ __forceinline__ bool mbar_wait_bounded(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) {
    return true;
  }
  const uint64_t start = global_timer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (global_timer_ns() - start > kWaitLimitNs) {
      return false;
    }
  }
  return true;
}

// Global -> shared bulk copy completing on an mbarrier. dst, src and bytes are multiples of 16.
__device__ __forceinline__ void bulk_load(void* dst_smem, const void* src_gmem, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(smem_addr(dst_smem)),
      "l"(src_gmem), "r"(bytes), "r"(smem_addr(bar))
      : "memory");
}

// Shared -> global bulk store, tracked by this thread's bulk groups.
__device__ __forceinline__ void bulk_store(void* dst_gmem, const void* src_smem, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst_gmem),
               "r"(smem_addr(src_smem)), "r"(bytes)
               : "memory");
}

// L2 cache policies for the bulk copies' cache hints: evict-last for data the kernel will read
// again soon (kept in L2 ahead of normal lines), evict-first for data it writes once.
__device__ __forceinline__ uint64_t l2_policy_evict_last() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
  return p;
}

__device__ __forceinline__ uint64_t l2_policy_evict_first() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}

// bulk_load with an L2 cache policy.
__device__ __forceinline__ void bulk_load_policy(void* dst_smem, const void* src_gmem,
                                                 uint32_t bytes, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], "
      "[%1], %2, [%3], %4;" ::"r"(smem_addr(dst_smem)),
      "l"(src_gmem), "r"(bytes), "r"(smem_addr(bar)), "l"(policy)
      : "memory");
}

// bulk_store with an L2 cache policy.
__device__ __forceinline__ void bulk_store_policy(void* dst_gmem, const void* src_smem,
                                                  uint32_t bytes, uint64_t policy) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group.L2::cache_hint [%0], [%1], %2, %3;" ::
                   "l"(dst_gmem),
               "r"(smem_addr(src_smem)), "r"(bytes), "l"(policy)
               : "memory");
}

__device__ __forceinline__ void bulk_commit() {
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// Waits until at most N of this thread's bulk groups still have to read their shared source.
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void bulk_wait_all() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// ---------------------------------------------------------------------------------------------
// Error word. The host passes either the caller's device int or the library's own per-device
// word (read back with svllm_read_device_error), so err is never null in a kernel.

__device__ __forceinline__ void raise_error(int* err, int bits) { atomicOr(err, bits); }

// ---------------------------------------------------------------------------------------------
// Reductions.

// Sum over aligned groups of G lanes (G a power of two, at most 32) by xor butterflies: every
// lane of a group ends with the same value.
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int offset = G / 2; offset > 0; offset /= 2) {
    v += __shfl_xor_sync(0xffffffffu, v, offset);
  }
  return v;
}

// The units a warp processes: a contiguous, balanced share of n units (interleave = false), or
// every warps_total-th unit starting at the warp's index (interleave = true), so that at any
// moment the grid streams through neighbouring units of memory together. On a B200 at 1M tokens
// the interleaved order measured 1-4% faster for the norm, rotary and SiLU kernels; the gather
// keeps contiguous shares so that a warp's ids arrive in coalesced batches.
struct WarpUnits {
  int64_t first;
  int64_t step;
  int64_t count;
  __device__ __forceinline__ int64_t at(int64_t j) const { return first + j * step; }
};

// Balanced contiguous partition of n units over `parts` workers: worker i gets [begin, end).
__device__ __forceinline__ void partition(int64_t n, int64_t parts, int64_t i, int64_t& begin,
                                          int64_t& end) {
  const int64_t base = n / parts;
  const int64_t rem = n % parts;
  begin = i * base + (i < rem ? i : rem);
  end = begin + base + (i < rem ? 1 : 0);
}

__device__ __forceinline__ WarpUnits warp_units(int64_t n, int64_t warps_total, int64_t gw,
                                                bool interleave) {
  if (interleave) {
    return {gw, warps_total, gw < n ? (n - gw + warps_total - 1) / warps_total : 0};
  }
  int64_t begin, end;
  partition(n, warps_total, gw, begin, end);
  return {begin, 1, end - begin};
}

}  // namespace svllm::k
