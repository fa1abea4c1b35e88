// ta_mx_device.cuh -- sm_100a device helpers of the matrix operators: mbarrier
// waits, tiled TMA loads, tcgen05 (tensor memory, matrix instructions) and the
// two shared-memory operand layouts they read.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ta {
namespace mx {

constexpr uint64_t kWaitLimitNs = 2000000000ull;  // every wait ends after 2 s
constexpr uint32_t kStatusTimeout = 2u;           // TA_STATUS_WAIT_TIMEOUT

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

// One lane of a converged warp. Code that issues TMA copies and matrix instructions keeps the whole
// warp on its path and issues from this lane: their operands then stay in uniform registers
// (from a single-lane branch each issue took about 250 cycles).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// ---- shared memory by address ----
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ void sts16(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}
template <int SIZE>
__device__ __forceinline__ uint32_t lds_elem(uint32_t a) {
  uint32_t v;
  if constexpr (SIZE == 4) {
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  } else {
    uint16_t h;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(a) : "memory");
    v = h;
  }
  return v;
}
template <int SIZE>
__device__ __forceinline__ void sts_elem(uint32_t a, uint32_t v) {
  if constexpr (SIZE == 4)
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
  else
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"((uint16_t)v) : "memory");
}

// ---- dependent launches ----
// A kernel of a chain starts while its predecessor drains: it sets itself up, then waits here
// before it touches memory that the predecessor reads or writes.
__device__ __forceinline__ void chain_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void chain_next() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ---- clusters --------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
// The shared::cluster address of `addr` (a shared address of this CTA) in CTA `rank`.
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
          : "memory");
}

// ---- mbarriers (by shared address) -----------------------------------------------
__device__ __forceinline__ void bar_init(uint32_t b, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(b), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_fence() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void bar_expect_tx(uint32_t b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(b), "r"(bytes)
               : "memory");
}
// Arrive on a barrier of any CTA of the cluster (shared::cluster address). What it orders is the
// thread's tensor-memory reads (behind tc_fence_before), not its global stores: a release at
// cluster scope would wait about 1000 cycles for those.
__device__ __forceinline__ void bar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t bar_try(uint32_t b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(b), "r"(parity), "r"(1000000u)  // may sleep for a millisecond
      : "memory");
  return ok;
}
// A wait that ends: false once kWaitLimitNs have passed, with the status bit set.
static __device__ __noinline__ bool bar_wait_on(uint32_t b, uint32_t parity, uint32_t* status) {
  const uint64_t t0 = now_ns();
  for (;;) {
    for (int i = 0; i < 16; ++i)
      if (bar_try(b, parity)) return true;
    if (now_ns() - t0 > kWaitLimitNs) {
      atomicOr(status, kStatusTimeout);
      return false;
    }
  }
}
__device__ __forceinline__ bool bar_wait(uint32_t b, uint32_t parity, uint32_t* status) {
  return bar_try(b, parity) || bar_wait_on(b, parity, status);
}

// ---- TMA -------------------------------------------------------------------
__device__ __forceinline__ void tma_prefetch(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
}
// One box of a 3-D tensor map into this CTA's shared memory; its bytes are counted on the
// barrier at shared::cluster address `bar`, of either CTA of the pair.
__device__ __forceinline__ void tma_load(const CUtensorMap* m, uint32_t dst, uint32_t bar, int x,
                                         int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::"
      "bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(m), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// The same of a 4-D map whose innermost dimension is taken whole.
__device__ __forceinline__ void tma_load4(const CUtensorMap* m, uint32_t dst, uint32_t bar, int y,
                                          int z, int t) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::"
      "bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(m), "r"(bar), "r"(0), "r"(y), "r"(z), "r"(t)
      : "memory");
}

// ---- tcgen05 (pairs of SMs) ----------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot),
               "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// D[tmem] (+)= A[smem] B[smem] on a pair of SMs, 16-bit operands, fp32 accumulators, K = 16.
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// Arrive on the barrier at `bar`'s offset in both CTAs of the pair when every matrix instruction
// issued so far by this thread has finished.
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(bar),
      "h"((uint16_t)3)
      : "memory");
}
// 32 consecutive columns of this warp's 32 tensor-memory lanes: lane l gets row l.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// Instruction descriptor of kind::f16: fp32 accumulators, both operands fp16 or both bf16,
// each K-major or MN-major (transposed), shape M x N.
__host__ __device__ constexpr uint32_t mma_idesc(bool bf16, bool a_mn, bool b_mn, int M, int N) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) |
         ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}
// Shared-memory descriptor of a 128 (rows) x 64 (k) operand tile of 16-bit elements in
// 128-byte swizzled rows. K-major: row r is 64 k's, 8-row groups 1024 bytes apart. MN-major:
// two chunks (8192 bytes apart) of 64 rows; row k of a chunk holds its 64 elements, 8-k groups
// 1024 bytes apart.
__device__ __forceinline__ uint64_t mma_smem_desc(uint32_t addr, bool mn) {
  const uint64_t lbo = mn ? (8192u >> 4) : 1u;
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (lbo << 16) | ((uint64_t)(1024u >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// What one instruction's 16 k's advance the descriptor's address field by.
__device__ __forceinline__ uint32_t mma_k_step(bool mn) { return (mn ? 2048u : 32u) >> 4; }

// ---- element types -----------------------------------------------------------
enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };  // TA_F32, TA_BF16, TA_F16

__device__ __forceinline__ float load_as_float(const void* p, int64_t i, int dt) {
  if (dt == DT_F32) return reinterpret_cast<const float*>(p)[i];
  if (dt == DT_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_from_float(void* p, int64_t i, int dt, float v) {
  if (dt == DT_F32)
    reinterpret_cast<float*>(p)[i] = v;
  else if (dt == DT_BF16)
    reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else
    reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf162(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, int dt) {
  return dt == DT_BF16 ? pack_bf162(lo, hi) : pack_half2(lo, hi);
}
__device__ __forceinline__ float2 unpack16(uint32_t u, int dt) {
  if (dt == DT_BF16) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<__half2*>(&u));
}

}  // namespace mx
}  // namespace ta
