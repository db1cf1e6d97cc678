// tcgen05 helpers of the 4-bit kernels: MMAs whose A operand lives in tensor memory, tensor-memory loads and
// stores, and waits that give up together.
#pragma once
#include "common.cuh"

namespace hla {
namespace tc {

// K-major SWIZZLE_128B operand in shared memory: rows of 128 B, 8-row groups 1024 B apart, 1024-byte aligned;
// a K step of 16 two-byte elements advances the address by 32 B.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t smem_addr) {
  return static_cast<uint64_t>((smem_addr & 0x3FFFF) >> 4) | (static_cast<uint64_t>(1) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
         (static_cast<uint64_t>(2) << 61);
}
// Byte offset of 16-byte chunk `chunk` of row `row` in such an operand (row < 16, 64 elements per row).
__device__ __forceinline__ uint32_t sw128(int row, int chunk) {
  return static_cast<uint32_t>((row >> 3) * 1024 + (row & 7) * 128 + ((chunk ^ (row & 7)) << 4));
}

// Instruction descriptor, fp32 accumulators: A and B both f16 (type 0) or both bf16 (type 1).
__host__ __device__ constexpr uint32_t idesc(int type, int m, int n) {
  return (1u << 4) | (uint32_t(type) << 7) | (uint32_t(type) << 10) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

// True in one lane of a converged warp.  MMAs are issued under this predicate and in unrolled code: the operands
// of tcgen05.mma are uniform registers, and under `lane == 0` or in a rolled loop the compiler moves them there one
// instruction after the other (150 and 100 clocks an MMA; 9 as written, for M = 128, N = 16 with A in tensor memory).
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile(
      "{\n"
      ".reg .pred q;\n"
      "elect.sync _|q, 0xffffffff;\n"
      "selp.u32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(p));
  return p != 0;
}
// D[tmem] (+)= A[tmem] . B[smem]^T
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void alloc(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void dealloc(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}

// Consecutive columns of this thread's lane.
__device__ __forceinline__ void st16(uint32_t a, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]));
}
__device__ __forceinline__ void ld16(uint32_t a, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(a));
}
__device__ __forceinline__ void ld8(uint32_t a, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(a));
}
__device__ __forceinline__ void st8(uint32_t a, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(a), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]));
}
// 16 lanes x 8 columns: thread 4 g + c holds columns 2c, 2c + 1 of lane g (r0, r1) and of lane g + 8 (r2, r3).
__device__ __forceinline__ void st_16x256(uint32_t a, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x1.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(r0), "r"(r1), "r"(r2), "r"(r3));
}

// The least limit of these kernels' waits.  They wait for nothing but their own copies and products, which take
// microseconds: when a wait runs out after this long, what was in flight has landed (the GPU ran something else
// meanwhile) or never will.  With a shorter limit a CTA could end before its copies.
constexpr uint64_t kLeastWaitNs = 100 * 1000 * 1000;

// Bounded waits of a CTA's roles.  The first that runs out records `code` in the error word and raises the shared abort
// flag; from then on every wait of the CTA returns once it has tried, so each role still takes all its steps (the
// barriers that count arrivals stay in step, nothing leaves a loop early) and the CTA ends with wrong values and an error
// code.  (Waits that say whether they ran out, for the copies to stop at, cost 1 to 5 % of every kernel here.)
struct Waits {
  int* abort_flag;  // shared memory, zeroed
  int* err;
  uint64_t limit_ns;
  __device__ __forceinline__ bool aborted() const { return *reinterpret_cast<volatile int*>(abort_flag) != 0; }
  // One try suspends the thread for up to 20 us: a waiting warp takes few issue slots from the working ones.
  __device__ __forceinline__ bool attempt(uint64_t* bar, uint32_t parity) const {
    uint32_t ok;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
        : "memory");
    return ok != 0;
  }
  __device__ __forceinline__ void operator()(uint64_t* bar, uint32_t parity, int code) const {
    if (!attempt(bar, parity)) retry(bar, parity, code);
  }
  __device__ __noinline__ void retry(uint64_t* bar, uint32_t parity, int code) const {
    const uint64_t t0 = global_ns();
    while (!attempt(bar, parity)) {
      if (aborted()) return;
      if (global_ns() - t0 > limit_ns) {
        record_error(err, code);
        atomicExch(abort_flag, 1);
        return;
      }
    }
  }
};

// Untiled bulk copy global -> this CTA's shared memory (16-byte aligned, size a multiple of 16), L2 policy hint.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

}  // namespace tc
}  // namespace hla
