// What one thread issues to the tensor cores in a loop that has some 500 cycles a step: a thread alone runs an instruction every five
// cycles or so, so a wait that is over costs one try, and a matrix descriptor one 32-bit addition.  Included inside the
// anonymous namespace of the kernels that use it, after tcgen05.cuh.
#pragma once

// The low half of a descriptor moves with the address (in units of 16 bytes; shared memory ends below its 14 bits), the high half
// is the same for all.
struct MatrixDesc {
  uint32_t lo, hi;
  __device__ __forceinline__ explicit MatrixDesc(uint32_t smem_addr) {
    const uint64_t d = umma_desc(smem_addr);
    lo = (uint32_t)d;
    hi = (uint32_t)(d >> 32);
  }
};
// wait_or_abort whose first try is inline
__device__ __forceinline__ bool quick_wait(uint64_t* bar, uint32_t parity, volatile int* failed) {
  uint32_t done;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done || wait_or_abort(bar, parity, failed);
}

#define FMS_ISSUE_HEAD "{\n.reg .pred p;\n.reg .b64 a, b;\nsetp.ne.b32 p, %5, 0;\nmov.b64 a, {%1, %2};\nmov.b64 b, {%3, %2};\n"
// e4m3, both operands in shared memory: 128 x N x 32 by one block
__device__ __forceinline__ void issue_e4m3(uint32_t tmem_d, uint32_t a_lo, uint32_t hi, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(FMS_ISSUE_HEAD "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %4, {%6, %6, %6, %6}, p;\n}\n" ::"r"(tmem_d), "r"(a_lo),
               "r"(hi), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(0)
               : "memory");
}
// 256 x N x 32 by a pair of blocks: A 128 rows from each block's shared memory, B N/2 rows from each
__device__ __forceinline__ void issue_e4m3_pair(uint32_t tmem_d, uint32_t a_lo, uint32_t hi, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(FMS_ISSUE_HEAD "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a, b, %4, {%6, %6, %6, %6, %6, %6, %6, %6}, p;\n}\n" ::"r"(tmem_d),
               "r"(a_lo), "r"(hi), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(0)
               : "memory");
}
#undef FMS_ISSUE_HEAD
#define FMS_ISSUE_HEAD "{\n.reg .pred p;\n.reg .b64 b;\nsetp.ne.b32 p, %5, 0;\nmov.b64 b, {%2, %3};\n"
// bfloat16, A in tensor memory (of a pair: in either block's): 128 x N x 16 by one block, 256 x N x 16 by a pair
__device__ __forceinline__ void issue_a_tmem(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(FMS_ISSUE_HEAD "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, {%6, %6, %6, %6}, p;\n}\n" ::"r"(tmem_d), "r"(tmem_a),
               "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(0)
               : "memory");
}
__device__ __forceinline__ void issue_a_tmem_pair(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(FMS_ISSUE_HEAD "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], b, %4, {%6, %6, %6, %6, %6, %6, %6, %6}, p;\n}\n" ::"r"(tmem_d),
               "r"(tmem_a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(0)
               : "memory");
}
#undef FMS_ISSUE_HEAD
