// Inline-PTX wrappers of the 5th-generation tensor cores: tensor memory, matrix descriptors,
// matrix products issued by one thread, loads and stores between tensor memory and registers.
#pragma once

#include <cstdint>

namespace gqa {

// ---- tensor memory -----------------------------------------------------------------------
// Whole warp. The address of the first column is left in shared memory at `dst`.
__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns)
                 : "memory");
}
__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// ---- descriptors -----------------------------------------------------------------------------
// Shared-memory matrix in 128-byte swizzled rows (atoms of 8 rows x 128 bytes, 1 KiB aligned).
// K-major operand (a row holds consecutive k): sbo = bytes between groups of 8 rows, lbo unused.
// MN-major operand (a row holds 64 consecutive m or n of one k): sbo = bytes between groups of 8 k,
// lbo = bytes between chunks of 64 m or n.
// The low word holds address and lbo and moves by bytes / 16 with the address; the high word is fixed.
__device__ __forceinline__ uint32_t matrix_lo(uint32_t addr, uint32_t lbo) {
    return (addr & 0x3ffffu) >> 4 | (lbo >> 4) << 16;
}
__host__ __device__ constexpr uint32_t matrix_hi(uint32_t sbo) { return sbo >> 4 | 1u << 14 | 2u << 29; }
// BF16 operands, FP32 accumulator, M x N; b_mn: B is MN-major.
__host__ __device__ constexpr uint32_t mma_shape(uint32_t m, uint32_t n, bool b_mn) {
    return 1u << 4 | 1u << 7 | 1u << 10 | (b_mn ? 1u << 16 : 0u) | (n >> 3) << 17 | (m >> 4) << 24;
}

// ---- products (one thread) ------------------------------------------------------------------------
// D[tmem] (+)= A[smem] B[smem], k = 16; `hi`: high word of both descriptors.
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t shape,
                                          bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b), "r"(hi), "r"(shape), "r"((uint32_t)accumulate)
        : "memory");
}
// D[tmem] (+)= A[tmem] B[smem], k = 16.
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t shape,
                                          bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b), "r"(hi), "r"(shape), "r"((uint32_t)accumulate)
        : "memory");
}
// Arrives on `bar` when all products this thread issued so far are complete.
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
                 : "memory");
}

// ---- tensor memory <-> registers (whole warp; lane l of warp w holds row 32 (w % 4) + l) -----------
#define GQA_R8(c, x, i) c(x[i]), c(x[i + 1]), c(x[i + 2]), c(x[i + 3]), c(x[i + 4]), c(x[i + 5]), c(x[i + 6]), c(x[i + 7])
#define GQA_R32(c, x) GQA_R8(c, x, 0), GQA_R8(c, x, 8), GQA_R8(c, x, 16), GQA_R8(c, x, 24)
#define GQA_OUT(v) "=r"(v)
#define GQA_IO(v) "+r"(v)
#define GQA_IN(v) "r"(v)
// 32 columns. The registers hold the values only after tmem_loaded() on them.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&x)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
        "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
        "%30, %31}, [%32];"
        : GQA_R32(GQA_OUT, x)
        : "r"(addr));
}
__device__ __forceinline__ void tmem_loaded(uint32_t (&x)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : GQA_R32(GQA_IO, x)::"memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&x)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
        "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
        "%30, %31, %32};"
        ::"r"(addr), GQA_R32(GQA_IN, x)
        : "memory");
}
__device__ __forceinline__ void tmem_stored() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
#undef GQA_R8
#undef GQA_R32
#undef GQA_OUT
#undef GQA_IO
#undef GQA_IN

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

}  // namespace gqa
