// tdc_tc.cuh — thin wrappers of the 5th-generation tensor core instructions:
// TMEM allocation, loads and stores, tcgen05.mma with A in TMEM or shared memory and
// B in shared memory, and untiled bulk copies.  Every instruction is spelled out.
#pragma once

#include "tdc_ptx.cuh"

namespace tdc {

// ---- TMEM --------------------------------------------------------------------
// 512 columns of 128 lanes x 32 bits; an address is lane << 16 | column.  A warp
// reaches the 32 lanes of its quadrant (warp number % 4): thread i lane i.
__device__ __forceinline__ void tmem_alloc(uint32_t result, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(result),
               "r"(columns)
               : "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns) {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns)
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}
// Loads come back complete: the wait is part of the statement, so no use of a
// value can be moved in front of it.
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
      "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
      "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, "
      "%36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, "
      "%53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]),
        "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]),
        "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]),
        "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]),
        "=r"(r[62]), "=r"(r[63])
      : "r"(at)
      : "memory");
}

// ---- matrix products ------------------------------------------------------------
// B operands are tiles of 64 rows of 16-bit elements in shared memory without a
// swizzle: 8 x 8 blocks of 128 contiguous bytes (8 rows of 16 bytes), blocks of
// the same 8 columns one after another (128 bytes apart), the next 8 columns
// behind all 64 rows (1024 bytes).  The same bytes serve with the rows as N
// (columns are the contraction) and with the columns as N (rows are).
constexpr uint32_t kRowBlock = 128, kColBlock = 1024;

// Descriptor of such a tile in two words.  Low: bits 0-13 start address / 16,
// 16-29 the leading byte offset / 16 (K-major: from 8 contraction columns to the
// next; N-major: from 8 contraction rows to the next).  High: bits 0-13 the
// stride byte offset / 16 (from 8 of N to the next), bit 14 set.  Adding bytes /
// 16 to the low word moves the start.
__device__ __forceinline__ uint32_t tile_desc(uint32_t addr, bool n_major) {
  return (addr >> 4) | ((n_major ? kRowBlock : kColBlock) >> 4) << 16;
}
__host__ __device__ constexpr uint32_t tile_desc_high(bool n_major) {
  return ((n_major ? kColBlock : kRowBlock) >> 4) | 1u << 14;
}
// The same for any tile of 8 x 8 blocks of 128 bytes: `lead` bytes from one to the
// next along the contraction, `stride` along M or N.
__device__ __forceinline__ uint32_t block_desc(uint32_t addr, uint32_t lead) {
  return (addr >> 4) | (lead >> 4) << 16;
}
__host__ __device__ constexpr uint32_t block_desc_high(uint32_t stride) {
  return (stride >> 4) | 1u << 14;
}
// bf16 operands, fp32 accumulators, M = 128.
__device__ __forceinline__ uint32_t mma_desc(uint32_t n, bool n_major, bool m_major = false) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(m_major) << 15) | (uint32_t(n_major) << 16) |
         ((n >> 3) << 17) | ((128u >> 4) << 24);
}
// d[128 x N] (+)= a[128 x 16] b[16 x N]; one thread issues it.
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t a, uint32_t b_low, uint32_t b_high,
                                       uint32_t desc, bool accumulate) {
  asm volatile(
      "{\n"
      " .reg .pred p;\n"
      " .reg .b64 b;\n"
      " setp.ne.b32 p, %5, 0;\n"
      " mov.b64 b, {%2, %3};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n"
      "}\n" ::"r"(d),
      "r"(a), "r"(b_low), "r"(b_high), "r"(desc), "r"(uint32_t(accumulate))
      : "memory");
}
// The same with A in shared memory.
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a_low, uint32_t a_high, uint32_t b_low,
                                          uint32_t b_high, uint32_t desc, bool accumulate) {
  asm volatile(
      "{\n"
      " .reg .pred p;\n"
      " .reg .b64 a, b;\n"
      " setp.ne.b32 p, %6, 0;\n"
      " mov.b64 a, {%1, %2};\n"
      " mov.b64 b, {%3, %4};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n"
      "}\n" ::"r"(d),
      "r"(a_low), "r"(a_high), "r"(b_low), "r"(b_high), "r"(desc), "r"(uint32_t(accumulate))
      : "memory");
}
// What this thread wrote to shared memory, before the products read it.
__device__ __forceinline__ void fence_proxy_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// One lane of a converged warp, the same one every time.  The products are
// issued under it in code that the whole warp runs: then their operands stay in
// uniform registers (32 cycles a product of N = 64; issued by `lane == 0` alone
// each took 64 to 120).
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n"
      " .reg .pred p;\n"
      " elect.sync _|p, 0xffffffff;\n"
      " selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(one));
  return one != 0;
}
// Arrives on `bar` once the products issued so far by this thread are done.
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
      : "memory");
}

// ---- untiled bulk copy, global -> shared (16-byte aligned, a multiple of 16 bytes) ----
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

}  // namespace tdc
