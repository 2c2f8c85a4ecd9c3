// tdc_seq_common.cuh — what the sequence kernels share: packed-batch lookups,
// slot indices, 16-byte vectors of 16-bit elements, warp matrix instructions
// and the split of an fp32 operand into three bf16 ones.
#pragma once

#include <cuda_bf16.h>

#include "tdc_ptx.cuh"

namespace tdc {

// ---- failed waits -----------------------------------------------------------
// Records that a pipeline wait gave up, as the depthwise kernels do: the first
// failure on the device in its status words {code, block, stage, load}, and in
// the device's slot of the mapped host page, code last.
__device__ __forceinline__ void record_wait_failure(int* words, int* host, int code, int block,
                                                    int stage, int64_t load) {
  if (atomicCAS(&words[0], 0, code) != 0) return;
  words[1] = block;
  words[2] = stage;
  words[3] = int(load);
  if (host == nullptr) return;
  volatile int* h = host;
  h[1] = block;
  h[2] = stage;
  h[3] = int(load);
  __threadfence_system();
  h[0] = code;
}

// ---- packed batches -----------------------------------------------------------
// Row offsets of a packed batch, int32 or int64, read as the header states:
// clamped to [0, T].
struct SeqTable {
  const void* cu;   // null: a [B, T] batch, every sequence has T rows
  int64_t n;        // number of sequences
  int64_t T;
  bool is64;

  __device__ __forceinline__ int64_t at(int64_t i) const {
    const int64_t v = is64 ? static_cast<const int64_t*>(cu)[i]
                           : int64_t(static_cast<const int32_t*>(cu)[i]);
    return v < 0 ? 0 : (v > T ? T : v);
  }
  // First sequence that ends behind row t (n if none does).
  __device__ __forceinline__ int64_t first_ending_after(int64_t t) const {
    int64_t lo = 0, hi = n;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (at(mid + 1) > t) hi = mid; else lo = mid + 1;
    }
    return lo;
  }
};

// ---- slots --------------------------------------------------------------------
// Slot of request b: >= 0 a state to update, -1 padding (zeros), -2 an index
// that no state may be read or written for (NaN).  An index that an earlier
// request has already is refused, so no two blocks update one state; every
// thread of the block calls this, and all get the same answer.
__device__ __forceinline__ int64_t slot_of(const void* idx, bool is64, int64_t b, int64_t slots,
                                           int tid, int threads) {
  if (idx == nullptr) return b < slots ? b : -2;
  auto get = [&](int64_t i) {
    return is64 ? static_cast<const int64_t*>(idx)[i]
                : int64_t(static_cast<const int32_t*>(idx)[i]);
  };
  const int64_t mine = get(b);
  bool again = false;
  for (int64_t i = tid; i < b; i += threads) again |= get(i) == mine;
  again = __syncthreads_or(again);
  if (mine < 0) return -1;
  return (again || mine >= slots) ? -2 : mine;
}

// ---- vectors --------------------------------------------------------------------
template <class E>
__device__ __forceinline__ void unpack8(const uint4& v, float f[8]) {
  unpack2<E>(v.x, f[0], f[1]);
  unpack2<E>(v.y, f[2], f[3]);
  unpack2<E>(v.z, f[4], f[5]);
  unpack2<E>(v.w, f[6], f[7]);
}

template <class E>
__device__ __forceinline__ uint4 pack8(const float f[8]) {
  return make_uint4(pack2_rn<E>(f[0], f[1]), pack2_rn<E>(f[2], f[3]), pack2_rn<E>(f[4], f[5]),
                    pack2_rn<E>(f[6], f[7]));
}

// d += a b for two fp32 values in one instruction.
__device__ __forceinline__ void fma_pair(float2& d, const float2& a, const float2& b) {
  asm("{\n"
      " .reg .b64 x, y, z;\n"
      " mov.b64 x, {%2, %3};\n"
      " mov.b64 y, {%4, %5};\n"
      " mov.b64 z, {%0, %1};\n"
      " fma.rn.f32x2 z, x, y, z;\n"
      " mov.b64 {%0, %1}, z;\n"
      "}\n"
      : "+f"(d.x), "+f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
}

template <class E>
__device__ __forceinline__ uint16_t nan16() {
  return std::is_same_v<E, BF16> ? 0x7FC0 : 0x7E00;
}

template <class E>
__device__ __forceinline__ float to_float(const void* p, int64_t i) {
  if constexpr (std::is_same_v<E, BF16>) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  else return __half2float(static_cast<const __half*>(p)[i]);
}

template <class E>
__device__ __forceinline__ void store_float(void* p, int64_t i, float v) {
  if constexpr (std::is_same_v<E, BF16>) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// 1 / (1 + exp(-z)), both steps in hardware's approximate forms (2^-21 or
// better); an overflowing exp gives 0, as the limit is.
__device__ __forceinline__ float sigmoid_f(float z) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + __expf(-z)));
  return r;
}

// ---- asynchronous copies ----------------------------------------------------------
// 16 bytes global -> shared; with `valid` false the destination gets zeros and
// nothing is read.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ---- warp matrix instructions -------------------------------------------------------
// Fragments of mma.m16n8k16 (g = lane / 4, t = lane % 4; a register holds two
// neighbouring columns of A, or rows of B):
//   A: a0 (g, 2t), a1 (g+8, 2t), a2 (g, 2t+8), a3 (g+8, 2t+8)
//   B: b0 (2t, g), b1 (2t+8, g);   C: c0,c1 (g, 2t), c2,c3 (g+8, 2t)
// so the C fragments of two neighbouring 8-column tiles are, once packed, the
// A fragment of a 16-deep step: products chain in registers.
__device__ __forceinline__ void mma_bf16(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Both operands in the element type (their products are exact in fp32).
template <class E>
__device__ __forceinline__ void mma_elem(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<E, BF16>) mma_bf16(c, a, b0, b1);
  else mma_f16(c, a, b0, b1);
}

__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void stsm4_t(uint32_t addr, const uint32_t r[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
               : "memory");
}

// An fp32 pair as three bf16 parts, each the remainder of those before it: 3 x 8
// bits hold fp32's 24, so nothing is lost (but what is below bf16's smallest values).
// A product with an exact bf16 operand costs three matrix instructions; one of two such
// operands six, without those of 2^-24 of its size and below.
__device__ __forceinline__ void split3(float x, float y, uint32_t r[3]) {
  r[0] = pack2_rn<BF16>(x, y);
  fma2<BF16>(r[0], 0xBF80BF80u, x, y);  // x - its part, exact (times -1, no unpacking)
  r[1] = pack2_rn<BF16>(x, y);
  fma2<BF16>(r[1], 0xBF80BF80u, x, y);
  r[2] = pack2_rn<BF16>(x, y);
}

// The first two of them: 16 bits of mantissa or more.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack2_rn<BF16>(x, y);
  fma2<BF16>(hi, 0xBF80BF80u, x, y);  // x - high part, exact (times -1, no unpacking)
  lo = pack2_rn<BF16>(x, y);
}

// A packed pair of elements as bf16 high parts and remainders: bf16 is itself;
// fp16's 11 bits fit the two exactly.
template <class E>
__device__ __forceinline__ void split_elem(uint32_t v, uint32_t& hi, uint32_t& lo) {
  if constexpr (std::is_same_v<E, BF16>) {
    hi = v;
    lo = 0;
  } else {
    float x, y;
    unpack2<E>(v, x, y);
    split2(x, y, hi, lo);
  }
}

// The A fragment of step `ks` from the C fragments of tiles 2ks, 2ks+1, split.
__device__ __forceinline__ void split_frag(const float c0[4], const float c1[4], uint32_t a[3][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float* c = i < 2 ? c0 : c1;
    uint32_t r[3];
    split3(c[2 * (i & 1)], c[2 * (i & 1) + 1], r);
#pragma unroll
    for (int x = 0; x < 3; ++x) a[x][i] = r[x];
  }
}

// c += A B, both split (b: registers at, at + 1 of each part), the small products first:
// an accumulator that is still small rounds off less.
__device__ __forceinline__ void mma_split(float c[4], const uint32_t a[3][4], const uint32_t b[3][4],
                                          int at) {
#pragma unroll
  for (int sum = 2; sum >= 0; --sum)
#pragma unroll
    for (int i = 0; i <= sum; ++i) mma_bf16(c, a[i], b[sum - i][at], b[sum - i][at + 1]);
}

// Addresses for ldmatrix.x4 over a row-major 16-bit tile with `ld` elements a
// row (ld * 2 bytes an odd multiple of 16, so that 8 rows hit all banks).
// B fragments of two 8-column tiles from a tile stored [n][k]:
//   r0,r1 = b0,b1 of columns n0..n0+7, r2,r3 of n0+8..n0+15.
__device__ __forceinline__ uint32_t addr_b(uint32_t base, int ld, int n0, int k0, int lane) {
  return base + 2 * ((n0 + (lane & 7) + ((lane >> 4) << 3)) * ld + k0 + ((lane >> 3) & 1) * 8);
}
// An A fragment from a tile stored [m][k].
__device__ __forceinline__ uint32_t addr_a(uint32_t base, int ld, int m0, int k0, int lane) {
  return base + 2 * ((m0 + (lane & 7) + ((lane >> 3) & 1) * 8) * ld + k0 + ((lane >> 4) << 3));
}
// An A fragment from a tile stored [k][m] (with .trans); as a store address
// for stmatrix.trans: C fragments of two neighbouring tiles into [col][row].
__device__ __forceinline__ uint32_t addr_at(uint32_t base, int ld, int m0, int k0, int lane) {
  return base + 2 * ((k0 + (lane & 7) + ((lane >> 4) << 3)) * ld + m0 + ((lane >> 3) & 1) * 8);
}

}  // namespace tdc
