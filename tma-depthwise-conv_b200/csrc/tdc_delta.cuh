// tdc_delta.cuh — the gated delta rule: chunked forward and gradients with
// warp matrix instructions, and the recurrence for running sequences.
//
// Chunks of C = 64 tokens.  With G the running sum of g in the chunk (fp64),
// gam = e^G, Gam_ij = e^(G_i - G_j) and w_i = e^(G_63 - G_i):
//   L = strictly lower part of (K K^T) * Gam      A = L diag(beta)
//   T = (I + A)^-1                                P = scale * lower(Q K^T) * Gam
//   X = V - diag(gam) K S,  U = T X,  V' = diag(beta) U
//   O = scale diag(gam) Q S + P V'                S <- gam_63 S + K^T diag(w) V'
// delta_prepare makes T and P of all chunks at once; delta_walk (its own file)
// walks the chunks of a sequence on the tensor cores.
//
// Precision: states, decays, sums and all accumulators are fp32.  An fp32
// operand of a matrix instruction is split into two bf16 parts (16 bits of
// mantissa or more; fp16 inputs are split as well, exactly), since one bf16
// rounding (2^-9) at each of the chain's operands would put about 3e-3 on
// every output, more than the output's own rounding, and the final state is
// fp32: with the split it is off by 4e-6.
#pragma once

#include "tdc_dwconv.h"
#include "tdc_seq_common.cuh"
#include "tdc_tc.cuh"

namespace tdc {

constexpr int kChunk = 64;
constexpr int kLdT = kChunk + 8;     // row of a [64][64] tile in shared memory
constexpr int kSq = kChunk * kChunk;  // elements of such a tile in the workspace

struct DeltaParams {
  const void *q, *k, *v, *beta;
  const float* g;
  const float* init;      // [N, HV, K, V] or null
  float* final_state;     // or null
  void* o;
  int64_t T;
  int H, HV, V, group;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh, g_sb, g_st, b_sb, b_st;
  SeqTable seq;
  int64_t chunks_per_b;   // batch form: chunks of each sequence
  int64_t max_chunks;     // chunks, or their upper bound in a packed batch
  // packed batches: filled by delta_plan
  int64_t* seq_lo;        // [N + 1] row offsets, not decreasing
  int64_t* seq_chunk;     // [N + 1] first chunk of each sequence
  bool beta_f32;
  float scale;
  // the forward in segments (segments > 1, batch form): see delta_walk_kernel
  int segments, segment_chunks, pass;
  float* seg_s;           // [N][HV][segments][K][V]: state before each
  float* seg_m;           // [N][HV][segments][K][K]: what a segment makes of a state
  // workspace of all chunks, [chunk][HV] each
  // (tiles in the order of WalkTiles; 8 x 8 blocks, see tdc_tc.cuh)
  __nv_bfloat16* tp;      // T and P, high parts and remainders: [4][64 x 64]
  float* coef;            // [3][64]: gam, w, beta
  unsigned char* kq;      // [chunk][H]: K and Q, [2][parts][64 x K]
  uint64_t timeout_ns;    // of the bounded waits
  int64_t withhold;       // first chunk of a sequence whose copies never come (-1: none)
  int *status_words, *status_host;
  // gradients
  // (32 channels together: [V / 32][2 parts][columns / 8][32][8])
  __nv_bfloat16* um;      // U^T, 64 columns
  __nv_bfloat16* xm;      // dX^T
  __nv_bfloat16* sm;      // S^T before the chunk, K columns
  __nv_bfloat16* dm;      // dS^T behind the chunk
  const void* d_o;
  int64_t do_sb, do_st, do_sh;
  const float* dfinal;
  void *dq, *dk, *dv, *dbeta;
  float *dg, *dinit;
};

// Where chunk c of the batch lies.
struct ChunkAt {
  int64_t n;      // sequence
  int64_t b;      // row of the batch
  int64_t t0;     // first row
  int rows;       // 0: no such chunk
};

__device__ __forceinline__ ChunkAt chunk_at(const DeltaParams& p, int64_t c) {
  ChunkAt r;
  if (p.seq.cu == nullptr) {
    r.n = r.b = c / p.chunks_per_b;
    r.t0 = (c % p.chunks_per_b) * kChunk;
    r.rows = int(min(int64_t(kChunk), p.T - r.t0));
    return r;
  }
  r.b = 0;
  int64_t lo = 0, hi = p.seq.n;  // last sequence whose first chunk is <= c
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (p.seq_chunk[mid] <= c) lo = mid; else hi = mid;
  }
  r.n = lo;
  r.t0 = p.seq_lo[lo] + (c - p.seq_chunk[lo]) * kChunk;
  const int64_t left = p.seq_lo[lo + 1] - r.t0;
  r.rows = int(max(int64_t(0), min(int64_t(kChunk), left)));
  return r;
}

// First chunk, number of chunks, first row and length of sequence n.
struct SeqAt {
  int64_t chunk0, lo, len, b;
};
__device__ __forceinline__ SeqAt seq_at(const DeltaParams& p, int64_t n) {
  if (p.seq.cu == nullptr) return {n * p.chunks_per_b, 0, p.T, n};
  return {p.seq_chunk[n], p.seq_lo[n], p.seq_lo[n + 1] - p.seq_lo[n], 0};
}

// ---- plan of a packed batch ------------------------------------------------------
// Block 0: running maximum of the clamped offsets, and the chunks before each
// sequence.  The other blocks zero the rows that no sequence owns.
struct ZeroRows {
  void* base[5];
  int64_t row_bytes[5];  // multiples of 2
};

__global__ void __launch_bounds__(1024) delta_plan_kernel(const SeqTable s, int64_t* seq_lo,
                                                          int64_t* seq_chunk, const ZeroRows z) {
  __shared__ int64_t sh[1024];
  __shared__ int64_t carry_lo, carry_chunk;
  const int tid = threadIdx.x;
  if (blockIdx.x != 0) {
    int64_t top = 0;
    for (int64_t i = tid; i <= s.n; i += 1024) top = max(top, s.at(i));
    sh[tid] = top;
    __syncthreads();
    for (int d = 512; d; d >>= 1) {
      if (tid < d) sh[tid] = max(sh[tid], sh[tid + d]);
      __syncthreads();
    }
    top = sh[0];
    const int64_t first = s.at(0), step = int64_t(gridDim.x - 1) * 1024;
    const int64_t at = int64_t(blockIdx.x - 1) * 1024 + tid;
    for (int i = 0; i < 5; ++i) {
      if (z.base[i] == nullptr) continue;
      uint16_t* base = static_cast<uint16_t*>(z.base[i]);
      const int64_t per = z.row_bytes[i] / 2;
      for (int64_t e = at; e < first * per; e += step) base[e] = 0;
      for (int64_t e = top * per + at; e < s.T * per; e += step) base[e] = 0;
    }
    return;
  }
  if (tid == 0) carry_lo = 0, carry_chunk = 0;
  for (int64_t i0 = 0; i0 <= s.n; i0 += 1024) {
    const int64_t i = i0 + tid;
    __syncthreads();
    sh[tid] = i <= s.n ? s.at(i) : 0;
    __syncthreads();
    for (int d = 1; d < 1024; d <<= 1) {
      const int64_t v = tid >= d ? sh[tid - d] : 0;
      __syncthreads();
      sh[tid] = max(sh[tid], v);
      __syncthreads();
    }
    const int64_t lo = max(sh[tid], carry_lo);
    const int64_t before = max(tid ? sh[tid - 1] : 0, carry_lo);
    __syncthreads();
    const bool ends = i >= 1 && i <= s.n;  // sequence i-1 is [before, lo)
    sh[tid] = ends ? (lo - before + kChunk - 1) / kChunk : 0;
    __syncthreads();
    for (int d = 1; d < 1024; d <<= 1) {
      const int64_t v = tid >= d ? sh[tid - d] : 0;
      __syncthreads();
      sh[tid] += v;
      __syncthreads();
    }
    if (i <= s.n) {
      seq_lo[i] = lo;
      seq_chunk[i] = carry_chunk + sh[tid];
    }
    __syncthreads();
    if (tid == 1023) carry_lo = lo, carry_chunk += sh[1023];
  }
}

// ---- shared pieces -------------------------------------------------------------------
// rows x (16 * vecs bytes) into shared memory with row stride ld elements;
// rows behind `valid` become zeros.
__device__ __forceinline__ void copy_rows(uint32_t dst, int ld, const uint16_t* src, int64_t stride,
                                          int rows, int valid, int vecs, int tid, int threads) {
  for (int i = tid; i < rows * vecs; i += threads) {
    const int r = i / vecs, c = i % vecs;
    cp_async16(dst + 2 * (r * ld + 8 * c), src + (r < valid ? r * stride : 0) + 8 * c, r < valid);
  }
}

__device__ __forceinline__ float load_beta(const DeltaParams& p, bool bf16, int64_t i) {
  if (p.beta_f32) return static_cast<const float*>(p.beta)[i];
  return bf16 ? to_float<BF16>(p.beta, i) : to_float<F16>(p.beta, i);
}

// Running sum of g over a chunk, by the first warp, two tokens a lane: in fp64,
// kept as a pair of fp32 values (differences of far sums have to keep fp32's
// precision).
struct Far {
  float hi, lo;
};
__device__ __forceinline__ Far to_far(double v) {
  const float hi = float(v);
  return {hi, float(v - double(hi))};
}
__device__ __forceinline__ float minus(const Far& a, const Far& b) {
  return (a.hi - b.hi) + (a.lo - b.lo);
}
__device__ __forceinline__ float2 load_decay(const DeltaParams& p, const ChunkAt& at, int hv,
                                             int lane) {
  float g[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = 2 * lane + i;
    g[i] = t < at.rows ? p.g[at.b * p.g_sb + (at.t0 + t) * p.g_st + hv] : 0.f;
    g[i] = g[i] < -200.f ? -200.f : g[i];
  }
  return make_float2(g[0], g[1]);
}
__device__ __forceinline__ void chunk_decay(const float2& g, Far* G, int lane) {
  double sum = double(g.x) + double(g.y);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const double o = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += o;
  }
  G[2 * lane + 1] = to_far(sum);
  G[2 * lane] = to_far(sum - double(g.y));
}

// ---- T and P of every chunk -------------------------------------------------------
// One block a chunk and key head; 4 warps, 16 rows each.  The triangular
// inverse: diagonal blocks of 16 by substitution in fp32, one column a thread,
// then joined twice with matrix instructions (split operands),
// inv([[P, 0], [B, R]]) = [[P', 0], [-R' B P', R']].  Only the 16 x 16 blocks
// on and below the diagonal of T and P are written, and none above is read.
//
// The fp32 rows (16 floats) of the diagonal blocks of A lie in the unused
// blocks above T's diagonal: row i of block w in row i or 16 + i of one part.
__device__ __forceinline__ int diag_offset(int w, int i) {
  return (w & 1) * kChunk * kLdT * 2 + ((w >> 1) * 16 + i) * kLdT * 2 + (w >> 1 ? 64 : 32);
}

template <int DK>
struct PrepareSmem {
  static constexpr int ld = DK + 8;
  static constexpr int part = kChunk * kLdT * 2;       // one [64][72] tile
  static constexpr int q = 0;                          // [64][ld], later T hi, lo and P hi
  static constexpr int k = kChunk * ld * 2;            // [64][ld]
  static constexpr int t = 0;
  static constexpr int p = 2 * part;
  static constexpr int a = 2 * kChunk * ld * 2 > 4 * part ? 2 * kChunk * ld * 2 : 4 * part;
  static constexpr int G = a + 2 * part;               // Far [64]
  static constexpr int beta = G + 64 * 8;
  static constexpr int bytes = beta + 64 * 4;
};

// Joins the inverses of two diagonal blocks of n columns at o and o + n: one
// warp makes 16 columns, from c0, of X = -R' B P'.  All operands are split tiles.
template <int n>
__device__ __forceinline__ void join_inverse(uint32_t a, uint32_t t, int o, int c0, int lane) {
  constexpr int part = kChunk * kLdT * 2, NT = n / 8, KS = n / 16;
  float w[NT][4] = {};  // (B P')^T: 16 columns of P' by the rows of B
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    if (16 * ks < c0) continue;  // P' is lower triangular: nothing is stored above
    uint32_t ph[4], pl[4];
    ldsm4_t(ph, addr_at(t, kLdT, o + c0, o + 16 * ks, lane));
    ldsm4_t(pl, addr_at(t + part, kLdT, o + c0, o + 16 * ks, lane));
#pragma unroll
    for (int np = 0; np < NT / 2; ++np) {
      uint32_t bh[4], bl[4];
      ldsm4(bh, addr_b(a, kLdT, o + n + 16 * np, o + 16 * ks, lane));
      ldsm4(bl, addr_b(a + part, kLdT, o + n + 16 * np, o + 16 * ks, lane));
#pragma unroll
      for (int i = 0; i < 2; ++i)
        mma_split(w[2 * np + i], ph, pl, bh[2 * i], bh[2 * i + 1], bl[2 * i], bl[2 * i + 1]);
    }
  }
  float x[NT][4] = {};
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    uint32_t wh[4], wl[4];
    split_frag(w[2 * ks], w[2 * ks + 1], wh, wl);
#pragma unroll
    for (int np = ks; np < NT / 2; ++np) {
      uint32_t rh[4], rl[4];
      ldsm4(rh, addr_b(t, kLdT, o + n + 16 * np, o + n + 16 * ks, lane));
      ldsm4(rl, addr_b(t + part, kLdT, o + n + 16 * np, o + n + 16 * ks, lane));
#pragma unroll
      for (int i = 0; i < 2; ++i)
        mma_split(x[2 * np + i], wh, wl, rh[2 * i], rh[2 * i + 1], rl[2 * i], rl[2 * i + 1]);
    }
  }
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {  // X^T's tiles into rows o + n .. of T
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float* v = x[2 * ks + i];
      split2(-v[0], -v[1], hi[2 * i], lo[2 * i]);
      split2(-v[2], -v[3], hi[2 * i + 1], lo[2 * i + 1]);
    }
    stsm4_t(addr_at(t, kLdT, o + c0, o + n + 16 * ks, lane), hi);
    stsm4_t(addr_at(t + part, kLdT, o + c0, o + n + 16 * ks, lane), lo);
  }
}

// Element offset of 16 bytes at row r, columns 8 c .. + 7 of a 64-row tile in
// 8 x 8 blocks.
__device__ __forceinline__ int block_offset(int r, int c) {
  return c * (kChunk * 8) + r * 8;
}

// Blocks on and below the diagonal of a split [64][64] tile, to [2][64 x 64].
__device__ __forceinline__ void store_lower(__nv_bfloat16* dst, const unsigned char* tile, int tid,
                                            int threads) {
  for (int e = tid; e < 2 * kChunk * 8; e += threads) {
    const int r = e & 63, c = (e >> 6) & 7, part = e >> 9;
    if (c < 2 * (r / 16 + 1))
      *reinterpret_cast<uint4*>(dst + part * kSq + block_offset(r, c)) =
          *reinterpret_cast<const uint4*>(tile + part * kChunk * kLdT * 2 + 2 * (r * kLdT + 8 * c));
  }
}

// A [64][DK] tile of the element type to its parts in 8 x 8 blocks.
template <class E, int DK>
__device__ __forceinline__ void store_keys(unsigned char* dst, const unsigned char* tile, int tid,
                                           int threads) {
  for (int e = tid; e < kChunk * (DK / 8); e += threads) {
    const int r = e & 63, c = e >> 6;
    const uint4 v = *reinterpret_cast<const uint4*>(tile + 2 * (r * (DK + 8) + 8 * c));
    uint4* d = reinterpret_cast<uint4*>(dst + 2 * block_offset(r, c));
    if constexpr (std::is_same_v<E, BF16>) {
      *d = v;
    } else {
      uint4 hi, lo;
      split_elem<E>(v.x, hi.x, lo.x);
      split_elem<E>(v.y, hi.y, lo.y);
      split_elem<E>(v.z, hi.z, lo.z);
      split_elem<E>(v.w, hi.w, lo.w);
      *d = hi;
      d[kChunk * DK / 8] = lo;
    }
  }
}

template <class E, int DK>
__global__ void __launch_bounds__(128) delta_prepare_kernel(const DeltaParams p) {
  extern __shared__ __align__(16) unsigned char raw[];
  using Sm = PrepareSmem<DK>;
  constexpr int ld = Sm::ld, part = Sm::part;
  const int64_t chunk = blockIdx.x;
  const int h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const ChunkAt at = chunk_at(p, chunk);
  if (at.rows == 0) return;
  const uint32_t sb = smem_addr(raw);
  Far* G = reinterpret_cast<Far*>(raw + Sm::G);
  float* sB = reinterpret_cast<float*>(raw + Sm::beta);
  const uint16_t* q = static_cast<const uint16_t*>(p.q) + at.b * p.q_sb + at.t0 * p.q_st + h * p.q_sh;
  const uint16_t* k = static_cast<const uint16_t*>(p.k) + at.b * p.k_sb + at.t0 * p.k_st + h * p.k_sh;
  copy_rows(sb + Sm::q, ld, q, p.q_st, kChunk, at.rows, DK / 8, tid, 128);
  copy_rows(sb + Sm::k, ld, k, p.k_st, kChunk, at.rows, DK / 8, tid, 128);
  cp_async_commit();
  // A head's decays (first warp) and betas (last two), loaded one head ahead.
  float2 decay = make_float2(0.f, 0.f);
  float beta = 0.f;
  auto fetch_gates = [&](int hv) {
    if (warp == 0) decay = load_decay(p, at, hv, lane);
    const int t = tid - 64;
    if (t >= 0)
      beta = t < at.rows ? load_beta(p, std::is_same_v<E, BF16>,
                                     at.b * p.b_sb + (at.t0 + t) * p.b_st + hv)
                         : 0.f;
  };
  fetch_gates(h * p.group);
  cp_async_wait<0>();
  __syncthreads();
  // Rows 16 warp .. + 15 of Q K^T and K K^T (both operands exact).
  float qk[8][4] = {}, kk[8][4] = {};
#pragma unroll
  for (int ks = 0; ks < DK / 16; ++ks) {
    uint32_t aq[4], ak[4];
    ldsm4(aq, addr_a(sb + Sm::q, ld, 16 * warp, 16 * ks, lane));
    ldsm4(ak, addr_a(sb + Sm::k, ld, 16 * warp, 16 * ks, lane));
#pragma unroll
    for (int np = 0; np < 4; ++np) {
      if (np > warp) break;  // columns behind the rows are not used
      uint32_t bk[4];
      ldsm4(bk, addr_b(sb + Sm::k, ld, 16 * np, 16 * ks, lane));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mma_elem<E>(qk[2 * np + i], aq, bk[2 * i], bk[2 * i + 1]);
        mma_elem<E>(kk[2 * np + i], ak, bk[2 * i], bk[2 * i + 1]);
      }
    }
  }
  {
    constexpr int64_t bytes = int64_t(std::is_same_v<E, BF16> ? 1 : 2) * kChunk * DK * 2;
    unsigned char* kq = p.kq + (chunk * p.H + h) * 2 * bytes;
    store_keys<E, DK>(kq, raw + Sm::k, tid, 128);
    store_keys<E, DK>(kq + bytes, raw + Sm::q, tid, 128);
  }
  const int g = lane >> 2, t2 = (lane & 3) * 2;
  for (int gi = 0; gi < p.group; ++gi) {
    const int hv = h * p.group + gi;
    const int64_t slot = chunk * p.HV + hv;
    __syncthreads();  // q and k, or the last head's tiles, are free
    if (warp == 0) chunk_decay(decay, G, lane);
    if (tid >= 64) sB[tid - 64] = beta;
    if (gi + 1 < p.group) fetch_gates(hv + 1);
    __syncthreads();
    if (tid < kChunk) {
      float* coef = p.coef + slot * 3 * kChunk;
      coef[tid] = expf(G[tid].hi + G[tid].lo);
      coef[kChunk + tid] = expf(minus(G[kChunk - 1], G[tid]));
      coef[2 * kChunk + tid] = sB[tid];
    }
    const Far Gi[2] = {G[16 * warp + g], G[16 * warp + g + 8]};
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
      if (nt > 2 * warp + 1) break;
      const int j = 8 * nt + t2;
      const float4 far2 = *reinterpret_cast<const float4*>(G + j);
      const Far Gj[2] = {{far2.x, far2.y}, {far2.z, far2.w}};
      const float2 be = *reinterpret_cast<const float2*>(sB + j);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int i = 16 * warp + g + 8 * half;
        float pv[2], av[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float gam = __expf(minus(Gi[half], Gj[u]));
          pv[u] = i >= j + u ? p.scale * gam * qk[nt][2 * half + u] : 0.f;
          av[u] = i > j + u ? kk[nt][2 * half + u] * gam * (u ? be.y : be.x) : 0.f;
        }
        if (nt >= 2 * warp)
          *reinterpret_cast<float2*>(raw + Sm::t + diag_offset(warp, g + 8 * half) +
                                     4 * (j - 16 * warp)) = make_float2(av[0], av[1]);
        uint32_t hi, lo;
        const int off = 2 * (i * kLdT + j);
        split2(pv[0], pv[1], hi, lo);
        *reinterpret_cast<uint32_t*>(raw + Sm::p + off) = hi;
        *reinterpret_cast<uint32_t*>(raw + Sm::p + part + off) = lo;
        split2(av[0], av[1], hi, lo);
        *reinterpret_cast<uint32_t*>(raw + Sm::a + off) = hi;
        *reinterpret_cast<uint32_t*>(raw + Sm::a + part + off) = lo;
      }
    }
    __syncwarp();
    if (lane < 16) {  // the warp's diagonal block, one column a lane
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float* d = reinterpret_cast<const float*>(raw + Sm::t + diag_offset(warp, i));
        float v = i == lane ? 1.f : 0.f;
#pragma unroll
        for (int m = 0; m < i; ++m) v = fmaf(-d[m], x[m], v);
        x[i] = v;
        const __nv_bfloat16 hi = __float2bfloat16_rn(v);
        __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(raw + Sm::t) +
                             (16 * warp + i) * kLdT + 16 * warp + lane;
        dst[0] = hi;
        dst[part / 2] = __float2bfloat16_rn(v - __bfloat162float(hi));
      }
    }
    __syncthreads();
    if (warp < 2) join_inverse<16>(sb + Sm::a, sb + Sm::t, 32 * warp, 0, lane);
    else store_lower(p.tp + slot * 4 * kSq + 2 * kSq, raw + Sm::p, tid - 64, 64);
    __syncthreads();
    if (warp < 2) join_inverse<32>(sb + Sm::a, sb + Sm::t, 0, 16 * warp, lane);
    __syncthreads();
    store_lower(p.tp + slot * 4 * kSq, raw + Sm::t, tid, 128);
  }
}

// ---- gradients of a chunk ------------------------------------------------------------
// One block a chunk and key head, all chunks at once.  With D = dO U^T and
// M = dX U^T (lower parts):
//   dQ = scale gam (dO S^T) + Dt K                     Dt = scale Gam beta_j D
//   dK = -gam (dX S^T) + w beta (U dS^T) + Dt^T Q + (N + N^T) K,  N = -M beta_j Gam
//   dbeta_j = sum_i (P_ij D_ij - M_ij L_ij) + w_j k_j.(U dS^T)_j
// The decay of row t stands in front of everything that reaches from before t to
// t or behind it, so with E_ij = beta_j (P_ij D_ij - M_ij L_ij), i > j,
//   dg_t = sum_{i >= t} (scale gam q.(dO S^T) - gam k.(dX S^T))_i
//        + sum_{j < t} (w beta k.(U dS^T))_j + sum_{i >= t > j} E_ij + gam_63 <dS, S>:
// no terms that cancel (a first token without a state gets exactly 0); the
// double sum grows by the column sum of E and falls by its row sum from row to row.
// 8 warps: 4 groups of 16 rows by 2 halves of the columns.  The value channels
// are walked in tiles of 32, of which the next is on its way while one is used,
// also from one head to the next, as bulk copies (through the load unit,
// cp.async, their issue took half of the kernel's time).
constexpr int kTile = 32;
template <int DK>
struct GradSmem {
  static constexpr int ld = DK + 8;
  static constexpr int ldo = kTile + 8;
  static constexpr int q = 0;
  static constexpr int k = q + kChunk * ld * 2;
  // a stage: S^T, dS^T, U^T, dX^T in two parts each, [columns / 8][32][8] as in the
  // workspace, and dO
  static constexpr int stages = k + kChunk * ld * 2;
  static constexpr int part = kTile * DK * 2, upart = kTile * kChunk * 2;
  static constexpr int s = 0;
  static constexpr int d = s + 2 * part;
  static constexpr int u = d + 2 * part;
  static constexpr int x = u + 2 * upart;
  static constexpr int o = x + 2 * upart;                 // [64][ldo]
  static constexpr int stage = o + kChunk * ldo * 2;
  static constexpr int dt = stages + 2 * stage;           // [2][64][72]
  static constexpr int nn = dt + 2 * kChunk * kLdT * 2;   // [2][64][72]
  static constexpr int G = nn + 2 * kChunk * kLdT * 2;    // Far [64]
  static constexpr int coef = G + 64 * 8;                 // [3][64]
  static constexpr int rows = coef + 3 * 64 * 4;          // [2][4][64]: row sums of both halves
  static constexpr int cols = rows + 2 * 4 * 64 * 4;      // [4][64]: column sums of the row groups
  static constexpr int diag = cols + 4 * 64 * 4;          // [64]
  static constexpr int dot = diag + 64 * 4;               // [8]
  static constexpr int dg = dot + 8 * 4;                  // [2][64]
  static constexpr int full = dg + 2 * 64 * 4;            // uint64 [2]
  static constexpr int bytes = full + 2 * 8;
};

// Addresses in a [columns / 8][32][8] tile: a B fragment pair with the channels as
// contraction, and an A fragment (both with .trans); 8 x 8 blocks of 128
// contiguous bytes, so no bank is hit twice.
__device__ __forceinline__ uint32_t addr_bt_blocks(uint32_t base, int n0, int k0, int lane) {
  return base + (n0 / 8 + (lane >> 4)) * (kTile * 16) + (k0 + (lane & 7) + ((lane >> 3) & 1) * 8) * 16;
}
__device__ __forceinline__ uint32_t addr_at_blocks(uint32_t base, int m0, int k0, int lane) {
  return base + (m0 / 8 + ((lane >> 3) & 1)) * (kTile * 16) + (k0 + (lane & 7) + (lane >> 4) * 8) * 16;
}

template <class E, int DK>
__global__ void __launch_bounds__(256, 1) delta_grad_kernel(const DeltaParams p) {
  extern __shared__ __align__(16) unsigned char raw[];
  using Sm = GradSmem<DK>;
  constexpr int ld = Sm::ld, NT = DK / 16;  // 8-column tiles of a half of K
  const int64_t chunk = blockIdx.x;
  const int h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rg = warp & 3, ch = warp >> 2;
  const ChunkAt at = chunk_at(p, chunk);
  if (at.rows == 0) return;
  const uint32_t sb = smem_addr(raw);
  Far* G = reinterpret_cast<Far*>(raw + Sm::G);
  float* coef = reinterpret_cast<float*>(raw + Sm::coef);
  float* rows = reinterpret_cast<float*>(raw + Sm::rows);
  float* cols = reinterpret_cast<float*>(raw + Sm::cols);
  float* dot = reinterpret_cast<float*>(raw + Sm::dot);
  float* diag = reinterpret_cast<float*>(raw + Sm::diag);
  float* dgs = reinterpret_cast<float*>(raw + Sm::dg);
  const uint16_t* q = static_cast<const uint16_t*>(p.q) + at.b * p.q_sb + at.t0 * p.q_st + h * p.q_sh;
  const uint16_t* k = static_cast<const uint16_t*>(p.k) + at.b * p.k_sb + at.t0 * p.k_st + h * p.k_sh;
  copy_rows(sb + Sm::q, ld, q, p.q_st, kChunk, at.rows, DK / 8, tid, 256);
  copy_rows(sb + Sm::k, ld, k, p.k_st, kChunk, at.rows, DK / 8, tid, 256);
  const int g = lane >> 2, t2 = (lane & 3) * 2;
  const int i0 = 16 * rg + g;        // this thread's rows: i0, i0 + 8
  const int kc0 = ch * (DK / 2);     // its half of K's columns
  float dq[NT][4] = {}, dk[NT][4] = {};

  const int per_head = p.V / kTile, tiles = p.group * per_head;
  uint64_t* full = reinterpret_cast<uint64_t*>(raw + Sm::full);
  if (tid == 0) {
    mbar_init(smem_addr(&full[0]), 1);
    mbar_init(smem_addr(&full[1]), 1);
    fence_mbar_init();
  }
  // Tiles come as four bulk copies, dO's rows through the load unit (one piece a
  // thread; rows behind the sequence's end become zeros).
  auto fetch = [&](int tile) {
    const int head = tile / per_head, v0 = (tile - head * per_head) * kTile;
    const int hv = h * p.group + head;
    const uint32_t st = sb + Sm::stages + (tile & 1) * Sm::stage, bar = smem_addr(&full[tile & 1]);
    if (tid == 0) {
      const int64_t at32 = ((chunk * p.HV + hv) * p.V + v0) / kTile;
      mbar_arrive_expect_tx(bar, 4 * Sm::part + 4 * Sm::upart);
      bulk_load(st + Sm::s, p.sm + at32 * Sm::part, 2 * Sm::part, bar);
      bulk_load(st + Sm::d, p.dm + at32 * Sm::part, 2 * Sm::part, bar);
      bulk_load(st + Sm::u, p.um + at32 * Sm::upart, 2 * Sm::upart, bar);
      bulk_load(st + Sm::x, p.xm + at32 * Sm::upart, 2 * Sm::upart, bar);
    }
    const uint16_t* d_o = static_cast<const uint16_t*>(p.d_o) + at.b * p.do_sb + at.t0 * p.do_st +
                          hv * p.do_sh + v0;
    copy_rows(st + Sm::o, Sm::ldo, d_o, p.do_st, kChunk, at.rows, kTile / 8, tid, 256);
    cp_async_commit();
  };
  __syncthreads();
  fetch(0);  // (Q and K go with its group)

  for (int gi = 0; gi < p.group; ++gi) {
    const int hv = h * p.group + gi;
    const int64_t slot = chunk * p.HV + hv;
    float os[NT][4] = {}, xs[NT][4] = {}, us[NT][4] = {}, D[4][4] = {}, M[4][4] = {};
    float dsum = 0.f;
    for (int vt = 0; vt < per_head; ++vt) {
      const int tile = gi * per_head + vt;
      __syncthreads();  // the other stage (and with a new head what is kept for one) is free
      if (tile + 1 < tiles) fetch(tile + 1);
      if (vt == 0) {
        if (warp == 0) chunk_decay(load_decay(p, at, hv, lane), G, lane);
        const float* src = p.coef + slot * 3 * kChunk;
        if (tid >= 64) coef[tid - 64] = src[tid - 64];
      }
      if (tile + 1 < tiles) cp_async_wait<1>(); else cp_async_wait<0>();
      // A copy that does not come ends the block (all its threads together).
      const bool ok = mbar_wait_bounded(smem_addr(&full[tile & 1]), uint32_t(tile >> 1) & 1u, nullptr,
                                        false, p.timeout_ns);
      if (!ok && tid == 0)
        record_wait_failure(p.status_words, p.status_host, TDC_DEVICE_FULL_TIMEOUT, int(blockIdx.x),
                            tile & 1, tile);
      if (!__syncthreads_and(ok)) {
        // the next tile's copies, if any are on their way, come to rest first
        if (tile + 1 < tiles)
          mbar_wait_bounded(smem_addr(&full[(tile + 1) & 1]), uint32_t((tile + 1) >> 1) & 1u, nullptr,
                            false, p.timeout_ns);
        return;
      }
      const unsigned char* stage = raw + Sm::stages + (tile & 1) * Sm::stage;
      const uint32_t st = smem_addr(stage);
      // <dS, S>
      for (int e = tid; e < kTile * DK / 8; e += 256) {  // 8 values at the same place of all four
        float a[2][8], b[2][8];
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          const int off = part * Sm::part + 16 * e;
          unpack8<BF16>(*reinterpret_cast<const uint4*>(stage + Sm::s + off), a[part]);
          unpack8<BF16>(*reinterpret_cast<const uint4*>(stage + Sm::d + off), b[part]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) dsum = fmaf(a[0][i] + a[1][i], b[0][i] + b[1][i], dsum);
      }
#pragma unroll 1
      for (int ks = 0; ks < kTile / 16; ++ks) {
        uint32_t a[4], oh[4], ol[4], xh[4], xl[4], uh[4], ul[4];
        ldsm4(a, addr_a(st + Sm::o, Sm::ldo, 16 * rg, 16 * ks, lane));
#pragma unroll
        for (int i = 0; i < 4; ++i) split_elem<E>(a[i], oh[i], ol[i]);
        ldsm4_t(xh, addr_at_blocks(st + Sm::x, 16 * rg, 16 * ks, lane));
        ldsm4_t(xl, addr_at_blocks(st + Sm::x + Sm::upart, 16 * rg, 16 * ks, lane));
        ldsm4_t(uh, addr_at_blocks(st + Sm::u, 16 * rg, 16 * ks, lane));
        ldsm4_t(ul, addr_at_blocks(st + Sm::u + Sm::upart, 16 * rg, 16 * ks, lane));
        // D and M: columns are tokens 32 ch .. + 31, from U^T [channel][token]
        {
          uint32_t bh[8], bl[8];
#pragma unroll
          for (int np = 0; np < 2; ++np) {
            ldsm4_t(bh + 4 * np, addr_bt_blocks(st + Sm::u, 32 * ch + 16 * np, 16 * ks, lane));
            ldsm4_t(bl + 4 * np, addr_bt_blocks(st + Sm::u + Sm::upart, 32 * ch + 16 * np, 16 * ks, lane));
          }
          if (32 * ch + 16 <= 16 * rg) {  // all four tiles reach below the diagonal
            mma_elem_split_n<E, 4>(D, oh, ol, bh, bl);
            mma_split_n<4>(M, xh, xl, bh, bl);
          } else if (32 * ch <= 16 * rg) {
            mma_elem_split_n<E, 2>(D, oh, ol, bh, bl);
            mma_split_n<2>(M, xh, xl, bh, bl);
          }
        }
        // dO S^T, dX S^T, U dS^T: columns kc0 .. of K, from S^T [channel][K], 32 at a time
#pragma unroll
        for (int nq = 0; nq < NT / 4; ++nq) {
          uint32_t bh[8], bl[8];
#pragma unroll
          for (int np = 0; np < 2; ++np) {
            ldsm4_t(bh + 4 * np, addr_bt_blocks(st + Sm::s, kc0 + 32 * nq + 16 * np, 16 * ks, lane));
            ldsm4_t(bl + 4 * np, addr_bt_blocks(st + Sm::s + Sm::part, kc0 + 32 * nq + 16 * np, 16 * ks, lane));
          }
          mma_elem_split_n<E, 4>(os + 4 * nq, oh, ol, bh, bl);
          mma_split_n<4>(xs + 4 * nq, xh, xl, bh, bl);
#pragma unroll
          for (int np = 0; np < 2; ++np) {
            ldsm4_t(bh + 4 * np, addr_bt_blocks(st + Sm::d, kc0 + 32 * nq + 16 * np, 16 * ks, lane));
            ldsm4_t(bl + 4 * np, addr_bt_blocks(st + Sm::d + Sm::part, kc0 + 32 * nq + 16 * np, 16 * ks, lane));
          }
          mma_split_n<4>(us + 4 * nq, uh, ul, bh, bl);
        }
      }
    }
    // Row sums with q and k, and the three products into dq and dk.
    float r[2][3] = {};  // [row i0 / i0 + 8][q.dOS, k.dXS, k.UdS]
    const float ga[2] = {coef[i0], coef[i0 + 8]};
    const float wb[2] = {coef[64 + i0] * coef[128 + i0], coef[64 + i0 + 8] * coef[128 + i0 + 8]};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int off = 2 * ((i0 + 8 * half) * ld + kc0 + 8 * nt + t2);
        float qv[2], kv[2];
        unpack2<E>(*reinterpret_cast<const uint32_t*>(raw + Sm::q + off), qv[0], qv[1]);
        unpack2<E>(*reinterpret_cast<const uint32_t*>(raw + Sm::k + off), kv[0], kv[1]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int e = 2 * half + u;
          r[half][0] = fmaf(qv[u], os[nt][e], r[half][0]);
          r[half][1] = fmaf(kv[u], xs[nt][e], r[half][1]);
          r[half][2] = fmaf(kv[u], us[nt][e], r[half][2]);
          dq[nt][e] = fmaf(p.scale * ga[half], os[nt][e], dq[nt][e]);
          dk[nt][e] += wb[half] * us[nt][e] - ga[half] * xs[nt][e];
        }
      }
    // Q K^T and K K^T once more, for this warp's 16 x 32 part.
    float qk[4][4] = {}, kk[4][4] = {};
#pragma unroll 2
    for (int ks = 0; ks < DK / 16; ++ks) {
      uint32_t aq[4], ak[4];
      ldsm4(aq, addr_a(sb + Sm::q, ld, 16 * rg, 16 * ks, lane));
      ldsm4(ak, addr_a(sb + Sm::k, ld, 16 * rg, 16 * ks, lane));
#pragma unroll
      for (int np = 0; np < 2; ++np) {
        uint32_t b[4];
        ldsm4(b, addr_b(sb + Sm::k, ld, 32 * ch + 16 * np, 16 * ks, lane));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          mma_elem<E>(qk[2 * np + i], aq, b[2 * i], b[2 * i + 1]);
          mma_elem<E>(kk[2 * np + i], ak, b[2 * i], b[2 * i + 1]);
        }
      }
    }
    float re[2] = {};  // row sums of E below the diagonal
#pragma unroll
    for (int nt = 0; nt < 4; ++nt) {
      float cs[2] = {};  // column sums of P D - M L below the diagonal, this thread's two rows
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int i = i0 + 8 * half, j = 32 * ch + 8 * nt + t2;
        float dt[2], nn[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int e = 2 * half + u;
          const float gam = i >= j + u ? __expf(minus(G[i], G[j + u])) : 0.f;
          const float be = coef[128 + j + u];
          const float dv = i >= j + u ? D[nt][e] : 0.f, mv = i > j + u ? M[nt][e] : 0.f;
          const float pd = p.scale * gam * qk[nt][e] * dv, ml = gam * kk[nt][e] * mv;
          if (i > j + u) {
            cs[u] += pd - ml;
            re[half] = fmaf(be, pd - ml, re[half]);
          } else if (i == j + u) {
            diag[i] = pd;
          }
          dt[u] = p.scale * gam * be * dv;
          nn[u] = -mv * be * gam;
        }
        uint32_t hi, lo;
        const int off = 2 * (i * kLdT + j);
        split2(dt[0], dt[1], hi, lo);
        *reinterpret_cast<uint32_t*>(raw + Sm::dt + off) = hi;
        *reinterpret_cast<uint32_t*>(raw + Sm::dt + 64 * kLdT * 2 + off) = lo;
        split2(nn[0], nn[1], hi, lo);
        *reinterpret_cast<uint32_t*>(raw + Sm::nn + off) = hi;
        *reinterpret_cast<uint32_t*>(raw + Sm::nn + 64 * kLdT * 2 + off) = lo;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          cs[u] += __shfl_xor_sync(0xffffffffu, cs[u], d);
        }
        if (g == 0) cols[rg * 64 + 32 * ch + 8 * nt + t2 + u] = cs[u];
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        re[half] += __shfl_xor_sync(0xffffffffu, re[half], d);
#pragma unroll
        for (int j = 0; j < 3; ++j) r[half][j] += __shfl_xor_sync(0xffffffffu, r[half][j], d);
      }
      if ((lane & 3) == 0) {
#pragma unroll
        for (int j = 0; j < 3; ++j) rows[(ch * 4 + j) * 64 + i0 + 8 * half] = r[half][j];
        rows[(ch * 4 + 3) * 64 + i0 + 8 * half] = re[half];
      }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) dsum += __shfl_xor_sync(0xffffffffu, dsum, d);
    if (lane == 0) dot[warp] = dsum;
    __syncthreads();
    // dq += Dt K; dk += Dt^T Q + (N + N^T) K
#pragma unroll 1
    for (int ks = 0; ks < 4; ++ks) {
      uint32_t ah[4], al[4], nh[4], nl[4];
      constexpr int part = kChunk * kLdT * 2;
      if (ks <= rg) {
        ldsm4(ah, addr_a(sb + Sm::dt, kLdT, 16 * rg, 16 * ks, lane));
        ldsm4(al, addr_a(sb + Sm::dt + part, kLdT, 16 * rg, 16 * ks, lane));
        ldsm4(nh, addr_a(sb + Sm::nn, kLdT, 16 * rg, 16 * ks, lane));
        ldsm4(nl, addr_a(sb + Sm::nn + part, kLdT, 16 * rg, 16 * ks, lane));
#pragma unroll
        for (int nq = 0; nq < NT / 4; ++nq) {
          uint32_t b[8];
#pragma unroll
          for (int np = 0; np < 2; ++np)
            ldsm4_t(b + 4 * np, addr_bt(sb + Sm::k, ld, kc0 + 32 * nq + 16 * np, 16 * ks, lane));
          mma_split_elem_n<E, 4>(dq + 4 * nq, ah, al, b);
          mma_split_elem_n<E, 4>(dk + 4 * nq, nh, nl, b);
        }
      }
      if (ks >= rg) {
        ldsm4_t(ah, addr_at(sb + Sm::dt, kLdT, 16 * rg, 16 * ks, lane));
        ldsm4_t(al, addr_at(sb + Sm::dt + part, kLdT, 16 * rg, 16 * ks, lane));
        ldsm4_t(nh, addr_at(sb + Sm::nn, kLdT, 16 * rg, 16 * ks, lane));
        ldsm4_t(nl, addr_at(sb + Sm::nn + part, kLdT, 16 * rg, 16 * ks, lane));
#pragma unroll
        for (int nq = 0; nq < NT / 4; ++nq) {
          uint32_t b[8], c[8];
#pragma unroll
          for (int np = 0; np < 2; ++np) {
            ldsm4_t(b + 4 * np, addr_bt(sb + Sm::q, ld, kc0 + 32 * nq + 16 * np, 16 * ks, lane));
            ldsm4_t(c + 4 * np, addr_bt(sb + Sm::k, ld, kc0 + 32 * nq + 16 * np, 16 * ks, lane));
          }
          mma_split_elem_n<E, 4>(dk + 4 * nq, ah, al, b);
          mma_split_elem_n<E, 4>(dk + 4 * nq, nh, nl, c);
        }
      }
    }
    // dbeta and dg
    if (tid < 64) {
      const int i = tid;
      const float ga1 = coef[i], w1 = coef[64 + i], be = coef[128 + i];
      float s0[4], c0 = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) s0[j] = rows[j * 64 + i] + rows[(4 + j) * 64 + i];
#pragma unroll
      for (int j = 0; j < 4; ++j) c0 += cols[j * 64 + i];
      if (i < at.rows) {
        const int64_t o = (at.b * p.T + at.t0 + i) * p.HV + hv;
        const float db = c0 + diag[i] + w1 * s0[2];
        if (p.beta_f32) static_cast<float*>(p.dbeta)[o] = db;
        else store_float<E>(p.dbeta, o, db);
      }
      dgs[i] = p.scale * ga1 * s0[0] - ga1 * s0[1];
      dgs[64 + i] = be * c0 - s0[3] + w1 * be * s0[2];
    }
    __syncthreads();
    if (warp == 0) {
      float ds = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ds += dot[i];
      ds *= coef[63];
      // sums from the row to the end, and over the rows before it
      const float a0 = dgs[2 * lane], a1 = dgs[2 * lane + 1];
      const float f0 = dgs[64 + 2 * lane], f1 = dgs[64 + 2 * lane + 1];
      float up = a0 + a1, down = f0 + f1;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const float x = __shfl_down_sync(0xffffffffu, up, d);
        const float y = __shfl_up_sync(0xffffffffu, down, d);
        if (lane + d < 32) up += x;
        if (lane >= d) down += y;
      }
      const float above = __shfl_down_sync(0xffffffffu, up, 1);
      float before = __shfl_up_sync(0xffffffffu, down, 1);
      if (lane == 0) before = 0.f;
      const int64_t o = (at.b * p.T + at.t0 + 2 * lane) * p.HV + hv;
      if (2 * lane < at.rows) p.dg[o] = up + before + ds;
      if (2 * lane + 1 < at.rows)
        p.dg[o + p.HV] = a1 + (lane < 31 ? above : 0.f) + before + f0 + ds;
    }
  }
  // dq and dk rows
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int i = i0 + 8 * half;
    if (i >= at.rows) continue;
    const int64_t o = ((at.b * p.T + at.t0 + i) * p.H + h) * DK + kc0 + t2;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.dq) + o + 8 * nt) =
          pack2_rn<E>(dq[nt][2 * half], dq[nt][2 * half + 1]);
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.dk) + o + 8 * nt) =
          pack2_rn<E>(dk[nt][2 * half], dk[nt][2 * half + 1]);
    }
  }
}

// ---- running sequences ---------------------------------------------------------------
// One block a request, value head and 32 value channels; a thread holds 4
// channels of DK / 16 rows of S.  Reads and writes the state once: bound by
// memory (8 bytes and 7 flops a value).  k.S~, q.S~ and q.k are summed over
// the rows together, so a token costs one exchange through shared memory:
//   o = scale (S~^T q + beta (q.k) u).
template <class E, int DK>
__global__ void __launch_bounds__(128) delta_step_kernel(const DeltaParams p, float* state,
                                                         const void* idx, bool idx64,
                                                         int64_t slots) {
  constexpr int R = DK / 16;  // rows a thread holds
  __shared__ float red[4][9][8];
  const int64_t b = blockIdx.x;
  const int hv = blockIdx.y, h = hv / p.group, tid = threadIdx.x;
  const int lane = tid & 31, warp = tid >> 5, cl = tid & 7, rgp = tid >> 3;
  const int vc = blockIdx.z * 32 + 4 * cl;
  const int64_t slot = slot_of(idx, idx64, b, slots, tid, 128);
  uint16_t* o = static_cast<uint16_t*>(p.o) + (b * p.T * p.HV + hv) * p.V + vc;
  const int64_t ostep = int64_t(p.HV) * p.V;
  if (slot < 0) {
    const uint32_t f = slot == -1 ? 0u : nan16<E>() * 0x10001u;
    if (rgp == 0)
      for (int64_t t = 0; t < p.T; ++t) *reinterpret_cast<uint2*>(o + t * ostep) = make_uint2(f, f);
    return;
  }
  float* sp = state + ((slot * p.HV + hv) * DK + rgp * R) * int64_t(p.V) + vc;
  float4 S[R];
#pragma unroll
  for (int r = 0; r < R; ++r) S[r] = *reinterpret_cast<const float4*>(sp + int64_t(r) * p.V);
  for (int64_t t = 0; t < p.T; ++t) {
    const float gr = p.g[b * p.g_sb + t * p.g_st + hv];
    const float decay = expf(gr < -200.f ? -200.f : gr);
    const float beta = load_beta(p, std::is_same_v<E, BF16>, b * p.b_sb + t * p.b_st + hv);
    const uint16_t* qp = static_cast<const uint16_t*>(p.q) + b * p.q_sb + t * p.q_st + h * p.q_sh + rgp * R;
    const uint16_t* kp = static_cast<const uint16_t*>(p.k) + b * p.k_sb + t * p.k_st + h * p.k_sh + rgp * R;
    float q[R], k[R], v[4];
#pragma unroll
    for (int r = 0; r < R; r += 4) {
      const uint2 a = *reinterpret_cast<const uint2*>(qp + r), c = *reinterpret_cast<const uint2*>(kp + r);
      unpack2<E>(a.x, q[r], q[r + 1]);
      unpack2<E>(a.y, q[r + 2], q[r + 3]);
      unpack2<E>(c.x, k[r], k[r + 1]);
      unpack2<E>(c.y, k[r + 2], k[r + 3]);
    }
    const uint2 vv = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.v) + b * p.v_sb +
                                                     t * p.v_st + hv * p.v_sh + vc);
    unpack2<E>(vv.x, v[0], v[1]);
    unpack2<E>(vv.y, v[2], v[3]);
    float a[9] = {};  // k.S~ (4), q.S~ (4), q.k
#pragma unroll
    for (int r = 0; r < R; ++r) {
      S[r].x *= decay, S[r].y *= decay, S[r].z *= decay, S[r].w *= decay;
      a[0] = fmaf(k[r], S[r].x, a[0]);
      a[1] = fmaf(k[r], S[r].y, a[1]);
      a[2] = fmaf(k[r], S[r].z, a[2]);
      a[3] = fmaf(k[r], S[r].w, a[3]);
      a[4] = fmaf(q[r], S[r].x, a[4]);
      a[5] = fmaf(q[r], S[r].y, a[5]);
      a[6] = fmaf(q[r], S[r].z, a[6]);
      a[7] = fmaf(q[r], S[r].w, a[7]);
      a[8] = fmaf(q[r], k[r], a[8]);
    }
#pragma unroll
    for (int i = 0; i < 9; ++i) {
      a[i] += __shfl_xor_sync(0xffffffffu, a[i], 8);
      a[i] += __shfl_xor_sync(0xffffffffu, a[i], 16);
    }
    __syncthreads();
    if (lane < 8) {
#pragma unroll
      for (int i = 0; i < 9; ++i) red[warp][i][lane] = a[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 9; ++i) a[i] = red[0][i][cl] + red[1][i][cl] + red[2][i][cl] + red[3][i][cl];
    float u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = beta * (v[i] - a[i]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      S[r].x = fmaf(k[r], u[0], S[r].x);
      S[r].y = fmaf(k[r], u[1], S[r].y);
      S[r].z = fmaf(k[r], u[2], S[r].z);
      S[r].w = fmaf(k[r], u[3], S[r].w);
    }
    if (rgp == 0) {
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = p.scale * fmaf(a[8], u[i], a[4 + i]);
      *reinterpret_cast<uint2*>(o + t * ostep) =
          make_uint2(pack2_rn<E>(y[0], y[1]), pack2_rn<E>(y[2], y[3]));
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) *reinterpret_cast<float4*>(sp + int64_t(r) * p.V) = S[r];
}

}  // namespace tdc
