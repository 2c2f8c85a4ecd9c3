// tdc_delta.cuh — the gated delta rule: what a chunk needs that depends on no state (with
// warp matrix instructions), and the recurrence for running sequences.
//
// Chunks of C = 64 tokens.  With G the running sum of g in the chunk (fp64),
// gam = e^G, Gam_ij = e^(G_i - G_j) and w_i = e^(G_63 - G_i):
//   L = strictly lower part of (K K^T) * Gam      A = L diag(beta)
//   T = (I + A)^-1                                P = scale * lower(Q K^T) * Gam
//   X = V - diag(gam) K S,  U = T X,  V' = diag(beta) U
//   O = scale diag(gam) Q S + P V'                S <- gam_63 S + K^T diag(w) V'
// delta_prepare makes T and P of all chunks at once; delta_walk (its own file)
// walks the chunks of a sequence on the tensor cores; the gradients of a chunk are
// in a third file.
//
// Precision: states, decays, sums and all accumulators are fp32.  An fp32
// operand of a matrix instruction is split into three bf16 parts, which hold it
// exactly (fp16 inputs into two, exactly too): one bf16 rounding (2^-9) at each of the
// chain's operands would put about 3e-3 on every output, and two parts 4e-6 on the
// fp32 final state, twenty times what fp32 throughout gives.  Two fp16 parts have
// nearly fp32's bits, but fp16's range would turn the products of keys with a norm far
// above 1 into infinities.
#pragma once

#include <cfloat>

#include "tdc_dwconv.h"
#include "tdc_seq_common.cuh"
#include "tdc_tc.cuh"

namespace tdc {

constexpr int kChunk = 64;
constexpr int kLdT = kChunk + 8;     // row of a [64][64] tile in shared memory
constexpr int kSq = kChunk * kChunk;  // elements of such a tile in the workspace
constexpr int kCoef = 3 * kChunk + 4;  // a slot's coefficients

// The gradients' workspace: for kTile value channels of a slot, transposed, what
// the gradients of a chunk need of them, in the order of a stage in shared memory
// (so that two copies bring it).  Each part is [columns / 8][kTile][8]; S, dS, U and dX
// have three parts (split3), dO what its type needs.  Two places of a stage hold zeros and
// are not in the workspace: bf16's second part of dO, and one between U's last
// part and dX's, which serves both as the other 64 rows of an operand.
constexpr int kTile = 16;
template <int KP, int DK>
struct GradTile {
  static constexpr int part = kTile * DK * 2, upart = kTile * kChunk * 2;  // bytes
  static constexpr int om = 0;              // dO^T, dX^T: second parts
  static constexpr int xm = om + upart;
  static constexpr int d = xm + upart;      // dS^T behind the chunk
  static constexpr int s = d + 5 * part;    // S^T before it: part i at s - i part
  static constexpr int u = s + part;        // U^T
  static constexpr int zero = u + 3 * upart;
  static constexpr int xl = zero + upart;   // dX^T: last part
  static constexpr int oh = xl + upart;     // dO^T, dX^T: first parts
  static constexpr int xh = oh + upart;
  static constexpr int stage = xh + upart;
  static constexpr int skip = KP == 1 ? upart : 0;
  static constexpr int front = zero - skip, back = stage - xl;  // the two copies
  static constexpr int bytes = front + back;
  static __host__ __device__ constexpr int x(int part) { return part == 0 ? xh : part == 1 ? xm : xl; }
  // where `off` of a stage lies in the workspace's tile
  static __host__ __device__ constexpr int at(int off) { return off - skip - (off > zero ? upart : 0); }
};

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
  __nv_bfloat16* tp;      // T in its three parts, then P: [6][64 x 64]
  float* coef;            // kCoef: gam, w, beta [64] each, and whether a key or a gate is not finite
  unsigned char* kq;      // [chunk][H]: [parts][K / 8][Q's 64 rows, K's 64 rows][8]
  uint64_t timeout_ns;    // of the bounded waits
  int64_t withhold;       // first chunk of a sequence whose copies never come (-1: none)
  int *status_words, *status_host;
  // gradients
  unsigned char* tiles;   // [chunk][HV][V / kTile] GradTile
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
    const uint32_t n = uint32_t(c) / uint32_t(p.chunks_per_b);  // (both below 2^31)
    r.n = r.b = n;
    r.t0 = (c - n * p.chunks_per_b) * kChunk;
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
// sequence.  The other blocks zero the rows that no sequence owns.  Bound by the
// latency of its steps: 5.3 us for 11 sequences with cold caches.
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
  double before = __shfl_up_sync(0xffffffffu, sum, 1);
  if (lane == 0) before = 0.0;
  G[2 * lane + 1] = to_far(sum);
  G[2 * lane] = to_far(before + double(g.x));  // (not sum - g.y: a NaN reaches no token before it)
}

// ---- T and P of every chunk -------------------------------------------------------
// One block a chunk and key head; 4 warps, 16 rows each.  The triangular
// inverse: diagonal blocks of 16 by substitution in fp32, one column a thread,
// then joined twice with matrix instructions (split operands),
// inv([[P, 0], [B, R]]) = [[P', 0], [-R' B P', R']].  Only the 16 x 16 blocks
// on and below the diagonal of T and P are written, and none above is read.
// Bound by the latency of the substitution and the two joins with 4 blocks an SM;
// 8192 tokens of 16 key and 32 value heads (263 MB) take 78 us, 3.4 TB/s.
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
  static constexpr int q = 0;                          // [64][ld]
  static constexpr int k = kChunk * ld * 2;            // [64][ld]
  static constexpr int t = 0;                          // T and A by parts, once Q and K are used
  static constexpr int a = 3 * part;
  static constexpr int G = a + 3 * part;               // Far [64]
  static_assert(2 * kChunk * ld * 2 <= G, "Q and K");
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
    uint32_t pp[3][4];
#pragma unroll
    for (int y = 0; y < 3; ++y)
      ldsm4_t(pp[y], addr_at(t + y * part, kLdT, o + c0, o + 16 * ks, lane));
#pragma unroll
    for (int np = 0; np < NT / 2; ++np) {
      uint32_t b[3][4];
#pragma unroll
      for (int y = 0; y < 3; ++y)
        ldsm4(b[y], addr_b(a + y * part, kLdT, o + n + 16 * np, o + 16 * ks, lane));
#pragma unroll
      for (int i = 0; i < 2; ++i) mma_split(w[2 * np + i], pp, b, 2 * i);
    }
  }
  float x[NT][4] = {};
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    uint32_t wp[3][4];
    split_frag(w[2 * ks], w[2 * ks + 1], wp);
#pragma unroll
    for (int np = ks; np < NT / 2; ++np) {
      uint32_t r[3][4];
#pragma unroll
      for (int y = 0; y < 3; ++y)
        ldsm4(r[y], addr_b(t + y * part, kLdT, o + n + 16 * np, o + n + 16 * ks, lane));
#pragma unroll
      for (int i = 0; i < 2; ++i) mma_split(x[2 * np + i], wp, r, 2 * i);
    }
  }
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {  // X^T's tiles into rows o + n .. of T
    float v[2][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i / 4][i % 4] = -x[2 * ks + i / 4][i % 4];
    uint32_t xp[3][4];
    split_frag(v[0], v[1], xp);
#pragma unroll
    for (int y = 0; y < 3; ++y)
      stsm4_t(addr_at(t + y * part, kLdT, o + c0, o + n + 16 * ks, lane), xp[y]);
  }
}

// Element offset of 16 bytes at row r, columns 8 c .. + 7 of a 64-row tile in
// 8 x 8 blocks.
__device__ __forceinline__ int block_offset(int r, int c) {
  return c * (kChunk * 8) + r * 8;
}

// Blocks on and below the diagonal of a split [64][64] tile, to [3][64 x 64].
__device__ __forceinline__ void store_lower(__nv_bfloat16* dst, const unsigned char* tile, int tid,
                                            int threads) {
  for (int e = tid; e < 3 * kChunk * 8; e += threads) {
    const int r = e & 63, c = (e >> 6) & 7, part = e >> 9;
    if (c < 2 * (r / 16 + 1))
      *reinterpret_cast<uint4*>(dst + part * kSq + block_offset(r, c)) =
          *reinterpret_cast<const uint4*>(tile + part * kChunk * kLdT * 2 + 2 * (r * kLdT + 8 * c));
  }
}

// Q's rows (threads 0-63) and K's to their parts, 8 columns of all rows together.
constexpr int kKeyBlock = 2 * kChunk * 16;  // bytes of 8 columns
template <class E, int DK>
__device__ __forceinline__ void store_keys(unsigned char* dst, const unsigned char* row, int tid) {
#pragma unroll
  for (int c = 0; c < DK / 8; ++c) {
    const uint4 v = *reinterpret_cast<const uint4*>(row + 16 * c);
    uint4* d = reinterpret_cast<uint4*>(dst + c * kKeyBlock + tid * 16);
    if constexpr (std::is_same_v<E, BF16>) {
      *d = v;
    } else {
      uint4 hi, lo;
      split_elem<E>(v.x, hi.x, lo.x);
      split_elem<E>(v.y, hi.y, lo.y);
      split_elem<E>(v.z, hi.z, lo.z);
      split_elem<E>(v.w, hi.w, lo.w);
      *d = hi;
      d[DK / 8 * kKeyBlock / 16] = lo;
    }
  }
}

template <class E, int DK>
__global__ void __launch_bounds__(128, 4) delta_prepare_kernel(const DeltaParams p) {
  extern __shared__ __align__(1024) unsigned char raw[];
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
    store_keys<E, DK>(kq, raw + (tid < kChunk ? Sm::q : Sm::k) + 2 * (tid & 63) * ld, tid);
  }
  const int g = lane >> 2, t2 = (lane & 3) * 2;
  bool odd_key = false;  // a key of this thread's that is not finite: k.k is not
#pragma unroll
  for (int nt = 0; nt < 8; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (8 * nt + t2 + (e & 1) == 16 * warp + g + 8 * (e >> 1)) odd_key |= !(fabsf(kk[nt][e]) <= FLT_MAX);
  for (int gi = 0; gi < p.group; ++gi) {
    const int hv = h * p.group + gi;
    const int64_t slot = chunk * p.HV + hv;
    __nv_bfloat16* tp = p.tp + slot * 6 * kSq;
    __syncthreads();  // q and k, or the last head's tiles, are free
    if (warp == 0) chunk_decay(decay, G, lane);
    if (tid >= 64) sB[tid - 64] = beta;
    if (gi + 1 < p.group) fetch_gates(hv + 1);
    __syncthreads();
    float* coef = p.coef + slot * kCoef;
    bool odd = odd_key;
    if (tid < kChunk) {
      odd |= !(fabsf(sB[tid]) <= FLT_MAX) || !(fabsf(G[tid].hi) <= FLT_MAX);
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
          // A row of T multiplies with the zeros behind its diagonal: what a NaN or infinite
          // key or decay leaves here would reach the rows before it.  Its own and later
          // rows get their NaN from X (delta_walk_kernel).
          const float l = kk[nt][2 * half + u] * gam;
          av[u] = i > j + u ? (fabsf(l) <= FLT_MAX ? l : 0.f) * (u ? be.y : be.x) : 0.f;
        }
        if (nt >= 2 * warp)
          *reinterpret_cast<float2*>(raw + Sm::t + diag_offset(warp, g + 8 * half) +
                                     4 * (j - 16 * warp)) = make_float2(av[0], av[1]);
        uint32_t pp[3], ap[3];
        split3(pv[0], pv[1], pp);
        split3(av[0], av[1], ap);
#pragma unroll
        for (int y = 0; y < 3; ++y) {  // (a warp's 8 rows of P are a whole line)
          *reinterpret_cast<uint32_t*>(tp + (3 + y) * kSq + block_offset(i, nt) + t2) = pp[y];
          *reinterpret_cast<uint32_t*>(raw + Sm::a + y * part + 2 * (i * kLdT + j)) = ap[y];
        }
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
        __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(raw + Sm::t) +
                             (16 * warp + i) * kLdT + 16 * warp + lane;
#pragma unroll
        for (int y = 0; y < 3; ++y) {
          const __nv_bfloat16 r = __float2bfloat16_rn(v);
          dst[y * (part / 2)] = r;
          v -= __bfloat162float(r);
        }
      }
    }
    odd = __syncthreads_or(odd);
    if (tid == 127) coef[3 * kChunk] = odd ? 1.f : 0.f;
    if (warp < 2) join_inverse<16>(sb + Sm::a, sb + Sm::t, 32 * warp, 0, lane);
    __syncthreads();
    if (warp < 2) join_inverse<32>(sb + Sm::a, sb + Sm::t, 0, 16 * warp, lane);
    __syncthreads();
    store_lower(tp, raw + Sm::t, tid, 128);
  }
}

// ---- running sequences ---------------------------------------------------------------
// One block a request, value head and 32 value channels; a thread holds 4
// channels of DK / 16 rows of S.  Reads and writes the state once: bound by
// memory (8 bytes and 7 flops a value).  k.S~, q.S~ and q.k are summed over
// the rows together, so a token costs one exchange through shared memory:
//   o = scale (S~^T q + beta (q.k) u).
// 192 requests of 32 heads of 128 x 128 (805 MB of states read and written):
// 135 us, 6.0 TB/s of the 6.46 that a copy reaches.  4 requests: 6.7 us with cold
// caches.
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
