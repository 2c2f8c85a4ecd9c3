// tdc_qknorm.cuh — norms of queries and keys for each head and the rotation
// of their positions, in one pass, with its gradients.
//
// One pass reads and writes each value once (4 bytes) and does about 8 flops
// on it: bound by memory, and at a few tokens by the launch.  A head row of D
// values is held by LANES neighbouring lanes, 8 values each, so the sum of
// squares is a few shuffles and a pair (i, i + R/2) of the half layout sits
// R/16 lanes apart (R % 16 == 0), again one shuffle a value; the pairs of the
// interleaved layout sit in one lane.
#pragma once

#include "tdc_seq_common.cuh"

namespace tdc {

struct QkParams {
  const void *q, *k, *qw, *kw;
  const float *cos, *sin;
  const void* pos;
  void *qo, *ko;
  int64_t T;
  int Hq, Hk, D, R;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, p_sb, p_st;
  int64_t table_rows, rows;  // rows: B * T
  bool pos64, interleaved;
  bool norm;
  float mul;                 // 1 / D (mean) or 1 (sum)
  float eps;
  // gradients
  const void *gq, *gk;
  void *dq, *dk;
  int64_t gq_sb, gq_st, gq_sh, gk_sb, gk_st, gk_sh;
  float* partial;            // [blocks][2][D]
  int rows_per_block;
};

template <int LANES>
__device__ __forceinline__ float lane_sum(float v) {
#pragma unroll
  for (int d = LANES / 2; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// How the pairs lie: no rotation, (i, i + R/2), (2i, 2i + 1).
enum { kNoTurn = 0, kHalves = 1, kPairs = 2 };

// cos and sin of the pairs that this lane's values belong to, for the angle
// (sign 1) or its opposite (-1): halves, 8 of each for pair (8 lane + i) mod R/2,
// the sine with the sign that this lane's half takes; pairs, 4 for 4 lane + i.
template <int TURN>
struct Turn {
  static constexpr int N = TURN == kPairs ? 4 : 8;
  float c[N], s[N];
};

template <int TURN>
__device__ __forceinline__ void load_turn(const QkParams& p, int64_t b, int64_t t, int lane,
                                          float sign, Turn<TURN>& r) {
  constexpr int N = Turn<TURN>::N;
  const int64_t pi = b * p.p_sb + t * p.p_st;
  const int64_t at = p.pos == nullptr ? t
                     : p.pos64        ? static_cast<const int64_t*>(p.pos)[pi]
                                      : int64_t(static_cast<const int32_t*>(p.pos)[pi]);
  const int half = p.R / 2;
  if (at < 0 || at >= p.table_rows) {
#pragma unroll
    for (int i = 0; i < N; ++i) r.c[i] = r.s[i] = __int_as_float(0x7fc00000);
    return;
  }
  int from = N * lane;
  if (TURN == kHalves) {
    if (from >= half) from -= half; else sign = -sign;
  }
  const int64_t o = at * half + from;
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 c = __ldg(reinterpret_cast<const float4*>(p.cos + o + i));
    const float4 s = __ldg(reinterpret_cast<const float4*>(p.sin + o + i));
    r.c[i] = c.x, r.c[i + 1] = c.y, r.c[i + 2] = c.z, r.c[i + 3] = c.w;
    r.s[i] = sign * s.x, r.s[i + 1] = sign * s.y, r.s[i + 2] = sign * s.z, r.s[i + 3] = sign * s.w;
  }
}

// Rotates the row that LANES lanes hold.  Lanes behind R keep their values;
// every lane takes part in the shuffles.
template <int LANES, int TURN>
__device__ __forceinline__ void rotate(const QkParams& p, const Turn<TURN>& r, int lane, float f[8]) {
  const bool in = 8 * lane < p.R;
  if constexpr (TURN == kPairs) {
    if (!in) return;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float a = f[i], b = f[i + 1];
      f[i] = a * r.c[i / 2] - b * r.s[i / 2];
      f[i + 1] = b * r.c[i / 2] + a * r.s[i / 2];
    }
  } else {
    const int step = p.R / 16;  // lanes from a value to its partner
    const int partner = !in ? lane : lane < step ? lane + step : lane - step;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float o = __shfl_sync(0xffffffffu, f[i], partner, LANES);
      if (in) f[i] = fmaf(f[i], r.c[i], o * r.s[i]);
    }
  }
}

__device__ __forceinline__ uint4 ldg16(const void* base, int64_t elem) {
  return __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + elem));
}

// 1 / sqrt(mean or sum of squares + eps) of the row.
template <int LANES>
__device__ __forceinline__ float inv_norm(const QkParams& p, const float f[8]) {
  float2 q = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 v = make_float2(f[i], f[i + 1]);
    fma_pair(q, v, v);
  }
  const float s = lane_sum<LANES>(q.x + q.y);
  return p.norm ? rsqrtf(fmaf(s, p.mul, p.eps)) : 1.f;
}

// Row (b, t) of the tensors, and the heads of a group of lanes in it: queries
// first, then keys, in elements.
struct RowAt {
  const uint16_t *q, *k;
  int64_t qh, kh;  // from head to head
  __device__ __forceinline__ const uint16_t* head(int h, int Hq) const {
    return h < Hq ? q + h * qh : k + (h - Hq) * kh;
  }
};
__device__ __forceinline__ RowAt row_of(const void* q, const void* k, int64_t b, int64_t t, int64_t qb,
                                        int64_t qt, int64_t qh, int64_t kb, int64_t kt, int64_t kh,
                                        int lane) {
  return {static_cast<const uint16_t*>(q) + b * qb + t * qt + 8 * lane,
          static_cast<const uint16_t*>(k) + b * kb + t * kt + 8 * lane, qh, kh};
}
__device__ __forceinline__ uint4 ldg16(const uint16_t* at) {
  return __ldg(reinterpret_cast<const uint4*>(at));
}

// A block takes one row of [B, T]; its groups of LANES lanes go over the heads,
// queries first, HEADS of a group's at a time: their loads are all under way
// before the first sum is needed.  Measured: 8192 rows of 32 + 8 heads of 128
// (bf16, RMS, 64 values rotated, 168 MB) 54 us, 3.1 TB/s, bound by the latency of
// load, sum, rotation and store in each of a block's few turns; 4999 rows of
// 16 + 16 heads in fp16, unit norm, no rotation (82 MB) 16.5 us, 5.0 TB/s; 64 rows
// 5.5 us with cold caches.
template <class E, int LANES, int HEADS, int TURN>
__global__ void __launch_bounds__(256, 4) qk_norm_rope_kernel(const QkParams p) {
  const uint32_t row = blockIdx.x;
  const uint32_t b = row / uint32_t(p.T), t = row - b * uint32_t(p.T);
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int groups = blockDim.x / LANES;
  const bool live = 8 * lane < p.D;
  const int heads = p.Hq + p.Hk;
  const RowAt in = row_of(p.q, p.k, b, t, p.q_sb, p.q_st, p.q_sh, p.k_sb, p.k_st, p.k_sh, lane);
  uint16_t* qo = static_cast<uint16_t*>(p.qo) + int64_t(row) * p.Hq * p.D + 8 * lane;
  uint16_t* ko = static_cast<uint16_t*>(p.ko) + int64_t(row) * p.Hk * p.D + 8 * lane;
  const int per_warp = 32 / LANES;
  // whole warps stay together in the shuffles, so a warp goes on while any of
  // its groups has a head left
  const int first = (group / per_warp) * per_warp, mine = group % per_warp;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  Turn<TURN> turn;
  for (int h0 = first; h0 < heads; h0 += HEADS * groups) {
    uint4 v[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const int h = h0 + mine + i * groups;
      v[i] = h < heads && live ? ldg16(in.head(h, p.Hq)) : zero;  // (lanes behind D hold zeros)
    }
    if (TURN != kNoTurn && h0 == first && 8 * lane < p.R) load_turn<TURN>(p, b, t, lane, 1.f, turn);
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      if (h0 + i * groups >= heads) break;
      const int h = h0 + mine + i * groups;
      const bool is_q = h < p.Hq;
      float f[8];
      unpack8<E>(v[i], f);
      const float inv = inv_norm<LANES>(p, f);
      const void* weight = is_q ? p.qw : p.kw;
      if (weight != nullptr) {
        float w[8];
        unpack8<E>(live ? ldg16(weight, 8 * lane) : zero, w);  // (from the cache)
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= inv * w[j];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= inv;
      }
      if constexpr (TURN != kNoTurn) rotate<LANES, TURN>(p, turn, lane, f);
      if (h < heads && live)
        *reinterpret_cast<uint4*>(is_q ? qo + h * p.D : ko + (h - p.Hq) * p.D) = pack8<E>(f);
    }
  }
}

// Gradients.  With y = R(x inv w) and xh = x inv: dy' = R^T dy,
// dw = sum dy' xh, dx = inv (dy' w - xh mean-or-sum(dy' w xh)).  A block takes
// rows_per_block rows; each group of lanes keeps its share of the two
// weights' gradients in registers, the block adds its groups in shared memory
// and writes one partial sum, which qk_wsum_kernel adds in block order.
// Measured at 8192 rows of 32 + 8 heads of 128 (bf16, 252 MB): 91 us, 2.8 TB/s,
// bound like the forward; qk_wsum_kernel: 7 us.
template <class E, int LANES, int HEADS, int TURN>
__global__ void __launch_bounds__(256) qk_norm_rope_bwd_kernel(const QkParams p) {
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int groups = blockDim.x / LANES, per_warp = 32 / LANES;
  const int first = (group / per_warp) * per_warp, mine = group % per_warp;
  const bool live = 8 * lane < p.D;
  const int heads = p.Hq + p.Hk;
  float dqw[8] = {}, dkw[8] = {};
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const uint4 wq = p.qw != nullptr && live ? ldg16(p.qw, 8 * lane) : zero;
  const uint4 wk = p.kw != nullptr && live ? ldg16(p.kw, 8 * lane) : zero;
  const uint32_t r0 = blockIdx.x * uint32_t(p.rows_per_block);
  const uint32_t r1 = min(r0 + uint32_t(p.rows_per_block), uint32_t(p.rows));
  for (uint32_t row = r0; row < r1; ++row) {
    const uint32_t b = row / uint32_t(p.T), t = row - b * uint32_t(p.T);
    const RowAt in = row_of(p.q, p.k, b, t, p.q_sb, p.q_st, p.q_sh, p.k_sb, p.k_st, p.k_sh, lane);
    const RowAt gr = row_of(p.gq, p.gk, b, t, p.gq_sb, p.gq_st, p.gq_sh, p.gk_sb, p.gk_st, p.gk_sh, lane);
    uint16_t* dq = static_cast<uint16_t*>(p.dq) + int64_t(row) * p.Hq * p.D + 8 * lane;
    uint16_t* dk = static_cast<uint16_t*>(p.dk) + int64_t(row) * p.Hk * p.D + 8 * lane;
    Turn<TURN> turn;
    for (int h0 = first; h0 < heads; h0 += HEADS * groups) {
      uint4 v[HEADS], g[HEADS];
#pragma unroll
      for (int i = 0; i < HEADS; ++i) {
        const int h = h0 + mine + i * groups;
        const bool go = h < heads && live;
        v[i] = go ? ldg16(in.head(h, p.Hq)) : zero;
        g[i] = go ? ldg16(gr.head(h, p.Hq)) : zero;
      }
      if (TURN != kNoTurn && h0 == first && 8 * lane < p.R) load_turn<TURN>(p, b, t, lane, -1.f, turn);
#pragma unroll
      for (int i = 0; i < HEADS; ++i) {
        if (h0 + i * groups >= heads) break;
        const int h = h0 + mine + i * groups;
        const bool is_q = h < p.Hq;
        float f[8], d[8];
        unpack8<E>(v[i], f);
        unpack8<E>(g[i], d);
        const float inv = inv_norm<LANES>(p, f);
        if constexpr (TURN != kNoTurn) rotate<LANES, TURN>(p, turn, lane, d);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= inv;
        if ((is_q ? p.qw : p.kw) != nullptr) {
          float w[8];
          unpack8<E>(is_q ? wq : wk, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float dw = d[j] * f[j];
            // (a spare group's row of zeros may have 0 * inf here)
            dqw[j] += is_q ? dw : 0.f;
            dkw[j] += is_q || h >= heads ? 0.f : dw;
            d[j] *= w[j];
          }
        }
        float2 q = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 8; j += 2)
          fma_pair(q, make_float2(d[j], d[j + 1]), make_float2(f[j], f[j + 1]));
        const float m = p.norm ? lane_sum<LANES>(q.x + q.y) * p.mul : 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = inv * fmaf(-f[j], m, d[j]);
        if (h < heads && live)
          *reinterpret_cast<uint4*>(is_q ? dq + h * p.D : dk + (h - p.Hq) * p.D) = pack8<E>(d);
      }
    }
  }
  if (p.partial == nullptr) return;
  __shared__ float red[2][256 * 8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    red[0][threadIdx.x * 8 + i] = dqw[i];
    red[1][threadIdx.x * 8 + i] = dkw[i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.D; i += blockDim.x) {
    const int which = i / p.D, d = i % p.D;
    float sum = 0.f;
    for (int g = 0; g < groups; ++g) sum += red[which][g * LANES * 8 + d];
    p.partial[int64_t(blockIdx.x) * 2 * p.D + i] = sum;
  }
}

template <class E>
__global__ void __launch_bounds__(256) qk_wsum_kernel(const float* partial, int64_t blocks, int D,
                                                      void* dqw, void* dkw) {
  // One warp a value: a lane adds every 32nd block, then the lanes are added.
  const int v = (blockIdx.x * blockDim.x + threadIdx.x) / 32, lane = threadIdx.x & 31;
  if (v >= 2 * D) return;
  float sum = 0.f;
  for (int64_t b = lane; b < blocks; b += 32) sum += partial[b * 2 * D + v];
  sum = lane_sum<32>(sum);
  if (lane != 0) return;
  if (v < D) {
    if (dqw != nullptr) store_float<E>(dqw, v, sum);
  } else if (dkw != nullptr) {
    store_float<E>(dkw, v - D, sum);
  }
}

}  // namespace tdc
