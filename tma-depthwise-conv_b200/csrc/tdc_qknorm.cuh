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
  int norm;                  // 0 none, 1 rms, 2 l2
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

// cos and sin of the pairs that this lane's 8 values belong to: in the half
// layout pair (8 * lane + i) mod R/2, in the interleaved one 4 * lane + i / 2.
struct Turn {
  float c[8], s[8];
};

__device__ __forceinline__ void load_turn(const QkParams& p, int64_t b, int64_t t, int lane,
                                          Turn& r) {
  const int64_t pi = b * p.p_sb + t * p.p_st;
  const int64_t at = p.pos == nullptr ? t
                     : p.pos64        ? static_cast<const int64_t*>(p.pos)[pi]
                                      : int64_t(static_cast<const int32_t*>(p.pos)[pi]);
  const int half = p.R / 2;
  if (at < 0 || at >= p.table_rows) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.c[i] = r.s[i] = __int_as_float(0x7fc00000);
    return;
  }
  if (p.interleaved) {
    const int64_t o = at * half + 4 * lane;
    const float4 c = __ldg(reinterpret_cast<const float4*>(p.cos + o));
    const float4 s = __ldg(reinterpret_cast<const float4*>(p.sin + o));
    r.c[0] = r.c[1] = c.x, r.c[2] = r.c[3] = c.y, r.c[4] = r.c[5] = c.z, r.c[6] = r.c[7] = c.w;
    r.s[0] = r.s[1] = s.x, r.s[2] = r.s[3] = s.y, r.s[4] = r.s[5] = s.z, r.s[6] = r.s[7] = s.w;
  } else {
    const int64_t o = at * half + (8 * lane) % half;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const float4 c = __ldg(reinterpret_cast<const float4*>(p.cos + o + i));
      const float4 s = __ldg(reinterpret_cast<const float4*>(p.sin + o + i));
      r.c[i] = c.x, r.c[i + 1] = c.y, r.c[i + 2] = c.z, r.c[i + 3] = c.w;
      r.s[i] = s.x, r.s[i + 1] = s.y, r.s[i + 2] = s.z, r.s[i + 3] = s.w;
    }
  }
}

// Rotates the row that LANES lanes hold, by the angle (sign 1) or back (-1).
// Lanes behind R keep their values; every lane takes part in the shuffles.
template <int LANES>
__device__ __forceinline__ void rotate(const QkParams& p, const Turn& r, int lane, float sign,
                                       float f[8]) {
  const bool in = 8 * lane < p.R;
  if (p.interleaved) {
    if (!in) return;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float a = f[i], b = f[i + 1];
      f[i] = a * r.c[i] - sign * b * r.s[i];
      f[i + 1] = b * r.c[i] + sign * a * r.s[i];
    }
    return;
  }
  const int step = p.R / 16;           // lanes from a value to its partner
  const bool low = lane < step;        // the first of the pair
  const int partner = low ? lane + step : lane - step;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float o = __shfl_sync(0xffffffffu, f[i], in ? partner : lane, LANES);
    if (in) f[i] = f[i] * r.c[i] + (low ? -sign : sign) * o * r.s[i];
  }
}

__device__ __forceinline__ uint4 ldg16(const void* base, int64_t elem) {
  return __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + elem));
}

// 1 / sqrt(mean or sum of squares + eps) of the row.
template <int LANES>
__device__ __forceinline__ float inv_norm(const QkParams& p, const float f[8]) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = fmaf(f[i], f[i], s);
  s = lane_sum<LANES>(s);
  if (p.norm == 0) return 1.f;
  return rsqrtf(p.norm == 1 ? s / float(p.D) + p.eps : s + p.eps);
}

// Where head h (queries first) of row (b, t) starts.
struct HeadAt {
  const void* in;
  int64_t at;
  bool is_q, has;
  int hh;
};
__device__ __forceinline__ HeadAt head_at(const QkParams& p, int64_t b, int64_t t, int h) {
  HeadAt r;
  r.has = h < p.Hq + p.Hk;
  r.is_q = h < p.Hq;
  r.hh = r.is_q ? h : h - p.Hq;
  r.in = r.is_q ? p.q : p.k;
  r.at = r.is_q ? b * p.q_sb + t * p.q_st + r.hh * p.q_sh : b * p.k_sb + t * p.k_st + r.hh * p.k_sh;
  return r;
}

// A block takes one row of [B, T]; its groups of LANES lanes go over the heads,
// queries first, HEADS of a group's at a time: their loads are all under way
// before the first sum is needed (one at a time left the pass waiting for
// memory at a third of its bandwidth).
template <class E, int LANES, int HEADS>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const QkParams p) {
  const int64_t row = blockIdx.x;
  const int64_t b = row / p.T, t = row % p.T;
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int groups = blockDim.x / LANES;
  const bool live = 8 * lane < p.D;
  const int heads = p.Hq + p.Hk;
  // whole warps stay together in the shuffles, so a warp goes on while any of
  // its groups has a head left
  const int per_warp = 32 / LANES, first = (group / per_warp) * per_warp;
  for (int h0 = first; h0 < heads; h0 += HEADS * groups) {
    uint4 v[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const HeadAt at = head_at(p, b, t, h0 + i * groups + group % per_warp);
      v[i] = at.has && live ? ldg16(at.in, at.at + 8 * lane) : make_uint4(0, 0, 0, 0);
    }
    Turn turn;
    if (p.R > 0 && 8 * lane < p.R) load_turn(p, b, t, lane, turn);
    uint4 wq = make_uint4(0, 0, 0, 0), wk = wq;  // (lanes behind D hold zeros)
    if (p.qw != nullptr && live) wq = ldg16(p.qw, 8 * lane);
    if (p.kw != nullptr && live) wk = ldg16(p.kw, 8 * lane);
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      if (h0 + i * groups >= heads) break;
      const HeadAt at = head_at(p, b, t, h0 + i * groups + group % per_warp);
      float f[8];
      unpack8<E>(v[i], f);
      const float inv = inv_norm<LANES>(p, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= inv;
      if ((at.is_q ? p.qw : p.kw) != nullptr) {
        float w[8];
        unpack8<E>(at.is_q ? wq : wk, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= w[j];
      }
      if (p.R > 0) rotate<LANES>(p, turn, lane, 1.f, f);
      if (at.has && live) {
        uint16_t* out = static_cast<uint16_t*>(at.is_q ? p.qo : p.ko) +
                        (row * (at.is_q ? p.Hq : p.Hk) + at.hh) * p.D + 8 * lane;
        *reinterpret_cast<uint4*>(out) = pack8<E>(f);
      }
    }
  }
}

// Gradients.  With y = R(x inv w) and xh = x inv: dy' = R^T dy,
// dw = sum dy' xh, dx = inv (dy' w - xh mean-or-sum(dy' w xh)).  A block takes
// rows_per_block rows; each group of lanes keeps its share of the two
// weights' gradients in registers, the block adds its groups in shared memory
// and writes one partial sum, which qk_wsum_kernel adds in block order.
template <class E, int LANES, int HEADS>
__global__ void __launch_bounds__(256) qk_norm_rope_bwd_kernel(const QkParams p) {
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int groups = blockDim.x / LANES, per_warp = 32 / LANES;
  const int first = (group / per_warp) * per_warp;
  const bool live = 8 * lane < p.D;
  const int heads = p.Hq + p.Hk;
  float dqw[8] = {}, dkw[8] = {};
  uint4 wq = make_uint4(0, 0, 0, 0), wk = wq;  // (lanes behind D hold zeros)
  if (p.qw != nullptr && live) wq = ldg16(p.qw, 8 * lane);
  if (p.kw != nullptr && live) wk = ldg16(p.kw, 8 * lane);
  const int64_t r0 = int64_t(blockIdx.x) * p.rows_per_block;
  const int64_t r1 = min(r0 + p.rows_per_block, p.rows);
  for (int64_t row = r0; row < r1; ++row) {
    const int64_t b = row / p.T, t = row % p.T;
    for (int h0 = first; h0 < heads; h0 += HEADS * groups) {
      uint4 v[HEADS], g[HEADS];
#pragma unroll
      for (int i = 0; i < HEADS; ++i) {
        const HeadAt at = head_at(p, b, t, h0 + i * groups + group % per_warp);
        const int64_t ga = at.is_q ? b * p.gq_sb + t * p.gq_st + at.hh * p.gq_sh
                                   : b * p.gk_sb + t * p.gk_st + at.hh * p.gk_sh;
        const bool go = at.has && live;
        v[i] = go ? ldg16(at.in, at.at + 8 * lane) : make_uint4(0, 0, 0, 0);
        g[i] = go ? ldg16(at.is_q ? p.gq : p.gk, ga + 8 * lane) : make_uint4(0, 0, 0, 0);
      }
      Turn turn;
      if (p.R > 0 && 8 * lane < p.R) load_turn(p, b, t, lane, turn);
#pragma unroll
      for (int i = 0; i < HEADS; ++i) {
        if (h0 + i * groups >= heads) break;
        const HeadAt at = head_at(p, b, t, h0 + i * groups + group % per_warp);
        float f[8], d[8];
        unpack8<E>(v[i], f);
        unpack8<E>(g[i], d);
        const float inv = inv_norm<LANES>(p, f);
        if (p.R > 0) rotate<LANES>(p, turn, lane, -1.f, d);
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= inv;
        if ((at.is_q ? p.qw : p.kw) != nullptr) {
          float w[8];
          unpack8<E>(at.is_q ? wq : wk, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float dw = d[j] * f[j];
            if (at.is_q) dqw[j] += dw; else dkw[j] += dw;
            d[j] *= w[j];
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaf(d[j], f[j], m);
        m = lane_sum<LANES>(m);
        m = p.norm == 0 ? 0.f : p.norm == 1 ? m / float(p.D) : m;
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = inv * (d[j] - f[j] * m);
        if (at.has && live) {
          uint16_t* out = static_cast<uint16_t*>(at.is_q ? p.dq : p.dk) +
                          (row * (at.is_q ? p.Hq : p.Hk) + at.hh) * p.D + 8 * lane;
          *reinterpret_cast<uint4*>(out) = pack8<E>(d);
        }
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
