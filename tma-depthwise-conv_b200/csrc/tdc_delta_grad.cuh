// tdc_delta_grad.cuh — gradients of a chunk of the gated delta rule, on the
// 5th-generation tensor cores.
//
// With D = dO U^T and M = dX U^T (lower parts):
//   dQ = scale gam (dO S^T) + Dt K                     Dt = scale Gam beta_j D
//   dK = -gam (dX S^T) + w beta (U dS^T) + Dt^T Q + (N + N^T) K,  N = -M beta_j Gam
//   dbeta_j = sum_i (P_ij D_ij - M_ij L_ij) + w_j k_j.(U dS^T)_j
// The decay of row t stands in front of everything that reaches from before t to
// t or behind it, so with E_ij = beta_j (P_ij D_ij - M_ij L_ij), i > j,
//   dg_t = sum_{i >= t} (scale gam q.(dO S^T) - gam k.(dX S^T))_i
//        + sum_{j < t} (w beta k.(U dS^T))_j + sum_{i >= t > j} E_ij + gam_63 <dS, S>:
// no terms that cancel (a first token without a state gets exactly 0); the
// double sum grows by the column sum of E and falls by its row sum from row to row.
//
// One block a chunk and key head.  Tokens are the rows of every product: lanes
// 0-63 of TMEM are the tokens of dO (and of what becomes dQ), lanes 64-127 those
// of dX (dK), so with M = 128
//   [dO; dX] S^T and [dO; dX] U^T      both halves at once,
//   [U_hi; U_lo] dS^T                  the two parts of U in the halves, added later,
//   [Q; K] K^T                         once a block,
//   [Dt; N] K                          into dQ and dK,
//   [Dt_hi; Dt_lo]^T Q + [N_hi; N_lo]^T K   into dK, again by parts.
// The walks left U, dX, dO, S and dS transposed, as [32 channels][8 columns]
// blocks that serve as A with the tokens and as B with the keys along them.  The
// channels are the contraction and come in tiles of 32 by bulk copies, two stages;
// meanwhile the threads sum <dS, S>.  A thread owns a lane and half of the
// columns; row sums are its own, column sums go through shuffles.
#pragma once

#include "tdc_delta.cuh"
#include "tdc_tc.cuh"

namespace tdc {

constexpr int kTile = 32;  // value channels of a stage

template <class E, int DK>
struct GradSmem {
  static constexpr int KP = std::is_same_v<E, BF16> ? 1 : 2;
  // rows of Q, then of K: [parts][DK / 8][128][8]
  static constexpr int qk = 0, qkpart = 2 * kChunk * DK * 2;
  // rows of Dt, then of N: [2 parts][8][128][8]
  static constexpr int dn = qk + KP * qkpart, dnpart = 2 * kChunk * kChunk * 2;
  static constexpr int stages = dn + 2 * dnpart;
  static constexpr int part = kTile * DK * 2, upart = kTile * kChunk * 2;
  static constexpr int s = 0;               // S^T, high parts and remainders
  static constexpr int d = s + 2 * part;    // dS^T
  static constexpr int u = d + 2 * part;    // U^T
  static constexpr int a = u + 2 * upart;   // dO^T and dX^T, then their remainders (dO's: 0 in bf16)
  static constexpr int stage = a + 4 * upart;
  static constexpr int sync = stages + 2 * stage;
};
struct GradSync {
  uint64_t full[2], used[2], keys, done, drain;
  uint32_t tmem;
  Far G[kChunk];
  float coef[3 * kChunk];      // gam, w, beta
  float sums[3][2][128];       // row sums by half of the columns: see kSum*
  float cols[4][kChunk];       // column sums of P D - M L below the diagonal, by 32 lanes
  float diag[kChunk];          // P D on it
  float dot[8];
  float dg[2][kChunk];
};
enum { kSumState = 0, kSumKey = 1, kSumE = 2 };
constexpr uint32_t kGradOX = 0, kGradDM = 128, kGradUS = 192, kGradGram = 320, kGradK = 384;

// d[128 x N] (+)= A B over 16 contraction rows; the operands are tiles
// [16 channels][8 columns] with the columns of 8 `step` bytes apart.
template <int N>
__device__ __forceinline__ void grad_product(uint32_t d, uint32_t a, uint32_t b, bool accumulate) {
  constexpr uint32_t high = block_desc_high(kTile * 16);
  tc_mma_ss(d, block_desc(a, kRowBlock), high, block_desc(b, kRowBlock), high, mma_desc(N, true, true),
            accumulate);
}

// 32 columns from c0 of a row of Q and K (row l of the 128), in fp32.
template <class E, int DK>
__device__ __forceinline__ void load_key_row(float (&f)[32], const unsigned char* qk, int l, int c0) {
  using Sm = GradSmem<E, DK>;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const unsigned char* src = qk + (c0 / 8 + c) * 2048 + l * 16;
    unpack8<BF16>(*reinterpret_cast<const uint4*>(src), f + 8 * c);
    if constexpr (Sm::KP == 2) {
      float lo[8];
      unpack8<BF16>(*reinterpret_cast<const uint4*>(src + Sm::qkpart), lo);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[8 * c + i] += lo[i];
    }
  }
}

template <class E, int DK>
__global__ void __launch_bounds__(256, 1) delta_grad_kernel(const DeltaParams p) {
  extern __shared__ __align__(1024) unsigned char raw[];
  using Sm = GradSmem<E, DK>;
  constexpr int KP = Sm::KP;
  const int64_t chunk = blockIdx.x;
  const int h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const ChunkAt at = chunk_at(p, chunk);
  if (at.rows == 0) return;
  const int wq = warp & 3, hc = warp >> 2;  // its lanes and its half of the columns
  const int l = 32 * wq + lane, i = l & 63;
  const bool upper = l >= 64;
  const int kc0 = hc * (DK / 2);
  const uint32_t sb = smem_addr(raw);
  GradSync* sy = reinterpret_cast<GradSync*>(raw + Sm::sync);
  const int per_head = p.V / kTile, tiles = p.group * per_head;
  if (tid == 0) {
    for (int x = 0; x < 2; ++x) mbar_init(smem_addr(&sy->full[x]), 1), mbar_init(smem_addr(&sy->used[x]), 1);
    mbar_init(smem_addr(&sy->keys), 1);
    mbar_init(smem_addr(&sy->done), 1);
    mbar_init(smem_addr(&sy->drain), 1);
    fence_mbar_init();
  }
  if (warp == 0) tmem_alloc(smem_addr(&sy->tmem), 512);
  if constexpr (KP == 1) {  // dO has no remainders
    for (int x = 0; x < 2; ++x)
      for (int e = 16 * tid; e < Sm::upart; e += 16 * 256)
        *reinterpret_cast<uint4*>(raw + Sm::stages + x * Sm::stage + Sm::a + 2 * Sm::upart + e) =
            make_uint4(0, 0, 0, 0);
    fence_proxy_async();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = sy->tmem, lanes = tm + (uint32_t(wq) << 21);

  auto fetch = [&](int tile) {  // one thread
    const int head = tile / per_head, v0 = (tile - head * per_head) * kTile;
    const int64_t at32 = ((chunk * p.HV + h * p.group + head) * p.V + v0) / kTile;
    const uint32_t st = sb + Sm::stages + (tile & 1) * Sm::stage, bar = smem_addr(&sy->full[tile & 1]);
    mbar_arrive_expect_tx(bar, 4 * Sm::part + (4 + KP) * Sm::upart);
    bulk_load(st + Sm::s, p.sm + at32 * Sm::part, 2 * Sm::part, bar);
    bulk_load(st + Sm::d, p.dm + at32 * Sm::part, 2 * Sm::part, bar);
    bulk_load(st + Sm::u, p.um + at32 * Sm::upart, 2 * Sm::upart, bar);
    const __nv_bfloat16* x = p.xm + at32 * Sm::upart;
    bulk_load(st + Sm::a + Sm::upart, x, Sm::upart, bar);
    bulk_load(st + Sm::a + 3 * Sm::upart, x + Sm::upart / 2, Sm::upart, bar);
    const __nv_bfloat16* o = p.om + at32 * (KP * Sm::upart / 2);
    bulk_load(st + Sm::a, o, Sm::upart, bar);
    if constexpr (KP == 2) bulk_load(st + Sm::a + 2 * Sm::upart, o + Sm::upart / 2, Sm::upart, bar);
  };
  int fetched = min(tiles, 2);  // (as warp 0 knows it)
  if (warp == 0) {
    // Q and K, 8 columns a copy: the two halves of the rows beside each other
    constexpr int keys = kChunk * DK * 2;
    if (lane == 0) mbar_arrive_expect_tx(smem_addr(&sy->keys), 2 * KP * keys);
    __syncwarp();
    const unsigned char* src = p.kq + (chunk * p.H + h) * (2 * KP * keys);
    for (int e = lane; e < 2 * KP * (DK / 8); e += 32) {
      const int c = e % (DK / 8), which = e / (DK / 8);  // K's parts, then Q's
      const int part = which % KP;
      bulk_load(sb + Sm::qk + part * Sm::qkpart + c * 2048 + (which < KP ? 1024 : 0),
                src + which * keys + c * 1024, 1024, smem_addr(&sy->keys));
    }
    if (lane == 0)
      for (int x = 0; x < fetched; ++x) fetch(x);
    __syncwarp();
  }
  auto wait = [&](uint64_t& bar, int phase, int code, int64_t load) {
    if (mbar_wait_bounded(smem_addr(&bar), uint32_t(phase) & 1u, nullptr, false, p.timeout_ns)) return true;
    record_wait_failure(p.status_words, p.status_host, code, int(blockIdx.x), phase & 1, load);
    return false;
  };
  bool ok = wait(sy->keys, 0, TDC_DEVICE_FULL_TIMEOUT, 0);
  float acc[DK / 2] = {}, acc2[DK / 2] = {};  // dQ or dK of the lane's token; dK, its parts
  int tile = 0;
  bool run = true;
  for (int gi = 0; gi < p.group && run; ++gi) {
    const int hv = h * p.group + gi;
    const int64_t slot = chunk * p.HV + hv;
    float dsum = 0.f;
    for (int vt = 0; vt < per_head; ++vt, ++tile) {
      const int x = tile & 1;
      ok = ok && wait(sy->full[x], tile >> 1, TDC_DEVICE_FULL_TIMEOUT, tile);
      const unsigned char* stage = raw + Sm::stages + x * Sm::stage;
      const uint32_t st = smem_addr(stage);
      if (warp == 0 && __all_sync(0xffffffffu, ok)) {
        tc_fence_after();
        if (elect_one()) {
          if (tile == 0) {
            // the rows of Q and K by those of K
#pragma unroll
            for (int y = 0; y < KP; ++y)
#pragma unroll
              for (int z = 0; z < KP - y; ++z)
#pragma unroll
                for (int ks = 0; ks < DK / 16; ++ks)
                  tc_mma_ss(tm + kGradGram, block_desc(sb + Sm::qk + y * Sm::qkpart + ks * 4096, 2048),
                            block_desc_high(kRowBlock),
                            block_desc(sb + Sm::qk + z * Sm::qkpart + 1024 + ks * 4096, 2048),
                            block_desc_high(kRowBlock), mma_desc(64, false, false), y + z + ks > 0);
          }
#pragma unroll
          for (int ks = 0; ks < kTile / 16; ++ks) {
            const bool on = vt + ks > 0;
            const uint32_t from = st + ks * 2 * kRowBlock;
            const uint32_t a = from + Sm::a, b = a + 2 * Sm::upart, u = from + Sm::u;
            grad_product<DK>(tm + kGradOX, a, from + Sm::s, on);
            grad_product<DK>(tm + kGradOX, b, from + Sm::s, true);
            grad_product<DK>(tm + kGradOX, a, from + Sm::s + Sm::part, true);
            grad_product<64>(tm + kGradDM, a, u, on);
            grad_product<64>(tm + kGradDM, b, u, true);
            grad_product<64>(tm + kGradDM, a, u + Sm::upart, true);
            grad_product<DK>(tm + kGradUS, u, from + Sm::d, on);
            grad_product<DK>(tm + kGradUS, u, from + Sm::d + Sm::part, true);
          }
          tc_commit(smem_addr(&sy->used[x]));
        }
        __syncwarp();
      }
      if (vt == 0) {
        if (warp == 1) chunk_decay(load_decay(p, at, hv, lane), sy->G, lane);
        const float* src = p.coef + slot * 3 * kChunk;
        if (tid >= 64) sy->coef[tid - 64] = src[tid - 64];
      }
      // <dS, S>: 8 values at the same place of all four
      for (int e = tid; e < kTile * DK / 8; e += 256) {
        float f[2][8], g[2][8];
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          const int off = part * Sm::part + 16 * e;
          unpack8<BF16>(*reinterpret_cast<const uint4*>(stage + Sm::s + off), f[part]);
          unpack8<BF16>(*reinterpret_cast<const uint4*>(stage + Sm::d + off), g[part]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) dsum = fmaf(f[0][j] + f[1][j], g[0][j] + g[1][j], dsum);
      }
      run = __syncthreads_and(ok);  // all have read the stage
      if (!run) break;
      if (warp == 0 && tile + 2 < tiles) {
        ok = __all_sync(0xffffffffu, wait(sy->used[x], tile >> 1, TDC_DEVICE_EMPTY_TIMEOUT, tile));
        if (ok) {
          if (lane == 0) fetch(tile + 2);
          fetched = tile + 3;
        }
        __syncwarp();
      }
    }
    if (!run) break;
    const int end = tile - 1;
    ok = ok && wait(sy->used[end & 1], end >> 1, TDC_DEVICE_EMPTY_TIMEOUT, end);
    run = __syncthreads_and(ok);
    if (!run) break;
    tc_fence_after();
    // Row sums with q and k, and what the products with the states add.
    const float* coef = sy->coef;
    const float gam = coef[i], be = coef[2 * kChunk + i], wb = coef[kChunk + i] * be;
    {
      const float by = upper ? -gam : p.scale * gam;
      float own = 0.f, key = 0.f;
#pragma unroll
      for (int x = 0; x < DK / 64; ++x) {
        uint32_t r[32];
        float f[32];
        tmem_ld(lanes + kGradOX + kc0 + 32 * x, r);
        load_key_row<E, DK>(f, raw + Sm::qk, l, kc0 + 32 * x);
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          own = fmaf(f[j], __uint_as_float(r[j]), own);
          acc[32 * x + j] = fmaf(by, __uint_as_float(r[j]), acc[32 * x + j]);
        }
        tmem_ld(lanes + kGradUS + kc0 + 32 * x, r);
        if (!upper) load_key_row<E, DK>(f, raw + Sm::qk, 64 + l, kc0 + 32 * x);
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          key = fmaf(f[j], __uint_as_float(r[j]), key);
          acc2[32 * x + j] = fmaf(wb, __uint_as_float(r[j]), acc2[32 * x + j]);
        }
      }
      sy->sums[kSumState][hc][l] = own;
      sy->sums[kSumKey][hc][l] = key;
    }
    // Dt and N, and the sums of E.
    {
      uint32_t r[32], g[32];
      tmem_ld(lanes + kGradDM + 32 * hc, r);
      tmem_ld(lanes + kGradGram + 32 * hc, g);
      const Far Gi = sy->G[i];
      const float sign = upper ? -1.f : p.scale;
      const int low = upper ? i : i + 1;  // columns below this are kept
      float row = 0.f, cs[32];
#pragma unroll
      for (int y = 0; y < 32; ++y) {
        const int j = 32 * hc + y;
        const float bj = coef[2 * kChunk + j];
        const bool in = j < low;
        const float v = in ? sign * __expf(minus(Gi, sy->G[j])) * __uint_as_float(r[y]) : 0.f;
        const float t = in ? v * __uint_as_float(g[y]) : 0.f;
        if (j == i && !upper) sy->diag[i] = t;
        cs[y] = j < i ? t : 0.f;
        row = fmaf(bj, cs[y], row);
        r[y] = __float_as_uint(in ? bj * v : 0.f);
      }
      sy->sums[kSumE][hc][l] = row;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int m = 0; m < 4; ++m)
          split2(__uint_as_float(r[8 * c + 2 * m]), __uint_as_float(r[8 * c + 2 * m + 1]), hi[m], lo[m]);
        unsigned char* dst = raw + Sm::dn + (4 * hc + c) * 2048 + l * 16;
        *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(dst + Sm::dnpart) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      fence_proxy_async();
      // column sums over the warp's lanes: lane j ends with column j
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        const bool up = lane & d;
#pragma unroll
        for (int y = 0; y < d; ++y) {
          const float send = up ? cs[y] : cs[y + d], keep = up ? cs[y + d] : cs[y];
          cs[y] = keep + __shfl_xor_sync(0xffffffffu, send, d);
        }
      }
      sy->cols[wq][32 * hc + lane] = cs[0];
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) dsum += __shfl_xor_sync(0xffffffffu, dsum, d);
    if (lane == 0) sy->dot[warp] = dsum;
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
      tc_fence_after();
      if (elect_one()) {
        // [Dt; N] K, then [Dt_hi; Dt_lo]^T Q + [N_hi; N_lo]^T K in the place of U dS^T
        constexpr uint32_t khigh = block_desc_high(2048), rhigh = block_desc_high(kRowBlock);
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int z = 0; z < KP; ++z) {
            if (y + z > 1) continue;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              tc_mma_ss(tm + kGradK, block_desc(sb + Sm::dn + y * Sm::dnpart + ks * 4096, 2048), rhigh,
                        block_desc(sb + Sm::qk + z * Sm::qkpart + 1024 + ks * 2 * kRowBlock, kRowBlock),
                        khigh, mma_desc(DK, true, false), y + z + ks > 0);
          }
#pragma unroll
        for (int z = 0; z < KP; ++z)
#pragma unroll
          for (int rows = 0; rows < 2; ++rows)  // of Dt and Q, of N and K
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              tc_mma_ss(tm + kGradUS,
                        block_desc(sb + Sm::dn + rows * 1024 + ks * 2 * kRowBlock, kRowBlock), khigh,
                        block_desc(sb + Sm::qk + z * Sm::qkpart + rows * 1024 + ks * 2 * kRowBlock,
                                   kRowBlock),
                        khigh, mma_desc(DK, true, true), z + rows + ks > 0);
        tc_commit(smem_addr(&sy->done));
      }
      __syncwarp();
    } else if (warp == 4 || warp == 5) {  // dbeta and dg
      const int t = tid - 128;
      auto sum = [&](int which, int from) { return sy->sums[which][0][from] + sy->sums[which][1][from]; };
      const float ga = coef[t], w = coef[kChunk + t], bt = coef[2 * kChunk + t];
      const float key = sum(kSumKey, t) + sum(kSumKey, 64 + t);
      const float col = (sy->cols[0][t] + sy->cols[1][t]) + (sy->cols[2][t] + sy->cols[3][t]);
      if (t < at.rows) {
        const int64_t o = (at.b * p.T + at.t0 + t) * p.HV + hv;
        const float db = col + sy->diag[t] + w * key;
        if (p.beta_f32) static_cast<float*>(p.dbeta)[o] = db;
        else store_float<E>(p.dbeta, o, db);
      }
      sy->dg[0][t] = p.scale * ga * sum(kSumState, t) - ga * sum(kSumState, 64 + t);
      sy->dg[1][t] = bt * col - (sum(kSumE, t) + sum(kSumE, 64 + t)) + w * bt * key;
      asm volatile("bar.sync 1, 64;" ::: "memory");
      if (warp == 4) {
        float ds = 0.f;
#pragma unroll
        for (int x = 0; x < 8; ++x) ds += sy->dot[x];
        ds *= coef[kChunk - 1];
        // sums from the row to the end, and over the rows before it
        const float a0 = sy->dg[0][2 * lane], a1 = sy->dg[0][2 * lane + 1];
        const float f0 = sy->dg[1][2 * lane], f1 = sy->dg[1][2 * lane + 1];
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
      __syncwarp();
    }
    ok = wait(sy->done, gi, TDC_DEVICE_EMPTY_TIMEOUT, tile);
    tc_fence_after();
#pragma unroll
    for (int x = 0; x < DK / 64; ++x) {
      uint32_t r[32];
      tmem_ld(lanes + kGradK + kc0 + 32 * x, r);
#pragma unroll
      for (int j = 0; j < 32; ++j) acc[32 * x + j] += __uint_as_float(r[j]);
      tmem_ld(lanes + kGradUS + kc0 + 32 * x, r);
#pragma unroll
      for (int j = 0; j < 32; ++j) acc2[32 * x + j] += __uint_as_float(r[j]);
    }
    tc_fence_before();
    run = __syncthreads_and(ok);
  }
  if (run) {
    // dK's parts of lanes 0-63 go to its lanes, through the first stage.
    float* x = reinterpret_cast<float*>(raw + Sm::stages) + i * (DK + 4) + kc0;
    if (!upper) {
#pragma unroll
      for (int j = 0; j < DK / 2; j += 4)
        *reinterpret_cast<float4*>(x + j) = make_float4(acc2[j], acc2[j + 1], acc2[j + 2], acc2[j + 3]);
    }
    __syncthreads();
    if (upper) {
#pragma unroll
      for (int j = 0; j < DK / 2; j += 4) {
        const float4 v = *reinterpret_cast<const float4*>(x + j);
        acc[j] += acc2[j] + v.x;
        acc[j + 1] += acc2[j + 1] + v.y;
        acc[j + 2] += acc2[j + 2] + v.z;
        acc[j + 3] += acc2[j + 3] + v.w;
      }
    }
    if (i < at.rows) {
      uint16_t* dst = static_cast<uint16_t*>(upper ? p.dk : p.dq) +
                      ((at.b * p.T + at.t0 + i) * p.H + h) * DK + kc0;
#pragma unroll
      for (int j = 0; j < DK / 2; j += 8) *reinterpret_cast<uint4*>(dst + j) = pack8<E>(acc + j);
    }
  } else if (warp == 0) {
    // A wait gave up: copies and products on their way come to rest first.
    for (int f = tile; f < fetched; ++f)
      mbar_wait_bounded(smem_addr(&sy->full[f & 1]), uint32_t(f >> 1) & 1u, nullptr, false, p.timeout_ns);
    if (elect_one()) tc_commit(smem_addr(&sy->drain));
    __syncwarp();
    mbar_wait_bounded(smem_addr(&sy->drain), 0, nullptr, false, p.timeout_ns);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_free(tm, 512);
}

}  // namespace tdc
