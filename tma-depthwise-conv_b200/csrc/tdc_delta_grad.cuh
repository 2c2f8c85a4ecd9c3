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
// A block takes chunks and key heads in turn, the tiles of the next one on their
// way while one is finished.  Tokens are the rows of every product: lanes
// 0-63 of TMEM are the tokens of dO (and of what becomes dQ), lanes 64-127 those
// of dX (dK), so with M = 128
//   [dO; dX] S^T and [dO; dX] U^T      both halves at once,
//   [U_1; U_2] dS^T, [U_3; 0] dS^T     parts of U in the halves, added later,
//   [Q; K] K^T                         once a block,
//   [Dt; N] K                          into dQ and dK,
//   [Dt_1; Dt_2]^T Q + [N_1; N_2]^T K  into dK, again by parts: the halves are added, so
//                                      with [Dt_2; Dt_3] too the second part counts twice
//                                      and is kept halved.
// The walks left U, dX, dO, S and dS transposed, as [kTile channels][8 columns]
// blocks that serve as A with the tokens and as B with the keys along them.  The
// channels are the contraction and come in tiles of kTile by bulk copies, as many
// stages as fit.
//
// Warps 0-7 sum <dS, S> while a head's tiles pass and finish the head: a thread
// owns a lane of TMEM and half of the columns; row sums are its own, column sums
// go through shuffles.  It puts the products with the states back scaled, so that
// the last products add to them in place.  Warp 8 issues the products, warp 9 the
// copies (also the next chunk's), warp 10 brings the decays.
//
// 8192 tokens of 16 key and 32 value heads of 128 x 128 (bf16): 1.28 GB of workspace
// in 376 us, 3.4 TB/s.  While a head is finished only the copies go on, and only as far
// as the stages hold (3 tiles of 8): TMEM has no room for the sums of two heads, shared
// memory none for more stages.  At 2048 tokens DRAM runs at 36 % of its peak rate and the
// tensor pipe is active 29 % of the time.  With operands in two parts instead of three it took 265 us, and
// dg was off by 7e-6 instead of 6e-7.
#pragma once

#include "tdc_delta_walk.cuh"

namespace tdc {

template <class E, int DK>
struct GradSmem {
  static constexpr int KP = std::is_same_v<E, BF16> ? 1 : 2;
  // rows of Q, then of K: [parts][DK / 8][128][8]
  using Tile = GradTile<KP, DK>;
  static constexpr int qk = 0, qkpart = DK / 8 * kKeyBlock;
  // rows of Dt, then of N: [3 parts][8][128][8], half of the second part
  static constexpr int dn = qk + KP * qkpart, dnpart = kChunk / 8 * kKeyBlock;
  static constexpr int stages = dn + 3 * dnpart, stage = Tile::stage;
  static constexpr int kMaxBytes = 232448 - 7168;  // of a block, less GradSync
  static constexpr int count = (kMaxBytes - stages) / stage < 6 ? (kMaxBytes - stages) / stage : 6;
  static constexpr int sync = stages + count * stage;
  static_assert(count >= 2, "one stage is read while another is filled");
};
struct GradSync {
  uint64_t full[6], used[6];   // stages: copied; read by the products and the 8 warps
  uint64_t keys;               // Q and K are there
  uint64_t gates;              // G and coef are
  uint64_t ready;              // products over the channels done
  uint64_t gram;               // products of Q and K with K done
  uint64_t dn;                 // Dt and N are stored
  uint64_t done;               // products with them done
  uint64_t swap;               // dK's parts of lanes 0-63 stored
  uint64_t next;               // the head is finished
  uint64_t drain;
  uint32_t tmem;
  int abort;
  Far G[kChunk];
  float coef[3 * kChunk];      // gam, w, beta
  float sums[3][2][128];       // row sums by half of the columns: see kSum*
  float cols[4][kChunk];       // column sums of P D - M L below the diagonal, by 32 lanes
  float diag[kChunk];          // P D on it
  float dot[8];
};
static_assert(sizeof(GradSync) <= 7168, "see kMaxBytes");
enum { kSumState = 0, kSumKey = 1, kSumE = 2 };
// TMEM columns; D and M stand behind the products with S (DK columns).  The tensor core
// cuts a sum's low bits off at each product it adds, so U dS's small products have a sum
// of their own (dbeta of 256 value channels: 1.1e-6 -> 6.7e-7 of the norm); there is
// no room for the others'.
constexpr uint32_t kGradOX = 0, kGradUS = 192, kGradGram = 320, kGradUS2 = 384;

// What a block works on: a chunk that has rows, and a key head; every gridDim.x-th.
struct GradItem {
  int64_t chunk;
  int head;
  ChunkAt at;

  __device__ __forceinline__ explicit GradItem(const DeltaParams& p) : chunk(blockIdx.x), head(0) {
    settle(p);
  }
  __device__ __forceinline__ bool here(const DeltaParams& p) const { return head < p.H; }
  __device__ __forceinline__ void next(const DeltaParams& p) {
    chunk += gridDim.x;
    settle(p);
  }
  __device__ __forceinline__ void settle(const DeltaParams& p) {
    for (;; chunk += gridDim.x) {
      while (chunk >= p.max_chunks) chunk -= p.max_chunks, ++head;
      if (head >= p.H) return;
      at = chunk_at(p, chunk);
      if (at.rows > 0) return;
    }
  }
};

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
    const unsigned char* src = qk + (c0 / 8 + c) * kKeyBlock + l * 16;
    unpack8<BF16>(*reinterpret_cast<const uint4*>(src), f + 8 * c);
    if constexpr (Sm::KP == 2) {
      float lo[8];
      unpack8<BF16>(*reinterpret_cast<const uint4*>(src + Sm::qkpart), lo);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[8 * c + i] += lo[i];
    }
  }
}

// Warp 9, one thread: the tiles of all items in turn, and each item's Q and K once
// the item before is finished.
template <class E, int DK>
__device__ __forceinline__ void grad_fetch(const DeltaParams& p, unsigned char* raw, GradSync* sy,
                                           const Waiter& wait) {
  using Sm = GradSmem<E, DK>;
  constexpr int KP = Sm::KP, NS = Sm::count;
  const uint32_t sb = smem_addr(raw);
  const int per_head = p.V / kTile, tiles = p.group * per_head;
  int n = 0, done = 0, sent = 0;  // tiles, items, and those whose Q and K are on their way
  bool ok = true;
  for (GradItem item(p); item.here(p) && ok; item.next(p), ++done) {
    const int64_t chunk = item.chunk;
    const int h = item.head;
    const int64_t tile0 = (chunk * p.HV + h * p.group) * per_head;
    for (int t = 0; t <= tiles && ok; ++t) {
      if (t == min(NS, tiles)) {
        if (done > 0) ok = wait(sy->next, uint32_t(done * p.group - 1), TDC_DEVICE_EMPTY_TIMEOUT, n);
        if (!ok) break;
        constexpr int bytes = KP * Sm::qkpart;
        mbar_arrive_expect_tx(smem_addr(&sy->keys), bytes);
        ++sent;
        bulk_load(sb + Sm::qk, p.kq + (chunk * p.H + h) * bytes, bytes, smem_addr(&sy->keys));
      }
      if (t == tiles) break;
      const int x = n % NS;
      if (n >= NS) ok = wait(sy->used[x], uint32_t(n / NS - 1), TDC_DEVICE_EMPTY_TIMEOUT, n);
      if (!ok) break;
      constexpr int bytes = Sm::Tile::bytes;
      const uint32_t bar = smem_addr(&sy->full[x]);
      const uint32_t dst = sb + Sm::stages + x * Sm::stage;
      const unsigned char* src = p.tiles + (tile0 + t) * bytes;
      mbar_arrive_expect_tx(bar, bytes);
      bulk_load(dst + Sm::Tile::skip, src, Sm::Tile::front, bar);
      bulk_load(dst + Sm::Tile::xl, src + Sm::Tile::front, Sm::Tile::back, bar);
      ++n;
    }
  }
  if (!*wait.abort) return;
  // A wait gave up: what is on its way comes to rest before the block ends.
  for (int f = max(0, n - NS); f < n; ++f)
    mbar_wait_bounded(smem_addr(&sy->full[f % NS]), uint32_t(f / NS) & 1u, nullptr, false, p.timeout_ns);
  if (sent > 0)
    mbar_wait_bounded(smem_addr(&sy->keys), uint32_t(sent - 1) & 1u, nullptr, false, p.timeout_ns);
}

// Warp 8: the products.
template <class E, int DK>
__device__ __forceinline__ void grad_issue(const DeltaParams& p, uint32_t sb, GradSync* sy,
                                           const Waiter& wait, uint32_t tm) {
  using Sm = GradSmem<E, DK>;
  constexpr int KP = Sm::KP, NS = Sm::count;
  constexpr uint32_t kGradDM = kGradOX + DK;
  constexpr uint32_t khigh = block_desc_high(kKeyBlock), rhigh = block_desc_high(kRowBlock);
  const int per_head = p.V / kTile;
  int x = 0, phase = 0, heads = 0, done = 0;
  for (GradItem item(p); item.here(p); item.next(p), ++done) {
    for (int gi = 0; gi < p.group; ++gi, ++heads) {
      if (heads > 0 && !warp_wait(wait, sy->next, heads - 1)) return;
      for (int vt = 0; vt < per_head; ++vt) {
        if (!warp_wait(wait, sy->full[x], phase)) return;
        tc_fence_after();
        const uint32_t st = sb + Sm::stages + x * Sm::stage;
        if (elect_one()) {
          using T = typename Sm::Tile;
          const uint32_t a = st + T::oh, b = st + T::om, c = st + T::zero;  // [dO; dX] by parts
          const uint32_t u = st + T::u, s = st + T::s, d = st + T::d;
          // by S and U together, where their parts lie beside each other; without the
          // products of 2^-24 and below
          grad_product<DK + 64>(tm + kGradOX, c, s, vt > 0);
          grad_product<DK>(tm + kGradOX, b, s - T::part, true);
          grad_product<64>(tm + kGradDM, b, u + T::upart, true);
          grad_product<DK>(tm + kGradOX, a, s - 2 * T::part, true);
          grad_product<64>(tm + kGradDM, a, u + 2 * T::upart, true);
          grad_product<DK + 64>(tm + kGradOX, b, s, true);
          grad_product<DK>(tm + kGradOX, a, s - T::part, true);
          grad_product<64>(tm + kGradDM, a, u + T::upart, true);
          grad_product<DK + 64>(tm + kGradOX, a, s, true);
          // [U's last part; 0], then its first two
          grad_product<DK>(tm + kGradUS2, u + 2 * T::upart, d, vt > 0);
          grad_product<DK>(tm + kGradUS2, u, d + 2 * T::part, true);
          grad_product<DK>(tm + kGradUS2, u, d + T::part, true);
          grad_product<DK>(tm + kGradUS, u, d, vt > 0);
          tc_commit(smem_addr(&sy->used[x]));
        }
        __syncwarp();
        if (++x == NS) x = 0, ++phase;
      }
      if (elect_one()) tc_commit(smem_addr(&sy->ready));
      __syncwarp();
      if (gi == 0) {
        if (!warp_wait(wait, sy->keys, done)) return;
        tc_fence_after();
        if (elect_one()) {  // the rows of Q and K by those of K
          uint32_t q = sb + Sm::qk;
          asm volatile("" : "+r"(q));
          const uint32_t k = q + 1024;
#pragma unroll
          for (int y = KP - 1; y >= 0; --y)
#pragma unroll
            for (int z = KP - 1; z >= 0; --z)
#pragma unroll
              for (int ks = 0; ks < DK / 16; ++ks)
                tc_mma_ss(tm + kGradGram, block_desc(q + y * Sm::qkpart + ks * 2 * kKeyBlock, kKeyBlock),
                          rhigh, block_desc(k + z * Sm::qkpart + ks * 2 * kKeyBlock, kKeyBlock), rhigh,
                          mma_desc(64, false, false), y + z < 2 * KP - 2 || ks > 0);
          tc_commit(smem_addr(&sy->gram));
        }
        __syncwarp();
      }
      if (!warp_wait(wait, sy->dn, heads)) return;
      tc_fence_after();
      if (elect_one()) {
        // (descriptors from an address of this turn: those of all products, kept over the
        // turns, did not fit the warp's registers)
        uint32_t q = sb + Sm::qk;
        asm volatile("" : "+r"(q));
        const uint32_t k = q + 1024, dn = q + (Sm::dn - Sm::qk);
        // [Dt; N] K onto the first (half of the second part twice), then two parts at a
        // time, the last two and the first two, [Dt; Dt]^T Q + [N; N]^T K onto the last
#pragma unroll
        for (int sum = 2; sum >= 0; --sum)
#pragma unroll
          for (int z = 0; z < KP && z <= sum; ++z)
#pragma unroll
            for (int twice = 0; twice < (sum - z == 1 ? 2 : 1); ++twice)
#pragma unroll
              for (int ks = 0; ks < 4; ++ks)
                tc_mma_ss(tm + kGradOX,
                          block_desc(dn + (sum - z) * Sm::dnpart + ks * 2 * kKeyBlock, kKeyBlock), rhigh,
                          block_desc(k + z * Sm::qkpart + ks * 2 * kRowBlock, kRowBlock), khigh,
                          mma_desc(DK, true, false), true);
#pragma unroll
        for (int z = KP - 1; z >= 0; --z)
#pragma unroll
          for (int y = 1; y >= 0; --y)
#pragma unroll
            for (int rows = 0; rows < 2; ++rows)  // of Dt and Q, of N and K
#pragma unroll
              for (int ks = 0; ks < 4; ++ks)
                tc_mma_ss(tm + kGradUS,
                          block_desc(dn + y * Sm::dnpart + rows * 1024 + ks * 2 * kRowBlock, kRowBlock), khigh,
                          block_desc(q + z * Sm::qkpart + rows * 1024 + ks * 2 * kRowBlock, kRowBlock),
                          khigh, mma_desc(DK, true, true), true);
        tc_commit(smem_addr(&sy->done));
      }
      __syncwarp();
    }
  }
}

// 32 columns of a thread's lane, scaled, back to TMEM.
__device__ __forceinline__ void put_scaled(uint32_t at, const uint32_t (&r)[32], float by) {
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    uint32_t v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(by * __uint_as_float(r[16 * x + j]));
    tmem_st(at + 16 * x, v);
  }
}

template <class E, int DK>
__global__ void __launch_bounds__(kWalkThreads, 1) delta_grad_kernel(const DeltaParams p) {
  extern __shared__ __align__(1024) unsigned char raw[];
  using Sm = GradSmem<E, DK>;
  constexpr int KP = Sm::KP, NS = Sm::count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  GradSync* sy = reinterpret_cast<GradSync*>(raw + Sm::sync);
  if (tid == 0) {
    for (int x = 0; x < NS; ++x) {
      mbar_init(smem_addr(&sy->full[x]), 1);
      mbar_init(smem_addr(&sy->used[x]), 9);
    }
    for (uint64_t* one : {&sy->keys, &sy->gates, &sy->ready, &sy->gram, &sy->done, &sy->drain})
      mbar_init(smem_addr(one), 1);
    for (uint64_t* all : {&sy->dn, &sy->swap, &sy->next}) mbar_init(smem_addr(all), 8);
    sy->abort = 0;
    fence_mbar_init();
  }
  if (warp == 8) tmem_alloc(smem_addr(&sy->tmem), kTmemColumns);
  {  // the stages' places of zeros
    constexpr int upart = Sm::Tile::upart;
    for (int e = 16 * tid; e < NS * upart; e += 16 * kWalkThreads) {
      unsigned char* at = raw + Sm::stages + e / upart * Sm::stage + e % upart;
      *reinterpret_cast<uint4*>(at + Sm::Tile::zero) = make_uint4(0, 0, 0, 0);
      if (KP == 1) *reinterpret_cast<uint4*>(at + Sm::Tile::om) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = sy->tmem;
  const Waiter wait{&sy->abort, p.timeout_ns, p.status_words, p.status_host, int(blockIdx.x)};
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    if (warp == 8) {
      grad_issue<E, DK>(p, smem_addr(raw), sy, wait, tm);
      if (elect_one()) tc_commit(smem_addr(&sy->drain));
      __syncwarp();
      mbar_wait_bounded(smem_addr(&sy->drain), 0, wait.abort, false, wait.timeout_ns);
    } else if (warp == 9) {
      if (lane == 0) grad_fetch<E, DK>(p, raw, sy, wait);
    } else if (warp == 10) {
      int heads = 0;
      bool ok = true;
      for (GradItem item(p); item.here(p) && ok; item.next(p)) {
        for (int gi = 0; gi < p.group && ok; ++gi, ++heads) {
          const int hv = item.head * p.group + gi;
          const float2 g = load_decay(p, item.at, hv, lane);
          const float2* src =
              reinterpret_cast<const float2*>(p.coef + (item.chunk * p.HV + hv) * kCoef);
          const float2 c[3] = {src[lane], src[32 + lane], src[64 + lane]};
          if (heads > 0) ok = warp_wait(wait, sy->next, heads - 1);
          chunk_decay(g, sy->G, lane);
#pragma unroll
          for (int x = 0; x < 3; ++x) reinterpret_cast<float2*>(sy->coef)[32 * x + lane] = c[x];
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_addr(&sy->gates));
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWalkRegs));
    const uint32_t lanes = tm + (uint32_t(warp & 3) << 21);
    const int wq = warp & 3, hc = warp >> 2;  // its lanes and its half of the columns
    const int l = 32 * wq + lane, i = l & 63;
    const bool upper = l >= 64;
    const int kc0 = hc * (DK / 2), per_head = p.V / kTile;
    const float* coef = sy->coef;
    auto all_wait = [&](uint64_t& bar, int phase) { return warp_wait(wait, bar, phase); };
    auto arrive = [&](uint64_t& bar) {
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&bar));
    };
    bool ok = true;
    int x = 0, phase = 0, heads = 0, done = 0;
    for (GradItem item(p); item.here(p) && ok; item.next(p), ++done) {
      const ChunkAt& at = item.at;
      const int h = item.head;
      float acc[DK / 2] = {};  // dQ (lanes 0-63) or dK of the lane's token
      for (int gi = 0; gi < p.group; ++gi, ++heads) {
        const int hv = h * p.group + gi;
        float dsum = 0.f;  // <dS, S>
        for (int vt = 0; vt < per_head; ++vt) {
          ok = all_wait(sy->full[x], phase);
          if (!ok) break;
          const unsigned char* stage = raw + Sm::stages + x * Sm::stage;
          for (int e = tid; e < kTile * DK / 8; e += 256) {  // 8 values at the same place of all six
            float f[8] = {}, g[8] = {};
#pragma unroll
            for (int part = 2; part >= 0; --part) {
              float a[8], b[8];
              unpack8<BF16>(*reinterpret_cast<const uint4*>(stage + Sm::Tile::s - part * Sm::Tile::part + 16 * e), a);
              unpack8<BF16>(*reinterpret_cast<const uint4*>(stage + Sm::Tile::d + part * Sm::Tile::part + 16 * e), b);
#pragma unroll
              for (int j = 0; j < 8; ++j) f[j] += a[j], g[j] += b[j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) dsum = fmaf(f[j], g[j], dsum);
          }
          arrive(sy->used[x]);
          if (++x == NS) x = 0, ++phase;
        }
        ok = ok && all_wait(sy->gates, heads) && all_wait(sy->keys, done) && all_wait(sy->ready, heads);
        if (!ok) break;
        tc_fence_after();
        // Row sums with q and k; the products with the states are scaled in place.
        const float gam = coef[i], be = coef[2 * kChunk + i], wb = coef[kChunk + i] * be;
        {
          const float by = upper ? -gam : p.scale * gam;
          float own = 0.f, key = 0.f;
#pragma unroll
          for (int y = 0; y < DK / 64; ++y) {
            uint32_t r[32];
            float f[32];
            tmem_ld(lanes + kGradOX + kc0 + 32 * y, r);
            load_key_row<E, DK>(f, raw + Sm::qk, l, kc0 + 32 * y);
#pragma unroll
            for (int j = 0; j < 32; ++j) own = fmaf(f[j], __uint_as_float(r[j]), own);
            put_scaled(lanes + kGradOX + kc0 + 32 * y, r, by);
            tmem_ld(lanes + kGradUS + kc0 + 32 * y, r);
#pragma unroll
            for (int x = 0; x < 2; ++x) {  // and the small products' sum
              uint32_t r2[16];
              tmem_ld(lanes + kGradUS2 + kc0 + 32 * y + 16 * x, r2);
#pragma unroll
              for (int j = 0; j < 16; ++j)
                r[16 * x + j] = __float_as_uint(__uint_as_float(r[16 * x + j]) + __uint_as_float(r2[j]));
            }
            load_key_row<E, DK>(f, raw + Sm::qk, 64 + i, kc0 + 32 * y);
#pragma unroll
            for (int j = 0; j < 32; ++j) key = fmaf(f[j], __uint_as_float(r[j]), key);
            put_scaled(lanes + kGradUS + kc0 + 32 * y, r, wb);
          }
          sy->sums[kSumState][hc][l] = own;
          sy->sums[kSumKey][hc][l] = key;
        }
        if (gi == 0) {
          ok = all_wait(sy->gram, done);
          if (!ok) break;
          tc_fence_after();
        }
        // Dt and N, and the sums of E.
        {
          uint32_t r[32], g[32];
          tmem_ld(lanes + kGradOX + DK + 32 * hc, r);
          tmem_ld(lanes + kGradGram + 32 * hc, g);
          const Far Gi = sy->G[i];
          const float sign = upper ? -1.f : p.scale;
          const int low = upper ? i : i + 1;  // columns below this are kept
          float row = 0.f, own = 0.f, cs[32];
#pragma unroll
          for (int y = 0; y < 32; y += 2) {
            const float4 far2 = *reinterpret_cast<const float4*>(sy->G + 32 * hc + y);
            const float2 be2 = *reinterpret_cast<const float2*>(coef + 2 * kChunk + 32 * hc + y);
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const int j = 32 * hc + y + z;
              const float bj = z ? be2.y : be2.x;
              const Far Gj = z ? Far{far2.z, far2.w} : Far{far2.x, far2.y};
              // (what is masked is replaced before it is used: no branches)
              const bool in = j < low;
              const float v =
                  sign * __expf(in ? minus(Gi, Gj) : 0.f) * __uint_as_float(in ? r[y + z] : 0u);
              const float t = v * __uint_as_float(in ? g[y + z] : 0u);
              own = j == i ? t : own;
              cs[y + z] = j < i ? t : 0.f;
              row = fmaf(bj, cs[y + z], row);
              r[y + z] = in ? __float_as_uint(bj * v) : 0u;
            }
          }
          sy->sums[kSumE][hc][l] = row;
          if (!upper && (i >> 5) == hc) sy->diag[i] = own;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t w[3][4];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              float v0 = __uint_as_float(r[8 * c + 2 * m]), v1 = __uint_as_float(r[8 * c + 2 * m + 1]);
              w[0][m] = pack2_rn<BF16>(v0, v1);
              fma2<BF16>(w[0][m], 0xBF80BF80u, v0, v1);  // less the part
              w[1][m] = pack2_rn<BF16>(0.5f * v0, 0.5f * v1);
              fma2<BF16>(w[1][m], 0xC000C000u, v0, v1);  // less twice its half
              w[2][m] = pack2_rn<BF16>(v0, v1);
            }
            unsigned char* dst = raw + Sm::dn + (4 * hc + c) * kKeyBlock + l * 16;
#pragma unroll
            for (int m = 0; m < 3; ++m)
              *reinterpret_cast<uint4*>(dst + m * Sm::dnpart) = make_uint4(w[m][0], w[m][1], w[m][2], w[m][3]);
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
        operand_ready(sy->dn, lane);
        if (warp == 4) {  // dbeta and dg of two tokens a lane
          ok = all_wait(sy->dn, heads);
          if (!ok) break;
          float a[2], f[2];  // of dg: for this token and those before it; for those behind it
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const int t = 2 * lane + z;
            auto sum = [&](int which, int from) {
              return sy->sums[which][0][from] + sy->sums[which][1][from];
            };
            const float ga = coef[t], w = coef[kChunk + t], bt = coef[2 * kChunk + t];
            const float key = sum(kSumKey, t) + sum(kSumKey, 64 + t);
            const float col = (sy->cols[0][t] + sy->cols[1][t]) + (sy->cols[2][t] + sy->cols[3][t]);
            if (t < at.rows) {
              const int64_t o = (at.b * p.T + at.t0 + t) * p.HV + hv;
              const float db = col + sy->diag[t] + w * key;
              if (p.beta_f32) static_cast<float*>(p.dbeta)[o] = db;
              else store_float<E>(p.dbeta, o, db);
            }
            a[z] = p.scale * ga * sum(kSumState, t) - ga * sum(kSumState, 64 + t);
            f[z] = bt * col - (sum(kSumE, t) + sum(kSumE, 64 + t)) + w * bt * key;
          }
          float ds = 0.f;
#pragma unroll
          for (int y = 0; y < 8; ++y) ds += sy->dot[y];
          ds *= coef[kChunk - 1];
          // sums from the row to the end, and over the rows before it
          float up = a[0] + a[1], down = f[0] + f[1];
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const float y = __shfl_down_sync(0xffffffffu, up, d);
            const float z = __shfl_up_sync(0xffffffffu, down, d);
            if (lane + d < 32) up += y;
            if (lane >= d) down += z;
          }
          const float above = __shfl_down_sync(0xffffffffu, up, 1);
          float before = __shfl_up_sync(0xffffffffu, down, 1);
          if (lane == 0) before = 0.f;
          const int64_t o = (at.b * p.T + at.t0 + 2 * lane) * p.HV + hv;
          if (2 * lane < at.rows) p.dg[o] = up + before + ds;
          if (2 * lane + 1 < at.rows)
            p.dg[o + p.HV] = a[1] + (lane < 31 ? above : 0.f) + before + f[0] + ds;
        }
        ok = all_wait(sy->done, heads);
        if (!ok) break;
        tc_fence_after();
        // dK's parts of lanes 0-63 go to its lanes, in the place of Dt and N (16 bytes
        // a place, spread over the banks).
        float4* parts = reinterpret_cast<float4*>(raw + Sm::dn) + i * (DK / 4);
#pragma unroll
        for (int y = 0; y < DK / 64; ++y) {
          uint32_t r[32];
          tmem_ld(lanes + kGradOX + kc0 + 32 * y, r);
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[32 * y + j] += __uint_as_float(r[j]);
          tmem_ld(lanes + kGradUS + kc0 + 32 * y, r);
          if (upper) {
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[32 * y + j] += __uint_as_float(r[j]);
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              parts[((kc0 + 32 * y + j) / 4) ^ (i & 7)] =
                  make_float4(__uint_as_float(r[j]), __uint_as_float(r[j + 1]), __uint_as_float(r[j + 2]),
                              __uint_as_float(r[j + 3]));
          }
        }
        tc_fence_before();
        arrive(sy->swap);
        if (upper) {
          ok = all_wait(sy->swap, heads);
          if (!ok) break;
#pragma unroll
          for (int j = 0; j < DK / 2; j += 4) {
            const float4 v = parts[((kc0 + j) / 4) ^ (i & 7)];
            acc[j] += v.x, acc[j + 1] += v.y, acc[j + 2] += v.z, acc[j + 3] += v.w;
          }
        }
        arrive(sy->next);
      }
      if (ok && i < at.rows) {
        uint16_t* dst = static_cast<uint16_t*>(upper ? p.dk : p.dq) +
                        ((at.b * p.T + at.t0 + i) * p.H + h) * DK + kc0;
#pragma unroll
        for (int j = 0; j < DK / 2; j += 8) *reinterpret_cast<uint4*>(dst + j) = pack8<E>(acc + j);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 8) tmem_free(tm, kTmemColumns);
}

}  // namespace tdc
