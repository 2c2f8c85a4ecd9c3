// tdc_delta_walk.cuh — the walk over a sequence's chunks, forward and back, on
// the 5th-generation tensor cores.
//
// The columns of S (the value channels) do not mix, so one block takes 128
// value channels of one head of one sequence and keeps S^T: one lane of TMEM
// a channel.  Every product of a chunk then has the state's side as its A
// operand (M = 128 channels, in TMEM) and a tile that all channels share as B
// (K, Q, T, P, in shared memory):
//   Y^T = S^T K^T                  X^T = V^T - gam Y^T
//   U^T = X^T T^T                  V'^T = beta U^T
//   O^T = scale gam (S^T Q^T) + V'^T P^T
//   S^T <- gam_63 S^T + (w V'^T) K
// A thread owns one channel and half of the columns, so scaling, splitting and
// the running state are thread-local; what a chunk costs is the chain of three
// dependent products (the walk is bound by its latency, with few sequences and
// heads, and by nothing else before the number of blocks passes the SMs).  Q's and
// P's products and the output run beside the chain.  8192 tokens of 32 heads of
// 128 x 128, as 4 sequences (128 blocks, 32 chunks each): 168 us forward, 168 when
// it stores U and S instead of making the output, 211 back, that is 5.2, 5.2 and 6.6 us
// a chunk (32 blocks alone: 4.0 forward).  With operands in two parts instead of
// three it took 109, 137 and 154, and was off by 4e-6 (see "Precision" in
// tdc_delta.cuh).  Two threads a channel measured best: with four (768 threads) one
// sequence of 8192 tokens took a fifth longer, since every exchange then waits for
// more warps.
//
// Warps 0-7 compute (warp % 4 picks the lanes, warp / 4 the half of the
// columns), warp 8 issues the products, warp 9 the bulk copies of the next
// chunk's tiles (two stages; delta_prepare has laid them out as the tensor
// cores read them, rows behind the sequence's end zeroed).  Every wait is
// bounded; a wait that gives up records the failure and ends the block.
#pragma once

#include "tdc_delta.cuh"
#include "tdc_tc.cuh"

namespace tdc {

// Tiles of a chunk in the workspace and in shared memory, in order.  KP: parts
// of an exact element (1 bf16, 2 fp16).
template <class E, int DK>
struct WalkTiles {
  static constexpr int KP = std::is_same_v<E, BF16> ? 1 : 2;
  static constexpr int keys = DK / 8 * kKeyBlock;     // one part of Q and K
  static constexpr int q = 0;
  static constexpr int k = kChunk * 16;
  static constexpr int t = KP * keys;
  static constexpr int p = t + 3 * kSq * 2;
  static constexpr int coef = p + 3 * kSq * 2;
  static constexpr int stage = coef + kCoef * 4;
};

// Shared memory behind the two stages.
struct WalkSync {
  uint64_t full[2], free[2];
  uint64_t y, u, q, s, o;                 // products done
  uint64_t sr, xr, vr, qr, gr;            // operands ready (or results read)
  uint64_t drain;
  uint32_t tmem;
  int abort;
  int bad[128];  // last chunk in which a channel's first 32 tokens spoil those behind
  int odd;       // whether anything so far was not finite (set before a chunk's sr)
};
static_assert(2 * WalkTiles<F16, 128>::stage + sizeof(WalkSync) <= 232448, "a block's shared memory");

// Three warpgroups; the third (products, copies) hands registers to the two that
// compute: 2 x 128 x 216 + 128 x 72 = 384 x 168, what the block starts with.
constexpr int kWalkThreads = 384, kWalkRegs = 216, kIssueRegs = 72;
constexpr uint32_t kTmemColumns = 512;

struct Waiter {
  volatile int* abort;
  uint64_t timeout_ns;
  int* words;
  int* host;
  int block;

  // False once the block has to end.
  __device__ __forceinline__ bool operator()(uint64_t& bar, uint32_t parity, int code, int64_t at) const {
    if (mbar_wait_bounded(smem_addr(&bar), parity & 1u, abort, true, timeout_ns)) return true;
    if (!*abort) {
      record_wait_failure(words, host, code, block, int(parity & 1u), at);
      *abort = 1;
    }
    return false;
  }
};

// v as three bf16 parts, 16 packed columns each: keep(part, columns) gets them one after
// another.  v is used up.  A part is the upper half of a value, cut and not rounded: 3 x 8
// bits hold it exactly all the same, and it takes one instruction instead of two slots.
template <class Keep>
__device__ __forceinline__ void split_parts(float (&v)[32], Keep keep) {
#pragma unroll
  for (int part = 0; part < 3; ++part) {
    uint32_t r[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      r[i] = __byte_perm(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]), 0x7632);
      if (part < 2) fma2<BF16>(r[i], 0xBF80BF80u, v[2 * i], v[2 * i + 1]);
    }
    keep(part, r);
  }
}
// The parts to TMEM columns at, at + step, at + 2 step.
__device__ __forceinline__ void split_to_tmem(float (&v)[32], uint32_t at, uint32_t step) {
  split_parts(v, [&](int part, const uint32_t (&r)[16]) { tmem_st(at + part * step, r); });
}

// For whole warps: all lanes go on, or none does.
__device__ __forceinline__ bool warp_wait(const Waiter& wait, uint64_t& bar, int phase) {
  const bool ok = wait(bar, uint32_t(phase), TDC_DEVICE_FULL_TIMEOUT, phase);
  return __all_sync(0xffffffffu, ok);
}

// Operands are stored: make them visible to the tensor core and tell warp 8.
__device__ __forceinline__ void operand_ready(uint64_t& bar, int lane) {
  tmem_wait_st();
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(smem_addr(&bar));
}

// Where the three parts of an A operand lie in TMEM, 8 columns a step of 16 of the
// contraction.  Of tokens: 32 columns a part.  The state's, in halves by the threads that
// own them: the first two parts of each in the columns of the update that the same
// threads read before, the third behind all of them.  Of tokens in halves: 48 columns a
// half.
struct TokenParts {
  static __device__ __forceinline__ constexpr uint32_t at(int part, int ks) { return 32 * part + 8 * ks; }
};
template <int DK>
struct StateParts {
  static __device__ __forceinline__ constexpr uint32_t at(int part, int ks) {
    constexpr int half = DK / 32;  // steps
    return part == 2 ? DK + 8 * ks : ks / half * (DK / 2) + part * (DK / 4) + ks % half * 8;
  }
};
struct HalfParts {
  static __device__ __forceinline__ constexpr uint32_t at(int part, int ks) {
    return ks / 2 * 48 + part * 16 + ks % 2 * 8;
  }
};

// d[128 x N] (+)= A B; A in three parts at a (Parts), B the rows of Q or K at b in BP
// parts bstep bytes apart, their tokens (n_major false) or their columns as N, DEPTH
// elements of the contraction.  Products of 2^-24 and below are left out, and the
// small ones come first: a sum that is still small rounds off less.
template <class Parts, int DEPTH, int N, bool N_MAJOR, int BP>
__device__ __forceinline__ void issue_product(uint32_t d, uint32_t a, uint32_t b, uint32_t bstep,
                                              bool accumulate) {
  const uint32_t low = block_desc(b, N_MAJOR ? kRowBlock : kKeyBlock);
  constexpr uint32_t high = block_desc_high(N_MAJOR ? kKeyBlock : kRowBlock);
  constexpr uint32_t kstep = (N_MAJOR ? 2 * kRowBlock : 2 * kKeyBlock) / 16;
#pragma unroll
  for (int sum = 2; sum >= 0; --sum)
#pragma unroll
    for (int j = 0; j < BP && j <= sum; ++j)
#pragma unroll
      for (int ks = 0; ks < DEPTH / 16; ++ks)
        tc_mma(d, a + Parts::at(sum - j, ks), low + j * (bstep / 16) + ks * kstep, high,
               mma_desc(N, N_MAJOR), accumulate || sum < 2 || j + ks > 0);
}

// d = A M^T (back: A M) for a lower triangular [64][64] tile M in three parts: only the
// blocks on and below the diagonal are read.  AP: parts of A, 32 columns each.
template <bool BACK, int AP>
__device__ __forceinline__ void issue_lower(uint32_t d, uint32_t a, uint32_t m) {
  const uint32_t low = tile_desc(m, BACK);
#pragma unroll
  for (int sum = 2; sum >= 0; --sum)
#pragma unroll
    for (int i = 0; i < AP && i <= sum; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int ks = BACK ? 3 - x : x;  // the step that fills all columns first
        const uint32_t n = BACK ? 16 * (ks + 1) : 64 - 16 * ks;
        const uint32_t from = BACK ? ks * 2 * kRowBlock : ks * (2 * kRowBlock + 2 * kColBlock);
        tc_mma(BACK ? d : d + 16 * ks, a + TokenParts::at(i, ks),
               low + (from + (sum - i) * kSq * 2) / 16, tile_desc_high(BACK), mma_desc(n, BACK),
               sum < 2 || i + x > 0);
      }
}

__device__ __forceinline__ void walk_setup(WalkSync* sy, int tid, int warp) {
  if (warp == 8) tmem_alloc(smem_addr(&sy->tmem), kTmemColumns);
  if (tid == 0) {
    for (uint64_t* b : {&sy->full[0], &sy->full[1], &sy->free[0], &sy->free[1], &sy->y, &sy->u,
                        &sy->q, &sy->s, &sy->o, &sy->drain})
      mbar_init(smem_addr(b), 1);
    for (uint64_t* b : {&sy->sr, &sy->xr, &sy->vr, &sy->qr, &sy->gr}) mbar_init(smem_addr(b), 8);
    sy->abort = 0;
    fence_mbar_init();
  }
  if (tid < 128) sy->bad[tid] = -1;
  if (tid == 0) sy->odd = 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
}

// Warp 9, one thread: the tiles of each chunk in turn.
template <class E, int DK, bool T_ONLY>
__device__ __forceinline__ void walk_fetch(const DeltaParams& p, unsigned char* raw, WalkSync* sy,
                                           const Waiter& wait, const SeqAt& s, int chunks, int h,
                                           int hv, bool back) {
  using W = WalkTiles<E, DK>;
  int issued = 0;
  for (int c = 0; c < chunks && c != p.withhold; ++c) {
    const int st = c & 1;
    if (c >= 2 && !wait(sy->free[st], uint32_t((c >> 1) - 1), TDC_DEVICE_EMPTY_TIMEOUT, c)) break;
    const int64_t chunk = s.chunk0 + (back ? chunks - 1 - c : c), slot = chunk * p.HV + hv;
    const uint32_t dst = smem_addr(raw) + st * W::stage, bar = smem_addr(&sy->full[st]);
    const unsigned char* keys = p.kq + (chunk * p.H + h) * (W::KP * W::keys);
    constexpr uint32_t kbytes = W::KP * W::keys;
    constexpr uint32_t tbytes = T_ONLY ? 3 * kSq * 2 : 6 * kSq * 2;
    mbar_arrive_expect_tx(bar, kbytes + tbytes + kCoef * 4);
    bulk_load(dst + W::q, keys, kbytes, bar);
    bulk_load(dst + W::t, p.tp + slot * (6 * kSq), tbytes, bar);
    bulk_load(dst + W::coef, p.coef + slot * kCoef, kCoef * 4, bar);
    issued = c + 1;
  }
  // No copy is in flight when the block ends.
  for (int c = issued > 2 ? issued - 2 : 0; c < issued; ++c)
    mbar_wait_bounded(smem_addr(&sy->full[c & 1]), uint32_t(c >> 1) & 1u, wait.abort, false,
                      wait.timeout_ns);
}

// S^T of this thread: its channel, DK / 2 keys from k0.
template <int DK>
__device__ __forceinline__ void walk_load(float (&S)[DK / 2], const float* src, int V, bool live) {
#pragma unroll
  for (int i = 0; i < DK / 2; ++i) S[i] = src != nullptr && live ? src[int64_t(i) * V] : 0.f;
}
template <int DK>
__device__ __forceinline__ void walk_store(float* dst, const float (&S)[DK / 2], int V, bool live) {
  if (!live) return;
#pragma unroll
  for (int i = 0; i < DK / 2; ++i) dst[int64_t(i) * V] = S[i];
}

// 32 tokens of this thread's channel, raw 16-bit, zeros behind `rows` (of the
// 32); stride in bytes.
__device__ __forceinline__ void walk_column(uint32_t (&v)[32], const void* src, uint32_t stride,
                                            int rows, bool live) {
  const char* at = static_cast<const char*>(src);
  if (live && rows >= 32) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      v[i] = *reinterpret_cast<const uint16_t*>(at + uint64_t(uint32_t(i)) * stride);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      v[i] = live && i < rows
                 ? *reinterpret_cast<const uint16_t*>(at + uint64_t(uint32_t(i)) * stride)
                 : 0u;
  }
}
// Tokens' results, rounded to the element type.
template <class E, int N>
__device__ __forceinline__ void walk_put(void* dst, uint32_t stride, const float (&x)[N], int rows,
                                         bool live) {
  char* at = static_cast<char*>(dst);
  if (live && rows >= N) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint32_t two = pack2_rn<E>(x[i], x[i + 1]);
      *reinterpret_cast<uint16_t*>(at + uint64_t(uint32_t(i)) * stride) = uint16_t(two);
      *reinterpret_cast<uint16_t*>(at + uint64_t(uint32_t(i + 1)) * stride) = uint16_t(two >> 16);
    }
  } else if (live) {
#pragma unroll 1
    for (int i = 0; i < rows; ++i) {
      float v = 0.f;
#pragma unroll
      for (int j = 0; j < N; ++j) v = j == i ? x[j] : v;
      *reinterpret_cast<uint16_t*>(at + uint64_t(uint32_t(i)) * stride) = uint16_t(pack2_rn<E>(v, 0.f));
    }
  }
}

// T's and P's rows multiply with the zeros behind their diagonals, so a NaN or an infinity
// in a row of X or V' would reach the tokens before its own.  It becomes 0 as an operand,
// and the results from its token on become NaN, as they are in the recurrence.  It comes
// from a value, from the chunk's keys and gates (delta_prepare looks at them) or from a
// state, so X and V' are looked at only from a block's first chunk with one of these on;
// values are while a thread waits for the state.
template <int N, class At>
__device__ __forceinline__ bool all_finite(At at) {
  float s[4] = {};
#pragma unroll
  for (int i = 0; i < N; ++i) s[i & 3] = fmaf(at(i), 0.f, s[i & 3]);  // 0 or NaN
  return (s[0] + s[1]) + (s[2] + s[3]) == 0.f;
}
// The first place of a thread's 32 that is not finite, 32 if none is; zeros in such places.
__device__ __forceinline__ int first_bad(float (&x)[32]) {
  int first = 32;
#pragma unroll
  for (int i = 31; i >= 0; --i) {
    if (fabsf(x[i]) <= FLT_MAX) continue;
    first = i;
    x[i] = 0.f;
  }
  return first;
}
// NaN from place `first` on.
template <class T>
__device__ __forceinline__ void spoil(T (&r)[32], int first) {
  if (__all_sync(0xffffffffu, first >= 32)) return;
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (i >= first) {
      if constexpr (std::is_same_v<T, float>) r[i] = __int_as_float(0x7fc00000);
      else r[i] = 0x7fc00000u;
    }
}

template <class E>
__device__ __forceinline__ float widen(uint32_t raw) {
  if constexpr (std::is_same_v<E, BF16>) return __uint_as_float(raw << 16);
  else return __half2float(__ushort_as_half(static_cast<unsigned short>(raw)));
}

// Where column `col` (a multiple of 8) of a channel (of all slots') lies in the
// gradients' workspace, in the part at `off` of its tile.
template <int KP, int DK>
__device__ __forceinline__ unsigned char* channel_at(unsigned char* base, int64_t channel, int off, int col) {
  using G = GradTile<KP, DK>;
  return base + channel / kTile * G::bytes + G::at(off) + int(channel % kTile) * 16 + col * (2 * kTile);
}
// 16 packed pairs (32 tokens or keys) of a channel there: a warp's stores are
// whole lines.
__device__ __forceinline__ void store_pairs(unsigned char* dst, const uint32_t (&r)[16], bool live) {
  if (!live) return;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *reinterpret_cast<uint4*>(dst + i * kTile * 16) =
        make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
}

// What a block of the forward walks.
struct Segment {
  enum { kWhole, kFromZero, kMap };  // as it is, from a state of 0, the identity with V = 0
  int64_t n;
  int index, role, v0, channels;
};
__device__ __forceinline__ Segment segment_of(const DeltaParams& p, int tiles, int DK) {
  Segment r{int64_t(blockIdx.x) / tiles, 0, Segment::kWhole, int(blockIdx.x % tiles) * 128, p.V};
  if (p.segments <= 1) return r;
  // pass 1: tiles of the first segment, of the inner ones, the inner ones' maps;
  // pass 2: tiles of all but the first
  const int inner = p.segments - 2;
  const int per = p.pass == 1 ? tiles * (1 + inner) + inner : tiles * (p.segments - 1);
  int j = int(blockIdx.x % per);
  r.n = blockIdx.x / per;
  if (p.pass == 1 && j >= tiles * (1 + inner)) {
    r.index = 1 + j - tiles * (1 + inner);
    r.role = Segment::kMap;
    r.v0 = 0;
    r.channels = DK;
    return r;
  }
  r.index = j / tiles + (p.pass == 1 ? 0 : 1);
  r.v0 = j % tiles * 128;
  if (p.pass == 1 && r.index > 0) r.role = Segment::kFromZero;
  return r;
}
__device__ __forceinline__ float* segment_state(const DeltaParams& p, float* base, int64_t n, int hv,
                                                int index, int K, int columns) {
  return base + ((n * p.HV + hv) * p.segments + index) * int64_t(K) * columns;
}

// The states between the segments, S_(i+1) = M_i S_i + N_i (N_i is in S_(i+1)'s
// place), in fp32: a block has 32 columns of a head's state, one a lane, a warp
// DK / 8 of its rows.  M comes through shared memory, in whole lines.  Bound by
// the latency of the segments one after another: 11 us for 3 segments of 32 heads
// (12 without the next one's M on its way).
template <int DK>
__global__ void __launch_bounds__(256) delta_join_kernel(const DeltaParams p) {
  constexpr int R = DK / 8;
  extern __shared__ __align__(16) float sh[];  // M [2][DK][DK], S [DK][32]
  float* S = sh + 2 * DK * DK;
  const int tid = threadIdx.x, lane = tid & 31, k0 = (tid >> 5) * R, v0 = blockIdx.y * 32;
  const int64_t n = blockIdx.x / p.HV;
  const int hv = int(blockIdx.x % p.HV);
  auto state = [&](int i) {
    return segment_state(p, p.seg_s, n, hv, i, DK, p.V) + int64_t(k0) * p.V + v0 + lane;
  };
  auto fetch = [&](int i) {  // M of inner segment i, one ahead
    const float* m = segment_state(p, p.seg_m, n, hv, i, DK, DK);
    const uint32_t dst = smem_addr(sh + (i & 1) * DK * DK);
    for (int e = 4 * tid; e < DK * DK; e += 4 * 256) cp_async16(dst + 4 * e, m + e, true);
    cp_async_commit();
  };
  float acc[R], next[R];
#pragma unroll
  for (int r = 0; r < R; ++r) next[r] = state(1)[int64_t(r) * p.V];
  for (int i = 1; i < p.segments; ++i) {
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = next[r];
    const bool more = i + 1 < p.segments;
    if (more) {
      fetch(i);
#pragma unroll
      for (int r = 0; r < R; ++r) next[r] = state(i + 1)[int64_t(r) * p.V];
    }
    if (i > 1) {
      if (more) cp_async_wait<1>(); else cp_async_wait<0>();
      __syncthreads();
      const float* m = sh + ((i - 1) & 1) * DK * DK;
      for (int x = 0; x < DK; x += 4) {
        float s[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) s[u] = S[(x + u) * 32 + lane];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float4 w = *reinterpret_cast<const float4*>(m + (k0 + r) * DK + x);
          acc[r] = fmaf(w.x, s[0], acc[r]);
          acc[r] = fmaf(w.y, s[1], acc[r]);
          acc[r] = fmaf(w.z, s[2], acc[r]);
          acc[r] = fmaf(w.w, s[3], acc[r]);
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) state(i)[int64_t(r) * p.V] = acc[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) S[(k0 + r) * 32 + lane] = acc[r];
    __syncthreads();
  }
}

// MODE 0: the forward (o and the final state).  MODE 1: the forward once more
// for the gradients: U of each chunk and the state before it.
//
// A long sequence with few heads leaves most SMs idle, so MODE 0 can walk its
// segments side by side.  A segment maps the state before it to M S + N: pass 1
// walks the first segment as it is and each inner one twice, from a state of 0
// (its end is N) and with V = 0 from the identity (its end is M, whose K columns
// stand in the channels' place); delta_join_kernel makes the states between the
// segments; pass 2 walks all but the first from them.  Two passes of a
// segment's length replace one of the whole: a call for one sequence of 8192 tokens with
// 32 heads takes 438 us (194 + 11 + 199 in these three launches) instead of 590.
template <class E, int DK, int MODE>
__global__ void __launch_bounds__(kWalkThreads, 1) delta_walk_kernel(const DeltaParams p) {
  extern __shared__ __align__(1024) unsigned char raw[];
  using W = WalkTiles<E, DK>;
  constexpr int KP = W::KP;
  using GT = GradTile<KP, DK>;
  WalkSync* sy = reinterpret_cast<WalkSync*>(raw + 2 * W::stage);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hv = blockIdx.y, h = hv / p.group;
  const int tiles = (p.V + 127) / 128;
  const Segment sg = MODE == 0 ? segment_of(p, tiles, DK) : Segment{};
  const int64_t n = MODE == 0 ? sg.n : blockIdx.x / tiles;
  const int v0 = MODE == 0 ? sg.v0 : int(blockIdx.x % tiles) * 128;
  const int V = MODE == 0 ? sg.channels : p.V;  // of the state that is walked
  SeqAt s = seq_at(p, n);
  if (MODE == 0 && p.segments > 1) {
    const int64_t from = int64_t(sg.index) * p.segment_chunks;
    s.chunk0 += from;
    s.lo += from * kChunk;
    s.len = max(int64_t(0), min(s.len - from * kChunk, int64_t(p.segment_chunks) * kChunk));
  }
  const int chunks = int((s.len + kChunk - 1) / kChunk);
  walk_setup(sy, tid, warp);
  const Waiter wait{&sy->abort, p.timeout_ns, p.status_words, p.status_host, int(blockIdx.x)};
  const uint32_t tm = sy->tmem;
  // TMEM columns: Y, then U; O; S^T parts, the first two then the state's update; X, then
  // w V'; V'
  constexpr uint32_t cY = 0, cO = 64, cS = 128, cX = 320, cV = 416;
  constexpr uint32_t sStep = DK / 4, xStep = 32;
  using SP = StateParts<DK>;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    if (warp == 9 && lane == 0) walk_fetch<E, DK, MODE == 1>(p, raw, sy, wait, s, chunks, h, hv, false);
    if (warp == 8) {
      for (int c = 0; c < chunks; ++c) {
        const uint32_t st = smem_addr(raw) + (c & 1) * W::stage;
        if (!warp_wait(wait, sy->full[c & 1], c >> 1) || !warp_wait(wait, sy->sr, c)) break;
        tc_fence_after();
        if (elect_one()) {
          issue_product<SP, DK, 64, false, KP>(tm + cY, tm + cS, st + W::k, W::keys, false);
          tc_commit(smem_addr(&sy->y));
        }
        __syncwarp();
        if (!warp_wait(wait, sy->xr, c)) break;
        tc_fence_after();
        if (elect_one()) {
          issue_lower<false, 3>(tm + cY, tm + cX, st + W::t);
          tc_commit(smem_addr(&sy->u));
          if constexpr (MODE == 0) {
            issue_product<SP, DK, 64, false, KP>(tm + cO, tm + cS, st + W::q, W::keys, false);
            tc_commit(smem_addr(&sy->q));
          }
        }
        __syncwarp();
        // (the update takes the place of the state's parts: Q's product is done with them)
        if (!warp_wait(wait, sy->vr, c) || (MODE == 0 && !warp_wait(wait, sy->q, c))) break;
        tc_fence_after();
        if (elect_one()) {
          issue_product<TokenParts, kChunk, DK, true, KP>(tm + cS, tm + cX, st + W::k, W::keys, false);
          tc_commit(smem_addr(&sy->s));
          if constexpr (MODE == 1) tc_commit(smem_addr(&sy->free[c & 1]));
        }
        __syncwarp();
        if constexpr (MODE == 0) {
          if (!warp_wait(wait, sy->qr, c)) break;
          tc_fence_after();
          if (elect_one()) {
            issue_lower<false, 3>(tm + cO, tm + cV, st + W::p);
            tc_commit(smem_addr(&sy->o));
            tc_commit(smem_addr(&sy->free[c & 1]));
          }
          __syncwarp();
        }
      }
      if (elect_one()) tc_commit(smem_addr(&sy->drain));
      __syncwarp();
      mbar_wait_bounded(smem_addr(&sy->drain), 0, wait.abort, false, wait.timeout_ns);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWalkRegs));
    const uint32_t lanes = tm + (uint32_t(warp & 3) << 21);  // 32 lanes a quadrant
    const int half = warp >> 2, ch = v0 + 32 * (warp & 3) + lane, t0 = 32 * half;
    const bool live = ch < V;
    const bool real = MODE != 0 || sg.role != Segment::kMap;  // V is read
    const bool out = MODE != 0 || sg.role == Segment::kWhole;  // o is written
    const int64_t state_at = ((n * p.HV + hv) * DK + half * (DK / 2)) * int64_t(V) + ch;
    const uint16_t* v = static_cast<const uint16_t*>(p.v) + s.b * p.v_sb + s.lo * p.v_st + hv * p.v_sh + ch;
    uint16_t* o = static_cast<uint16_t*>(p.o) + ((s.b * p.T + s.lo) * p.HV + hv) * p.V + ch;
    float S[DK / 2];
    if (MODE == 0 && p.segments > 1) {
      if (sg.role == Segment::kMap) {
#pragma unroll
        for (int i = 0; i < DK / 2; ++i) S[i] = half * (DK / 2) + i == ch ? 1.f : 0.f;
      } else {
        const float* from = sg.role == Segment::kFromZero ? nullptr
                            : sg.index == 0
                                ? (p.init == nullptr ? nullptr : p.init + state_at)
                                : segment_state(p, p.seg_s, n, hv, sg.index, DK, V) +
                                      int64_t(half * (DK / 2)) * V + ch;
        walk_load<DK>(S, from, V, live);
      }
    } else {
      walk_load<DK>(S, p.init == nullptr ? nullptr : p.init + state_at, p.V, live);
    }
    uint32_t vr[32];
    const uint32_t vstep = uint32_t(p.v_st * 2), ostep = uint32_t(p.HV * p.V * 2);
    auto rows_of = [&](int c) {  // of this thread's 32 tokens
      return int(min(int64_t(32), s.len - int64_t(c) * kChunk - t0));
    };
    walk_column(vr, v + t0 * p.v_st, vstep, rows_of(0), live && real);
    float qs[32];     // scale gam S^T Q^T of the chunk
    float last = 1.f; // gam_63 of the chunk before
    const int own = 32 * (warp & 3) + lane;
    int bad = 32, bad_out = 32;  // first of this thread's tokens that are spoiled, and outputs
    bool look = false;
    auto odd_values = [&] { return !all_finite<32>([&](int i) { return widen<E>(vr[i]); }); };
    if (odd_values() || !all_finite<DK / 2>([&](int i) { return S[i]; })) sy->odd = 1;
    bool ok = true;
    // Output of a chunk: qs plus P's product.
    auto put_out = [&](int c) {
      if (look && half) {  // (the other half's tokens come first)
        ok = warp_wait(wait, sy->qr, c);
        if (!ok) return;
        if (sy->bad[own] == c) bad_out = 0;
      }
      ok = warp_wait(wait, sy->o, c);
      if (!ok) return;
      tc_fence_after();
      uint32_t r[32];
      tmem_ld(lanes + cO + t0, r);
#pragma unroll
      for (int i = 0; i < 32; ++i) qs[i] += __uint_as_float(r[i]);
      if (look) spoil(qs, bad_out);
      walk_put<E>(o + (int64_t(c) * kChunk + t0) * p.HV * p.V, ostep, qs, rows_of(c), live && out);
    };
    // The state after the chunk before: gam_63 S + its update.
    auto advance = [&](int c) {
      ok = warp_wait(wait, sy->s, c);
      if (!ok) return;
      tc_fence_after();
      uint32_t r[DK / 2];
      tmem_ld(lanes + cS + half * (DK / 2), r);
#pragma unroll
      for (int i = 0; i < DK / 2; ++i) S[i] = fmaf(last, S[i], __uint_as_float(r[i]));
    };
    for (int c = 0; chunks > 0; ++c) {  // (behind the last chunk: its state and output)
      const float* coef =
          reinterpret_cast<const float*>(raw + (c & 1) * W::stage + W::coef);
      const int64_t slot = (s.chunk0 + c) * p.HV + hv;
      if (c > 0) {
        if (c < chunks && odd_values()) sy->odd = 1;
        advance(c - 1);
        if (!ok) break;
      }
      if (MODE == 1 && c == chunks) break;
#pragma unroll
      for (int x = 0; x < DK / 64; ++x) {
        float w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) w[i] = S[32 * x + i];
        split_parts(w, [&](int part, const uint32_t (&r)[16]) {
          tmem_st(lanes + cS + 16 * x + (part == 2 ? DK + half * sStep : half * (DK / 2) + part * sStep), r);
          if constexpr (MODE == 1)
            store_pairs(channel_at<KP, DK>(p.tiles, slot * p.V + ch, GT::s - part * GT::part,
                                           half * (DK / 2) + 32 * x), r, live);
        });
      }
      operand_ready(sy->sr, lane);
      if (MODE == 0 && c > 0) {
        put_out(c - 1);
        if (!ok) break;
      }
      if (c == chunks) break;
      // X = V - gam Y
      ok = warp_wait(wait, sy->full[c & 1], c >> 1) &&  // (the coefficients)
           warp_wait(wait, sy->sr, c);                  // (the other half's word on the state)
      if (!ok) break;
      look = *const_cast<volatile int*>(&sy->odd) != 0 || coef[3 * kChunk] != 0.f;  // (all threads)
      if (look) sy->odd = 1;
      bad = 32;
      ok = warp_wait(wait, sy->y, c);
      if (!ok) break;
      tc_fence_after();
      {
        uint32_t r[32];
        tmem_ld(lanes + cY + t0, r);
        float x[32];
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 gam = *reinterpret_cast<const float4*>(coef + t0 + i);
          x[i] = widen<E>(vr[i]) - gam.x * __uint_as_float(r[i]);
          x[i + 1] = widen<E>(vr[i + 1]) - gam.y * __uint_as_float(r[i + 1]);
          x[i + 2] = widen<E>(vr[i + 2]) - gam.z * __uint_as_float(r[i + 2]);
          x[i + 3] = widen<E>(vr[i + 3]) - gam.w * __uint_as_float(r[i + 3]);
        }
        if (look) {
          bad = first_bad(x);
          if (!half && bad < 32) sy->bad[own] = c;
        }
        split_to_tmem(x, lanes + cX + t0 / 2, xStep);
      }
      operand_ready(sy->xr, lane);
      if (c + 1 < chunks)
        walk_column(vr, v + (int64_t(c + 1) * kChunk + t0) * p.v_st, vstep, rows_of(c + 1),
                    live && real);
      // V' = beta U and w V'
      if (look && half) {
        ok = warp_wait(wait, sy->xr, c);
        if (!ok) break;
        if (sy->bad[own] == c) bad = 0;
      }
      ok = warp_wait(wait, sy->u, c);
      if (!ok) break;
      tc_fence_after();
      last = coef[kChunk - 1];
      {
        uint32_t r[32];
        tmem_ld(lanes + cY + t0, r);
        if (look) spoil(r, bad);
        float u[32], x[32];
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 w = *reinterpret_cast<const float4*>(coef + kChunk + t0 + i);
          const float4 be = *reinterpret_cast<const float4*>(coef + 2 * kChunk + t0 + i);
          u[i] = be.x * __uint_as_float(r[i]);
          u[i + 1] = be.y * __uint_as_float(r[i + 1]);
          u[i + 2] = be.z * __uint_as_float(r[i + 2]);
          u[i + 3] = be.w * __uint_as_float(r[i + 3]);
          x[i] = w.x * u[i];
          x[i + 1] = w.y * u[i + 1];
          x[i + 2] = w.z * u[i + 2];
          x[i + 3] = w.w * u[i + 3];
        }
        split_to_tmem(x, lanes + cX + t0 / 2, xStep);
        operand_ready(sy->vr, lane);
        if constexpr (MODE == 1) {
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(r[i]);
          split_parts(x, [&](int part, const uint32_t (&b)[16]) {
            store_pairs(channel_at<KP, DK>(p.tiles, slot * p.V + ch, GT::u + part * GT::upart, t0), b, live);
          });
        }
        if constexpr (MODE == 0) {
          // beside the chain: V' for the output, and Q's product
          bad_out = 32;
          if (look) {
            bad_out = first_bad(u);  // (U's NaN among them)
            if (!half && bad_out < 32) sy->bad[own] = c;
          }
          split_to_tmem(u, lanes + cV + t0 / 2, xStep);
          ok = warp_wait(wait, sy->q, c);
          if (!ok) break;
          tc_fence_after();
          tmem_ld(lanes + cO + t0, r);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 gam = *reinterpret_cast<const float4*>(coef + t0 + i);
            qs[i] = p.scale * gam.x * __uint_as_float(r[i]);
            qs[i + 1] = p.scale * gam.y * __uint_as_float(r[i + 1]);
            qs[i + 2] = p.scale * gam.z * __uint_as_float(r[i + 2]);
            qs[i + 3] = p.scale * gam.w * __uint_as_float(r[i + 3]);
          }
          operand_ready(sy->qr, lane);
        }
      }
    }
    if (MODE == 0 && ok) {
      float* to = nullptr;
      if (p.segments <= 1 || sg.index == p.segments - 1)
        to = p.final_state == nullptr ? nullptr : p.final_state + state_at;
      else if (sg.role == Segment::kMap)
        to = segment_state(p, p.seg_m, n, hv, sg.index, DK, DK) + int64_t(half * (DK / 2)) * DK + ch;
      else if (p.pass == 1)  // the state behind the first segment, N of an inner one
        to = segment_state(p, p.seg_s, n, hv, sg.index + 1, DK, V) + int64_t(half * (DK / 2)) * V + ch;
      if (to != nullptr) walk_store<DK>(to, S, V, live);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 8) tmem_free(tm, kTmemColumns);
}

// The walk back:
//   dV' = P^T dO + w (K dS)        dX = T^T (beta dV')  (= dV)
//   dS <- gam_63 dS + scale Q^T (gam dO) - K^T (gam dX)
// with dS^T in the lanes.  dS behind each chunk, dX and dO^T go to the workspace
// (671 MB at 8192 tokens of 32 heads of 128 x 128: 3.2 TB/s beside the chain).
template <class E, int DK>
__global__ void __launch_bounds__(kWalkThreads, 1) delta_walk_back_kernel(const DeltaParams p) {
  extern __shared__ __align__(1024) unsigned char raw[];
  using W = WalkTiles<E, DK>;
  constexpr int KP = W::KP;
  using GT = GradTile<KP, DK>;
  WalkSync* sy = reinterpret_cast<WalkSync*>(raw + 2 * W::stage);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hv = blockIdx.y, h = hv / p.group;
  const int tiles = (p.V + 127) / 128;
  const int64_t n = blockIdx.x / tiles;
  const int v0 = int(blockIdx.x % tiles) * 128;
  const SeqAt s = seq_at(p, n);
  const int chunks = int((s.len + kChunk - 1) / kChunk);
  walk_setup(sy, tid, warp);
  const Waiter wait{&sy->abort, p.timeout_ns, p.status_words, p.status_host, int(blockIdx.x)};
  const uint32_t tm = sy->tmem;
  // TMEM columns: K dS, then dX; dS^T parts, the first two then the state's update; P^T dO
  // and, once a half of it is read, that half of gam dO; dO (exact); beta dV', then -gam dX
  constexpr uint32_t cY = 0, cS = 64, cG = 256, cP = cG + 16, cO = 352, cX = 416;
  constexpr uint32_t sStep = DK / 4, xStep = 32;
  using SP = StateParts<DK>;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    if (warp == 9 && lane == 0) walk_fetch<E, DK, false>(p, raw, sy, wait, s, chunks, h, hv, true);
    if (warp == 8) {
      for (int c = 0; c < chunks; ++c) {
        const uint32_t st = smem_addr(raw) + (c & 1) * W::stage;
        // (P^T dO takes the place of gam dO: the last chunk's products are done with it)
        if (!warp_wait(wait, sy->full[c & 1], c >> 1) || !warp_wait(wait, sy->gr, c) ||
            (c > 0 && !warp_wait(wait, sy->s, c - 1)))
          break;
        tc_fence_after();
        if (elect_one()) issue_lower<true, KP>(tm + cP, tm + cO, st + W::p);
        __syncwarp();
        if (!warp_wait(wait, sy->sr, c)) break;
        tc_fence_after();
        if (elect_one()) {
          issue_product<SP, DK, 64, false, KP>(tm + cY, tm + cS, st + W::k, W::keys, false);
          tc_commit(smem_addr(&sy->y));
        }
        __syncwarp();
        if (!warp_wait(wait, sy->xr, c)) break;
        tc_fence_after();
        if (elect_one()) {
          issue_lower<true, 3>(tm + cY, tm + cX, st + W::t);
          tc_commit(smem_addr(&sy->u));
        }
        __syncwarp();
        // (xr stands behind y: K dS has read dS^T's parts, the update may take their place)
        if (!warp_wait(wait, sy->qr, c)) break;
        tc_fence_after();
        if (elect_one())
          issue_product<HalfParts, kChunk, DK, true, KP>(tm + cS, tm + cG, st + W::q, W::keys, false);
        __syncwarp();
        if (!warp_wait(wait, sy->vr, c)) break;
        tc_fence_after();
        if (elect_one()) {
          issue_product<TokenParts, kChunk, DK, true, KP>(tm + cS, tm + cX, st + W::k, W::keys, true);
          tc_commit(smem_addr(&sy->s));
          tc_commit(smem_addr(&sy->free[c & 1]));
        }
        __syncwarp();
      }
      if (elect_one()) tc_commit(smem_addr(&sy->drain));
      __syncwarp();
      mbar_wait_bounded(smem_addr(&sy->drain), 0, wait.abort, false, wait.timeout_ns);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWalkRegs));
    const uint32_t lanes = tm + (uint32_t(warp & 3) << 21);
    const int half = warp >> 2, ch = v0 + 32 * (warp & 3) + lane, t0 = 32 * half;
    const bool live = ch < p.V;
    const int64_t state_at = ((n * p.HV + hv) * DK + half * (DK / 2)) * int64_t(p.V) + ch;
    const uint16_t* d_o = static_cast<const uint16_t*>(p.d_o) + s.b * p.do_sb + s.lo * p.do_st +
                          hv * p.do_sh + ch;
    uint16_t* dv = static_cast<uint16_t*>(p.dv) + ((s.b * p.T + s.lo) * p.HV + hv) * p.V + ch;
    float D[DK / 2];
    walk_load<DK>(D, p.dfinal == nullptr ? nullptr : p.dfinal + state_at, p.V, live);
    uint32_t vr[32], hi[16], lo[16];
    const uint32_t dostep = uint32_t(p.do_st * 2), dvstep = uint32_t(p.HV * p.V * 2);
    auto rows_of = [&](int cc) { return int(min(int64_t(32), s.len - int64_t(cc) * kChunk - t0)); };
    auto fetch_do = [&](int c) {  // c counts from the end
      const int cc = chunks - 1 - c;
      walk_column(vr, d_o + (int64_t(cc) * kChunk + t0) * p.do_st, dostep, rows_of(cc), live);
    };
    if (chunks > 0) fetch_do(0);
    float last = 1.f;
    bool ok = true;
    auto advance = [&](int c) {
      ok = warp_wait(wait, sy->s, c);
      if (!ok) return;
      tc_fence_after();
      uint32_t r[DK / 2];
      tmem_ld(lanes + cS + half * (DK / 2), r);
#pragma unroll
      for (int i = 0; i < DK / 2; ++i) D[i] = fmaf(last, D[i], __uint_as_float(r[i]));
    };
    for (int c = 0; c < chunks; ++c) {
      const int cc = chunks - 1 - c;
      const float* coef =
          reinterpret_cast<const float*>(raw + (c & 1) * W::stage + W::coef);
      const int64_t slot = (s.chunk0 + cc) * p.HV + hv;
      // dO as it is (the last chunk's product with it was done before its update)
#pragma unroll
      for (int i = 0; i < 16; ++i) split_elem<E>(vr[2 * i] | vr[2 * i + 1] << 16, hi[i], lo[i]);
      tmem_st(lanes + cO + t0 / 2, hi);
      if constexpr (KP == 2) tmem_st(lanes + cO + xStep + t0 / 2, lo);
      operand_ready(sy->gr, lane);
      {
        store_pairs(channel_at<KP, DK>(p.tiles, slot * p.V + ch, GT::oh, t0), hi, live);
        if constexpr (KP == 2)
          store_pairs(channel_at<KP, DK>(p.tiles, slot * p.V + ch, GT::om, t0), lo, live);
      }
      if (c > 0) {
        advance(c - 1);
        if (!ok) break;
      }
#pragma unroll
      for (int x = 0; x < DK / 64; ++x) {
        float w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) w[i] = D[32 * x + i];
        split_parts(w, [&](int part, const uint32_t (&r)[16]) {
          tmem_st(lanes + cS + 16 * x + (part == 2 ? DK + half * sStep : half * (DK / 2) + part * sStep), r);
          store_pairs(channel_at<KP, DK>(p.tiles, slot * p.V + ch, GT::d + part * GT::part,
                                         half * (DK / 2) + 32 * x), r, live);
        });
      }
      operand_ready(sy->sr, lane);
      // beta dV'
      ok = warp_wait(wait, sy->full[c & 1], c >> 1);  // (the coefficients)
      if (!ok) break;
      ok = warp_wait(wait, sy->y, c);
      if (!ok) break;
      tc_fence_after();
      {
        uint32_t r[32], r2[32];
        tmem_ld(lanes + cY + t0, r);
        tmem_ld(lanes + cP + t0, r2);
        float x[32];
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 w = *reinterpret_cast<const float4*>(coef + kChunk + t0 + i);
          const float4 be = *reinterpret_cast<const float4*>(coef + 2 * kChunk + t0 + i);
          x[i] = be.x * fmaf(w.x, __uint_as_float(r[i]), __uint_as_float(r2[i]));
          x[i + 1] = be.y * fmaf(w.y, __uint_as_float(r[i + 1]), __uint_as_float(r2[i + 1]));
          x[i + 2] = be.z * fmaf(w.z, __uint_as_float(r[i + 2]), __uint_as_float(r2[i + 2]));
          x[i + 3] = be.w * fmaf(w.w, __uint_as_float(r[i + 3]), __uint_as_float(r2[i + 3]));
        }
        split_to_tmem(x, lanes + cX + t0 / 2, xStep);
      }
      operand_ready(sy->xr, lane);
      {  // gam dO beside the chain, where this thread has just read P^T dO
        float x[32];
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 gam = *reinterpret_cast<const float4*>(coef + t0 + i);
          x[i] = p.scale * gam.x * widen<E>(vr[i]);
          x[i + 1] = p.scale * gam.y * widen<E>(vr[i + 1]);
          x[i + 2] = p.scale * gam.z * widen<E>(vr[i + 2]);
          x[i + 3] = p.scale * gam.w * widen<E>(vr[i + 3]);
        }
        split_to_tmem(x, lanes + cG + half * 48, 16);
        operand_ready(sy->qr, lane);
      }
      if (c + 1 < chunks) fetch_do(c + 1);
      // dX
      ok = warp_wait(wait, sy->u, c);
      if (!ok) break;
      tc_fence_after();
      last = coef[kChunk - 1];
      {
        uint32_t r[32];
        tmem_ld(lanes + cY + t0, r);
        float x[32];
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 gam = *reinterpret_cast<const float4*>(coef + t0 + i);
          x[i] = -gam.x * __uint_as_float(r[i]);
          x[i + 1] = -gam.y * __uint_as_float(r[i + 1]);
          x[i + 2] = -gam.z * __uint_as_float(r[i + 2]);
          x[i + 3] = -gam.w * __uint_as_float(r[i + 3]);
        }
        split_to_tmem(x, lanes + cX + t0 / 2, xStep);
        operand_ready(sy->vr, lane);
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(r[i]);
        walk_put<E>(dv + (int64_t(cc) * kChunk + t0) * p.HV * p.V, dvstep, x, rows_of(cc), live);
        split_parts(x, [&](int part, const uint32_t (&b)[16]) {
          store_pairs(channel_at<KP, DK>(p.tiles, slot * p.V + ch, GT::x(part), t0), b, live);
        });
      }
    }
    if (ok && chunks > 0) advance(chunks - 1);
    if (ok && p.dinit != nullptr) walk_store<DK>(p.dinit + state_at, D, p.V, live);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 8) tmem_free(tm, kTmemColumns);
}

}  // namespace tdc
