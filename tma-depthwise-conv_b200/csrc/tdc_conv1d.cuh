// tdc_conv1d.cuh — causal depthwise convolution over [B, T, C]: forward,
// gradients and the step of running sequences.
//
// The forward moves 4 bytes per element and does 2K flops on them, so it is
// bound by memory.  A thread owns 8 channels (one 16-byte vector) and slides
// down a run of rows with the last K-1 inputs in registers, as packed pairs
// that fma.rn.f32.{f16,bf16} takes without conversion; consecutive threads own
// consecutive channels, so every access of a warp is whole 128-byte lines and
// needs no shared memory.  Four rows are loaded ahead of their use.
// Measured (K = 4, SiLU): 8192 rows of 8192 channels in bf16 (268 MB) 50 us,
// 5.3 TB/s of the 6.46 that a copy reaches; 5003 packed rows of 2560 in fp16
// (51 MB) 14.5 us, the latency of a wave of blocks: 285 that make the outputs and 34 that
// copy final states, of which 11 find a place at once.
#pragma once

#include "tdc_seq_common.cuh"

namespace tdc {

struct Conv1dParams {
  const void* x;
  const void* w;
  const void* bias;
  const void* init;      // [N, K-1, C] or null
  void* final_state;     // [N, K-1, C] or null
  void* y;
  SeqTable seq;          // seq.n = N
  int64_t B, T, C;
  int64_t x_sb, x_st;
  int64_t runs_per_b;    // runs of `run` rows in each batch row
  int run;
  int64_t main_threads;  // B * runs_per_b * C / 8; the threads behind it copy final states
  // backward
  const void* dy;
  int64_t dy_sb, dy_st;
  const void* dfinal;
  void* dx;
  void* dinit;
  float* partial;        // [groups][K + 1][C]
  int64_t groups;
  // step
  void* state;
  const void* idx;
  int64_t slots;
  bool idx64;
};

// The sequence that owns row t of batch row b.  covered: rows [lo, hi) belong
// to sequence n; otherwise no sequence owns rows t .. hi-1.
struct SeqSpan {
  int64_t n, lo, hi;
  bool covered;
};

__device__ __forceinline__ SeqSpan span_from(const SeqTable& s, int64_t n, int64_t t) {
  while (n < s.n && s.at(n + 1) <= t) ++n;
  SeqSpan r;
  r.n = n;
  if (n >= s.n) {
    r.covered = false;
    r.lo = t;
    r.hi = s.T;
    return r;
  }
  const int64_t lo = s.at(n);
  r.covered = lo <= t;
  r.lo = r.covered ? lo : t;
  r.hi = r.covered ? s.at(n + 1) : lo;
  return r;
}

__device__ __forceinline__ SeqSpan span_at(const SeqTable& s, int64_t b, int64_t t) {
  if (s.cu == nullptr) return {b, 0, s.T, true};
  return span_from(s, s.first_ending_after(t), t);
}

__device__ __forceinline__ uint4 ld16(const void* base, int64_t elem) {
  return __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + elem));
}
__device__ __forceinline__ void st16(void* base, int64_t elem, const uint4& v) {
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + elem) = v;
}

// Row t as an input of sequence s: from x, or for t < lo from the initial
// state (zeros without one).
__device__ __forceinline__ uint4 conv_input(const Conv1dParams& p, int taps, const SeqSpan& s,
                                            int64_t xbase, int64_t t, int64_t c) {
  if (t >= s.lo) return ld16(p.x, xbase + t * p.x_st + c);
  const int64_t row = t - s.lo + taps - 1;
  if (p.init == nullptr || row < 0) return make_uint4(0, 0, 0, 0);
  return ld16(p.init, (s.n * (taps - 1) + row) * p.C + c);
}

template <class E, int K>
__device__ __forceinline__ void conv_dot(float z[8], const uint4 win[K], const uint4 w[K]) {
#pragma unroll
  for (int j = 0; j < K; ++j) {
    fma2<E>(win[j].x, w[j].x, z[0], z[1]);
    fma2<E>(win[j].y, w[j].y, z[2], z[3]);
    fma2<E>(win[j].z, w[j].z, z[4], z[5]);
    fma2<E>(win[j].w, w[j].w, z[6], z[7]);
  }
}

// PACKED: sequences may end inside a run (cu_seqlens).
template <class E, int K, bool SILU, bool PACKED>
__global__ void __launch_bounds__(256, 2) conv1d_fwd_kernel(const Conv1dParams p) {
  const int64_t id = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t vecs = p.C / 8;
  if (id >= p.main_threads) {
    // The last K-1 inputs of each sequence, one vector a thread.
    const int64_t r = id - p.main_threads;
    if (p.final_state == nullptr || r >= p.seq.n * (K - 1) * vecs) return;
    const int64_t c = (r % vecs) * 8, j = (r / vecs) % (K - 1), n = r / (vecs * (K - 1));
    SeqSpan s{n, 0, p.T, true};
    int64_t xbase = n * p.x_sb;
    if (PACKED) {
      s.lo = p.seq.at(n);
      s.hi = max(s.lo, p.seq.at(n + 1));
      xbase = 0;
    }
    const uint4 v = conv_input(p, K, s, xbase, s.hi - (K - 1) + j, c);
    st16(p.final_state, (n * (K - 1) + j) * p.C + c, v);
    return;
  }
  const int64_t c = (id % vecs) * 8, run = id / vecs;
  const int64_t b = run / p.runs_per_b, t0 = (run % p.runs_per_b) * p.run;
  const int rows = int(min(int64_t(p.run), p.T - t0));
  const int64_t xbase = b * p.x_sb;
  const uint16_t* x = static_cast<const uint16_t*>(p.x) + xbase + t0 * p.x_st + c;
  uint16_t* y = static_cast<uint16_t*>(p.y) + (b * p.T + t0) * p.C + c;
  // win: the K-1 inputs before the first of 4 rows, then those rows.  What does not
  // depend on the sequences is on its way before they are looked up.
  uint4 win[K + 3], next[4], w[K];
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (u < rows) next[u] = ld16(x, u * p.x_st);
#pragma unroll
  for (int j = 0; j < K - 1; ++j)
    if (t0 >= K - 1 - j) win[j] = ld16(x, (j - (K - 1)) * p.x_st);
#pragma unroll
  for (int j = 0; j < K; ++j) w[j] = ld16(p.w, j * p.C + c);
  uint4 b8 = make_uint4(0, 0, 0, 0);
  if (p.bias != nullptr) b8 = ld16(p.bias, c);
  SeqSpan s{b, 0, p.T, true};
  if (PACKED) s = span_at(p.seq, b, t0);
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    if (!s.covered) win[j] = make_uint4(0, 0, 0, 0);
    else if (t0 - (K - 1) + j < s.lo) win[j] = conv_input(p, K, s, xbase, t0 - (K - 1) + j, c);
  }
  float bias[8];
  unpack8<E>(b8, bias);

  for (int t = 0; t < rows; t += 4) {
#pragma unroll
    for (int u = 0; u < 4; ++u) win[K - 1 + u] = next[u];
    x += 4 * p.x_st;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (t + 4 + u < rows) next[u] = ld16(x, u * p.x_st);
    auto put = [&](int u, bool covered) {
      float z[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = bias[i];
      conv_dot<E, K>(z, win + u, w);
      if constexpr (SILU) {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] *= sigmoid_f(z[i]);
      }
      st16(y, 0, covered ? pack8<E>(z) : make_uint4(0, 0, 0, 0));
      y += p.C;
    };
    if (t + 4 <= rows && (!PACKED || (s.covered && t0 + t + 4 <= s.hi))) {
      // in the inside of a run and a sequence: no tests between the rows
#pragma unroll
      for (int u = 0; u < 4; ++u) put(u, true);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (t + u < rows) {
          if (PACKED && t0 + t + u >= s.hi) {  // the next sequence (or gap) starts here
            s = span_from(p.seq, s.n, t0 + t + u);
            if (s.covered) {
#pragma unroll
              for (int j = 0; j < K - 1; ++j)
                win[u + j] = conv_input(p, K, s, xbase, s.lo - (K - 1) + j, c);
            }
          }
          put(u, s.covered);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < K - 1; ++j) win[j] = win[j + 4];
  }
}

// ---- gradients -----------------------------------------------------------------
// With dz = dy * act'(z): dx[t] = sum_j w[j] dz[t + K-1-j] within the sequence
// (plus dfinal where the row is among the sequence's last K-1 inputs), dw[j] =
// sum_t dz[t] x[t-(K-1)+j], dbias = sum dz.  z is recomputed from x, so the
// pass reads x and dy and writes dx: bound by memory.  A thread owns 4 channels
// (8 would not leave registers for the taps' sums) and a run of rows.  The last
// K inputs and the K unfinished rows of dx sit in rings of registers whose
// places are fixed by unrolling K rows; dz[t] is added to the rows it reaches.
// Rows in the inside of a sequence and a run go through the loop without a test.
// The K-1 values of dz behind the run are recomputed.  The runs of a block are
// added in shared memory and one partial sum per block goes to the workspace,
// which conv1d_wsum_kernel adds in a fixed order.
// Measured (K = 4, SiLU, bf16, 8192 rows of 8192 channels, 403 MB): 101 us,
// 4.0 TB/s; what is left is latency, with the 512 threads an SM that the taps'
// sums leave room for.  conv1d_wsum_kernel: 5.6 us.
constexpr int kGradVec = 4;

struct Quad {  // 4 channels
  float2 a, b;
};
template <class E>
__device__ __forceinline__ Quad unpack4(const uint2& v) {
  Quad q;
  unpack2<E>(v.x, q.a.x, q.a.y);
  unpack2<E>(v.y, q.b.x, q.b.y);
  return q;
}
__device__ __forceinline__ void fma4(Quad& d, const Quad& x, const Quad& y) {
  fma_pair(d.a, x.a, y.a);
  fma_pair(d.b, x.b, y.b);
}
__device__ __forceinline__ Quad zero4() { return {make_float2(0.f, 0.f), make_float2(0.f, 0.f)}; }
__device__ __forceinline__ uint2 ld8(const void* base, int64_t elem) {
  return __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + elem));
}
template <class E>
__device__ __forceinline__ void st8(void* base, int64_t elem, const Quad& f) {
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + elem) =
      make_uint2(pack2_rn<E>(f.a.x, f.a.y), pack2_rn<E>(f.b.x, f.b.y));
}

__device__ __forceinline__ uint2 conv_input4(const Conv1dParams& p, int taps, const SeqSpan& s,
                                             int64_t xbase, int64_t t, int64_t c) {
  if (t >= s.lo) return ld8(p.x, xbase + t * p.x_st + c);
  const int64_t row = t - s.lo + taps - 1;
  if (p.init == nullptr || row < 0) return make_uint2(0, 0);
  return ld8(p.init, (s.n * (taps - 1) + row) * p.C + c);
}

// dz = dy act'(z), z from the inputs at(0) .. at(K-1) (the last is the row's own).
__device__ __forceinline__ float dsilu(float dy, float z) {
  const float sg = sigmoid_f(z);
  return dy * (sg * fmaf(z, 1.f - sg, 1.f));
}
template <int K, bool SILU, class At>
__device__ __forceinline__ Quad conv_dz(At at, const Quad w[K], const Quad& bias, const Quad& dy) {
  if constexpr (!SILU) {
    return dy;
  } else {
    Quad z = bias;
#pragma unroll
    for (int j = 0; j < K; ++j) fma4(z, at(j), w[j]);
    return {make_float2(dsilu(dy.a.x, z.a.x), dsilu(dy.a.y, z.a.y)),
            make_float2(dsilu(dy.b.x, z.b.x), dsilu(dy.b.y, z.b.y))};
  }
}

template <class E, int K, bool SILU, bool PACKED>
__global__ void __launch_bounds__(256, K <= 4 ? 2 : 1) conv1d_bwd_kernel(const Conv1dParams p) {
  __shared__ __align__(16) float red[256 * kGradVec];  // [blockDim.y][blockDim.x * 4]
  const int64_t c = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * kGradVec;
  const int64_t run = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
  const int64_t b = run / p.runs_per_b;
  const bool live = c < p.C && b < p.B;
  Quad dw[K], db = zero4();
#pragma unroll
  for (int j = 0; j < K; ++j) dw[j] = zero4();
  if (live) {
    const int64_t t0 = (run % p.runs_per_b) * p.run, t1 = min(t0 + p.run, p.T);
    const int64_t xbase = b * p.x_sb;
    Quad w[K], bias = zero4();
#pragma unroll
    for (int j = 0; j < K; ++j) w[j] = unpack4<E>(ld8(p.w, j * p.C + c));
    if (p.bias != nullptr) bias = unpack4<E>(ld8(p.bias, c));
    SeqSpan s{b, 0, p.T, true};
    if (PACKED) s = span_at(p.seq, b, t0);
    int64_t a = t0;
    while (a < t1) {  // the part [a, e) of the run that lies in one sequence (or gap)
      const int64_t e = min(t1, s.hi);
      const uint16_t* x = static_cast<const uint16_t*>(p.x) + xbase + a * p.x_st + c;
      const uint16_t* dy = static_cast<const uint16_t*>(p.dy) + b * p.dy_sb + a * p.dy_st + c;
      uint16_t* dx = static_cast<uint16_t*>(p.dx) + (b * p.T + a) * p.C + c;
      if (PACKED && !s.covered) {
        for (int64_t t = a; t < e; ++t, dx += p.C) st8<E>(dx, 0, zero4());
      } else {
        const int own = int(e - a);                                       // rows of dx
        const int known = int(min(int64_t(own + K - 1), s.hi - a));       // rows of dz
        const int64_t to_final = K - 1 - (s.hi - a);  // row i is row i + to_final of final_state
        // Rows before `inside` need no test: dz is known K rows ahead, and no row is one of
        // the final state's.
        const int inside = min(own, known - K);
        uint2 xn[K], dn[K];
        Quad xr[K], acc[K];
        // row a - (K-1) + j has place (j + 1) % K
        xr[0] = zero4();
#pragma unroll
        for (int j = 0; j < K - 1; ++j)
          xr[j + 1] = unpack4<E>(conv_input4(p, K, s, xbase, a - (K - 1) + j, c));
#pragma unroll
        for (int u = 0; u < K; ++u) {
          acc[u] = zero4();
          if (u < known) {
            xn[u] = ld8(x, u * p.x_st);
            dn[u] = ld8(dy, u * p.dy_st);
          }
        }
        // Row i takes place u of both rings; K rows on its place is loaded again.
        auto row = [&](int i, int u, auto tested) {
          constexpr bool TEST = decltype(tested)::value;
          acc[u] = zero4();
          if (TEST && p.dfinal != nullptr && i < own && i + to_final >= 0)
            acc[u] = unpack4<E>(ld8(p.dfinal, (s.n * (K - 1) + i + to_final) * p.C + c));
          if (!TEST || i < known) {
            xr[u] = unpack4<E>(xn[u]);
            const Quad dyv = unpack4<E>(dn[u]);
            if (!TEST || i + K < known) {
              xn[u] = ld8(x, u * p.x_st);
              dn[u] = ld8(dy, u * p.dy_st);
            }
            const Quad dz =
                conv_dz<K, SILU>([&](int j) -> const Quad& { return xr[(u + 1 + j) % K]; }, w, bias, dyv);
            if (!TEST || i < own) {
#pragma unroll
              for (int j = 0; j < K; ++j) fma4(dw[j], dz, xr[(u + 1 + j) % K]);
              db.a.x += dz.a.x, db.a.y += dz.a.y, db.b.x += dz.b.x, db.b.y += dz.b.y;
            }
#pragma unroll
            for (int j = 0; j < K; ++j) fma4(acc[(u + 1 + j) % K], w[j], dz);  // row i - (K-1) + j
          }
          if (!TEST || (i >= K - 1 && i < own + K - 1)) {
            st8<E>(dx, 0, acc[(u + 1) % K]);
            dx += p.C;
          }
        };
        int i0 = 0;
        for (; i0 < own + K - 1; i0 += K) {
          x += K * p.x_st;
          dy += K * p.dy_st;
          if (i0 > 0 && i0 + K <= inside) {
#pragma unroll
            for (int u = 0; u < K; ++u) row(i0 + u, u, std::false_type{});
          } else {
#pragma unroll
            for (int u = 0; u < K; ++u) row(i0 + u, u, std::true_type{});
          }
        }
      }
      a = e;
      if (PACKED && a < t1) s = span_from(p.seq, s.n, a);
    }
  }
  // Add the block's runs, tap by tap (K is the bias).
  const int width = blockDim.x * kGradVec;
#pragma unroll
  for (int j = 0; j <= K; ++j) {
    __syncthreads();
    const Quad part = j < K ? dw[j < K ? j : 0] : db;
    *reinterpret_cast<float4*>(red + threadIdx.y * width + threadIdx.x * kGradVec) =
        make_float4(part.a.x, part.a.y, part.b.x, part.b.y);
    __syncthreads();
    for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < width; i += blockDim.x * blockDim.y) {
      const int64_t cc = int64_t(blockIdx.y) * width + i;
      if (cc >= p.C) continue;
      float sum = 0.f;
      for (int r = 0; r < int(blockDim.y); ++r) sum += red[r * width + i];
      p.partial[(int64_t(blockIdx.x) * (K + 1) + j) * p.C + cc] = sum;
    }
  }
}

// dw [K, C] and dbias [C] from the blocks' partial sums, in block order.
template <class E>
__global__ void __launch_bounds__(256) conv1d_wsum_kernel(const float* partial, int64_t groups,
                                                          int64_t taps, int64_t C, void* dw,
                                                          void* dbias) {
  // 8 threads a value: each adds every 8th group, then the 8 are added.
  const int64_t v = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) / 8;
  const int part = threadIdx.x & 7;
  const int64_t total = (taps + 1) * C;
  float sum = 0.f;
  if (v < total)
    for (int64_t g = part; g < groups; g += 8) sum += partial[g * total + v];
  sum += __shfl_xor_sync(0xffffffffu, sum, 1);
  sum += __shfl_xor_sync(0xffffffffu, sum, 2);
  sum += __shfl_xor_sync(0xffffffffu, sum, 4);
  if (v >= total || part != 0) return;
  if (v < taps * C) store_float<E>(dw, v, sum);
  else if (dbias != nullptr) store_float<E>(dbias, v - taps * C, sum);
}

// Gradient of the initial states: row r of sequence n is input t = lo-(K-1)+r,
// reached by dz[lo .. lo+r].
template <class E, int K, bool SILU>
__global__ void __launch_bounds__(128) conv1d_dinit_kernel(const Conv1dParams p) {
  const int64_t vecs = p.C / 4;
  const int64_t id = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (id >= p.seq.n * vecs) return;
  const int64_t c = (id % vecs) * 4, n = id / vecs;
  SeqSpan s{n, 0, p.T, true};
  int64_t b = n;
  if (p.seq.cu != nullptr) {
    s.lo = p.seq.at(n);
    s.hi = max(s.lo, p.seq.at(n + 1));
    b = 0;
  }
  const int64_t len = s.hi - s.lo;
  Quad w[K], win[2 * K - 2], d[K - 1], bias = zero4();
#pragma unroll
  for (int j = 0; j < K; ++j) w[j] = unpack4<E>(ld8(p.w, j * p.C + c));
  if (p.bias != nullptr) bias = unpack4<E>(ld8(p.bias, c));
  // input r + len of the K-1 + len ones is row r of final_state
#pragma unroll
  for (int r = 0; r < K - 1; ++r)
    d[r] = p.dfinal != nullptr && r >= len
               ? unpack4<E>(ld8(p.dfinal, (n * (K - 1) + r - len) * p.C + c))
               : zero4();
#pragma unroll
  for (int j = 0; j < K - 1; ++j)
    win[j] = unpack4<E>(conv_input4(p, K, s, b * p.x_sb, s.lo - (K - 1) + j, c));
#pragma unroll
  for (int t = 0; t < K - 1; ++t) {
    if (t < len) {
      win[K - 1 + t] = unpack4<E>(ld8(p.x, b * p.x_sb + (s.lo + t) * p.x_st + c));
      const Quad dz = conv_dz<K, SILU>(
          [&](int j) -> const Quad& { return win[t + j]; }, w, bias,
          unpack4<E>(ld8(p.dy, b * p.dy_sb + (s.lo + t) * p.dy_st + c)));
      // dz[t] reaches inputs t .. t+K-1 through w[0 .. K-1]
#pragma unroll
      for (int r = t; r < K - 1; ++r) fma4(d[r], w[r - t], dz);
    }
  }
#pragma unroll
  for (int r = 0; r < K - 1; ++r) st8<E>(p.dinit, (n * (K - 1) + r) * p.C + c, d[r]);
}

// ---- running sequences ---------------------------------------------------------
// One thread takes 8 channels of one request: K-1 state rows in, T inputs
// through the window, K-1 rows out.  Bound by latency at the usual sizes: all
// loads of a thread are independent.  4 requests of 8192 channels: 4.7 us with
// cold caches, less than the call takes on the host.
template <class E, int K, bool SILU>
__global__ void __launch_bounds__(128) conv1d_step_kernel(const Conv1dParams p) {
  const int64_t b = blockIdx.x;
  const int64_t c = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 8;
  const int64_t slot = slot_of(p.idx, p.idx64, b, p.slots, threadIdx.x, blockDim.x);
  if (c >= p.C) return;
  const int64_t ybase = b * p.T * p.C + c;
  if (slot < 0) {
    const uint32_t nan2 = nan16<E>() * 0x10001u, fill = slot == -1 ? 0u : nan2;
    for (int64_t t = 0; t < p.T; ++t) st16(p.y, ybase + t * p.C, make_uint4(fill, fill, fill, fill));
    return;
  }
  uint4 w[K], win[K];
  const int64_t sbase = slot * (K - 1) * p.C + c;
#pragma unroll
  for (int j = 0; j < K; ++j) w[j] = ld16(p.w, j * p.C + c);
#pragma unroll
  for (int j = 0; j < K - 1; ++j)
    win[j] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.state) + sbase + j * p.C);
  float bias[8] = {};
  if (p.bias != nullptr) unpack8<E>(ld16(p.bias, c), bias);
  for (int64_t t = 0; t < p.T; ++t) {
    win[K - 1] = ld16(p.x, b * p.x_sb + t * p.x_st + c);
    float z[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = bias[i];
    conv_dot<E, K>(z, win, w);
    if constexpr (SILU) {
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] *= sigmoid_f(z[i]);
    }
    st16(p.y, ybase + t * p.C, pack8<E>(z));
#pragma unroll
    for (int j = 0; j < K - 1; ++j) win[j] = win[j + 1];
  }
#pragma unroll
  for (int j = 0; j < K - 1; ++j) st16(p.state, sbase + j * p.C, win[j]);
}

}  // namespace tdc
