// tdc_sequence.cu — host half of the sequence operators: argument checks,
// launch shapes and workspaces behind the C ABI of include/tdc_sequence.h.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstring>

#include "tdc_sequence.h"
#include "tdc_conv1d.cuh"
#include "tdc_delta_grad.cuh"
#include "tdc_delta_walk.cuh"
#include "tdc_host.h"
#include "tdc_qknorm.cuh"

namespace {

using tdc::host::cuda_fail;
using tdc::host::prepare_device;

constexpr int64_t kMaxDim = int64_t(1) << 40;
constexpr int64_t kMaxRow = int64_t(1) << 31;  // elements of 2 bytes
constexpr int64_t kMaxSize = int64_t(1) << 46;  // elements of a tensor, channels of all chunks

// a * b > limit, without the product (all at least 0)
bool exceeds(int64_t a, int64_t b, int64_t limit) { return b > 0 && a > limit / b; }

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }
bool bad_stride(int64_t s) { return s % 8 != 0; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TDC_OK : cuda_fail(int(e));
}

template <class K>
int allow_smem(K kernel, size_t bytes) {
  // Idempotent and cheap (no device work); kernels below 48 KB need none.
  if (bytes <= 48 * 1024) return TDC_OK;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
  return e == cudaSuccess ? TDC_OK : cuda_fail(int(e));
}

// ---- causal depthwise convolution ---------------------------------------------
int check_conv(int64_t B, int64_t T, int64_t C, int64_t K, int64_t dtype, int64_t act,
               int64_t x_sb, int64_t x_st) {
  if (dtype != TDC_F16 && dtype != TDC_BF16) return TDC_ERR_UNSUPPORTED;
  if (act != TDC_ACT_NONE && act != TDC_ACT_SILU) return TDC_ERR_ACT;
  if (B < 0 || T < 0 || C < 0) return TDC_ERR_BAD_SHAPE;
  if (K < 2 || K > 8) return TDC_ERR_FILTER_SHAPE;
  if (C % 8 != 0) return TDC_ERR_CHANNELS;
  if (B > kMaxDim || T > kMaxDim || C > kMaxDim) return TDC_ERR_TOO_LARGE;
  if (exceeds(B, T, kMaxDim) || exceeds(B, C, kMaxSize) || exceeds(B * T, C, kMaxSize))
    return TDC_ERR_TOO_LARGE;
  if (bad_stride(x_sb) || bad_stride(x_st)) return TDC_ERR_ALIGNMENT;
  return TDC_OK;
}

int check_conv_args(const tdc_conv1d_args* a) {
  if (a == nullptr) return TDC_ERR_NULL_POINTER;
  const int rc = check_conv(a->B, a->T, a->C, a->K, a->dtype, a->act, a->x_sb, a->x_st);
  if (rc != TDC_OK) return rc;
  if (a->cu_seqlens != nullptr && (a->B != 1 || a->num_seqs < 1)) return TDC_ERR_BAD_SHAPE;
  if (a->cu_seqlens != nullptr && exceeds(a->num_seqs, std::max<int64_t>(1, a->C), kMaxSize))
    return TDC_ERR_TOO_LARGE;
  return TDC_OK;
}

tdc::Conv1dParams conv_params(const tdc_conv1d_args* a) {
  tdc::Conv1dParams p;
  std::memset(&p, 0, sizeof p);
  p.x = a->x;
  p.w = a->w;
  p.bias = a->bias;
  p.init = a->initial_state;
  p.final_state = a->final_state;
  p.y = a->y;
  p.seq.cu = a->cu_seqlens;
  p.seq.n = a->cu_seqlens != nullptr ? a->num_seqs : a->B;
  p.seq.T = a->T;
  p.seq.is64 = a->cu_is_64 != 0;
  p.B = a->B;
  p.T = a->T;
  p.C = a->C;
  p.x_sb = a->x_sb;
  p.x_st = a->x_st;
  return p;
}

template <class E, int K>
int conv_fwd_k(const tdc::Conv1dParams& p, bool silu, int64_t blocks, cudaStream_t st) {
  const bool packed = p.seq.cu != nullptr;
  auto* k = silu ? (packed ? &tdc::conv1d_fwd_kernel<E, K, true, true>
                           : &tdc::conv1d_fwd_kernel<E, K, true, false>)
                 : (packed ? &tdc::conv1d_fwd_kernel<E, K, false, true>
                           : &tdc::conv1d_fwd_kernel<E, K, false, false>);
  k<<<unsigned(blocks), 256, 0, st>>>(p);
  return launched();
}

constexpr int kSms = 148;  // a B200's

// Backward launch shape: a block is LX vectors of 4 channels by 256 / LX runs.
struct ConvBwdPlan {
  int lx, run;
  int64_t runs_per_b, groups, cblocks;
};

ConvBwdPlan conv_bwd_plan(const tdc_conv1d_args* a) {
  ConvBwdPlan pl;
  const int64_t vecs = a->C / tdc::kGradVec;
  pl.lx = vecs >= 32 ? 32 : vecs >= 16 ? 16 : 8;
  pl.cblocks = ceil_div(vecs, pl.lx);
  // One wave on 148 SMs (2 blocks each, 1 beyond 4 taps); a run of at least 8 rows, or
  // the K-1 rows that it recomputes behind its end would cost more than they save.
  const int64_t blocks = 148 * (a->K <= 4 ? 2 : 1);
  const int64_t rows = std::max<int64_t>(1, a->B * a->T);
  const int64_t groups = std::max<int64_t>(1, blocks / pl.cblocks);
  int64_t run = std::max<int64_t>(8, ceil_div(rows, groups * (256 / pl.lx)));
  run = std::min(run, std::max<int64_t>(1, a->T));
  pl.runs_per_b = ceil_div(std::max<int64_t>(1, a->T), run);
  pl.run = int(std::min<int64_t>(ceil_div(std::max<int64_t>(1, a->T), pl.runs_per_b), 1 << 30));
  pl.groups = std::max<int64_t>(1, ceil_div(a->B * pl.runs_per_b, 256 / pl.lx));
  return pl;
}

template <class E, int K, bool SILU>
int conv_bwd_t(const tdc::Conv1dParams& p, const ConvBwdPlan& pl, void* dw, void* dbias,
               cudaStream_t st) {
  const dim3 block(pl.lx, 256 / pl.lx), grid(unsigned(pl.groups), unsigned(pl.cblocks));
  auto* k = p.seq.cu != nullptr ? &tdc::conv1d_bwd_kernel<E, K, SILU, true>
                                : &tdc::conv1d_bwd_kernel<E, K, SILU, false>;
  k<<<grid, block, 0, st>>>(p);
  int rc = launched();
  if (rc != TDC_OK) return rc;
  const int64_t values = (K + 1) * p.C;
  tdc::conv1d_wsum_kernel<E><<<unsigned(ceil_div(values, 32)), 256, 0, st>>>(p.partial, pl.groups, K,
                                                                          p.C, dw, dbias);
  rc = launched();
  if (rc != TDC_OK || p.dinit == nullptr || p.seq.n == 0) return rc;
  tdc::conv1d_dinit_kernel<E, K, SILU>
      <<<unsigned(ceil_div(p.seq.n * (p.C / 4), 128)), 128, 0, st>>>(p);
  return launched();
}

template <class E, int K>
int conv_step_k(const tdc::Conv1dParams& p, bool silu, cudaStream_t st) {
  const int threads = p.C / 8 >= 128 ? 128 : p.C / 8 > 32 ? 64 : 32;
  const dim3 grid(unsigned(p.B), unsigned(ceil_div(p.C / 8, threads)));
  if (silu) tdc::conv1d_step_kernel<E, K, true><<<grid, threads, 0, st>>>(p);
  else tdc::conv1d_step_kernel<E, K, false><<<grid, threads, 0, st>>>(p);
  return launched();
}

// f<E, K>(...) for a call's element type and number of taps.
#define TDC_FOR_TAPS(E, K_, CALL)   \
  switch (K_) {                     \
    case 2: return CALL(E, 2);      \
    case 3: return CALL(E, 3);      \
    case 4: return CALL(E, 4);      \
    case 5: return CALL(E, 5);      \
    case 6: return CALL(E, 6);      \
    case 7: return CALL(E, 7);      \
    default: return CALL(E, 8);     \
  }
#define TDC_FOR_CONV(DTYPE, K_, CALL)                                        \
  do {                                                                       \
    if ((DTYPE) == TDC_BF16) { TDC_FOR_TAPS(tdc::BF16, K_, CALL) }           \
    TDC_FOR_TAPS(tdc::F16, K_, CALL)                                         \
  } while (0)

int conv_fwd_any(const tdc::Conv1dParams& p, int64_t K, int64_t dtype, bool silu, int64_t blocks,
                 cudaStream_t st) {
#define TDC_CALL(E, K_) conv_fwd_k<E, K_>(p, silu, blocks, st)
  TDC_FOR_CONV(dtype, K, TDC_CALL);
#undef TDC_CALL
}
int conv_bwd_any(const tdc::Conv1dParams& p, const ConvBwdPlan& pl, int64_t K, int64_t dtype,
                 bool silu, void* dw, void* db, cudaStream_t st) {
#define TDC_CALL(E, K_) \
  (silu ? conv_bwd_t<E, K_, true>(p, pl, dw, db, st) : conv_bwd_t<E, K_, false>(p, pl, dw, db, st))
  TDC_FOR_CONV(dtype, K, TDC_CALL);
#undef TDC_CALL
}
int conv_step_any(const tdc::Conv1dParams& p, int64_t K, int64_t dtype, bool silu, cudaStream_t st) {
#define TDC_CALL(E, K_) conv_step_k<E, K_>(p, silu, st)
  TDC_FOR_CONV(dtype, K, TDC_CALL);
#undef TDC_CALL
}

// ---- norms and rotation -----------------------------------------------------------
int check_qk(const tdc_qk_args* a) {
  if (a == nullptr) return TDC_ERR_NULL_POINTER;
  if (a->dtype != TDC_F16 && a->dtype != TDC_BF16) return TDC_ERR_UNSUPPORTED;
  if (a->norm < TDC_NORM_NONE || a->norm > TDC_NORM_L2) return TDC_ERR_UNSUPPORTED;
  if (a->B < 0 || a->T < 0 || a->Hq < 0 || a->Hk < 0) return TDC_ERR_BAD_SHAPE;
  if (a->Hq > 65535 || a->Hk > 65535 || a->B > kMaxDim || a->T > kMaxDim) return TDC_ERR_TOO_LARGE;
  if (a->T > 0 && a->B > ((int64_t(1) << 31) - 1) / a->T) return TDC_ERR_TOO_LARGE;
  if (a->D < 8 || a->D > 256 || a->D % 8 != 0) return TDC_ERR_CHANNELS;
  if (a->R < 0 || a->R > a->D || a->R % 16 != 0) return TDC_ERR_BAD_SHAPE;
  if (a->R > 0) {
    if (a->cos == nullptr || a->sin == nullptr) return TDC_ERR_NULL_POINTER;
    if (a->table_rows < 0) return TDC_ERR_BAD_SHAPE;
    if (misaligned(a->cos) || misaligned(a->sin)) return TDC_ERR_ALIGNMENT;
  }
  if (!(a->eps >= 0)) return TDC_ERR_BAD_SHAPE;
  for (int64_t s : {a->q_sb, a->q_st, a->q_sh, a->k_sb, a->k_st, a->k_sh})
    if (bad_stride(s)) return TDC_ERR_ALIGNMENT;
  if ((a->Hq > 0 && misaligned(a->q)) || (a->Hk > 0 && misaligned(a->k)) ||
      misaligned(a->q_weight) || misaligned(a->k_weight))
    return TDC_ERR_ALIGNMENT;
  return TDC_OK;
}

tdc::QkParams qk_params(const tdc_qk_args* a) {
  tdc::QkParams p;
  std::memset(&p, 0, sizeof p);
  p.q = a->q, p.k = a->k, p.qw = a->q_weight, p.kw = a->k_weight;
  p.cos = a->cos, p.sin = a->sin, p.pos = a->positions;
  p.qo = a->q_out, p.ko = a->k_out;
  p.T = a->T;
  p.Hq = int(a->Hq), p.Hk = int(a->Hk), p.D = int(a->D), p.R = int(a->R);
  p.q_sb = a->q_sb, p.q_st = a->q_st, p.q_sh = a->q_sh;
  p.k_sb = a->k_sb, p.k_st = a->k_st, p.k_sh = a->k_sh;
  p.p_sb = a->p_sb, p.p_st = a->p_st;
  p.table_rows = a->table_rows;
  p.rows = a->B * a->T;
  p.pos64 = a->positions_are_64 != 0;
  p.interleaved = a->interleaved != 0;
  p.norm = a->norm != TDC_NORM_NONE;
  p.mul = a->norm == TDC_NORM_RMS ? 1.f / float(a->D) : 1.f;
  p.eps = float(a->eps);
  return p;
}

int qk_lanes(int64_t D) { return D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32; }

// Threads of a block: its groups take `heads` heads each, so that what a block
// does once (places, the angle) is spread over several.
int qk_threads(const tdc_qk_args* a, int64_t heads) {
  const int64_t want = ceil_div(a->Hq + a->Hk, heads) * qk_lanes(a->D);
  return int(std::min<int64_t>(256, std::max<int64_t>(1, ceil_div(want, 32)) * 32));
}

// Blocks of the gradient kernel: 4 on each of 148 SMs, or one for each row.
int64_t qk_bwd_rows(const tdc_qk_args* a) {
  return std::max<int64_t>(1, ceil_div(a->B * a->T, 148 * 4));
}
int64_t qk_bwd_blocks(const tdc_qk_args* a) { return ceil_div(a->B * a->T, qk_bwd_rows(a)); }

template <class E, int LANES>
int qk_fwd_l(const tdc::QkParams& p, int threads, cudaStream_t st) {
  auto* k = p.R == 0        ? &tdc::qk_norm_rope_kernel<E, LANES, 4, tdc::kNoTurn>
            : p.interleaved ? &tdc::qk_norm_rope_kernel<E, LANES, 4, tdc::kPairs>
                            : &tdc::qk_norm_rope_kernel<E, LANES, 4, tdc::kHalves>;
  k<<<unsigned(p.rows), threads, 0, st>>>(p);
  return launched();
}

template <class E, int LANES>
int qk_bwd_l(const tdc::QkParams& p, int threads, int64_t blocks, cudaStream_t st) {
  auto* k = p.R == 0        ? &tdc::qk_norm_rope_bwd_kernel<E, LANES, 3, tdc::kNoTurn>
            : p.interleaved ? &tdc::qk_norm_rope_bwd_kernel<E, LANES, 3, tdc::kPairs>
                            : &tdc::qk_norm_rope_bwd_kernel<E, LANES, 3, tdc::kHalves>;
  k<<<unsigned(blocks), threads, 0, st>>>(p);
  return launched();
}

template <class E>
int qk_fwd_e(const tdc::QkParams& p, int threads, cudaStream_t st) {
  switch (qk_lanes(p.D)) {
    case 4: return qk_fwd_l<E, 4>(p, threads, st);
    case 8: return qk_fwd_l<E, 8>(p, threads, st);
    case 16: return qk_fwd_l<E, 16>(p, threads, st);
    default: return qk_fwd_l<E, 32>(p, threads, st);
  }
}

template <class E>
int qk_bwd_e(const tdc::QkParams& p, int threads, int64_t blocks, void* dqw, void* dkw,
             cudaStream_t st) {
  int rc;
  switch (qk_lanes(p.D)) {
    case 4: rc = qk_bwd_l<E, 4>(p, threads, blocks, st); break;
    case 8: rc = qk_bwd_l<E, 8>(p, threads, blocks, st); break;
    case 16: rc = qk_bwd_l<E, 16>(p, threads, blocks, st); break;
    default: rc = qk_bwd_l<E, 32>(p, threads, blocks, st); break;
  }
  if (rc != TDC_OK || p.partial == nullptr) return rc;
  tdc::qk_wsum_kernel<E><<<unsigned(ceil_div(2 * p.D, 8)), 256, 0, st>>>(p.partial, blocks, p.D, dqw,
                                                                         dkw);
  return launched();
}

// ---- gated delta rule -------------------------------------------------------------
int64_t delta_seqs(const tdc_delta_args* a) { return a->cu_seqlens != nullptr ? a->num_seqs : a->B; }
int64_t delta_chunks(const tdc_delta_args* a) {
  return a->cu_seqlens != nullptr ? a->T / tdc::kChunk + a->num_seqs
                                  : a->B * ceil_div(a->T, tdc::kChunk);
}

int check_delta(const tdc_delta_args* a) {
  if (a == nullptr) return TDC_ERR_NULL_POINTER;
  if (a->dtype != TDC_F16 && a->dtype != TDC_BF16) return TDC_ERR_UNSUPPORTED;
  if (a->B < 0 || a->T < 0 || a->H < 1 || a->HV < 1 || a->HV % a->H != 0) return TDC_ERR_BAD_SHAPE;
  if (a->K != 64 && a->K != 128) return TDC_ERR_CHANNELS;
  if (a->V != 64 && a->V != 128 && a->V != 256) return TDC_ERR_CHANNELS;
  if (a->HV > 65535 || a->B > (int64_t(1) << 24) || a->T > (int64_t(1) << 36))
    return TDC_ERR_TOO_LARGE;
  if (a->cu_seqlens != nullptr && (a->B != 1 || a->num_seqs < 1)) return TDC_ERR_BAD_SHAPE;
  if (a->num_seqs > (int64_t(1) << 24)) return TDC_ERR_TOO_LARGE;
  // The workspace's size, at most 2.6 KB a value channel of a chunk, fits 64 bits.
  if (exceeds(delta_chunks(a), a->HV * a->V, kMaxSize)) return TDC_ERR_TOO_LARGE;
  for (int64_t s : {a->q_sb, a->q_st, a->q_sh, a->k_sb, a->k_st, a->k_sh, a->v_sb, a->v_st, a->v_sh})
    if (bad_stride(s)) return TDC_ERR_ALIGNMENT;
  // rows of v and o are addressed by 32-bit byte strides in a chunk
  if (a->v_st < 0 || a->v_st >= kMaxRow || a->HV * a->V >= kMaxRow) return TDC_ERR_TOO_LARGE;
  if (misaligned(a->q) || misaligned(a->k) || misaligned(a->v)) return TDC_ERR_ALIGNMENT;
  return TDC_OK;
}

int delta_wait_record(tdc::DeltaParams* p) {
  tdc::host::WaitRecord r;
  const int rc = tdc::host::wait_record(&r);
  if (rc != TDC_OK) return rc;
  p->timeout_ns = r.timeout_ns;
  p->status_words = r.words;
  p->status_host = r.host;
  return TDC_OK;
}

// Segments that the forward walks side by side (1: none): as many as give every
// block of both passes an SM of its own, if two passes over a segment and what joins
// them are shorter than one over the whole.  In chunks' times the second launch and
// the join's start are 3, and each product of the join 5/3 with K = 128, 1/2 with K = 64.
// Packed batches' lengths are not known here: they are walked whole.
// Whole and split calls, us (bf16, K = V = 128, one sequence): 4 heads, 13 chunks whole 67,
// 10 segments 104; 16 chunks 79 and 68; 40 chunks 177 and 104 (13 segments 129).
// 32 heads, 16 chunks 86; 20 chunks 115 and 107; 40 chunks 212 and 181.  Two sequences of
// 4 heads of 64 (fp16), 10 chunks 47 and 38; 40 chunks 153 and 68.
int delta_segments(const tdc_delta_args* a) {
  if (a->cu_seqlens != nullptr) return 1;
  const int64_t chunks = ceil_div(a->T, tdc::kChunk), heads = a->B * a->HV;
  const int64_t walks = heads * ceil_div(a->V, 128);
  const int64_t product = a->K == 128 ? 10 : 3;
  int best = 1;
  int64_t cost = 6 * chunks;
  for (int p = 3; p <= 16; ++p) {
    if (walks + (p - 2) * (walks + heads) > kSms || walks * (p - 1) > kSms) break;
    const int64_t c = 6 * (2 * ceil_div(chunks, p) + 3) + (p - 2) * product;
    if (c < cost) best = p, cost = c;
  }
  return best;
}

// Lays the workspace out (base may be null: only the size is wanted).
int64_t delta_layout(const tdc_delta_args* a, bool grads, unsigned char* base, tdc::DeltaParams* p) {
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    unsigned char* r = base + at;
    at += ceil_div(bytes, 256) * 256;
    return r;
  };
  const int64_t slots = delta_chunks(a) * a->HV;
  unsigned char* plan = take(2 * (delta_seqs(a) + 1) * 8);
  unsigned char* tp = take(slots * 6 * tdc::kSq * 2);
  const int64_t parts = a->dtype == TDC_BF16 ? 1 : 2;
  unsigned char* kq = take(delta_chunks(a) * a->H * 2 * parts * tdc::kChunk * a->K * 2);
  unsigned char* coef = take(slots * tdc::kCoef * 4);
  unsigned char* tiles = nullptr;
  unsigned char *seg_s = nullptr, *seg_m = nullptr;
  const int segments = grads ? 1 : delta_segments(a);
  if (segments > 1) {
    seg_s = take(a->B * a->HV * segments * a->K * a->V * 4);
    seg_m = take(a->B * a->HV * segments * a->K * a->K * 4);
  }
  if (grads) {
    // (GradTile: S, dS, U and dX in three parts, dO in `parts`)
    tiles = take(slots * a->V * 2 * (6 * a->K + (6 + parts) * tdc::kChunk));
  }
  if (p != nullptr) {
    p->seq_lo = reinterpret_cast<int64_t*>(plan);
    p->seq_chunk = p->seq_lo + delta_seqs(a) + 1;
    p->tp = reinterpret_cast<__nv_bfloat16*>(tp);
    p->kq = kq;
    p->segments = segments;
    p->segment_chunks = int(ceil_div(ceil_div(a->T, tdc::kChunk), segments));
    p->seg_s = reinterpret_cast<float*>(seg_s);
    p->seg_m = reinterpret_cast<float*>(seg_m);
    p->coef = reinterpret_cast<float*>(coef);
    p->tiles = tiles;
  }
  return at;
}

tdc::DeltaParams delta_params(const tdc_delta_args* a) {
  tdc::DeltaParams p;
  std::memset(&p, 0, sizeof p);
  p.q = a->q, p.k = a->k, p.v = a->v, p.beta = a->beta, p.g = a->g;
  p.init = a->initial_state, p.final_state = a->final_state, p.o = a->o;
  p.T = a->T;
  p.H = int(a->H), p.HV = int(a->HV), p.V = int(a->V), p.group = int(a->HV / a->H);
  p.q_sb = a->q_sb, p.q_st = a->q_st, p.q_sh = a->q_sh;
  p.k_sb = a->k_sb, p.k_st = a->k_st, p.k_sh = a->k_sh;
  p.v_sb = a->v_sb, p.v_st = a->v_st, p.v_sh = a->v_sh;
  p.g_sb = a->g_sb, p.g_st = a->g_st, p.b_sb = a->b_sb, p.b_st = a->b_st;
  p.seq.cu = a->cu_seqlens;
  p.seq.n = delta_seqs(a);
  p.seq.T = a->T;
  p.seq.is64 = a->cu_is_64 != 0;
  p.chunks_per_b = ceil_div(a->T, tdc::kChunk);
  p.max_chunks = delta_chunks(a);
  p.beta_f32 = a->beta_is_f32 != 0;
  p.scale = float(a->scale);
  p.withhold = -1;
  return p;
}

int delta_plan(const tdc::DeltaParams& p, const tdc::ZeroRows& z, cudaStream_t st) {
  if (p.seq.cu == nullptr) return TDC_OK;
  tdc::delta_plan_kernel<<<33, 1024, 0, st>>>(p.seq, p.seq_lo, p.seq_chunk, z);
  return launched();
}

template <class E, int DK>
int delta_prepare(const tdc::DeltaParams& p, cudaStream_t st) {
  if (p.max_chunks == 0) return TDC_OK;
  auto* k = &tdc::delta_prepare_kernel<E, DK>;
  const size_t smem = tdc::PrepareSmem<DK>::bytes;
  const int rc = allow_smem(k, smem);
  if (rc != TDC_OK) return rc;
  k<<<dim3(unsigned(p.max_chunks), unsigned(p.H)), 128, smem, st>>>(p);
  return launched();
}

// `blocks` blocks for each head: 128 value channels of a sequence (or segment) each.
template <class E, int DK, class Kernel>
int delta_walk(Kernel* k, const tdc::DeltaParams& p, int64_t blocks, cudaStream_t st) {
  if (p.seq.n == 0) return TDC_OK;
  const size_t smem = 2 * tdc::WalkTiles<E, DK>::stage + sizeof(tdc::WalkSync);
  const int rc = allow_smem(k, smem);
  if (rc != TDC_OK) return rc;
  k<<<dim3(unsigned(blocks), unsigned(p.HV)), tdc::kWalkThreads, smem, st>>>(p);
  return launched();
}

template <class E, int DK>
int delta_fwd_t(tdc::DeltaParams& p, cudaStream_t st) {
  int rc = delta_prepare<E, DK>(p, st);
  if (rc != TDC_OK) return rc;
  auto* k = &tdc::delta_walk_kernel<E, DK, 0>;
  const int64_t tiles = ceil_div(p.V, 128);
  if (p.segments <= 1) return delta_walk<E, DK>(k, p, p.seq.n * tiles, st);
  const int64_t inner = p.segments - 2;
  p.pass = 1;
  rc = delta_walk<E, DK>(k, p, p.seq.n * (tiles * (1 + inner) + inner), st);
  if (rc != TDC_OK) return rc;
  const size_t smem = (2 * DK * DK + DK * 32) * sizeof(float);
  rc = allow_smem(&tdc::delta_join_kernel<DK>, smem);
  if (rc != TDC_OK) return rc;
  tdc::delta_join_kernel<DK>
      <<<dim3(unsigned(p.seq.n * p.HV), unsigned(p.V / 32)), 256, smem, st>>>(p);
  rc = launched();
  p.pass = 2;
  return rc != TDC_OK ? rc : delta_walk<E, DK>(k, p, p.seq.n * tiles * (p.segments - 1), st);
}

template <class E, int DK>
int delta_bwd_t(const tdc::DeltaParams& p, cudaStream_t st) {
  int rc = delta_prepare<E, DK>(p, st);
  const int64_t blocks = p.seq.n * ceil_div(p.V, 128);
  if (rc == TDC_OK) rc = delta_walk<E, DK>(&tdc::delta_walk_kernel<E, DK, 1>, p, blocks, st);
  if (rc == TDC_OK) rc = delta_walk<E, DK>(&tdc::delta_walk_back_kernel<E, DK>, p, blocks, st);
  if (rc != TDC_OK || p.max_chunks == 0) return rc;
  auto* k = &tdc::delta_grad_kernel<E, DK>;
  const size_t smem = tdc::GradSmem<E, DK>::sync + sizeof(tdc::GradSync);
  rc = allow_smem(k, smem);
  if (rc != TDC_OK) return rc;
  k<<<unsigned(std::min<int64_t>(kSms, p.max_chunks * p.H)), tdc::kWalkThreads, smem, st>>>(p);
  return launched();
}

template <class E, int DK>
int delta_step_t(const tdc::DeltaParams& p, int64_t B, float* state, int64_t slots, const void* idx,
                 bool idx64, cudaStream_t st) {
  tdc::delta_step_kernel<E, DK>
      <<<dim3(unsigned(B), unsigned(p.HV), unsigned(p.V / 32)), 128, 0, st>>>(p, state, idx, idx64,
                                                                             slots);
  return launched();
}

int delta_fwd(const tdc_delta_args* a, void* workspace, int64_t workspace_bytes, int64_t withhold,
              int64_t timeout_ns, void* stream) {
  int rc = check_delta(a);
  if (rc != TDC_OK) return rc;
  if (workspace == nullptr) return TDC_ERR_NULL_POINTER;
  if (workspace_bytes < tdc_delta_fwd_workspace(a)) return TDC_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return TDC_ERR_ALIGNMENT;
  if (a->B * a->T > 0 && (a->q == nullptr || a->k == nullptr || a->v == nullptr ||
                          a->g == nullptr || a->beta == nullptr || a->o == nullptr))
    return TDC_ERR_NULL_POINTER;
  if (misaligned(a->o) || misaligned(a->initial_state) || misaligned(a->final_state))
    return TDC_ERR_ALIGNMENT;
  rc = prepare_device();
  if (rc != TDC_OK) return rc;
  tdc::DeltaParams p = delta_params(a);
  delta_layout(a, false, static_cast<unsigned char*>(workspace), &p);
  if (p.max_chunks > 0x7fffffff) return TDC_ERR_TOO_LARGE;
  auto st = static_cast<cudaStream_t>(stream);
  tdc::ZeroRows z = {};
  z.base[0] = a->o, z.row_bytes[0] = a->HV * a->V * 2;
  rc = delta_wait_record(&p);
  p.withhold = withhold;
  if (timeout_ns > 0) p.timeout_ns = uint64_t(timeout_ns);
  if (rc == TDC_OK) rc = delta_plan(p, z, st);
  if (rc != TDC_OK) return rc;
  if (a->dtype == TDC_BF16)
    return a->K == 128 ? delta_fwd_t<tdc::BF16, 128>(p, st) : delta_fwd_t<tdc::BF16, 64>(p, st);
  return a->K == 128 ? delta_fwd_t<tdc::F16, 128>(p, st) : delta_fwd_t<tdc::F16, 64>(p, st);
}

}  // namespace

extern "C" {

TDC_API int tdc_conv1d_fwd(const tdc_conv1d_args* a, void* stream) {
  int rc = check_conv_args(a);
  if (rc != TDC_OK) return rc;
  tdc::Conv1dParams p = conv_params(a);
  const int64_t vecs = a->C / 8;
  const bool rows = a->B > 0 && a->T > 0;
  if (vecs == 0 || (!rows && (a->final_state == nullptr || p.seq.n == 0))) return TDC_OK;
  if ((rows && (a->x == nullptr || a->w == nullptr || a->y == nullptr))) return TDC_ERR_NULL_POINTER;
  if (misaligned(a->x) || misaligned(a->w) || misaligned(a->y) || misaligned(a->bias) ||
      misaligned(a->initial_state) || misaligned(a->final_state))
    return TDC_ERR_ALIGNMENT;
  // Runs that fill the SMs with one wave of blocks (2 of 256 threads on each), or
  // with several equal ones if they were longer than 128 rows.  Against the shortest
  // runs that give each SM 1024 threads (at most 32 rows), K = 4: 1500 rows of 2560
  // channels 14.1 -> 11.4 us a call, 5003 rows 20.5 -> 16.4 (then 15 with loads before the
  // sequences are looked up), 9000 rows of 8192 61.4 -> 57.8.
  const int64_t wave = 2 * kSms * 256, work = a->B * a->T * vecs;
  const int64_t waves = std::max<int64_t>(1, ceil_div(work, wave * 128));
  p.runs_per_b = ceil_div(a->T, std::max<int64_t>(1, ceil_div(work, wave * waves)));
  p.run = int(std::min<int64_t>(ceil_div(a->T, std::max<int64_t>(1, p.runs_per_b)), 1 << 30));
  p.main_threads = a->B * p.runs_per_b * vecs;
  const int64_t tail = a->final_state != nullptr ? p.seq.n * (a->K - 1) * vecs : 0;
  const int64_t blocks = ceil_div(p.main_threads + tail, 256);
  if (blocks > 0x7fffffff) return TDC_ERR_TOO_LARGE;
  rc = prepare_device();
  if (rc != TDC_OK) return rc;
  return conv_fwd_any(p, a->K, a->dtype, a->act == TDC_ACT_SILU, blocks,
                      static_cast<cudaStream_t>(stream));
}

TDC_API int64_t tdc_conv1d_bwd_workspace(const tdc_conv1d_args* a) {
  const int rc = check_conv_args(a);
  if (rc != TDC_OK) return rc;
  return std::max<int64_t>(16, conv_bwd_plan(a).groups * (a->K + 1) * a->C * 4);
}

TDC_API int tdc_conv1d_bwd(const tdc_conv1d_args* a, const void* dy, int64_t dy_sb, int64_t dy_st,
                           const void* dfinal, void* dx, void* dw, void* dbias, void* dinitial,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_conv_args(a);
  if (rc != TDC_OK) return rc;
  if (a->C == 0) return TDC_OK;
  if (a->w == nullptr || dw == nullptr || workspace == nullptr) return TDC_ERR_NULL_POINTER;
  if (a->B * a->T > 0 && (a->x == nullptr || dy == nullptr || dx == nullptr))
    return TDC_ERR_NULL_POINTER;
  if (a->bias != nullptr && dbias == nullptr) return TDC_ERR_NULL_POINTER;
  if (workspace_bytes < tdc_conv1d_bwd_workspace(a)) return TDC_ERR_WORKSPACE;
  if (bad_stride(dy_sb) || bad_stride(dy_st)) return TDC_ERR_ALIGNMENT;
  for (const void* q : {a->x, a->w, a->bias, a->initial_state, dy, dfinal,
                        static_cast<const void*>(dx), static_cast<const void*>(dinitial),
                        static_cast<const void*>(workspace)})
    if (misaligned(q)) return TDC_ERR_ALIGNMENT;
  const ConvBwdPlan pl = conv_bwd_plan(a);
  if (pl.groups > 0x7fffffff || pl.cblocks > 65535) return TDC_ERR_TOO_LARGE;
  tdc::Conv1dParams p = conv_params(a);
  p.run = pl.run;
  p.runs_per_b = pl.runs_per_b;
  if (a->T == 0) p.B = 0;  // no rows: only zero weight gradients and the states'
  p.dy = dy, p.dy_sb = dy_sb, p.dy_st = dy_st;
  p.dfinal = dfinal, p.dx = dx, p.dinit = dinitial;
  p.partial = static_cast<float*>(workspace);
  p.groups = pl.groups;
  rc = prepare_device();
  if (rc != TDC_OK) return rc;
  return conv_bwd_any(p, pl, a->K, a->dtype, a->act == TDC_ACT_SILU, dw,
                      a->bias != nullptr ? dbias : nullptr, static_cast<cudaStream_t>(stream));
}

TDC_API int tdc_conv1d_step(const tdc_conv1d_step_args* a, void* stream) {
  if (a == nullptr) return TDC_ERR_NULL_POINTER;
  int rc = check_conv(a->B, a->T, a->C, a->K, a->dtype, a->act, a->x_sb, a->x_st);
  if (rc != TDC_OK) return rc;
  if (a->slots < 0) return TDC_ERR_BAD_SHAPE;
  if (a->B == 0 || a->T == 0 || a->C == 0) return TDC_OK;
  if (a->B > 0x7fffffff || a->C > 65535 * 256) return TDC_ERR_TOO_LARGE;
  if (a->x == nullptr || a->w == nullptr || a->y == nullptr ||
      (a->state == nullptr && a->slots > 0))
    return TDC_ERR_NULL_POINTER;
  for (const void* q : {a->x, a->w, a->bias, static_cast<const void*>(a->state),
                        static_cast<const void*>(a->y)})
    if (misaligned(q)) return TDC_ERR_ALIGNMENT;
  tdc::Conv1dParams p;
  std::memset(&p, 0, sizeof p);
  p.x = a->x, p.w = a->w, p.bias = a->bias, p.y = a->y;
  p.B = a->B, p.T = a->T, p.C = a->C, p.x_sb = a->x_sb, p.x_st = a->x_st;
  p.state = a->state, p.idx = a->state_indices, p.slots = a->slots;
  p.idx64 = a->indices_are_64 != 0;
  rc = prepare_device();
  if (rc != TDC_OK) return rc;
  return conv_step_any(p, a->K, a->dtype, a->act == TDC_ACT_SILU, static_cast<cudaStream_t>(stream));
}

TDC_API int tdc_qk_norm_rope(const tdc_qk_args* a, void* stream) {
  int rc = check_qk(a);
  if (rc != TDC_OK) return rc;
  if (a->B * a->T == 0 || a->Hq + a->Hk == 0) return TDC_OK;
  if ((a->Hq > 0 && (a->q == nullptr || a->q_out == nullptr)) ||
      (a->Hk > 0 && (a->k == nullptr || a->k_out == nullptr)))
    return TDC_ERR_NULL_POINTER;
  if (misaligned(a->q_out) || misaligned(a->k_out)) return TDC_ERR_ALIGNMENT;
  rc = prepare_device();
  if (rc != TDC_OK) return rc;
  const tdc::QkParams p = qk_params(a);
  auto st = static_cast<cudaStream_t>(stream);
  return a->dtype == TDC_BF16 ? qk_fwd_e<tdc::BF16>(p, qk_threads(a, 4), st)
                              : qk_fwd_e<tdc::F16>(p, qk_threads(a, 4), st);
}

TDC_API int64_t tdc_qk_norm_rope_bwd_workspace(const tdc_qk_args* a) {
  const int rc = check_qk(a);
  if (rc != TDC_OK) return rc;
  return std::max<int64_t>(16, qk_bwd_blocks(a) * 2 * a->D * 4);
}

TDC_API int tdc_qk_norm_rope_bwd(const tdc_qk_args* a, const tdc_qk_grad_args* g, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  int rc = check_qk(a);
  if (rc != TDC_OK) return rc;
  if (g == nullptr) return TDC_ERR_NULL_POINTER;
  const bool weights = a->q_weight != nullptr || a->k_weight != nullptr;
  if ((a->q_weight != nullptr && g->dq_weight == nullptr) ||
      (a->k_weight != nullptr && g->dk_weight == nullptr))
    return TDC_ERR_NULL_POINTER;
  if (weights && workspace == nullptr) return TDC_ERR_NULL_POINTER;
  if (weights && workspace_bytes < tdc_qk_norm_rope_bwd_workspace(a)) return TDC_ERR_WORKSPACE;
  const bool rows = a->B * a->T > 0 && a->Hq + a->Hk > 0;
  if (!rows && !weights) return TDC_OK;
  if (rows && ((a->Hq > 0 && (a->q == nullptr || g->dq == nullptr || g->dq_out == nullptr)) ||
               (a->Hk > 0 && (a->k == nullptr || g->dk == nullptr || g->dk_out == nullptr))))
    return TDC_ERR_NULL_POINTER;
  for (int64_t s : {g->gq_sb, g->gq_st, g->gq_sh, g->gk_sb, g->gk_st, g->gk_sh})
    if (bad_stride(s)) return TDC_ERR_ALIGNMENT;
  for (const void* q : {g->dq_out, g->dk_out, static_cast<const void*>(g->dq),
                        static_cast<const void*>(g->dk)})
    if (misaligned(q)) return TDC_ERR_ALIGNMENT;
  rc = prepare_device();
  if (rc != TDC_OK) return rc;
  tdc::QkParams p = qk_params(a);
  p.gq = g->dq_out, p.gk = g->dk_out, p.dq = g->dq, p.dk = g->dk;
  p.gq_sb = g->gq_sb, p.gq_st = g->gq_st, p.gq_sh = g->gq_sh;
  p.gk_sb = g->gk_sb, p.gk_st = g->gk_st, p.gk_sh = g->gk_sh;
  p.partial = weights ? static_cast<float*>(workspace) : nullptr;
  p.rows_per_block = int(std::min<int64_t>(qk_bwd_rows(a), 0x7fffffff));
  auto st = static_cast<cudaStream_t>(stream);
  const int64_t blocks = std::max<int64_t>(1, qk_bwd_blocks(a));  // no rows: zero weight gradients
  return a->dtype == TDC_BF16
             ? qk_bwd_e<tdc::BF16>(p, qk_threads(a, 1), blocks, g->dq_weight, g->dk_weight, st)
             : qk_bwd_e<tdc::F16>(p, qk_threads(a, 1), blocks, g->dq_weight, g->dk_weight, st);
}

TDC_API int64_t tdc_delta_fwd_workspace(const tdc_delta_args* a) {
  const int rc = check_delta(a);
  return rc != TDC_OK ? rc : delta_layout(a, false, nullptr, nullptr);
}

TDC_API int64_t tdc_delta_bwd_workspace(const tdc_delta_args* a) {
  const int rc = check_delta(a);
  return rc != TDC_OK ? rc : delta_layout(a, true, nullptr, nullptr);
}

TDC_API int tdc_delta_fwd(const tdc_delta_args* a, void* workspace, int64_t workspace_bytes,
                          void* stream) {
  return delta_fwd(a, workspace, workspace_bytes, -1, 0, stream);
}

TDC_API int tdc_delta_fwd_withhold(const tdc_delta_args* a, void* workspace,
                                   int64_t workspace_bytes, int64_t withhold_chunk,
                                   int64_t timeout_ns, void* stream) {
  if (withhold_chunk < 0 || timeout_ns <= 0) return TDC_ERR_BAD_SHAPE;
  return delta_fwd(a, workspace, workspace_bytes, withhold_chunk, timeout_ns, stream);
}

TDC_API int tdc_delta_bwd(const tdc_delta_args* a, const tdc_delta_grad_args* g, void* workspace,
                          int64_t workspace_bytes, void* stream) {
  int rc = check_delta(a);
  if (rc != TDC_OK) return rc;
  if (g == nullptr || workspace == nullptr) return TDC_ERR_NULL_POINTER;
  if (workspace_bytes < tdc_delta_bwd_workspace(a)) return TDC_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return TDC_ERR_ALIGNMENT;
  if (a->B * a->T > 0 &&
      (a->q == nullptr || a->k == nullptr || a->v == nullptr || a->g == nullptr ||
       a->beta == nullptr || g->d_o == nullptr || g->dq == nullptr || g->dk == nullptr ||
       g->dv == nullptr || g->dg == nullptr || g->dbeta == nullptr))
    return TDC_ERR_NULL_POINTER;
  for (int64_t s : {g->do_sb, g->do_st, g->do_sh})
    if (bad_stride(s)) return TDC_ERR_ALIGNMENT;
  if (g->do_st < 0 || g->do_st >= kMaxRow) return TDC_ERR_TOO_LARGE;
  for (const void* q : {g->d_o, static_cast<const void*>(g->dq), static_cast<const void*>(g->dk),
                        static_cast<const void*>(g->dv)})
    if (misaligned(q)) return TDC_ERR_ALIGNMENT;
  rc = prepare_device();
  if (rc != TDC_OK) return rc;
  tdc::DeltaParams p = delta_params(a);
  delta_layout(a, true, static_cast<unsigned char*>(workspace), &p);
  if (p.max_chunks > 0x7fffffff) return TDC_ERR_TOO_LARGE;
  p.d_o = g->d_o;
  p.do_sb = g->do_sb, p.do_st = g->do_st, p.do_sh = g->do_sh;
  p.dfinal = g->dfinal, p.dq = g->dq, p.dk = g->dk, p.dv = g->dv;
  p.dg = g->dg, p.dbeta = g->dbeta, p.dinit = g->dinitial;
  auto st = static_cast<cudaStream_t>(stream);
  tdc::ZeroRows z = {};
  z.base[0] = g->dq, z.row_bytes[0] = a->H * a->K * 2;
  z.base[1] = g->dk, z.row_bytes[1] = a->H * a->K * 2;
  z.base[2] = g->dv, z.row_bytes[2] = a->HV * a->V * 2;
  z.base[3] = g->dg, z.row_bytes[3] = a->HV * 4;
  z.base[4] = g->dbeta, z.row_bytes[4] = a->HV * (a->beta_is_f32 ? 4 : 2);
  rc = delta_wait_record(&p);
  if (rc == TDC_OK) rc = delta_plan(p, z, st);
  if (rc != TDC_OK) return rc;
  if (a->dtype == TDC_BF16)
    return a->K == 128 ? delta_bwd_t<tdc::BF16, 128>(p, st) : delta_bwd_t<tdc::BF16, 64>(p, st);
  return a->K == 128 ? delta_bwd_t<tdc::F16, 128>(p, st) : delta_bwd_t<tdc::F16, 64>(p, st);
}

TDC_API int tdc_delta_step(const tdc_delta_args* a, float* state, int64_t slots,
                           const void* state_indices, int64_t indices_are_64, void* stream) {
  int rc = check_delta(a);
  if (rc != TDC_OK) return rc;
  if (slots < 0) return TDC_ERR_BAD_SHAPE;
  if (a->B == 0 || a->T == 0) return TDC_OK;
  if (a->q == nullptr || a->k == nullptr || a->v == nullptr || a->g == nullptr ||
      a->beta == nullptr || a->o == nullptr || (state == nullptr && slots > 0))
    return TDC_ERR_NULL_POINTER;
  if (misaligned(a->o) || misaligned(state)) return TDC_ERR_ALIGNMENT;
  rc = prepare_device();
  if (rc != TDC_OK) return rc;
  tdc::DeltaParams p = delta_params(a);
  auto st = static_cast<cudaStream_t>(stream);
  const bool i64 = indices_are_64 != 0;
  if (a->dtype == TDC_BF16)
    return a->K == 128 ? delta_step_t<tdc::BF16, 128>(p, a->B, state, slots, state_indices, i64, st)
                       : delta_step_t<tdc::BF16, 64>(p, a->B, state, slots, state_indices, i64, st);
  return a->K == 128 ? delta_step_t<tdc::F16, 128>(p, a->B, state, slots, state_indices, i64, st)
                     : delta_step_t<tdc::F16, 64>(p, a->B, state, slots, state_indices, i64, st);
}

}  // extern "C"
