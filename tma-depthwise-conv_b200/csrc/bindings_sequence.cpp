// bindings_sequence.cpp — the sequence operators of the `_tma_dwconv_C`
// extension: tensors in, tensors out, on torch's current stream of their
// device, through the C ABI of include/tdc_sequence.h.  Argument errors raise
// RuntimeError (TORCH_CHECK); outputs and workspaces come from torch's caching
// allocator, so calls can be captured into CUDA graphs.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <optional>
#include <tuple>

#include "bindings_common.h"
#include "tdc_sequence.h"

namespace tma_dwconv {
namespace {

using OptTensor = std::optional<torch::Tensor>;

int64_t dtype_of(const torch::Tensor& x, const char* name) {
  TORCH_CHECK(x.scalar_type() == torch::kHalf || x.scalar_type() == torch::kBFloat16, name,
              " must be fp16 or bf16");
  return x.scalar_type() == torch::kBFloat16 ? TDC_BF16 : TDC_F16;
}

// The other checks come first, so that they hold on any host.
c10::Device cuda_device(const torch::Tensor& x) {
  TORCH_CHECK(x.is_cuda(), "the tensors must be CUDA tensors");
  return x.device();
}

void check_like(const torch::Tensor& t, const torch::Tensor& x, const char* name, const char* xname) {
  TORCH_CHECK(t.device() == x.device(), name, " and ", xname, " must be on the same device");
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), name, " must have ", xname, "'s dtype");
}

void check_f32(const torch::Tensor& t, const torch::Tensor& x, const char* name) {
  TORCH_CHECK(t.device() == x.device(), name, " must be on the inputs' device");
  TORCH_CHECK(t.scalar_type() == torch::kFloat, name, " must be fp32");
}

bool is_index64(const torch::Tensor& t, const torch::Tensor& x, const char* name) {
  TORCH_CHECK(t.device() == x.device(), name, " must be on the inputs' device");
  TORCH_CHECK(t.scalar_type() == torch::kInt || t.scalar_type() == torch::kLong, name,
              " must be int32 or int64");
  return t.scalar_type() == torch::kLong;
}

// A tensor that the vectorised kernels read in place: last dimension
// contiguous, the other strides multiples of 8 elements (a stride of a
// dimension of one entry does not matter), the base 16-byte aligned.
// Anything else is copied.
torch::Tensor in_place(const torch::Tensor& t) {
  bool ok = (t.stride(-1) == 1 || t.size(-1) <= 1) &&
            reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t i = 0; ok && i + 1 < t.dim(); ++i) ok = t.size(i) <= 1 || t.stride(i) % 8 == 0;
  return ok || t.numel() == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}

torch::Tensor aligned(const torch::Tensor& t) {
  auto c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c
                                                             : c.clone(at::MemoryFormat::Contiguous);
}

// (strides without an element do not matter either)
int64_t stride_of(const torch::Tensor& t, int64_t dim) {
  return t.size(dim) <= 1 || t.numel() == 0 ? 0 : t.stride(dim);
}

const void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }

torch::Tensor bytes_on(const torch::Tensor& x, int64_t n) {
  return torch::empty({n}, torch::TensorOptions().dtype(torch::kByte).device(x.device()));
}

// `t` was written in place: a tensor that a backward pass saved before raises there, as
// after any in-place operation of torch (inference tensors have no versions).
void written(const torch::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void check_cu(const OptTensor& cu, const torch::Tensor& x) {
  if (!cu) return;
  is_index64(*cu, x, "cu_seqlens");
  TORCH_CHECK(cu->dim() == 1 && cu->size(0) >= 2 && cu->is_contiguous(),
              "cu_seqlens must be a contiguous vector of at least 2 offsets");
  TORCH_CHECK(x.size(0) == 1, "a packed batch (cu_seqlens) has a batch dimension of 1");
}

void check_state_indices(const OptTensor& idx, const torch::Tensor& x, int64_t batch) {
  if (!idx) return;
  is_index64(*idx, x, "state_indices");
  TORCH_CHECK(idx->dim() == 1 && idx->size(0) == batch && idx->is_contiguous(),
              "state_indices must be a contiguous vector with one slot for each request");
}

// ---- causal depthwise convolution ---------------------------------------------
struct ConvCall {
  tdc_conv1d_args a{};
  torch::Tensor x, w, bias, init, cu;  // kept alive over the call
  int64_t seqs = 0;
};

ConvCall conv_call(const torch::Tensor& x, const torch::Tensor& w, const OptTensor& bias,
                   const OptTensor& init, const OptTensor& cu, int64_t act) {
  ConvCall c;
  c.a.dtype = dtype_of(x, "x");
  TORCH_CHECK(x.dim() == 3, "x must be [B,T,C]");
  TORCH_CHECK(w.dim() == 2, "w must be [K,C]");
  check_like(w, x, "w", "x");
  const int64_t B = x.size(0), T = x.size(1), C = x.size(2), K = w.size(0);
  TORCH_CHECK(w.size(1) == C, "w and x must agree on C");
  TORCH_CHECK(C % 8 == 0, "C must be a multiple of 8");
  TORCH_CHECK(K >= 2 && K <= 8, "K must be 2 to 8, got ", K);
  check_cu(cu, x);
  c.seqs = cu ? cu->size(0) - 1 : B;
  c.x = in_place(x);
  c.w = aligned(w);
  if (bias) {
    check_like(*bias, x, "bias", "x");
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == C, "bias must be [C]");
    c.bias = aligned(*bias);
    c.a.bias = c.bias.data_ptr();
  }
  if (init) {
    check_like(*init, x, "initial_state", "x");
    TORCH_CHECK(init->dim() == 3 && init->size(0) == c.seqs && init->size(1) == K - 1 &&
                    init->size(2) == C,
                "initial_state must be [sequences, K-1, C]");
    c.init = aligned(*init);
    c.a.initial_state = c.init.data_ptr();
  }
  if (cu) {
    c.cu = *cu;
    c.a.cu_seqlens = cu->data_ptr();
    c.a.num_seqs = c.seqs;
    c.a.cu_is_64 = cu->scalar_type() == torch::kLong;
  }
  c.a.x = c.x.data_ptr();
  c.a.w = c.w.data_ptr();
  c.a.B = B, c.a.T = T, c.a.C = C, c.a.K = K;
  c.a.x_sb = stride_of(c.x, 0), c.a.x_st = stride_of(c.x, 1);
  c.a.act = act;
  return c;
}

std::tuple<torch::Tensor, OptTensor> causal_conv1d(torch::Tensor x, torch::Tensor w, OptTensor bias,
                                                   OptTensor init, OptTensor cu, int64_t act,
                                                   bool want_final) {
  auto c = conv_call(x, w, bias, init, cu, act);
  const c10::cuda::CUDAGuard guard(cuda_device(x));
  auto y = torch::empty({c.a.B, c.a.T, c.a.C}, x.options());
  OptTensor fin;
  if (want_final) {
    fin = torch::empty({c.seqs, c.a.K - 1, c.a.C}, x.options());
    c.a.final_state = fin->data_ptr();
  }
  c.a.y = y.data_ptr();
  check_status(tdc_conv1d_fwd(&c.a, stream_of(x)), "causal_conv1d");
  return {y, fin};
}

// (dx, dw, dbias or None, dinitial or None)
std::tuple<torch::Tensor, torch::Tensor, OptTensor, OptTensor> causal_conv1d_bwd(
    torch::Tensor x, torch::Tensor w, OptTensor bias, OptTensor init, OptTensor cu, int64_t act,
    torch::Tensor dy, OptTensor dfinal) {
  auto c = conv_call(x, w, bias, init, cu, act);
  check_like(dy, x, "dy", "x");
  TORCH_CHECK(dy.sizes() == x.sizes(), "dy must have x's shape");
  auto d = in_place(dy);
  torch::Tensor df;
  if (dfinal) {
    check_like(*dfinal, x, "dfinal", "x");
    TORCH_CHECK(dfinal->dim() == 3 && dfinal->size(0) == c.seqs && dfinal->size(1) == c.a.K - 1 &&
                    dfinal->size(2) == c.a.C,
                "dfinal must be [sequences, K-1, C]");
    df = aligned(*dfinal);
  }
  const c10::cuda::CUDAGuard guard(cuda_device(x));
  auto dx = torch::empty({c.a.B, c.a.T, c.a.C}, x.options());
  auto dw = torch::empty({c.a.K, c.a.C}, x.options());
  OptTensor db, di;
  if (bias) db = torch::empty({c.a.C}, x.options());
  if (init) di = torch::empty({c.seqs, c.a.K - 1, c.a.C}, x.options());
  const int64_t need = tdc_conv1d_bwd_workspace(&c.a);
  if (need < 0) check_status(int(need), "causal_conv1d_bwd");
  auto ws = bytes_on(x, need);
  check_status(tdc_conv1d_bwd(&c.a, d.data_ptr(), stride_of(d, 0), stride_of(d, 1),
                              dfinal ? df.data_ptr() : nullptr, dx.data_ptr(), dw.data_ptr(),
                              db ? db->data_ptr() : nullptr, di ? di->data_ptr() : nullptr,
                              ws.data_ptr(), need, stream_of(x)),
               "causal_conv1d_bwd");
  return {dx, dw, db, di};
}

torch::Tensor causal_conv1d_step(torch::Tensor x, torch::Tensor w, OptTensor bias,
                                 torch::Tensor state, OptTensor idx, int64_t act) {
  TORCH_CHECK(x.dim() == 3, "x must be [B,T,C]");
  auto c = conv_call(x, w, bias, std::nullopt, std::nullopt, act);
  check_like(state, x, "state", "x");
  TORCH_CHECK(state.dim() == 3 && state.size(1) == c.a.K - 1 && state.size(2) == c.a.C,
              "state must be [slots, K-1, C]");
  TORCH_CHECK(state.is_contiguous(), "state must be contiguous (it is updated in place)");
  check_state_indices(idx, x, c.a.B);
  TORCH_CHECK(idx || state.size(0) >= c.a.B, "state has fewer slots than there are requests");
  const c10::cuda::CUDAGuard guard(cuda_device(state));
  auto y = torch::empty({c.a.B, c.a.T, c.a.C}, x.options());
  tdc_conv1d_step_args s{};
  s.x = c.a.x, s.w = c.a.w, s.bias = c.a.bias;
  s.state = state.data_ptr();
  s.state_indices = ptr(idx);
  s.y = y.data_ptr();
  s.B = c.a.B, s.T = c.a.T, s.C = c.a.C, s.K = c.a.K;
  s.x_sb = c.a.x_sb, s.x_st = c.a.x_st;
  s.slots = state.size(0);
  s.indices_are_64 = idx && idx->scalar_type() == torch::kLong;
  s.dtype = c.a.dtype, s.act = act;
  check_status(tdc_conv1d_step(&s, stream_of(x)), "causal_conv1d_step");
  written(state);
  return y;
}

// ---- norms and rotation -----------------------------------------------------------
struct QkCall {
  tdc_qk_args a{};
  torch::Tensor q, k, qw, kw, cos, sin, pos;
};

QkCall qk_call(const torch::Tensor& q, const torch::Tensor& k, const OptTensor& qw,
               const OptTensor& kw, const OptTensor& cos, const OptTensor& sin,
               const OptTensor& pos, int64_t norm, double eps, bool interleaved) {
  QkCall c;
  c.a.dtype = dtype_of(q, "q");
  check_like(k, q, "k", "q");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4, "q and k must be [B,T,H,D]");
  TORCH_CHECK(q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3),
              "q and k must agree on B, T and D");
  const int64_t D = q.size(3);
  TORCH_CHECK(D >= 8 && D <= 256 && D % 8 == 0, "D must be a multiple of 8 from 8 to 256, got ", D);
  TORCH_CHECK(cos.has_value() == sin.has_value(), "cos and sin come together");
  TORCH_CHECK(!pos || cos, "positions need cos and sin");
  c.q = in_place(q);
  c.k = in_place(k);
  auto weight = [&](const OptTensor& w, const char* name, torch::Tensor& keep) -> const void* {
    if (!w) return nullptr;
    check_like(*w, q, name, "q");
    TORCH_CHECK(w->dim() == 1 && w->size(0) == D, name, " must be [D]");
    keep = aligned(*w);
    return keep.data_ptr();
  };
  c.a.q_weight = weight(qw, "q_weight", c.qw);
  c.a.k_weight = weight(kw, "k_weight", c.kw);
  if (cos) {
    check_f32(*cos, q, "cos");
    check_f32(*sin, q, "sin");
    TORCH_CHECK(cos->dim() == 2 && sin->sizes() == cos->sizes(),
                "cos and sin must be [positions, R/2] of one shape");
    const int64_t R = 2 * cos->size(1);
    TORCH_CHECK(R % 16 == 0 && R >= 16 && R <= D,
                "the rotated part 2 * cos.shape[1] must be a multiple of 16, at most D");
    c.cos = aligned(*cos);
    c.sin = aligned(*sin);
    c.a.cos = c.cos.data_ptr<float>();
    c.a.sin = c.sin.data_ptr<float>();
    c.a.R = R;
    c.a.table_rows = cos->size(0);
    if (pos) {
      c.a.positions_are_64 = is_index64(*pos, q, "positions");
      TORCH_CHECK((pos->dim() == 1 && pos->size(0) == q.size(1)) ||
                      (pos->dim() == 2 && pos->size(0) == q.size(0) && pos->size(1) == q.size(1)),
                  "positions must be [T] or [B,T]");
      c.pos = *pos;
      c.a.positions = pos->data_ptr();
      c.a.p_sb = pos->dim() == 2 ? pos->stride(0) : 0;
      c.a.p_st = pos->stride(-1);
    } else {
      TORCH_CHECK(c.a.table_rows >= q.size(1), "cos and sin have fewer rows than there are tokens");
    }
  }
  c.a.q = c.q.data_ptr();
  c.a.k = c.k.data_ptr();
  c.a.B = q.size(0), c.a.T = q.size(1), c.a.Hq = q.size(2), c.a.Hk = k.size(2), c.a.D = D;
  c.a.q_sb = stride_of(c.q, 0), c.a.q_st = stride_of(c.q, 1), c.a.q_sh = stride_of(c.q, 2);
  c.a.k_sb = stride_of(c.k, 0), c.a.k_st = stride_of(c.k, 1), c.a.k_sh = stride_of(c.k, 2);
  c.a.norm = norm;
  c.a.eps = eps;
  c.a.interleaved = interleaved;
  return c;
}

std::tuple<torch::Tensor, torch::Tensor> qk_norm_rope(torch::Tensor q, torch::Tensor k, OptTensor qw,
                                                      OptTensor kw, OptTensor cos, OptTensor sin,
                                                      OptTensor pos, int64_t norm, double eps,
                                                      bool interleaved) {
  auto c = qk_call(q, k, qw, kw, cos, sin, pos, norm, eps, interleaved);
  const c10::cuda::CUDAGuard guard(cuda_device(q));
  auto qo = torch::empty(q.sizes(), q.options()), ko = torch::empty(k.sizes(), k.options());
  c.a.q_out = qo.data_ptr();
  c.a.k_out = ko.data_ptr();
  check_status(tdc_qk_norm_rope(&c.a, stream_of(q)), "qk_norm_rope");
  return {qo, ko};
}

std::tuple<torch::Tensor, torch::Tensor, OptTensor, OptTensor> qk_norm_rope_bwd(
    torch::Tensor q, torch::Tensor k, OptTensor qw, OptTensor kw, OptTensor cos, OptTensor sin,
    OptTensor pos, int64_t norm, double eps, bool interleaved, torch::Tensor dq_out,
    torch::Tensor dk_out) {
  auto c = qk_call(q, k, qw, kw, cos, sin, pos, norm, eps, interleaved);
  check_like(dq_out, q, "dq_out", "q");
  check_like(dk_out, q, "dk_out", "q");
  TORCH_CHECK(dq_out.sizes() == q.sizes() && dk_out.sizes() == k.sizes(),
              "dq_out and dk_out must have q's and k's shapes");
  const c10::cuda::CUDAGuard guard(cuda_device(q));
  auto gq = in_place(dq_out), gk = in_place(dk_out);
  auto dq = torch::empty(q.sizes(), q.options()), dk = torch::empty(k.sizes(), k.options());
  OptTensor dqw, dkw;
  if (qw) dqw = torch::empty({c.a.D}, q.options());
  if (kw) dkw = torch::empty({c.a.D}, q.options());
  tdc_qk_grad_args g{};
  g.dq_out = gq.data_ptr(), g.dk_out = gk.data_ptr();
  g.dq = dq.data_ptr(), g.dk = dk.data_ptr();
  g.dq_weight = dqw ? dqw->data_ptr() : nullptr;
  g.dk_weight = dkw ? dkw->data_ptr() : nullptr;
  g.gq_sb = stride_of(gq, 0), g.gq_st = stride_of(gq, 1), g.gq_sh = stride_of(gq, 2);
  g.gk_sb = stride_of(gk, 0), g.gk_st = stride_of(gk, 1), g.gk_sh = stride_of(gk, 2);
  const int64_t need = tdc_qk_norm_rope_bwd_workspace(&c.a);
  if (need < 0) check_status(int(need), "qk_norm_rope_bwd");
  auto ws = bytes_on(q, need);
  check_status(tdc_qk_norm_rope_bwd(&c.a, &g, ws.data_ptr(), need, stream_of(q)),
               "qk_norm_rope_bwd");
  return {dq, dk, dqw, dkw};
}

// ---- gated delta rule -------------------------------------------------------------
struct DeltaCall {
  tdc_delta_args a{};
  torch::Tensor q, k, v, g, beta, init, cu;
  int64_t seqs = 0;
};

DeltaCall delta_call(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                     const torch::Tensor& g, const torch::Tensor& beta, double scale,
                     const OptTensor& init, const OptTensor& cu) {
  DeltaCall c;
  c.a.dtype = dtype_of(q, "q");
  check_like(k, q, "k", "q");
  check_like(v, q, "v", "q");
  check_f32(g, q, "g");
  TORCH_CHECK(beta.device() == q.device(), "beta must be on the inputs' device");
  TORCH_CHECK(beta.scalar_type() == torch::kFloat || beta.scalar_type() == q.scalar_type(),
              "beta must be fp32 or have q's dtype");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4,
              "q, k must be [B,T,H,K] and v [B,T,HV,V]");
  TORCH_CHECK(g.dim() == 3 && beta.dim() == 3, "g and beta must be [B,T,HV]");
  const int64_t B = q.size(0), T = q.size(1), H = q.size(2), K = q.size(3);
  const int64_t HV = v.size(2), V = v.size(3);
  TORCH_CHECK(k.sizes() == q.sizes(), "k must have q's shape");
  TORCH_CHECK(v.size(0) == B && v.size(1) == T, "v must agree with q on B and T");
  TORCH_CHECK(g.size(0) == B && g.size(1) == T && g.size(2) == HV && beta.sizes() == g.sizes(),
              "g and beta must be [B,T,HV]");
  TORCH_CHECK(H >= 1 && HV >= 1 && HV % H == 0, "the value heads must be a multiple of the key heads");
  TORCH_CHECK(K == 64 || K == 128, "the key head size must be 64 or 128, got ", K);
  TORCH_CHECK(V == 64 || V == 128 || V == 256, "the value head size must be 64, 128 or 256, got ", V);
  check_cu(cu, q);
  c.seqs = cu ? cu->size(0) - 1 : B;
  c.q = in_place(q);
  c.k = in_place(k);
  c.v = in_place(v);
  c.g = g.stride(2) == 1 || HV == 1 ? g : g.contiguous();
  c.beta = beta.stride(2) == 1 || HV == 1 ? beta : beta.contiguous();
  if (init) {
    check_f32(*init, q, "initial_state");
    TORCH_CHECK(init->dim() == 4 && init->size(0) == c.seqs && init->size(1) == HV &&
                    init->size(2) == K && init->size(3) == V,
                "initial_state must be [sequences, HV, K, V]");
    c.init = aligned(*init);
    c.a.initial_state = c.init.data_ptr<float>();
  }
  if (cu) {
    c.cu = *cu;
    c.a.cu_seqlens = cu->data_ptr();
    c.a.num_seqs = c.seqs;
    c.a.cu_is_64 = cu->scalar_type() == torch::kLong;
  }
  c.a.q = c.q.data_ptr(), c.a.k = c.k.data_ptr(), c.a.v = c.v.data_ptr();
  c.a.g = c.g.data_ptr<float>(), c.a.beta = c.beta.data_ptr();
  c.a.B = B, c.a.T = T, c.a.H = H, c.a.HV = HV, c.a.K = K, c.a.V = V;
  c.a.q_sb = stride_of(c.q, 0), c.a.q_st = stride_of(c.q, 1), c.a.q_sh = stride_of(c.q, 2);
  c.a.k_sb = stride_of(c.k, 0), c.a.k_st = stride_of(c.k, 1), c.a.k_sh = stride_of(c.k, 2);
  c.a.v_sb = stride_of(c.v, 0), c.a.v_st = stride_of(c.v, 1), c.a.v_sh = stride_of(c.v, 2);
  c.a.g_sb = stride_of(c.g, 0), c.a.g_st = stride_of(c.g, 1);
  c.a.b_sb = stride_of(c.beta, 0), c.a.b_st = stride_of(c.beta, 1);
  c.a.beta_is_f32 = beta.scalar_type() == torch::kFloat;
  c.a.scale = scale;
  return c;
}

std::tuple<torch::Tensor, OptTensor> gated_delta_rule(torch::Tensor q, torch::Tensor k,
                                                      torch::Tensor v, torch::Tensor g,
                                                      torch::Tensor beta, double scale,
                                                      OptTensor init, OptTensor cu,
                                                      bool want_final, int64_t withhold_chunk,
                                                      int64_t timeout_ns) {
  auto c = delta_call(q, k, v, g, beta, scale, init, cu);
  const c10::cuda::CUDAGuard guard(cuda_device(q));
  auto o = torch::empty(v.sizes(), v.options());
  OptTensor fin;
  if (want_final) {
    fin = torch::empty({c.seqs, c.a.HV, c.a.K, c.a.V}, g.options());
    c.a.final_state = fin->data_ptr<float>();
  }
  c.a.o = o.data_ptr();
  const int64_t need = tdc_delta_fwd_workspace(&c.a);
  if (need < 0) check_status(int(need), "gated_delta_rule");
  auto ws = bytes_on(q, need);
  check_status(withhold_chunk < 0
                   ? tdc_delta_fwd(&c.a, ws.data_ptr(), need, stream_of(q))
                   : tdc_delta_fwd_withhold(&c.a, ws.data_ptr(), need, withhold_chunk, timeout_ns,
                                            stream_of(q)),
               "gated_delta_rule");
  return {o, fin};
}

// (dq, dk, dv, dg, dbeta, dinitial or None)
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, OptTensor>
gated_delta_rule_bwd(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor g,
                     torch::Tensor beta, double scale, OptTensor init, OptTensor cu,
                     torch::Tensor d_o, OptTensor dfinal) {
  auto c = delta_call(q, k, v, g, beta, scale, init, cu);
  check_like(d_o, q, "d_o", "q");
  TORCH_CHECK(d_o.sizes() == v.sizes(), "d_o must have v's shape");
  auto d = in_place(d_o);
  torch::Tensor df;
  if (dfinal) {
    check_f32(*dfinal, q, "dfinal");
    TORCH_CHECK(dfinal->dim() == 4 && dfinal->size(0) == c.seqs && dfinal->size(1) == c.a.HV &&
                    dfinal->size(2) == c.a.K && dfinal->size(3) == c.a.V,
                "dfinal must be [sequences, HV, K, V]");
    df = aligned(*dfinal);
  }
  const c10::cuda::CUDAGuard guard(cuda_device(q));
  auto dq = torch::empty(q.sizes(), q.options()), dk = torch::empty(k.sizes(), k.options());
  auto dv = torch::empty(v.sizes(), v.options());
  auto dg = torch::empty(g.sizes(), g.options()), db = torch::empty(beta.sizes(), beta.options());
  OptTensor di;
  if (init) di = torch::empty(init->sizes(), init->options());
  tdc_delta_grad_args r{};
  r.d_o = d.data_ptr();
  r.dfinal = dfinal ? df.data_ptr<float>() : nullptr;
  r.dq = dq.data_ptr(), r.dk = dk.data_ptr(), r.dv = dv.data_ptr();
  r.dg = dg.data_ptr<float>(), r.dbeta = db.data_ptr();
  r.dinitial = di ? di->data_ptr<float>() : nullptr;
  r.do_sb = stride_of(d, 0), r.do_st = stride_of(d, 1), r.do_sh = stride_of(d, 2);
  const int64_t need = tdc_delta_bwd_workspace(&c.a);
  if (need < 0) check_status(int(need), "gated_delta_rule_bwd");
  auto ws = bytes_on(q, need);
  check_status(tdc_delta_bwd(&c.a, &r, ws.data_ptr(), need, stream_of(q)), "gated_delta_rule_bwd");
  return {dq, dk, dv, dg, db, di};
}

torch::Tensor gated_delta_step(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor g,
                               torch::Tensor beta, double scale, torch::Tensor state,
                               OptTensor idx) {
  auto c = delta_call(q, k, v, g, beta, scale, std::nullopt, std::nullopt);
  check_f32(state, q, "state");
  TORCH_CHECK(state.dim() == 4 && state.size(1) == c.a.HV && state.size(2) == c.a.K &&
                  state.size(3) == c.a.V,
              "state must be [slots, HV, K, V]");
  TORCH_CHECK(state.is_contiguous(), "state must be contiguous (it is updated in place)");
  check_state_indices(idx, q, c.a.B);
  TORCH_CHECK(idx || state.size(0) >= c.a.B, "state has fewer slots than there are requests");
  const c10::cuda::CUDAGuard guard(cuda_device(state));
  auto o = torch::empty(v.sizes(), v.options());
  c.a.o = o.data_ptr();
  check_status(tdc_delta_step(&c.a, state.data_ptr<float>(), state.size(0), ptr(idx),
                              idx && idx->scalar_type() == torch::kLong, stream_of(q)),
               "gated_delta_step");
  written(state);
  return o;
}

}  // namespace

void bind_sequence(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("causal_conv1d", &causal_conv1d,
        "Causal depthwise convolution over [B,T,C]: (y, final state or None).", py::arg("x"),
        py::arg("w"), py::arg("bias"), py::arg("initial_state"), py::arg("cu_seqlens"),
        py::arg("act"), py::arg("want_final"));
  m.def("causal_conv1d_bwd", &causal_conv1d_bwd,
        "Its gradients: (dx, dw, dbias or None, dinitial or None).", py::arg("x"), py::arg("w"),
        py::arg("bias"), py::arg("initial_state"), py::arg("cu_seqlens"), py::arg("act"),
        py::arg("dy"), py::arg("dfinal"));
  m.def("causal_conv1d_step", &causal_conv1d_step,
        "The next tokens of running sequences; updates state in place.", py::arg("x"), py::arg("w"),
        py::arg("bias"), py::arg("state"), py::arg("state_indices"), py::arg("act"));
  m.def("qk_norm_rope", &qk_norm_rope, "Norms of queries and keys and the position rotation.",
        py::arg("q"), py::arg("k"), py::arg("q_weight"), py::arg("k_weight"), py::arg("cos"),
        py::arg("sin"), py::arg("positions"), py::arg("norm"), py::arg("eps"),
        py::arg("interleaved"));
  m.def("qk_norm_rope_bwd", &qk_norm_rope_bwd,
        "Its gradients: (dq, dk, dq_weight or None, dk_weight or None).", py::arg("q"), py::arg("k"),
        py::arg("q_weight"), py::arg("k_weight"), py::arg("cos"), py::arg("sin"),
        py::arg("positions"), py::arg("norm"), py::arg("eps"), py::arg("interleaved"),
        py::arg("dq_out"), py::arg("dk_out"));
  m.def("gated_delta_rule", &gated_delta_rule,
        "Gated delta rule over whole sequences: (o, final state or None).  withhold_chunk >= 0 "
        "makes the copies of that chunk never come (tests the failure path; see device_status).",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("g"), py::arg("beta"), py::arg("scale"),
        py::arg("initial_state"), py::arg("cu_seqlens"), py::arg("want_final"),
        py::arg("withhold_chunk") = -1, py::arg("timeout_ns") = 0);
  m.def("gated_delta_rule_bwd", &gated_delta_rule_bwd,
        "Its gradients: (dq, dk, dv, dg, dbeta, dinitial or None).", py::arg("q"), py::arg("k"),
        py::arg("v"), py::arg("g"), py::arg("beta"), py::arg("scale"), py::arg("initial_state"),
        py::arg("cu_seqlens"), py::arg("d_o"), py::arg("dfinal"));
  m.def("gated_delta_step", &gated_delta_step,
        "The next tokens of running sequences; updates state in place.", py::arg("q"), py::arg("k"),
        py::arg("v"), py::arg("g"), py::arg("beta"), py::arg("scale"), py::arg("state"),
        py::arg("state_indices"));
}

}  // namespace tma_dwconv
