"""Sequence operators next to the depthwise convolutions: what a mixer layer of
a language model runs between its two matrix products.

* ``causal_conv1d(x, w, ...)`` — causal depthwise convolution over [B, T, C]
  (2 to 8 taps, bias, SiLU), with states that carry a sequence from one call to
  the next, packed batches of ragged sequences and all gradients;
  ``causal_conv1d_step`` — the next tokens of running sequences, whose states
  stay in a pool of slots.
* ``qk_norm_rope(q, k, ...)`` — the norm of every query and key head (RMS or
  unit length, with or without weights) and the rotation of its position in the
  same pass, with gradients; ``rotary_table`` makes the cos / sin tables, also
  stretched for contexts longer than the model was trained on.
* ``gated_delta_rule(q, k, v, g, beta, ...)`` — the recurrence
  ``S = e^g S;  S = S + beta k (v - S^T k)^T;  o = scale S^T q`` over whole
  sequences, in chunks of 64 tokens, with all gradients, initial and final
  states and packed batches; ``gated_delta_step`` — the recurrence for the next
  tokens of running sequences.
* ``GatedDeltaMixer`` — the layer made of them, for training, prefill and
  token-by-token decoding.

Inputs are fp16 or bf16 CUDA tensors; states and decays are fp32, and every sum
is.  Wrong arguments raise ``ValueError`` or ``RuntimeError`` before anything
runs.  The functions run on torch's current stream of their tensors' device,
take their workspaces from torch's allocator (so they can be captured into CUDA
graphs) and give the same bits every run.  They have first derivatives in
reverse mode; second and forward-mode ones raise ``RuntimeError``.  Under
``torch.compile`` they are the custom ops ``torch.ops.tdc.causal_conv1d``,
``tdc.qk_norm_rope`` and ``tdc.gated_delta_rule``; in eager mode lighter
autograd Functions call the same kernels.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch
from torch import Tensor, nn
from torch.autograd import forward_ad as fwAD
from torch.autograd.function import once_differentiable

import _tma_dwconv_C as _C  # type: ignore

__all__ = ["causal_conv1d", "causal_conv1d_step", "qk_norm_rope", "rotary_table",
           "gated_delta_rule", "gated_delta_step", "GatedDeltaMixer", "MixerState",
           "CONV_ACTIVATIONS", "NORMS"]

#: Activations of the causal convolution.
CONV_ACTIVATIONS = {"none": 0, "silu": 3}
#: Norms of ``qk_norm_rope``: none, x / sqrt(mean(x^2) + eps), x / sqrt(sum(x^2) + eps).
NORMS = {"none": 0, "rms": 1, "l2": 2}


def _needs_grad(*tensors: Optional[Tensor]) -> bool:
    if fwAD._current_level >= 0 and any(t is not None and fwAD.unpack_dual(t).tangent is not None
                                        for t in tensors):
        raise RuntimeError("the sequence operators have no forward-mode derivatives")
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _code(table: dict, name: str, what: str) -> int:
    if name not in table:
        raise ValueError(f"{what} must be one of {sorted(table)}, got {name!r}")
    return table[name]


def _sequences(x: Tensor, cu_seqlens: Optional[Tensor]) -> int:
    return x.shape[0] if cu_seqlens is None else cu_seqlens.shape[0] - 1


def _or_empty(t: Optional[Tensor], like: Tensor) -> Tensor:
    return like.new_empty(0) if t is None else t


# --------------------------- causal convolution -------------------------------

class _Conv1dFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, initial_state, cu_seqlens, act, want_final):
        y, final = _C.causal_conv1d(x, w, bias, initial_state, cu_seqlens, act, want_final)
        ctx.save_for_backward(x, w, bias, initial_state, cu_seqlens)
        ctx.act = act
        ctx.set_materialize_grads(False)
        return y, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal):
        x, w, bias, initial_state, cu = ctx.saved_tensors
        if dy is None:
            if dfinal is None:
                return (None,) * 7
            dy = torch.zeros_like(x)
        dx, dw, db, ds = _C.causal_conv1d_bwd(x, w, bias, initial_state, cu, ctx.act,
                                              dy.to(x.dtype), dfinal)
        return dx, dw, db, ds, None, None, None


@torch.library.custom_op("tdc::causal_conv1d", mutates_args=())
def causal_conv1d_op(x: Tensor, w: Tensor, bias: Optional[Tensor],
                     initial_state: Optional[Tensor], cu_seqlens: Optional[Tensor], act: int,
                     want_final: bool) -> tuple[Tensor, Tensor]:
    """(y, final state; empty if not wanted)."""
    y, final = _C.causal_conv1d(x, w, bias, initial_state, cu_seqlens, act, want_final)
    return y, _or_empty(final, x)


@causal_conv1d_op.register_fake
def _(x, w, bias, initial_state, cu_seqlens, act, want_final):
    n = _sequences(x, cu_seqlens)
    final = x.new_empty((n, w.shape[0] - 1, x.shape[2])) if want_final else x.new_empty(0)
    return x.new_empty(x.shape), final


@torch.library.custom_op("tdc::causal_conv1d_bwd", mutates_args=())
def causal_conv1d_bwd_op(x: Tensor, w: Tensor, bias: Optional[Tensor],
                         initial_state: Optional[Tensor], cu_seqlens: Optional[Tensor], act: int,
                         dy: Tensor, dfinal: Optional[Tensor]
                         ) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(dx, dw, dbias, dinitial; the last two empty without bias or state)."""
    dx, dw, db, ds = _C.causal_conv1d_bwd(x, w, bias, initial_state, cu_seqlens, act,
                                          dy.to(x.dtype), dfinal)
    return dx, dw, _or_empty(db, x), _or_empty(ds, x)


@causal_conv1d_bwd_op.register_fake
def _(x, w, bias, initial_state, cu_seqlens, act, dy, dfinal):
    return (x.new_empty(x.shape), w.new_empty(w.shape),
            x.new_empty(0 if bias is None else bias.shape),
            x.new_empty(0 if initial_state is None else initial_state.shape))


def _conv_setup(ctx, inputs, output):
    x, w, bias, initial_state, cu_seqlens, act, want_final = inputs
    ctx.save_for_backward(x, w, bias, initial_state, cu_seqlens)
    ctx.act, ctx.want_final = act, want_final


def _conv_backward(ctx, dy, dfinal):
    x, w, bias, initial_state, cu = ctx.saved_tensors
    dy = torch.zeros_like(x) if dy is None else dy
    dx, dw, db, ds = causal_conv1d_bwd_op(x, w, bias, initial_state, cu, ctx.act, dy,
                                          dfinal if ctx.want_final else None)
    return (dx, dw, None if bias is None else db, None if initial_state is None else ds, None,
            None, None)


causal_conv1d_op.register_autograd(_conv_backward, setup_context=_conv_setup)


def causal_conv1d(x: Tensor, w: Tensor, bias: Optional[Tensor] = None, activation: str = "none",
                  initial_state: Optional[Tensor] = None, cu_seqlens: Optional[Tensor] = None,
                  output_final_state: bool = False):
    """Causal depthwise convolution: ``y[b,t] = act(bias + sum_j w[j] x[b, t-(K-1)+j])``.

    Args:
        x: [B, T, C] fp16 or bf16, C % 8 == 0; any strides whose last is 1 and
            whose others are multiples of 8 are read in place.
        w: [K, C] of x's dtype, 2 <= K <= 8.
        bias: [C] or None.
        activation: "none" or "silu".
        initial_state: [N, K-1, C], the inputs before each sequence (oldest
            first); zeros if None.
        cu_seqlens: int32 or int64 [N+1] row offsets of a packed batch (B = 1).
            Rows that no sequence owns give zeros.
        output_final_state: also return [N, K-1, C], each sequence's last K-1
            inputs.

    Differentiable in x, w, bias and initial_state, also through the final state.
    """
    act = _code(CONV_ACTIVATIONS, activation, "activation")
    if torch.compiler.is_compiling():
        y, final = causal_conv1d_op(x, w, bias, initial_state, cu_seqlens, act, output_final_state)
    elif _needs_grad(x, w, bias, initial_state):
        y, final = _Conv1dFunction.apply(x, w, bias, initial_state, cu_seqlens, act,
                                         output_final_state)
    else:
        y, final = _C.causal_conv1d(x, w, bias, initial_state, cu_seqlens, act, output_final_state)
    return (y, final) if output_final_state else y


def causal_conv1d_step(x: Tensor, w: Tensor, bias: Optional[Tensor], state: Tensor,
                       activation: str = "none",
                       state_indices: Optional[Tensor] = None) -> Tensor:
    """The convolution for the next T tokens (usually 1) of B running sequences.

    x is [B, T, C] or [B, C]; state [slots, K-1, C] is updated in place.
    Request b continues slot ``state_indices[b]`` (int32 or int64; slot b
    without indices).  A negative index is padding: zeros, and no state is
    touched.  An index >= slots, and one that an earlier request of the call
    has, gives NaN and touches no state.  Not differentiable.
    """
    act = _code(CONV_ACTIVATIONS, activation, "activation")
    if _needs_grad(x, w, bias, state):
        raise RuntimeError("causal_conv1d_step updates its state in place and has no gradients; "
                           "call it under torch.no_grad()")
    if x.dim() == 2:
        return _C.causal_conv1d_step(x.unsqueeze(1), w, bias, state, state_indices, act)[:, 0]
    return _C.causal_conv1d_step(x, w, bias, state, state_indices, act)


# --------------------------- norms and rotation ---------------------------------

def rotary_table(rotary_dim: int, length: int, base: float = 10000.0, scaling: str = "none",
                 factor: float = 1.0, original_length: Optional[int] = None,
                 beta_fast: float = 32.0, beta_slow: float = 1.0, device=None
                 ) -> tuple[Tensor, Tensor]:
    """(cos, sin), fp32 [length, rotary_dim / 2], of position times
    ``base^(-2 i / rotary_dim)``, from angles in fp64.

    ``scaling`` stretches the table by ``factor`` for contexts longer than the
    trained ``original_length``: "linear" divides every frequency; "base"
    enlarges the base so that the lowest frequency is divided by the factor and
    the highest is kept; "parts" keeps the frequencies that turn more than
    ``beta_fast`` times within original_length, divides those that turn less
    than ``beta_slow`` times, blends linearly between, and multiplies cos and
    sin by ``0.1 ln(factor) + 1``.
    """
    if rotary_dim < 16 or rotary_dim % 16:
        raise ValueError(f"rotary_dim must be a positive multiple of 16, got {rotary_dim}")
    if length < 0:
        raise ValueError(f"length must not be negative, got {length}")
    if scaling not in ("none", "linear", "base", "parts"):
        raise ValueError(f"scaling must be 'none', 'linear', 'base' or 'parts', got {scaling!r}")
    if scaling != "none" and not factor >= 1.0:
        raise ValueError(f"factor must be at least 1, got {factor}")
    if scaling == "parts" and (original_length is None or original_length < 1):
        raise ValueError("scaling 'parts' needs original_length")
    half = rotary_dim // 2
    i = torch.arange(half, dtype=torch.float64, device=device)
    size = 1.0
    if scaling == "base":
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-i / half)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "parts":
        # index of the frequency as a real number at which `beta` turns happen
        at = [half * math.log(original_length / (b * 2 * math.pi)) / math.log(base)
              for b in (beta_fast, beta_slow)]
        # (the blend may end behind the last pair, where that one still turns beta_slow times)
        low, high = max(math.floor(at[0]), 0), math.ceil(at[1])
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        size = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * freq
    return (angle.cos() * size).float(), (angle.sin() * size).float()


class _QkFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, cos, sin, positions, norm, eps, interleaved):
        qo, ko = _C.qk_norm_rope(q, k, qw, kw, cos, sin, positions, norm, eps, interleaved)
        ctx.save_for_backward(q, k, qw, kw, cos, sin, positions)
        ctx.conf = (norm, eps, interleaved)
        ctx.set_materialize_grads(False)
        return qo, ko

    @staticmethod
    @once_differentiable
    def backward(ctx, dqo, dko):
        q, k, qw, kw, cos, sin, positions = ctx.saved_tensors
        if dqo is None and dko is None:
            return (None,) * 10
        dqo = torch.zeros_like(q) if dqo is None else dqo.to(q.dtype)
        dko = torch.zeros_like(k) if dko is None else dko.to(k.dtype)
        return (*_C.qk_norm_rope_bwd(q, k, qw, kw, cos, sin, positions, *ctx.conf, dqo, dko),
                None, None, None, None, None, None)


@torch.library.custom_op("tdc::qk_norm_rope", mutates_args=())
def qk_norm_rope_op(q: Tensor, k: Tensor, q_weight: Optional[Tensor], k_weight: Optional[Tensor],
                    cos: Optional[Tensor], sin: Optional[Tensor], positions: Optional[Tensor],
                    norm: int, eps: float, interleaved: bool) -> tuple[Tensor, Tensor]:
    """(q, k) normed and rotated."""
    return _C.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, norm, eps, interleaved)


@qk_norm_rope_op.register_fake
def _(q, k, q_weight, k_weight, cos, sin, positions, norm, eps, interleaved):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.custom_op("tdc::qk_norm_rope_bwd", mutates_args=())
def qk_norm_rope_bwd_op(q: Tensor, k: Tensor, q_weight: Optional[Tensor],
                        k_weight: Optional[Tensor], cos: Optional[Tensor], sin: Optional[Tensor],
                        positions: Optional[Tensor], norm: int, eps: float, interleaved: bool,
                        dq_out: Tensor, dk_out: Tensor) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(dq, dk, dq_weight, dk_weight; the last two empty without weights)."""
    dq, dk, dqw, dkw = _C.qk_norm_rope_bwd(q, k, q_weight, k_weight, cos, sin, positions, norm, eps,
                                           interleaved, dq_out.to(q.dtype), dk_out.to(k.dtype))
    return dq, dk, _or_empty(dqw, q), _or_empty(dkw, q)


@qk_norm_rope_bwd_op.register_fake
def _(q, k, q_weight, k_weight, cos, sin, positions, norm, eps, interleaved, dq_out, dk_out):
    return (q.new_empty(q.shape), k.new_empty(k.shape),
            q.new_empty(0 if q_weight is None else q_weight.shape),
            q.new_empty(0 if k_weight is None else k_weight.shape))


def _qk_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:7])
    ctx.conf = inputs[7:]


def _qk_backward(ctx, dqo, dko):
    saved = ctx.saved_tensors
    dqo = torch.zeros_like(saved[0]) if dqo is None else dqo
    dko = torch.zeros_like(saved[1]) if dko is None else dko
    dq, dk, dqw, dkw = qk_norm_rope_bwd_op(*saved, *ctx.conf, dqo, dko)
    return (dq, dk, None if saved[2] is None else dqw, None if saved[3] is None else dkw,
            None, None, None, None, None, None)


qk_norm_rope_op.register_autograd(_qk_backward, setup_context=_qk_setup)


def qk_norm_rope(q: Tensor, k: Tensor, q_weight: Optional[Tensor] = None,
                 k_weight: Optional[Tensor] = None, norm: str = "rms", eps: float = 1e-6,
                 cos: Optional[Tensor] = None, sin: Optional[Tensor] = None,
                 positions: Optional[Tensor] = None, interleaved: bool = False
                 ) -> tuple[Tensor, Tensor]:
    """Norm of each query and key head, then the rotation of its position, in one pass.

    Args:
        q, k: [B, T, Hq, D] and [B, T, Hk, D] fp16 or bf16 (8 <= D <= 256, D % 8
            == 0); views of a packed projection are read in place.
        q_weight, k_weight: [D] of q's dtype, or None.
        norm: "rms", "l2" (unit length) or "none"; eps is added to the mean or
            sum of squares.
        cos, sin: fp32 [positions, R/2] tables (``rotary_table``), or None for no
            rotation.  The first R values of a head are rotated, R % 16 == 0.
        positions: int32 or int64 [T] or [B, T]; 0 .. T-1 if None.  A position
            outside the table gives NaN in the rotated values.
        interleaved: pairs are (2i, 2i+1) instead of (i, i + R/2).

    Returns new contiguous tensors.  Differentiable in q, k and the weights.
    """
    code = _code(NORMS, norm, "norm")
    args = (q, k, q_weight, k_weight, cos, sin, positions, code, float(eps), bool(interleaved))
    if torch.compiler.is_compiling():
        return qk_norm_rope_op(*args)
    if _needs_grad(q, k, q_weight, k_weight):
        return _QkFunction.apply(*args)
    return _C.qk_norm_rope(*args)


# --------------------------- gated delta rule -----------------------------------

class _DeltaFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, scale, initial_state, cu_seqlens, want_final):
        o, final = _C.gated_delta_rule(q, k, v, g, beta, scale, initial_state, cu_seqlens,
                                       want_final)
        ctx.save_for_backward(q, k, v, g, beta, initial_state, cu_seqlens)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, final

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o, dfinal):
        q, k, v, g, beta, initial_state, cu = ctx.saved_tensors
        if d_o is None:
            if dfinal is None:
                return (None,) * 9
            d_o = torch.zeros_like(v)
        dq, dk, dv, dg, db, ds = _C.gated_delta_rule_bwd(q, k, v, g, beta, ctx.scale, initial_state,
                                                         cu, d_o.to(v.dtype), dfinal)
        return dq, dk, dv, dg, db, None, ds, None, None


@torch.library.custom_op("tdc::gated_delta_rule", mutates_args=())
def gated_delta_rule_op(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, scale: float,
                        initial_state: Optional[Tensor], cu_seqlens: Optional[Tensor],
                        want_final: bool) -> tuple[Tensor, Tensor]:
    """(o, final state; empty if not wanted)."""
    o, final = _C.gated_delta_rule(q, k, v, g, beta, scale, initial_state, cu_seqlens, want_final)
    return o, _or_empty(final, g)


@gated_delta_rule_op.register_fake
def _(q, k, v, g, beta, scale, initial_state, cu_seqlens, want_final):
    n = _sequences(q, cu_seqlens)
    final = (g.new_empty((n, v.shape[2], q.shape[3], v.shape[3])) if want_final
             else g.new_empty(0))
    return v.new_empty(v.shape), final


@torch.library.custom_op("tdc::gated_delta_rule_bwd", mutates_args=())
def gated_delta_rule_bwd_op(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, scale: float,
                            initial_state: Optional[Tensor], cu_seqlens: Optional[Tensor],
                            d_o: Tensor, dfinal: Optional[Tensor]
                            ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(dq, dk, dv, dg, dbeta, dinitial; the last empty without a state)."""
    dq, dk, dv, dg, db, ds = _C.gated_delta_rule_bwd(q, k, v, g, beta, scale, initial_state,
                                                     cu_seqlens, d_o.to(v.dtype), dfinal)
    return dq, dk, dv, dg, db, _or_empty(ds, g)


@gated_delta_rule_bwd_op.register_fake
def _(q, k, v, g, beta, scale, initial_state, cu_seqlens, d_o, dfinal):
    return (q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape), g.new_empty(g.shape),
            beta.new_empty(beta.shape),
            g.new_empty(0 if initial_state is None else initial_state.shape))


def _delta_setup(ctx, inputs, output):
    q, k, v, g, beta, scale, initial_state, cu_seqlens, want_final = inputs
    ctx.save_for_backward(q, k, v, g, beta, initial_state, cu_seqlens)
    ctx.scale, ctx.want_final = scale, want_final


def _delta_backward(ctx, d_o, dfinal):
    q, k, v, g, beta, initial_state, cu = ctx.saved_tensors
    d_o = torch.zeros_like(v) if d_o is None else d_o
    *grads, ds = gated_delta_rule_bwd_op(q, k, v, g, beta, ctx.scale, initial_state, cu, d_o,
                                         dfinal if ctx.want_final else None)
    return (*grads, None, None if initial_state is None else ds, None, None)


gated_delta_rule_op.register_autograd(_delta_backward, setup_context=_delta_setup)


def gated_delta_rule(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor,
                     scale: Optional[float] = None, initial_state: Optional[Tensor] = None,
                     cu_seqlens: Optional[Tensor] = None, output_final_state: bool = False):
    """The gated delta rule over whole sequences.

    For each value head, with S [K, V] from ``initial_state`` (or zeros), token
    by token: ``S = e^g S``, ``S = S + beta k (v - S^T k)^T``, ``o = scale S^T q``.

    Args:
        q, k: [B, T, H, K] fp16 or bf16, K 64 or 128.  Keys should have a norm
            of about 1 (``qk_norm_rope(..., norm="l2")``).
        v: [B, T, HV, V], V 64, 128 or 256, HV a multiple of H: value head i
            uses query and key head i // (HV // H).
        g: [B, T, HV] fp32, the logarithm of the decay (at most 0 as a rule).
        beta: [B, T, HV] fp32 or of q's dtype, in [0, 2).
        scale: K^-0.5 if None.
        initial_state: [N, HV, K, V] fp32 or None.
        cu_seqlens: int32 or int64 [N+1] row offsets of a packed batch (B = 1).
        output_final_state: also return the states [N, HV, K, V] behind the
            last tokens.

    Differentiable in all tensors, also through the final state.
    """
    scale = float(q.shape[-1]) ** -0.5 if scale is None else float(scale)
    args = (q, k, v, g, beta, scale, initial_state, cu_seqlens, output_final_state)
    if torch.compiler.is_compiling():
        o, final = gated_delta_rule_op(*args)
    elif _needs_grad(q, k, v, g, beta, initial_state):
        o, final = _DeltaFunction.apply(*args)
    else:
        o, final = _C.gated_delta_rule(*args)
    return (o, final) if output_final_state else o


def gated_delta_step(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, state: Tensor,
                     scale: Optional[float] = None,
                     state_indices: Optional[Tensor] = None) -> Tensor:
    """The gated delta rule for the next T tokens (usually 1) of B running
    sequences: shapes as for ``gated_delta_rule``, state [slots, HV, K, V] fp32,
    updated in place.  Slots and their indices as for ``causal_conv1d_step``.
    Not differentiable."""
    if _needs_grad(q, k, v, g, beta, state):
        raise RuntimeError("gated_delta_step updates its state in place and has no gradients; "
                           "call it under torch.no_grad()")
    scale = float(q.shape[-1]) ** -0.5 if scale is None else float(scale)
    return _C.gated_delta_step(q, k, v, g, beta, scale, state, state_indices)


# --------------------------- the layer --------------------------------------------

@dataclass
class MixerState:
    """What a ``GatedDeltaMixer`` carries of its running sequences, one slot each:
    the convolution's last inputs [slots, taps-1, channels] and the delta rule's
    states [slots, value heads, K, V] (fp32)."""
    conv: Tensor
    delta: Tensor


class GatedDeltaMixer(nn.Module):
    """A sequence mixer for fp16 or bf16 inputs [B, T, hidden]: one projection to
    queries, keys, values, an output gate and the two gates of the delta rule; a
    causal depthwise convolution with SiLU over queries, keys and values; unit
    queries and keys (rotated if ``rotary_dim`` is given); the gated delta rule;
    the heads' RMS norm times the output gate; the output projection.

    ``forward`` is for training and prefill (also of packed batches), ``step``
    for the next tokens of running sequences; ``new_state`` makes their slots.
    """

    def __init__(self, hidden: int, key_heads: int, value_heads: Optional[int] = None,
                 key_dim: int = 128, value_dim: int = 128, taps: int = 4, rotary_dim: int = 0,
                 rotary_base: float = 10000.0, max_positions: int = 0, eps: float = 1e-6,
                 device=None, dtype=torch.bfloat16):
        super().__init__()
        value_heads = key_heads if value_heads is None else value_heads
        if key_dim not in (64, 128) or value_dim not in (64, 128, 256):
            raise ValueError(f"key_dim must be 64 or 128 and value_dim 64, 128 or 256, got "
                             f"{key_dim}, {value_dim}")
        if key_heads < 1 or value_heads < 1 or value_heads % key_heads:
            raise ValueError(f"value_heads must be a multiple of key_heads, got {value_heads}, "
                             f"{key_heads}")
        if not 2 <= taps <= 8:
            raise ValueError(f"taps must be 2 to 8, got {taps}")
        if rotary_dim % 16 or not 0 <= rotary_dim <= key_dim:
            raise ValueError(f"rotary_dim must be a multiple of 16 up to key_dim, got {rotary_dim}")
        if rotary_dim and max_positions < 1:
            raise ValueError("rotary_dim needs max_positions")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"dtype must be float16 or bfloat16, got {dtype}")
        self.key_heads, self.value_heads = key_heads, value_heads
        self.key_dim, self.value_dim, self.taps, self.eps = key_dim, value_dim, taps, eps
        self.sizes = (key_heads * key_dim, key_heads * key_dim, value_heads * value_dim)
        self.channels = sum(self.sizes)
        inner = value_heads * value_dim
        # the gates' columns are padded to 8, so that every part of a row stays aligned
        self.gates = -(-2 * value_heads // 8) * 8
        make = dict(device=device, dtype=dtype)
        self.in_proj = nn.Linear(hidden, self.channels + inner + self.gates, bias=False, **make)
        self.conv_weight = nn.Parameter(torch.empty(taps, self.channels, **make))
        nn.init.uniform_(self.conv_weight, -taps ** -0.5, taps ** -0.5)
        # decay e^(-exp(log_rate) softplus(a + step_bias)): rates of 1 to 16, steps of 1e-3 to 0.1
        rate = torch.empty(value_heads, device=device, dtype=torch.float32).uniform_(1, 16)
        step = torch.exp(torch.empty(value_heads, device=device, dtype=torch.float32).uniform_(
            math.log(1e-3), math.log(0.1)))
        self.log_rate = nn.Parameter(rate.log())
        self.step_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))
        self.norm_weight = nn.Parameter(torch.ones(value_dim, **make))
        self.out_proj = nn.Linear(inner, hidden, bias=False, **make)
        self.rotary_dim = rotary_dim
        if rotary_dim:
            self.table_args = (rotary_dim, max_positions, rotary_base)
            cos, sin = rotary_table(*self.table_args, device=device)
            self.register_buffer("cos", cos, persistent=False)
            self.register_buffer("sin", sin, persistent=False)

    def _apply(self, fn, *args, **kwargs):
        # .to(dtype) casts floating buffers as well: the tables are fp32 in any case
        tables = {n: getattr(self, n) for n in ("cos", "sin") if self.rotary_dim}
        super()._apply(fn, *args, **kwargs)
        for n, t in tables.items():
            device = getattr(self, n).device
            if t.is_meta and device.type != "meta":   # (to_empty: they are in no state dict)
                t = rotary_table(*self.table_args, device=device)[n == "sin"]
            setattr(self, n, t.to(device))
        return self

    def new_state(self, slots: int) -> MixerState:
        w = self.conv_weight
        return MixerState(
            torch.zeros(slots, self.taps - 1, self.channels, device=w.device, dtype=w.dtype),
            torch.zeros(slots, self.value_heads, self.key_dim, self.value_dim, device=w.device,
                        dtype=torch.float32))

    def _project(self, x: Tensor):
        p = self.in_proj(x)
        mixed, gate, ab = p.split((self.channels, self.value_heads * self.value_dim, self.gates), -1)
        a, b = ab[..., :self.value_heads], ab[..., self.value_heads:2 * self.value_heads]
        g = -self.log_rate.float().exp() * nn.functional.softplus(a.float() + self.step_bias.float())
        return mixed, gate, g, torch.sigmoid(b)

    def _heads(self, mixed: Tensor, positions: Optional[Tensor]):
        q, k, v = mixed.split(self.sizes, -1)
        q = q.unflatten(-1, (self.key_heads, self.key_dim))
        k = k.unflatten(-1, (self.key_heads, self.key_dim))
        v = v.unflatten(-1, (self.value_heads, self.value_dim))
        cos, sin = (self.cos, self.sin) if self.rotary_dim else (None, None)
        q, k = qk_norm_rope(q, k, norm="l2", eps=self.eps, cos=cos, sin=sin,
                            positions=positions if self.rotary_dim else None)
        return q, k, v

    def _finish(self, o: Tensor, gate: Tensor) -> Tensor:
        o, _ = qk_norm_rope(o, o[:, :, :0], self.norm_weight, norm="rms", eps=self.eps)
        return self.out_proj(o.flatten(-2) * nn.functional.silu(gate))

    def forward(self, x: Tensor, state: Optional[MixerState] = None,
                cu_seqlens: Optional[Tensor] = None, positions: Optional[Tensor] = None,
                output_state: bool = False):
        """y [B, T, hidden]; with ``output_state`` also the ``MixerState`` behind
        the last tokens, one slot a sequence.  ``state`` continues earlier tokens.
        ``positions`` ([T] or [B, T], for the rotation) default to 0 .. T-1, the row
        of a packed batch too; with ``rotary_dim`` they have to be given where that
        cannot be right: with a ``state``, and for the states of a packed batch."""
        if self.rotary_dim and positions is None and (
                state is not None or (output_state and cu_seqlens is not None)):
            raise ValueError("a rotated layer needs positions with a state, and for the states of "
                             "a packed batch")
        mixed, gate, g, beta = self._project(x)
        conv_state, delta_state = (None, None) if state is None else (state.conv, state.delta)
        out = causal_conv1d(mixed, self.conv_weight, activation="silu", initial_state=conv_state,
                            cu_seqlens=cu_seqlens, output_final_state=output_state)
        mixed, conv_final = out if output_state else (out, None)
        q, k, v = self._heads(mixed, positions)
        out = gated_delta_rule(q, k, v, g, beta, initial_state=delta_state, cu_seqlens=cu_seqlens,
                               output_final_state=output_state)
        o, delta_final = out if output_state else (out, None)
        y = self._finish(o, gate)
        return (y, MixerState(conv_final, delta_final)) if output_state else y

    @torch.no_grad()
    def step(self, x: Tensor, state: MixerState, state_indices: Optional[Tensor] = None,
             positions: Optional[Tensor] = None) -> Tensor:
        """The next tokens x [B, T, hidden] (T usually 1) of B running sequences,
        whose slots are updated in place (``causal_conv1d_step`` says how slots
        are picked).  With ``rotary_dim`` the tokens' ``positions`` ([B, T], or [T]
        for all alike) have to be given."""
        if self.rotary_dim and positions is None:
            raise ValueError("a rotated layer needs the tokens' positions")
        mixed, gate, g, beta = self._project(x)
        mixed = causal_conv1d_step(mixed, self.conv_weight, None, state.conv, activation="silu",
                                   state_indices=state_indices)
        q, k, v = self._heads(mixed, positions)
        o = gated_delta_step(q, k, v, g, beta, state.delta, state_indices=state_indices)
        return self._finish(o, gate)

    def extra_repr(self) -> str:
        return (f"key_heads={self.key_heads}, value_heads={self.value_heads}, "
                f"key_dim={self.key_dim}, value_dim={self.value_dim}, taps={self.taps}, "
                f"rotary_dim={self.rotary_dim}")
