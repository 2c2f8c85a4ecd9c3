"""Calls that the sequence operators refuse, without a GPU: nothing runs before the refusal."""
import pytest
import torch
from torch.autograd import forward_ad as fwAD

import tdc_sequence as S


def test_forward_mode_derivatives():
    # a dual tensor of any argument that has gradients: no result without its tangent
    x, w = torch.randn(2, 5, 64).half(), torch.randn(4, 64).half()
    q, v = torch.randn(1, 5, 2, 64).half(), torch.randn(1, 5, 2, 64).half()
    g, s = -torch.rand(1, 5, 2), torch.zeros(1, 2, 64, 64)
    with fwAD.dual_level():
        d = lambda t: fwAD.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: S.causal_conv1d(d(x), w),
                     lambda: S.causal_conv1d(x, d(w)),
                     lambda: S.causal_conv1d_step(d(x), w, None, torch.zeros(2, 3, 64).half()),
                     lambda: S.qk_norm_rope(q, d(q)),
                     lambda: S.qk_norm_rope(q, q, d(torch.ones(64).half())),
                     lambda: S.gated_delta_rule(q, q, d(v), g, g),
                     lambda: S.gated_delta_rule(q, q, v, g, g, initial_state=d(s)),
                     lambda: S.gated_delta_step(q, q, v, d(g), g, s)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="CUDA"):       # others go on to their checks
            S.causal_conv1d(x, w)


def test_rotated_layer_without_positions():
    # its states hold keys turned by their positions: 0 .. T-1 cannot be right for more tokens
    m = S.GatedDeltaMixer(64, 1, key_dim=64, value_dim=64, rotary_dim=32, max_positions=100)
    x, state = torch.randn(2, 3, 64).bfloat16(), m.new_state(2)
    with pytest.raises(ValueError, match="positions"):
        m.step(x, state)
    with pytest.raises(ValueError, match="positions"):
        m(x, state)
    with pytest.raises(ValueError, match="positions"):
        m(x[:1], cu_seqlens=torch.tensor([0, 1, 3]), output_state=True)
    for call in (lambda: m.step(x, state, positions=torch.arange(3)),
                 lambda: m(x, output_state=True),
                 lambda: m(x[:1], cu_seqlens=torch.tensor([0, 1, 3]))):
        with pytest.raises(RuntimeError, match="CUDA"):       # go on to the operators
            call()
    plain = S.GatedDeltaMixer(64, 1, key_dim=64, value_dim=64)
    with pytest.raises(RuntimeError, match="CUDA"):
        plain.step(x, plain.new_state(2))
