"""Calls that the sequence operators refuse, without a GPU: nothing runs before the refusal."""
import os

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


def test_sizes_whose_workspace_has_no_number():
    # products of sizes that pass 64 bits: refused, not a small or negative size
    import test_seq_host as H
    import ctypes as C
    lib = C.CDLL(os.path.join(H.REPO, "tma-depthwise-conv_b200", "libtdc_sm100.so"))
    sizes = ("tdc_conv1d_bwd_workspace", "tdc_delta_fwd_workspace", "tdc_delta_bwd_workspace")
    for f in sizes:
        getattr(lib, f).restype = C.c_int64
    large, p = H.CODES["TDC_ERR_TOO_LARGE"], C.c_void_p(H.P)
    big = 1 << 40
    for over in (dict(B=big, T=big), dict(B=1 << 20, T=1 << 20, C=1 << 20),
                 dict(B=1, cu_seqlens=H.P, num_seqs=1 << 62)):
        a = H._conv(**over)
        assert lib.tdc_conv1d_bwd_workspace(C.byref(a)) == large
        assert lib.tdc_conv1d_fwd(C.byref(a), None) == large
    for over in (dict(B=1 << 24, T=1 << 36, HV=65534, V=256, K=128, v_sb=0, v_st=0),
                 dict(B=1 << 24, T=1, HV=65534, V=256), dict(B=1 << 20, T=1 << 30)):
        a = H._delta(**over)
        for f in sizes[1:]:
            assert getattr(lib, f)(C.byref(a)) == large
        assert lib.tdc_delta_fwd(C.byref(a), p, C.c_int64(1 << 40), None) == large


def test_workspace_error_names_no_other_operation():
    import test_seq_host as H
    import ctypes as C
    lib = C.CDLL(os.path.join(H.REPO, "tma-depthwise-conv_b200", "libtdc_sm100.so"))
    lib.tdc_strerror.restype = C.c_char_p
    text = lib.tdc_strerror(H.CODES["TDC_ERR_WORKSPACE"]).decode()
    assert "workspace" in text and "dwconv3x3" not in text
