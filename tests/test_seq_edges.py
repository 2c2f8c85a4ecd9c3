"""Calls of the sequence operators at their edges: no eps, NaN and infinities, states that
an earlier call saved, forward-mode derivatives, views without rows, long runs."""
import pytest
import torch

import seq_reference as R
import tdc_sequence as S
import test_seq_delta as D
import test_seq_qk as Q


@pytest.mark.gpu
@pytest.mark.parametrize("H,HK,dim", [(4, 1, 128), (1, 1, 64), (3, 0, 64), (0, 1, 128), (9, 2, 32)])
@pytest.mark.parametrize("norm", ["rms", "l2"])
def test_weight_gradients_without_eps(H, HK, dim, norm):
    # totals of heads that leave some lanes of a warp without one: what they hold counts nowhere
    c = Q._case(2, 5, H, HK, dim, 16, "bf16", True, "batch", seed=H)
    Q._check(Q._run(c, norm, False, 0.0), Q._want(c, norm, False, 0.0))
