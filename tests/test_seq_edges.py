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


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["q", "k", "v", "g", "beta"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("T,t", [(100, 1), (100, 37), (100, 63), (100, 64), (100, 99), (1700, 901)])
@pytest.mark.parametrize("K,V,dtype", [(64, 64, "bf16"), (128, 256, "fp16")])
def test_what_is_not_finite_reaches_no_token_before_it(name, bad, T, t, K, V, dtype):
    # as in the recurrence: a padded batch may hold anything behind its last token.
    # (1700 tokens are walked in segments; a decay is never +inf)
    bad = float("nan") if name == "g" else bad
    c = D._case(2, T, 1, 2, K, V, dtype, state=True, beta_f32=True)
    a = {n: c[n].detach().clone().cuda() for n in ("q", "k", "v", "g", "beta")}
    run = lambda: S.gated_delta_rule(*a.values(), initial_state=c["state"].cuda())  # noqa: E731
    want = run()
    a[name][(0, t) + {"q": (0, 5), "k": (0, 5), "v": (1, 7), "g": (1,), "beta": (1,)}[name]] = bad
    got = run()
    reached = torch.zeros_like(got, dtype=torch.bool)    # head 0 shares q and k with head 1
    heads, channels = {"q": (slice(None),) * 2, "k": (slice(None),) * 2}.get(name, (1, slice(None)))
    reached[0, slice(t, t + 1 if name == "q" else None), heads, 7 if name == "v" else channels] = True
    assert torch.equal(got[~reached], want[~reached])
    assert not torch.isfinite(got[reached]).any()


@pytest.mark.gpu
def test_states_saved_for_a_backward_pass_and_stepped_since():
    # as after any in-place operation: the backward pass refuses instead of using the new state
    x = torch.randn(2, 5, 64, device="cuda").half()
    w = torch.randn(4, 64, device="cuda").half().requires_grad_()
    pool = torch.randn(2, 3, 64, device="cuda").half()
    y = S.causal_conv1d(x, w, initial_state=pool)
    with torch.no_grad():
        S.causal_conv1d_step(x[:, :1], w, None, pool)
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.sum().backward()
    c = D._case(2, 5, 1, 1, 64, 64)
    a = [c[n].cuda() for n in ("q", "k", "v", "g", "beta")]
    pool = torch.randn(2, 1, 64, 64, device="cuda")
    o = S.gated_delta_rule(*(t.clone().requires_grad_() for t in a), initial_state=pool)
    S.gated_delta_step(*(t[:, :1] for t in a), pool)
    with pytest.raises(RuntimeError, match="inplace operation"):
        o.sum().backward()
    with torch.inference_mode():
        pool = torch.randn(2, 1, 64, 64, device="cuda")
    S.gated_delta_step(*(t[:, :1] for t in a), pool)          # (has no version)


@pytest.mark.gpu
def test_views_without_rows():
    # strides of a view that has no element are no reason to refuse it
    odd = lambda *s: torch.randn(*s, 68, device="cuda").half()[..., :64]  # noqa: E731
    w, state = torch.randn(4, 64, device="cuda").half(), torch.randn(2, 3, 64, device="cuda").half()
    y, last = S.causal_conv1d(odd(2, 5)[:, :0], w, initial_state=state, output_final_state=True)
    assert y.shape == (2, 0, 64) and torch.equal(last, state)
    assert S.causal_conv1d_step(odd(2, 5)[:, :0], w, None, state).shape == (2, 0, 64)
    q, k = S.qk_norm_rope(odd(2, 5, 3)[:, :0], odd(2, 5, 1)[:, :0])
    assert q.shape == (2, 0, 3, 64) and k.shape == (2, 0, 1, 64)
    q, k = S.qk_norm_rope(torch.randn(2, 5, 1, 64, device="cuda").half(), odd(2, 5, 3)[:, :, :0])
    assert k.shape == (2, 5, 0, 64)
    q, g = odd(2, 5, 2)[:, :0], torch.rand(2, 5, 2, device="cuda")[:, :0]
    pool = torch.randn(2, 2, 64, 64, device="cuda")
    o, last = S.gated_delta_rule(q, q, q, g, g, initial_state=pool, output_final_state=True)
    assert o.shape == q.shape and torch.equal(last, pool)
    assert S.gated_delta_step(q, q, q, g, g, pool).shape == q.shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,T,H,HV,K,V", [(4, 1, 2, 4, 128, 128), (2, 3, 1, 2, 64, 256)])
def test_steps_with_fp32_betas(B, T, H, HV, K, V, dtype):
    c = D._case(B, T, H, HV, K, V, dtype, state=True, beta_f32=True, seed=T)
    pool = c["state"].clone().cuda()
    names = ("q", "k", "v", "g", "beta")
    o = S.gated_delta_step(*(c[n].cuda() for n in names), pool)
    want, final = R.delta(*(c[n].double() for n in names), K ** -0.5, c["state"].double(), None)
    R.close(o, want, D.STEP * want.abs().max().item(), "o")
    R.close(pool, final, D.STEP * final.abs().max().item(), "state")


@pytest.mark.gpu
@pytest.mark.parametrize("T,t", [(100, 37), (200, 70), (200, 128)])
@pytest.mark.parametrize("K,V,dtype", [(64, 64, "bf16"), (128, 256, "fp16")])
def test_gradients_before_a_value_that_is_not_finite(T, t, K, V, dtype):
    # a loss that takes nothing from token t on: what stands there does not reach the
    # gradients before it (values enter no gradient of the state)
    c = D._case(2, T, 1, 2, K, V, dtype, state=True, beta_f32=True)
    c["do"][:, t:] = 0
    want = D._run(c, final=False)
    c["v"] = c["v"].detach().clone()
    c["v"][0, t:, 1, 7] = float("nan")
    c["v"][1, t:] = float("inf")
    got = D._run(c, final=False)
    for n in ("dq", "dk", "dv", "dg", "dbeta"):
        assert torch.equal(got[n][:, :t], want[n][:, :t]), n
    assert torch.equal(got["dstate"], want["dstate"])
