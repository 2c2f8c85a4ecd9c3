"""The causal depthwise convolution against its definition in fp64.

Tolerance: a value is a sum of K products that are exact in fp32, then bias and
SiLU, so it is off by its own rounding plus at most (K + 4) fp32 roundings of
the sum's largest term and the error of exp and the division (2^-20 of the
value): below 2^-18 of the largest magnitude.  A gradient of the weights is a
sum over all rows, in fp32: rows * 2^-24 of the largest term, below 2^-12 of the
largest result at these sizes."""
import pytest
import torch

import seq_reference as R
import tdc_sequence as S

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _case(B, T, C, K, dtype, bias, state, cu, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = B if cu is None else len(cu) - 1
    rnd = lambda *s: torch.randn(*s, generator=g).to(DT[dtype])  # noqa: E731
    return dict(x=rnd(B, T, C), w=rnd(K, C) * K ** -0.5, bias=rnd(C) if bias else None,
                state=rnd(n, K - 1, C) if state else None, dy=rnd(B, T, C), df=rnd(n, K - 1, C),
                cu=cu)


def _run(c, act, final=True, grads=True, cu_dtype=torch.int32):
    dev = {k: t.cuda() if isinstance(t, torch.Tensor) else t for k, t in c.items()}
    leaves = {k: dev[k].requires_grad_(grads) for k in ("x", "w", "bias", "state")
              if dev[k] is not None}
    cu = None if c["cu"] is None else torch.tensor(c["cu"], dtype=cu_dtype, device="cuda")
    out = S.causal_conv1d(dev["x"], dev["w"], dev["bias"], act, dev["state"], cu, final)
    y, f = out if final else (out, None)
    got = {"y": y, "final": f}
    if grads:
        outs, gs = ([y, f], [dev["dy"], dev["df"]]) if final else ([y], [dev["dy"]])
        got.update(zip(["d" + k for k in leaves], torch.autograd.grad(outs, list(leaves.values()), gs)))
    return got


def _want(c, act, final=True):
    ref = {k: t.double().requires_grad_() if isinstance(t, torch.Tensor) else t
           for k, t in c.items()}
    leaves = {k: ref[k] for k in ("x", "w", "bias", "state") if ref[k] is not None}
    y, f = R.conv(ref["x"], ref["w"], ref["bias"], act, ref["state"], c["cu"])
    loss = (y * c["dy"].double()).sum() + ((f * c["df"].double()).sum() if final else 0)
    grads = torch.autograd.grad(loss, list(leaves.values()), allow_unused=True)
    want = {"y": y, "final": f if final else None}
    want.update(zip(["d" + k for k in leaves],
                    [torch.zeros_like(t) if g is None else g for t, g in zip(leaves.values(), grads)]))
    return want


def _check(got, want):
    assert set(got) == set(want)
    for k, w in want.items():
        if w is None:
            assert got[k] is None
            continue
        top = w.abs().max().item() if w.numel() else 0.0
        R.close(got[k], w, (2 ** -12 if k in ("dw", "dbias") else 2 ** -18) * top + 1e-30, k)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("K", [2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("act,bias,state", [("silu", True, True), ("none", False, False)])
def test_taps(K, dtype, act, bias, state):
    c = _case(2, 37, 72, K, dtype, bias, state, None)
    _check(_run(c, act), _want(c, act))


@pytest.mark.parametrize("B,T,C", [(1, 1, 8), (3, 1, 64), (2, 2, 16), (1, 3, 256), (1, 130, 8),
                                   (2, 65, 264), (1, 513, 40), (5, 17, 520)])
@pytest.mark.parametrize("state", [False, True])
def test_sizes(B, T, C, state):
    c = _case(B, T, C, 4, "bf16", True, state, None, seed=T)
    _check(_run(c, "silu"), _want(c, "silu"))


@pytest.mark.parametrize("cu", [[0, 1, 3, 3, 20, 52, 53, 100], [0, 0, 0, 64], [0, 100], [3, 40, 90],
                                [0, 0], [0, 17, 34, 51, 68, 85, 100, 100, 100]])
@pytest.mark.parametrize("state,dtype", [(True, "bf16"), (False, "fp16")])
def test_packed(cu, state, dtype):
    # [3, 40, 90] leaves rows in front and behind without a sequence: zeros
    c = _case(1, 100, 48, 4, dtype, True, state, cu, seed=len(cu))
    _check(_run(c, "silu", cu_dtype=torch.int64 if state else torch.int32), _want(c, "silu"))


@pytest.mark.parametrize("B,T,C,cu", [(1, 5000, 1024, None), (3, 1700, 1024, None),
                                      (1, 5000, 1024, [2, 3, 9, 9, 17, 40, 1000, 1001, 1007, 2500, 4321, 4990]),
                                      (1, 5000, 1024, [0, 8, 12, 16, 20, 21, 22, 23, 24, 36, 4996, 5000])])
@pytest.mark.parametrize("K,dtype,state", [(2, "bf16", True), (4, "fp16", False), (8, "bf16", True)])
def test_forward_in_runs_of_several_rows(B, T, C, cu, K, dtype, state):
    c = _case(B, T, C, K, dtype, True, state, cu, seed=K)
    got = _run(c, "silu", grads=False)
    y, f = R.conv(*(None if c[n] is None else c[n].double() for n in ("x", "w", "bias")), "silu",
                  None if c["state"] is None else c["state"].double(), cu)
    _check(got, {"y": y, "final": f})


def test_no_rows_gives_the_state_back():
    c = _case(2, 0, 16, 4, "fp16", True, True, None)
    got = _run(c, "silu")
    assert got["y"].shape == (2, 0, 16)
    assert torch.equal(got["final"].cpu(), c["state"].detach())
    assert torch.equal(got["dstate"].cpu(), c["df"]) and not got["dw"].any()


def test_without_gradients_and_without_final_state():
    c = _case(2, 50, 64, 4, "bf16", False, False, None)
    _check(_run(c, "silu", final=False), _want(c, "silu", final=False))
    with_grad = _run(c, "silu", final=False)["y"]
    with torch.no_grad():
        assert torch.equal(_run(c, "silu", grads=False)["y"], with_grad)


def test_strided_input_and_expanded_gradient():
    wide = torch.randn(2, 60, 3 * 64, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    x = wide[..., 64:128]
    w = torch.randn(4, 64).bfloat16().cuda()
    y = S.causal_conv1d(x, w, activation="silu")
    assert torch.equal(y, S.causal_conv1d(x.contiguous(), w, activation="silu"))
    odd = torch.randn(2, 60, 65).bfloat16().cuda()[..., 1:]     # rows that are not aligned
    assert torch.equal(S.causal_conv1d(odd, w), S.causal_conv1d(odd.contiguous(), w))
    xr = x.detach().clone().requires_grad_()
    S.causal_conv1d(xr, w).sum().backward()                      # a gradient of stride 0
    want = torch.autograd.grad(S.causal_conv1d(xr, w), xr, torch.ones_like(xr))[0]
    assert torch.equal(xr.grad, want)


def test_inputs_far_behind_32_bits():
    # rows whose offsets pass 2^31 elements, by stride
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    big = torch.zeros((1 << 32) + 4096, dtype=torch.float16, device="cuda")
    x = big.as_strided((2, 33, 64), (1 << 32, 64, 1))
    x.copy_(torch.randn(2, 33, 64))
    w = torch.randn(4, 64).half().cuda()
    assert torch.equal(S.causal_conv1d(x, w), S.causal_conv1d(x.contiguous(), w))


def test_nan_outside_the_sequences_and_in_a_neighbour():
    cu = [3, 40, 70, 90]
    c = _case(1, 100, 16, 4, "bf16", True, True, cu)
    want = _run(c, "silu")
    bad = {k: t.detach().clone() if isinstance(t, torch.Tensor) else t for k, t in c.items()}
    for k in ("x", "dy"):
        bad[k][0, :3] = float("nan")
        bad[k][0, 90:] = float("nan")
    got = _run(bad, "silu")                      # rows that no sequence owns are not used
    for k in want:
        assert torch.equal(got[k], want[k]), k
    bad["x"][0, 40:70] = float("nan")
    got = _run(bad, "silu")
    for lo, hi in ((0, 40), (70, 100)):          # a sequence's NaN stays its own
        assert torch.equal(got["y"][0, lo:hi], want["y"][0, lo:hi])
        assert torch.equal(got["dx"][0, lo:hi], want["dx"][0, lo:hi])


def test_infinities_stay_in_their_channel_and_reach():
    x = torch.randn(1, 40, 16, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    w = torch.rand(4, 16).bfloat16().cuda() + 0.5
    want = S.causal_conv1d(x, w)
    bad = x.clone()
    bad[0, 10, 3] = float("inf")
    bad[0, 20, 5] = float("nan")
    got = S.causal_conv1d(bad, w)
    touched = torch.zeros(40, 16, dtype=torch.bool)
    touched[10:14, 3] = True
    touched[20:24, 5] = True
    assert torch.equal(got[0][~touched.cuda()], want[0][~touched.cuda()])
    assert not torch.isfinite(got[0][touched.cuda()]).any()


@pytest.mark.parametrize("B,T,C,K", [(1, 1, 8, 2), (5, 1, 264, 4), (3, 2, 64, 4), (2, 7, 40, 5),
                                     (130, 1, 1032, 4), (4, 1, 48, 8)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_step_continues_a_sequence(B, T, C, K, dtype):
    c = _case(B, T, C, K, dtype, True, True, None, seed=B)
    slots = B + 3
    idx = torch.randperm(slots, generator=torch.Generator().manual_seed(1))[:B]
    pool = torch.randn(slots, K - 1, C).to(DT[dtype])
    before = pool.clone()
    pool = pool.cuda()
    y = S.causal_conv1d_step(c["x"].cuda(), c["w"].cuda(), c["bias"].cuda(), pool, "silu",
                             idx.to(torch.int32 if B % 2 else torch.int64).cuda())
    want, final = R.conv(c["x"].double(), c["w"].double(), c["bias"].double(), "silu",
                         before[idx].double(), None)
    R.close(y, want, 2 ** -18 * want.abs().max().item(), "y")
    before[idx] = final.to(DT[dtype])
    assert torch.equal(pool.cpu(), before)                       # the other slots as they were


def test_step_matches_the_whole_sequence():
    c = _case(2, 20, 64, 4, "bf16", True, True, None)
    whole, final = S.causal_conv1d(c["x"].cuda(), c["w"].cuda(), c["bias"].cuda(), "silu",
                                   c["state"].cuda(), output_final_state=True)
    state = c["state"].cuda()
    got = [S.causal_conv1d_step(c["x"][:, t].cuda(), c["w"].cuda(), c["bias"].cuda(), state, "silu")
           for t in range(20)]
    assert torch.equal(torch.stack(got, 1), whole) and torch.equal(state, final)


def test_step_padding_bad_and_repeated_slots():
    x = torch.randn(6, 1, 16).half().cuda()
    w = torch.randn(4, 16).half().cuda()
    pool = torch.randn(3, 3, 16).half().cuda()
    before = pool.clone()
    y = S.causal_conv1d_step(x, w, None, pool, "none",
                             torch.tensor([2, -1, 2, 3, 0, 1 << 30], dtype=torch.int32).cuda())
    alone = before.clone()
    want = S.causal_conv1d_step(x[[0, 4]], w, None, alone, "none", torch.tensor([2, 0]).cuda())
    assert torch.equal(y[[0, 4]], want) and torch.equal(pool, alone)
    assert not y[1].any() and torch.isnan(y[[2, 3, 5]]).all()
    assert torch.equal(pool[1], before[1])


def test_captured_and_on_another_stream():
    c = _case(2, 90, 64, 4, "bf16", True, False, None)
    x, w, b = (c[k].cuda() for k in ("x", "w", "bias"))
    want = S.causal_conv1d(x, w, b, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(S.causal_conv1d(x, w, b, "silu"), want)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = S.causal_conv1d(x, w, b, "silu")
    x.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, S.causal_conv1d(x, w, b, "silu"))


def test_gradients_are_the_same_every_run():
    c = _case(4, 700, 256, 4, "bf16", True, True, None)
    a, b = _run(c, "silu"), _run(c, "silu")
    for k in a:
        assert torch.equal(a[k], b[k]), k
