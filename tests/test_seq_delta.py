"""The gated delta rule against the recurrence in fp64.

Tolerance of the chunked form: every fp32 operand of a matrix instruction is
split into two bf16 parts that keep it to 2^-17, and the product of the two
remainders (2^-18) is left out.  A value comes through at most 8 such products
one after another; unit keys keep their sums from growing, and a factor of 2
allows for cancellation: 8 * 2^-17 * 2 = 2^-13 of the tensor's largest value,
plus the output's own rounding.  The recurrent form works in fp32 throughout:
its sums over K = 128 and a few tokens stay below 2^-18."""
import os
import subprocess
import sys

import pytest
import torch

import seq_reference as R
import tdc_sequence as S

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
CHUNKED, STEP = 2 ** -13, 2 ** -18


def _case(B, T, H, HV, K, V, dtype="bf16", state=False, cu=None, beta_f32=False, seed=0, rate=1.0):
    g = torch.Generator().manual_seed(seed)
    n = B if cu is None else len(cu) - 1
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    unit = lambda x: (x / x.norm(dim=-1, keepdim=True)).to(DT[dtype])  # noqa: E731
    return dict(q=unit(rnd(B, T, H, K)), k=unit(rnd(B, T, H, K) + 0.7 * rnd(B, 1, H, K)),
                v=rnd(B, T, HV, V).to(DT[dtype]),
                g=-rate * torch.nn.functional.softplus(rnd(B, T, HV) - 2),
                beta=torch.sigmoid(rnd(B, T, HV)).to(torch.float32 if beta_f32 else DT[dtype]),
                state=0.3 * rnd(n, HV, K, V) if state else None, do=rnd(B, T, HV, V).to(DT[dtype]),
                df=0.3 * rnd(n, HV, K, V), cu=cu)


LEAVES = ("q", "k", "v", "g", "beta", "state")


def _run(c, scale=None, final=True, cu_dtype=torch.int32):
    d = {k: t.cuda() if isinstance(t, torch.Tensor) else t for k, t in c.items()}
    leaves = {k: d[k].requires_grad_() for k in LEAVES if d[k] is not None}
    cu = None if c["cu"] is None else torch.tensor(c["cu"], dtype=cu_dtype, device="cuda")
    out = S.gated_delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], scale, d["state"], cu, final)
    o, f = out if final else (out, None)
    grads = torch.autograd.grad([o, f] if final else [o], list(leaves.values()),
                                [d["do"], d["df"]] if final else [d["do"]])
    return {"o": o, "final": f, **{"d" + k: x for k, x in zip(leaves, grads)}}


def _want(c, scale=None, final=True):
    d = {k: t.double() if isinstance(t, torch.Tensor) else t for k, t in c.items()}
    leaves = {k: d[k].requires_grad_() for k in LEAVES if d[k] is not None}
    scale = c["q"].shape[-1] ** -0.5 if scale is None else scale
    o, f = R.delta(d["q"], d["k"], d["v"], d["g"], d["beta"], scale, d["state"], c["cu"])
    loss = (o * d["do"]).sum() + ((f * d["df"]).sum() if final else 0)
    loss = loss + 0 * sum(t.sum() for t in leaves.values())      # (a graph even without a row)
    grads = torch.autograd.grad(loss, list(leaves.values()), allow_unused=True)
    grads = [torch.zeros_like(t) if x is None else x for t, x in zip(leaves.values(), grads)]
    return {"o": o, "final": f if final else None, **{"d" + k: x for k, x in zip(leaves, grads)}}


def _check(got, want, tol=CHUNKED):
    assert set(got) == set(want)
    for k, w in want.items():
        if w is None:
            assert got[k] is None
            continue
        top = w.abs().max().item() if w.numel() else 0.0
        R.close(got[k], w, tol * top + 1e-30, k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("K,V", [(64, 64), (64, 128), (64, 256), (128, 64), (128, 128), (128, 256)])
def test_head_sizes(K, V, dtype):
    c = _case(1, 100, 2, 2, K, V, dtype, state=True)
    _check(_run(c), _want(c))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 15, 16, 63, 64, 65, 127, 128, 129, 200])
@pytest.mark.parametrize("state", [False, True])
def test_lengths(T, state):
    c = _case(2, T, 1, 2, 64, 64, "bf16", state=state, seed=T)
    _check(_run(c), _want(c))


@pytest.mark.gpu
@pytest.mark.parametrize("H,HV", [(1, 1), (1, 4), (2, 6), (3, 3)])
def test_shared_key_heads(H, HV):
    c = _case(2, 70, H, HV, 128, 64, "bf16", state=True, beta_f32=True, seed=HV)
    _check(_run(c), _want(c))


@pytest.mark.gpu
@pytest.mark.parametrize("cu", [[0, 1, 3, 3, 20, 85, 86, 150], [0, 0, 0, 150], [0, 150], [5, 70, 140],
                                [0, 0], [0, 64, 128, 150, 150]])
@pytest.mark.parametrize("state,dtype", [(True, "bf16"), (False, "fp16")])
def test_packed(cu, state, dtype):
    # [5, 70, 140] leaves rows in front and behind without a sequence: zeros
    c = _case(1, 150, 1, 2, 64, 64, dtype, state=state, cu=cu, seed=len(cu))
    _check(_run(c, cu_dtype=torch.int64 if state else torch.int32), _want(c))


@pytest.mark.gpu
def test_many_sequences_in_one_plan():
    lens = [(i * 7) % 5 for i in range(2500)]          # more than one block's sweep of offsets
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    c = _case(1, cu[-1], 1, 1, 64, 64, "bf16", cu=cu)
    d = {k: t.cuda() if isinstance(t, torch.Tensor) else t for k, t in c.items()}
    got, f = S.gated_delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"],
                                cu_seqlens=torch.tensor(cu).cuda(), output_final_state=True)
    want, wf = R.delta(*(c[k].double() for k in ("q", "k", "v", "g", "beta")), 64 ** -0.5, None, cu)
    R.close(got, want, CHUNKED * want.abs().max().item(), "o")
    R.close(f, wf, CHUNKED * wf.abs().max().item(), "final")


@pytest.mark.gpu
@pytest.mark.parametrize("walks", [1, 80, 160])
def test_every_block_size_of_the_walk(walks):
    # 2, 4 and 8 warps a block, by the number of sequences and heads
    c = _case(walks, 66, 1, 1, 64, 128, "bf16", state=True, seed=walks)
    _check(_run(c), _want(c))


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,H,HV,K,V", [(1, 1601, 1, 1, 64, 64), (2, 2048, 1, 2, 128, 128),
                                          (1, 1537, 2, 2, 64, 256), (1, 4000, 1, 1, 128, 64),
                                          (1, 1984, 16, 32, 64, 64)])
@pytest.mark.parametrize("state,dtype", [(True, "bf16"), (False, "fp16")])
def test_long_sequences_in_segments(B, T, H, HV, K, V, state, dtype):
    c = _case(B, T, H, HV, K, V, dtype, state=state, seed=T)
    c["g"] *= 0.05                                   # states that last over several segments
    args = [c[k] for k in ("q", "k", "v", "g", "beta")]
    o, f = S.gated_delta_rule(*(t.cuda() for t in args), None,
                              c["state"].cuda() if state else None, None, True)
    # the recurrence in fp64 (on the GPU: thousands of tokens)
    d = [t.double().cuda() for t in args]
    q, k = (t.repeat_interleave(HV // H, 2) for t in d[:2])
    s = (c["state"].double().cuda() if state else torch.zeros(B, HV, K, V, dtype=torch.float64).cuda())
    rows = []
    for t in range(T):
        s = s * d[3][:, t].exp()[..., None, None]
        u = (d[2][:, t] - torch.einsum("bhkv,bhk->bhv", s, k[:, t])) * d[4][:, t][..., None]
        s = s + k[:, t][..., None] * u[:, :, None, :]
        rows.append(torch.einsum("bhkv,bhk->bhv", s, q[:, t]) * K ** -0.5)
    want = torch.stack(rows, 1)
    R.close(o, want, CHUNKED * want.abs().max().item(), "o")
    R.close(f, s, CHUNKED * s.abs().max().item(), "final")
    # the same without segments: a packed batch of the sequences
    cu = torch.arange(B + 1).cuda() * T
    o2, f2 = S.gated_delta_rule(*(t.cuda().flatten(0, 1)[None] for t in args), None,
                                c["state"].cuda() if state else None, cu, True)
    assert (f2 - f).abs().max().item() <= 2 * CHUNKED * s.abs().max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,H,HV,K,V,dtype,cu", [
    (3, 200, 14, 28, 64, 64, "bf16", None),               # 168 chunks and key heads
    (2, 640, 16, 16, 128, 64, "fp16", None),              # 320, several a block
    (1, 330, 30, 30, 128, 256, "bf16", None),             # 180, 16 tiles of channels a head
    (1, 260, 31, 31, 64, 128, "fp16", [0, 1, 1, 70, 200, 200, 255]),
    (1, 40, 8, 16, 64, 64, "bf16", [min(i, 40) for i in range(60)]),  # most have no rows
    (1, 64, 1, 8, 128, 128, "fp16", None)])               # one of 8 heads
def test_gradients_of_more_chunks_and_heads_than_blocks(B, T, H, HV, K, V, dtype, cu):
    c = _case(B, T, H, HV, K, V, dtype, state=True, cu=cu, seed=T)
    _check(_run(c), _want(c))


@pytest.mark.gpu
def test_no_rows_gives_the_state_back():
    c = _case(2, 0, 1, 2, 64, 64, "bf16", state=True)
    got = _run(c)
    assert got["o"].shape == (2, 0, 2, 64)
    assert torch.equal(got["final"].cpu(), c["state"].detach())
    assert torch.equal(got["dstate"].cpu(), c["df"])


@pytest.mark.gpu
def test_decays_of_every_size():
    # rates from none to a reset at a token, -inf among them: exp(-inf) = 0
    c = _case(1, 130, 1, 3, 64, 64, "bf16", state=True, rate=0.0)
    c["g"][0, :, 1] = torch.where(torch.arange(130) % 13 == 5, -80.0, -0.01)
    c["g"][0, :, 2] = -30.0
    _check(_run(c), _want(c))
    c["g"][0, 77, 0] = -float("inf")
    got = _run(c)
    ref = dict(c, g=c["g"].clamp_min(-200.0))
    _check(got, _want(ref))


@pytest.mark.gpu
def test_beta_zero_leaves_the_state_and_one_replaces():
    c = _case(1, 90, 1, 2, 64, 64, "bf16", state=True, beta_f32=True)
    c["beta"][0, :, 0] = 0.0
    c["beta"][0, :, 1] = 1.0
    _check(_run(c), _want(c))


@pytest.mark.gpu
def test_equal_keys():
    # one key for all tokens: the triangular system is as full as it gets
    c = _case(1, 128, 1, 1, 64, 64, "bf16")
    c["k"][:] = c["k"][:, :1]
    _check(_run(c), _want(c))


@pytest.mark.gpu
@pytest.mark.parametrize("K,V", [(64, 64), (128, 128)])
def test_decay_of_a_first_token_without_state_has_no_effect(K, V):
    # nothing stands behind it: its gradient is exactly zero, not a rounding
    c = _case(3, 1, 2, 4, K, V, "bf16")
    got = _run(c)
    assert not got["dg"].any() and got["dv"].any()
    c = _case(1, 150, 1, 2, K, V, "bf16", cu=[0, 1, 2, 70, 71, 150])
    got = _run(c)
    assert not got["dg"][0, [0, 1, 2, 70, 71]].any() and got["dg"][0, 3:70].any()


@pytest.mark.gpu
def test_scale_and_no_final_state():
    c = _case(1, 80, 1, 1, 128, 64, "fp16")
    _check(_run(c, scale=1.0, final=False), _want(c, scale=1.0, final=False))


@pytest.mark.gpu
def test_strided_inputs():
    c = _case(2, 70, 2, 2, 64, 64, "bf16")
    packed = torch.randn(2, 70, 6 * 64).bfloat16().cuda()
    q, k, v = (t.view(2, 70, 2, 64) for t in packed.split(128, -1))
    k = k / 8
    g, beta = c["g"].cuda(), c["beta"].cuda()
    a = S.gated_delta_rule(q, k, v, g, beta)
    b = S.gated_delta_rule(q.contiguous(), k.contiguous(), v.contiguous(), g, beta)
    assert torch.equal(a, b)
    gates = torch.stack([g, g], -1)[..., 0]                     # heads two apart
    assert torch.equal(S.gated_delta_rule(q, k, v, gates, beta), a)


@pytest.mark.gpu
def test_nan_stays_in_its_sequence_and_head():
    c = _case(2, 100, 1, 2, 64, 64, "bf16")
    d = {k: t.cuda() if isinstance(t, torch.Tensor) else t for k, t in c.items()}
    args = lambda: (d["q"], d["k"], d["v"], d["g"], d["beta"])  # noqa: E731
    want = S.gated_delta_rule(*args())
    d["v"] = d["v"].clone()
    d["v"][0, 30, 1, 7] = float("nan")
    got = S.gated_delta_rule(*args())
    clean = torch.ones(2, 100, 2, 64, dtype=torch.bool)
    clean[0, :, 1, 7] = False                                    # value channels do not mix
    assert torch.equal(got[clean.cuda()], want[clean.cuda()])
    assert torch.isnan(got[0, 64:, 1, 7]).all()


@pytest.mark.gpu
def test_nan_outside_the_sequences_and_in_a_neighbour():
    # rows that no sequence owns are not read; one sequence's NaN stays its own, also
    # where it ends inside the next one's first chunk
    cu = [7, 40, 110, 131]
    c = _case(1, 140, 1, 2, 64, 64, "bf16", state=True, cu=cu)
    want = _run(c)
    bad = {k: t.detach().clone() if isinstance(t, torch.Tensor) else t for k, t in c.items()}
    for k in ("q", "k", "v", "g", "beta", "do"):
        bad[k][0, :7] = float("nan")
        bad[k][0, 131:] = float("nan")
        bad[k][0, 40:110] = float("nan")
    got = _run(bad)
    for k in ("o", "dq", "dk", "dv", "dg", "dbeta"):
        a, b = got[k][0], want[k][0]
        for lo, hi in ((0, 40), (110, 140)):
            assert torch.equal(a[lo:hi], b[lo:hi]), k
    for k in ("final", "dstate"):
        assert torch.equal(got[k][[0, 2]], want[k][[0, 2]]), k


@pytest.mark.gpu
def test_first_call_of_a_process_inside_a_capture():
    code = """
import sys; sys.path.insert(0, %r)
import torch, tdc_sequence as S
q = torch.randn(1, 100, 1, 64, device="cuda").bfloat16() / 8
v = torch.randn(1, 100, 1, 64, device="cuda").bfloat16()
g, b = -torch.rand(1, 100, 1, device="cuda"), torch.rand(1, 100, 1, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    o = S.gated_delta_rule(q, q, v, g, b)
    x = S.causal_conv1d(v.flatten(2), torch.ones(4, 64, device="cuda").bfloat16(), activation="silu")
graph.replay()
torch.cuda.synchronize()
assert torch.equal(o, S.gated_delta_rule(q, q, v, g, b)) and torch.isfinite(x).all()
""" % os.path.dirname(S.__file__)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.gpu
def test_no_second_derivatives():
    c = _case(1, 20, 1, 1, 64, 64)
    q, k, v, g, b = (c[n].cuda().requires_grad_() for n in ("q", "k", "v", "g", "beta"))
    o = S.gated_delta_rule(q, k, v, g, b)
    d, = torch.autograd.grad(o.float().square().sum(), v, create_graph=True)
    with pytest.raises(RuntimeError):
        d.float().sum().backward()


@pytest.mark.gpu
def test_gradients_match_differences():
    # central differences of the fp64 loss of the kernel's outputs; the final state
    # is fp32, so a step of 1/64 leaves its rounding far below the tolerance
    c = _case(1, 70, 1, 1, 64, 64, "bf16", state=True, beta_f32=True)
    d = {k: t.cuda() if isinstance(t, torch.Tensor) else t for k, t in c.items()}
    w = d["df"].double()
    def loss(**over):
        a = {**d, **over}
        _, f = S.gated_delta_rule(a["q"], a["k"], a["v"], a["g"], a["beta"], None, a["state"], None,
                                  True)
        return (f.double() * w).sum().item()
    for name in ("g", "beta", "state"):
        leaf = d[name].clone().requires_grad_()
        a = {**d, name: leaf}
        _, f = S.gated_delta_rule(a["q"], a["k"], a["v"], a["g"], a["beta"], None, a["state"], None,
                                  True)
        f.backward(d["df"])
        top = leaf.grad.abs().max().item()
        for i in range(0, leaf.numel(), leaf.numel() // 7):
            up, down = d[name].clone(), d[name].clone()
            up.view(-1)[i] += 1 / 64
            down.view(-1)[i] -= 1 / 64
            diff = (loss(**{name: up}) - loss(**{name: down})) * 32
            # the third derivatives are of the size of the first: 2^-12 / 6 of it, and
            # the outputs' error of 2^-13 over a difference of 2^-5
            assert abs(diff - leaf.grad.view(-1)[i].item()) < 0.02 * top + 1e-4, (name, i)


@pytest.mark.gpu
def test_same_bits_every_run_and_on_another_stream():
    c = _case(2, 300, 2, 4, 128, 128, "bf16", state=True)
    a = _run(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = _run(c)
    torch.cuda.synchronize()
    for k in a:
        assert torch.equal(a[k], b[k]), k


@pytest.mark.gpu
def test_captured_forward_and_backward():
    c = _case(2, 100, 1, 2, 64, 64, "bf16", state=True)
    d = {k: t.cuda() if isinstance(t, torch.Tensor) else t for k, t in c.items()}
    leaves = [d[k].requires_grad_() for k in LEAVES]
    def step():
        o, f = S.gated_delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], None, d["state"], None,
                                  True)
        return (o, f, *torch.autograd.grad([o, f], leaves, [d["do"], d["df"]]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        d["v"].mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,T,H,HV,K,V", [(1, 1, 1, 1, 64, 64), (5, 1, 2, 4, 128, 128),
                                          (3, 2, 1, 2, 128, 256), (2, 6, 2, 2, 64, 128)])
def test_step_continues_a_sequence(B, T, H, HV, K, V, dtype):
    c = _case(B, T, H, HV, K, V, dtype, seed=B)
    slots = B + 2
    idx = torch.randperm(slots, generator=torch.Generator().manual_seed(1))[:B]
    pool = torch.randn(slots, HV, K, V, generator=torch.Generator().manual_seed(2))
    before = pool.clone()
    pool = pool.cuda()
    o = S.gated_delta_step(*(c[k].cuda() for k in ("q", "k", "v", "g", "beta")), pool,
                           state_indices=idx.to(torch.int32 if B % 2 else torch.int64).cuda())
    want, final = R.delta(*(c[k].double() for k in ("q", "k", "v", "g", "beta")), K ** -0.5,
                          before[idx].double(), None)
    R.close(o, want, STEP * want.abs().max().item(), "o")
    R.close(pool[idx.cuda()], final, STEP * final.abs().max().item(), "state")
    rest = [i for i in range(slots) if i not in idx.tolist()]
    assert torch.equal(pool[rest].cpu(), before[rest])


@pytest.mark.gpu
def test_step_matches_the_whole_sequence():
    c = _case(2, 80, 1, 2, 128, 64, "bf16", state=True)
    d = {k: t.cuda() if isinstance(t, torch.Tensor) else t for k, t in c.items()}
    whole, final = S.gated_delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], None, d["state"],
                                      None, True)
    pool = d["state"].clone()
    got = torch.cat([S.gated_delta_step(*(d[k][:, t:t + 1] for k in ("q", "k", "v", "g", "beta")), pool)
                     for t in range(80)], 1)
    # both are off the truth by their tolerances, and both round
    top = whole.abs().max().item()
    assert (got.double() - whole.double()).abs().max().item() <= (CHUNKED + STEP + 2 ** -8) * top
    R.close(pool, final.double(), 2 * CHUNKED * final.abs().max().item(), "state")


@pytest.mark.gpu
def test_step_padding_bad_and_repeated_slots():
    c = _case(6, 1, 1, 2, 64, 64, "fp16")
    d = {k: t.cuda() if isinstance(t, torch.Tensor) else t for k, t in c.items()}
    pool = torch.randn(3, 2, 64, 64).cuda()
    before = pool.clone()
    names = ("q", "k", "v", "g", "beta")
    o = S.gated_delta_step(*(d[k] for k in names), pool,
                           state_indices=torch.tensor([2, -1, 2, 3, 0, 1 << 30]).cuda())
    alone = before.clone()
    want = S.gated_delta_step(*(d[k][[0, 4]] for k in names), alone,
                              state_indices=torch.tensor([2, 0]).cuda())
    assert torch.equal(o[[0, 4]], want) and torch.equal(pool, alone)
    assert not o[1].any() and torch.isnan(o[[2, 3, 5]]).all()
    assert torch.equal(pool[1], before[1])
