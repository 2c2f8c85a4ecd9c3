"""Norms of queries and keys with the position rotation, against fp64.

Tolerance: a value is its input times an inverse root (fp32, a few roundings of
2^-24 and rsqrt's 2^-22), a weight, and a rotation of two such products: below
2^-19 of the largest magnitude, plus the output's own rounding.  A weight's
gradient sums fp32 terms over all rows and heads: below 2^-12 of the largest
result at these sizes."""
import pytest
import torch

import seq_reference as R
import tdc_sequence as S

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _case(B, T, H, HK, D, rotary, dtype, weights, positions, seed=0, far=200):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g).to(DT[dtype])  # noqa: E731
    c = dict(q=rnd(B, T, H, D), k=rnd(B, T, HK, D), gq=rnd(B, T, H, D), gk=rnd(B, T, HK, D),
             qw=rnd(D) if weights else None, kw=rnd(D) if weights else None, cos=None, sin=None,
             positions=None)
    if rotary:
        c["cos"], c["sin"] = S.rotary_table(rotary, far + T)
        if positions == "batch":
            c["positions"] = torch.randint(0, far + T, (B, T), generator=g)
        elif positions == "row":
            c["positions"] = torch.arange(T, dtype=torch.int32) + far
    return c


def _run(c, norm, interleaved, eps=1e-6):
    d = {k: t.cuda() if t is not None else None for k, t in c.items()}
    leaves = {k: d[k].requires_grad_() for k in ("q", "k", "qw", "kw") if d[k] is not None}
    q, k = S.qk_norm_rope(d["q"], d["k"], d["qw"], d["kw"], norm, eps, d["cos"], d["sin"],
                          d["positions"], interleaved)
    grads = torch.autograd.grad([q, k], list(leaves.values()), [d["gq"], d["gk"]])
    return {"q": q, "k": k, **{"d" + n: g for n, g in zip(leaves, grads)}}


def _want(c, norm, interleaved, eps=1e-6):
    d = {k: t.double() if t is not None and t.is_floating_point() else t for k, t in c.items()}
    leaves = {k: d[k].requires_grad_() for k in ("q", "k", "qw", "kw") if d[k] is not None}
    B, T = d["q"].shape[:2]
    pos = torch.arange(T) if d["positions"] is None else d["positions"].long()
    pos = pos.expand(B, T)
    out = {n: R.norm_rope(d[n], d[n + "w"], norm, eps, d["cos"], d["sin"], pos, interleaved)
           for n in ("q", "k")}
    grads = torch.autograd.grad([out["q"], out["k"]], list(leaves.values()), [d["gq"], d["gk"]])
    return {**out, **{"d" + n: g for n, g in zip(leaves, grads)}}


def _check(got, want):
    for k, w in want.items():
        top = w.abs().max().item() if w.numel() else 0.0
        R.close(got[k], w, (2 ** -12 if k in ("dqw", "dkw") else 2 ** -19) * top + 1e-30, k)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("norm", ["rms", "l2", "none"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("weights", [False, True])
def test_norms_and_layouts(norm, interleaved, weights, dtype):
    c = _case(2, 5, 6, 2, 128, 64, dtype, weights, "batch")
    _check(_run(c, norm, interleaved), _want(c, norm, interleaved))


@pytest.mark.parametrize("D,rotary", [(8, 0), (16, 16), (24, 16), (32, 32), (40, 16), (64, 64),
                                      (96, 32), (96, 96), (128, 16), (192, 64), (256, 256), (256, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_head_sizes(D, rotary, interleaved):
    c = _case(1, 7, 3, 1, D, rotary, "bf16", True, "row", seed=D)
    _check(_run(c, "rms", interleaved), _want(c, "rms", interleaved))


@pytest.mark.parametrize("B,T,H,HK", [(1, 1, 1, 1), (3, 1, 32, 8), (1, 300, 4, 4), (2, 9, 5, 0),
                                      (2, 9, 0, 7), (1, 1300, 1, 1), (2, 3, 0, 0)])
def test_heads_and_lengths(B, T, H, HK):
    c = _case(B, T, H, HK, 64, 32, "bf16", True, None, seed=T)
    _check(_run(c, "rms", False), _want(c, "rms", False))


def test_no_rows():
    c = _case(2, 0, 4, 2, 64, 32, "bf16", True, None)
    got = _run(c, "rms", False)
    assert got["q"].shape == (2, 0, 4, 64) and not got["dqw"].any() and not got["dkw"].any()


def test_zero_rows_give_zero_not_nan():
    c = _case(1, 4, 2, 2, 64, 64, "bf16", False, None)
    c["q"][0, 1] = 0
    for norm in ("rms", "l2"):
        _check(_run(c, norm, False), _want(c, norm, False))


def test_views_of_a_packed_projection_and_odd_strides():
    packed = torch.randn(2, 9, 8 * 64).bfloat16().cuda()
    q, k = packed[..., :256].view(2, 9, 4, 64), packed[..., 256:384].view(2, 9, 2, 64)
    cos, sin = (t.cuda() for t in S.rotary_table(32, 16))
    a = S.qk_norm_rope(q, k, cos=cos, sin=sin)
    b = S.qk_norm_rope(q.contiguous(), k.contiguous(), cos=cos, sin=sin)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    t = torch.randn(2, 64, 4, 9).bfloat16().cuda().permute(0, 3, 2, 1)     # last stride not 1
    a, _ = S.qk_norm_rope(t, k[:, :, :0], norm="l2")
    b, _ = S.qk_norm_rope(t.contiguous(), k[:, :, :0], norm="l2")
    assert torch.equal(a, b)


def test_positions_outside_the_table_are_nan_in_the_rotated_part():
    q = torch.randn(1, 3, 2, 64).bfloat16().cuda()
    cos, sin = (t.cuda() for t in S.rotary_table(32, 10))
    pos = torch.tensor([5, 10, -1]).cuda()
    out, _ = S.qk_norm_rope(q, q, cos=cos, sin=sin, positions=pos)
    assert torch.isfinite(out[0, 0]).all() and torch.isfinite(out[..., 32:]).all()
    assert torch.isnan(out[0, 1:, :, :32]).all()


def test_far_positions():
    c = _case(1, 3, 2, 1, 64, 64, "bf16", False, "row", far=200000)
    _check(_run(c, "rms", False), _want(c, "rms", False))


def test_gradients_match_differences():
    # central differences of the kernel's own fp16 outputs: a step of 2^-3 moves an
    # output by about 2^-5, of which its rounding (2^-12) is below 1 %
    c = _case(1, 2, 1, 1, 16, 16, "fp16", False, None)
    q = c["q"].cuda()
    cos, sin = c["cos"].cuda(), c["sin"].cuda()
    w = c["gq"].cuda().double()
    def loss(t):
        return (S.qk_norm_rope(t, t, cos=cos, sin=sin)[0].double() * w).sum().item()
    x = q.clone().requires_grad_()
    S.qk_norm_rope(x, x.detach(), cos=cos, sin=sin)[0].backward(w.half())
    for i in range(0, 32, 5):
        up, down = q.clone(), q.clone()
        up.view(-1)[i] += 0.125
        down.view(-1)[i] -= 0.125
        diff = (loss(up) - loss(down)) / (up.view(-1)[i] - down.view(-1)[i]).item()
        # third-order term of the norm: 0.125^2 / 6 times derivatives of order 10
        assert abs(diff - x.grad.view(-1)[i].item()) < 0.06


def test_captured():
    c = _case(2, 9, 4, 2, 64, 32, "bf16", True, "row")
    d = {k: t.cuda() if t is not None else None for k, t in c.items()}
    def call():
        return S.qk_norm_rope(d["q"], d["k"], d["qw"], d["kw"], "rms", 1e-6, d["cos"], d["sin"],
                              d["positions"])
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, k = call()
    d["q"].mul_(3)
    d["positions"].sub_(4)
    graph.replay()
    torch.cuda.synchronize()
    want = call()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
