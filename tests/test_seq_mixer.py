"""The sequence operators as a layer uses them: GatedDeltaMixer against the same
layer in plain fp64, prefill and steps against the whole sequence, packed
batches, torch.compile, and the failure path of the walk's waits.

Tolerance against fp64: the layer has 7 roundings to bf16 one after another
(projection, convolution, queries and keys, delta rule, norm, gate product,
output projection), each off by 2^-9 of its value at most; sums over independent
terms do not add them up fully, and 4 allows for the norms' and gates' slopes:
4 * 7 * 2^-9 of the largest output.  Gradients pass them twice."""
import pytest
import torch

import seq_reference as R
import tdc_sequence as S
import tma_dwconv as T

pytestmark = pytest.mark.gpu
TOL = 4 * 7 * 2 ** -9


def _layer(seed=0, **over):
    torch.manual_seed(seed)
    conf = dict(hidden=96, key_heads=2, value_heads=4, key_dim=64, value_dim=64, taps=4)
    conf.update(over)
    return S.GatedDeltaMixer(**conf, device="cuda")


def _plain(m, x, cu=None, positions=None):
    """The layer in fp64 from its parameters (leaves p) and x."""
    p = {n: t.detach().double().cpu().requires_grad_() for n, t in m.named_parameters()}
    proj = x @ p["in_proj.weight"].T
    inner = m.value_heads * m.value_dim
    mixed, gate, ab = proj.split((m.channels, inner, m.gates), -1)
    a, b = ab[..., :m.value_heads], ab[..., m.value_heads:2 * m.value_heads]
    g = -p["log_rate"].exp() * torch.nn.functional.softplus(a + p["step_bias"])
    mixed, _ = R.conv(mixed, p["conv_weight"], None, "silu", None, cu)
    q, k, v = mixed.split(m.sizes, -1)
    q, k = (t.unflatten(-1, (m.key_heads, m.key_dim)) for t in (q, k))
    pos = torch.arange(x.shape[1]).expand(x.shape[:2]) if positions is None else positions
    cos, sin = (m.cos.double().cpu(), m.sin.double().cpu()) if m.rotary_dim else (None, None)
    q, k = (R.norm_rope(t, None, "l2", m.eps, cos, sin, pos, False) for t in (q, k))
    o, _ = R.delta(q, k, v.unflatten(-1, (m.value_heads, m.value_dim)), g, torch.sigmoid(b),
                   m.key_dim ** -0.5, None, cu)
    o = R.norm_rope(o, p["norm_weight"], "rms", m.eps, None, None, None, False)
    return (o.flatten(-2) * torch.nn.functional.silu(gate)) @ p["out_proj.weight"].T, p


@pytest.mark.parametrize("rotary", [0, 32])
def test_layer_and_its_gradients(rotary):
    m = _layer(rotary_dim=rotary, max_positions=200)
    x = torch.randn(2, 75, 96, generator=torch.Generator().manual_seed(1)).bfloat16()
    xd = x.cuda().requires_grad_()
    y = m(xd)
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(2)).bfloat16()
    y.backward(dy.cuda())
    xr = x.double().requires_grad_()
    want, p = _plain(m, xr)
    want.backward(dy.double())
    R.close(y, want, TOL * want.abs().max().item(), "y")
    R.close(xd.grad, xr.grad, 2 * TOL * xr.grad.abs().max().item(), "dx")
    for n, t in m.named_parameters():
        assert t.grad is not None and t.grad.dtype == t.dtype
        R.close(t.grad, p[n].grad, 2 * TOL * p[n].grad.abs().max().item(), n)


def test_prefill_then_steps_is_the_whole_sequence():
    m = _layer(rotary_dim=32, max_positions=100).eval()
    x = torch.randn(3, 90, 96, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    with torch.no_grad():
        whole = m(x)
        y, state = m(x[:, :70], output_state=True)
        pool = m.new_state(5)
        slots = torch.tensor([4, 0, 2], device="cuda")
        pool.conv[slots], pool.delta[slots] = state.conv, state.delta
        got = [y]
        for t in range(70, 90, 2):                       # two tokens a step
            pos = torch.arange(t, t + 2, device="cuda").expand(3, 2)
            got.append(m.step(x[:, t:t + 2], pool, slots, pos))
    got = torch.cat(got, 1)
    assert torch.equal(got[:, :70], whole[:, :70])       # the same kernels on the same rows
    top = whole.abs().max().item()
    assert (got.double() - whole.double()).abs().max().item() <= 2 * TOL * top


def test_segments_continue_one_another():
    m = _layer().eval()
    x = torch.randn(1, 200, 96, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    with torch.no_grad():
        whole = m(x)
        a, s = m(x[:, :77], output_state=True)
        b, s = m(x[:, 77:130], state=s, output_state=True)
        c, _ = m(x[:, 130:], state=s, output_state=True)
    got = torch.cat([a, b, c], 1)
    assert (got.double() - whole.double()).abs().max().item() <= 2 * TOL * whole.abs().max().item()


def test_packed_batch_is_its_sequences():
    m = _layer(rotary_dim=64, max_positions=100).eval()
    cu = [0, 1, 40, 40, 104, 130]
    x = torch.randn(1, 130, 96, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    pos = torch.cat([torch.arange(b - a) for a, b in zip(cu, cu[1:])]).cuda()
    with torch.no_grad():
        y, state = m(x, cu_seqlens=torch.tensor(cu).cuda(), positions=pos, output_state=True)
        for i, (lo, hi) in enumerate(zip(cu, cu[1:])):
            if lo == hi:
                assert not state.delta[i].any() and not state.conv[i].any()
                continue
            one, s = m(x[:, lo:hi], output_state=True)
            top = one.abs().max().item()
            assert (y[:, lo:hi].double() - one.double()).abs().max().item() <= TOL * top
            assert torch.equal(state.conv[i], s.conv[0])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_compiled_layer_gives_the_eager_results(dtype):
    torch._dynamo.reset()
    m = _layer(dtype=dtype, rotary_dim=32, max_positions=64)
    compiled = torch.compile(m, backend="aot_eager", fullgraph=True)
    x = torch.randn(2, 50, 96, device="cuda", dtype=dtype)
    xe, xc = x.clone().requires_grad_(), x.clone().requires_grad_()
    ye, yc = m(xe), compiled(xc)
    assert torch.equal(ye, yc)
    dy = torch.randn_like(ye)
    ge = torch.autograd.grad(ye, [xe, *m.parameters()], dy)
    gc = torch.autograd.grad(yc, [xc, *m.parameters()], dy)
    for a, b in zip(ge, gc):
        assert torch.equal(a, b)


def test_captured_steps():
    m = _layer().eval()
    pool, alone = m.new_state(4), m.new_state(4)
    x = torch.randn(2, 1, 96).bfloat16().cuda()
    slots = torch.tensor([3, 1], device="cuda")
    m.step(x, m.new_state(4), slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m.step(x, pool, slots)
    pool.conv.zero_(), pool.delta.zero_()
    for t in range(5):
        x.normal_()
        graph.replay()
        assert torch.equal(y, m.step(x, alone, slots))
    assert torch.equal(pool.delta, alone.delta) and torch.equal(pool.conv, alone.conv)


def test_two_graphs_and_streams_do_not_share_workspaces():
    m = _layer().eval()
    xs = [torch.randn(1, 150, 96).bfloat16().cuda() for _ in range(2)]
    with torch.no_grad():
        want = [m(x) for x in xs]
        graphs, outs = [], []
        torch.cuda.synchronize()
        for x in xs:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                outs.append(m(x))
        streams = [torch.cuda.Stream() for _ in xs]
        torch.cuda.synchronize()
        for _ in range(10):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
    for a, b in zip(outs, want):
        assert torch.equal(a, b)


def test_moving_the_layer_keeps_the_tables_fp32():
    m = _layer(rotary_dim=32, max_positions=50).to(torch.float16)
    assert m.cos.dtype == torch.float32 and m.conv_weight.dtype == torch.float16
    assert torch.isfinite(m(torch.randn(1, 40, 96, device="cuda").half())).all()


def test_a_copy_that_never_comes_is_reported():
    # The walk's waits are bounded: the launch ends, the next call is refused until the
    # record is cleared, and then everything runs again.
    q = torch.randn(1, 300, 1, 64, device="cuda").bfloat16() / 8
    v = torch.randn(1, 300, 2, 64, device="cuda").bfloat16()
    g, beta = -torch.rand(1, 300, 2, device="cuda"), torch.rand(1, 300, 2, device="cuda")
    want = S.gated_delta_rule(q, q, v, g, beta)
    T.device_status()
    try:
        for chunk in (0, 1, 3):
            S._C.gated_delta_rule(q, q, v, g, beta, 0.125, None, None, True, chunk, 2_000_000)
            torch.cuda.synchronize()
            with pytest.raises(RuntimeError, match="gave up waiting"):
                S.gated_delta_rule(q, q, v, g, beta)
            code, *_ = T.device_status()
            assert code in (1, 2)
    finally:
        T.device_status()
    assert torch.equal(S.gated_delta_rule(q, q, v, g, beta), want)
