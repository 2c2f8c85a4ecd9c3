"""Plain forms of the sequence operators in fp64, for the tests: written from
the definitions, token by token, with gradients by torch's autograd."""
import torch


def pieces(batch, tokens, cu):
    """(batch row, first, last + 1) of every sequence."""
    if cu is None:
        return [(b, 0, tokens) for b in range(batch)]
    return [(0, cu[i], cu[i + 1]) for i in range(len(cu) - 1)]


def conv(x, w, bias, act, state, cu):
    """(y, final): y[t] = act(bias + sum_j w[j] x[t-(K-1)+j])."""
    taps = w.shape[0]
    y = torch.zeros_like(x)
    finals = []
    for n, (b, lo, hi) in enumerate(pieces(x.shape[0], x.shape[1], cu)):
        past = x.new_zeros(taps - 1, x.shape[2]) if state is None else state[n]
        xs = torch.cat([past, x[b, lo:hi]])
        rows = []
        for t in range(hi - lo):
            z = (xs[t:t + taps] * w).sum(0)
            if bias is not None:
                z = z + bias
            rows.append(z * torch.sigmoid(z) if act == "silu" else z)
        if rows:
            y = torch.cat([y[:b], torch.cat([y[b, :lo], torch.stack(rows), y[b, hi:]])[None],
                           y[b + 1:]])
        finals.append(xs[hi - lo:])
    return y, torch.stack(finals)


def norm_rope(x, weight, norm, eps, cos, sin, positions, interleaved):
    """x [B, T, H, D] normed, weighted and rotated pair by pair."""
    d = x.shape[-1]
    if norm == "rms":
        x = x / ((x * x).sum(-1, keepdim=True) / d + eps).sqrt()
    elif norm == "l2":
        x = x / ((x * x).sum(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        x = x * weight
    if cos is None:
        return x
    cols = list(x.unbind(-1))
    half = cos.shape[1]
    for i in range(half):
        c, s = cos[positions, i][..., None], sin[positions, i][..., None]
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        u, v = cols[a], cols[b]
        cols[a], cols[b] = u * c - v * s, v * c + u * s
    return torch.stack(cols, -1)


def delta(q, k, v, g, beta, scale, state, cu):
    """(o, final): the recurrence, token after token."""
    group = v.shape[2] // q.shape[2]
    q, k = q.repeat_interleave(group, 2), k.repeat_interleave(group, 2)
    rows = [[torch.zeros_like(v[b, t]) for t in range(v.shape[1])] for b in range(v.shape[0])]
    finals = []
    for n, (b, lo, hi) in enumerate(pieces(v.shape[0], v.shape[1], cu)):
        s = (v.new_zeros(v.shape[2], q.shape[3], v.shape[3]) if state is None else state[n])
        for t in range(lo, hi):
            s = s * g[b, t].exp()[:, None, None]
            u = v[b, t] - torch.einsum("hkv,hk->hv", s, k[b, t])
            s = s + beta[b, t][:, None, None] * k[b, t][:, :, None] * u[:, None, :]
            rows[b][t] = scale * torch.einsum("hkv,hk->hv", s, q[b, t])
        finals.append(s)
    o = torch.stack([torch.stack(r) if r else v[b] for b, r in enumerate(rows)])
    return o, torch.stack(finals)


def close(got, want, atol, name=""):
    """got's rounding to its type (half a step of the value) plus atol."""
    assert got.shape == want.shape, name
    if got.numel() == 0:
        return
    got, half = got.detach(), torch.finfo(got.dtype).eps / 2
    got, want = got.double().cpu(), want.detach().double().cpu()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    off = (got - want).abs() - half * want.abs()
    worst = off.max().item()
    assert worst <= atol, f"{name}: off by {worst:.3g} beyond its rounding, allowed {atol:.3g}"
