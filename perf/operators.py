"""Measured cases of the sequence operators: the causal depthwise convolution,
the head norms with the position rotation, and the gated delta rule.

``listed()`` names the cases, ``draw`` gives more of the same ranges,
``prepare`` makes a case's inputs, ``run`` is one pass (the plain form in
elementary torch operations, or with ``own`` set the package's operators), and
``exact`` the operator's definition in 64 bits.
"""
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _ops():
    """The package's module of sequence operators."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "tma-depthwise-conv_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tdc_sequence
    return tdc_sequence


# ------------------------------- the cases -----------------------------------

def listed():
    return [
        # A training step of the short convolution over the packed q | k | v
        # projections of a mixer with 16 key and 32 value heads of 128.
        {"name": "conv_train", "op": "conv", "mode": "train", "dtype": "bf16", "batch": 2,
         "tokens": 4096, "channels": 8192, "taps": 4, "bias": False, "act": "silu",
         "sequences": 0, "split": 0, "states": False},
        # Prefill of a ragged packed batch that continues earlier segments:
        # states in and out, a bias, an odd number of tokens.
        {"name": "conv_prefill_ragged", "op": "conv", "mode": "infer", "dtype": "fp16", "batch": 1,
         "tokens": 5003, "channels": 2560, "taps": 4, "bias": True, "act": "silu",
         "sequences": 9, "split": 3, "states": True},
        # One decoded token for each of 4 requests, in a pool of 16 slots.
        {"name": "conv_step_4", "op": "conv_step", "dtype": "bf16", "batch": 4, "tokens": 1,
         "channels": 8192, "taps": 4, "bias": False, "act": "silu", "slots": 16},
        # Norms and partial rotation of a training step's queries and keys
        # (grouped heads of 128, half of each rotated, weights trained).
        {"name": "qk_train", "op": "qk", "mode": "train", "dtype": "bf16", "batch": 2,
         "tokens": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 64, "norm": "rms",
         "weights": True, "interleaved": False, "far": 0},
        # The same for 64 decoded tokens far into long contexts; q and k are
        # views of one packed projection, adjacent pairs are rotated.
        {"name": "qk_decode_64", "op": "qk", "mode": "infer", "dtype": "bf16", "batch": 64,
         "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "norm": "rms",
         "weights": True, "interleaved": True, "far": 120000},
        # Unit queries and keys for the delta rule, no weights, no rotation.
        {"name": "qk_unit_prefill", "op": "qk", "mode": "infer", "dtype": "fp16", "batch": 1,
         "tokens": 4999, "heads": 16, "kv_heads": 16, "dim": 128, "rotary": 0, "norm": "l2",
         "weights": False, "interleaved": False, "far": 0},
        # Prefill of one long prompt: few sequences, so the chunks of a
        # sequence run one after another in few blocks.
        {"name": "delta_prefill_long", "op": "delta", "mode": "infer", "dtype": "bf16", "batch": 1,
         "tokens": 8192, "heads": 16, "value_heads": 32, "key_dim": 128, "value_dim": 128,
         "sequences": 0, "split": 0, "states": False},
        # Prefill of a ragged packed batch that continues earlier segments.
        {"name": "delta_prefill_ragged", "op": "delta", "mode": "infer", "dtype": "bf16",
         "batch": 1, "tokens": 6007, "heads": 16, "value_heads": 32, "key_dim": 128,
         "value_dim": 128, "sequences": 11, "split": 5, "states": True},
        # A training step: all gradients.
        {"name": "delta_train", "op": "delta", "mode": "train", "dtype": "bf16", "batch": 4,
         "tokens": 2048, "heads": 16, "value_heads": 32, "key_dim": 128, "value_dim": 128,
         "sequences": 0, "split": 0, "states": False},
        # A small model's training step in fp16: heads of 64, an odd length,
        # states in and out with their gradients.
        {"name": "delta_train_small", "op": "delta", "mode": "train", "dtype": "fp16", "batch": 2,
         "tokens": 777, "heads": 4, "value_heads": 4, "key_dim": 64, "value_dim": 64,
         "sequences": 0, "split": 0, "states": True},
        # One decoded token for each of 4 requests, in a pool of 16 slots ...
        {"name": "delta_step_4", "op": "delta_step", "dtype": "bf16", "batch": 4, "tokens": 1,
         "heads": 16, "value_heads": 32, "key_dim": 128, "value_dim": 128, "slots": 16},
        # ... and for each of 192, where the states' traffic is the time.
        {"name": "delta_step_192", "op": "delta_step", "dtype": "bf16", "batch": 192, "tokens": 1,
         "heads": 16, "value_heads": 32, "key_dim": 128, "value_dim": 128, "slots": 200},
    ]


def _log(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["conv", "conv", "conv_step", "qk", "qk", "delta", "delta", "delta",
                     "delta_step"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    case = {"op": op, "dtype": dtype}
    if op in ("conv", "conv_step"):
        case.update(channels=8 * _log(rng, 8, 1024), taps=rng.choice([2, 3, 4, 4, 5, 8]),
                    bias=rng.random() < 0.5, act=rng.choice(["silu", "silu", "none"]))
    if op in ("conv_step", "delta_step"):
        batch = _log(rng, 1, 192)
        case.update(batch=batch, tokens=rng.choice([1, 1, 1, 2, 5]),
                    slots=batch + rng.randrange(0, 9))
    if op == "conv":
        tokens = _log(rng, 1, 8192)
        ragged = rng.random() < 0.5
        case.update(mode=rng.choice(["train", "infer"]), tokens=tokens,
                    batch=1 if ragged else rng.randint(1, max(1, min(4, 8192 // tokens))),
                    sequences=_log(rng, 1, 24) if ragged else 0, split=rng.randrange(1000),
                    states=rng.random() < 0.5)
    if op == "qk":
        tokens, dim = _log(rng, 1, 8192), rng.choice([64, 128, 128, 256])
        heads = rng.choice([4, 8, 16, 32])
        case.update(mode=rng.choice(["train", "infer"]), tokens=tokens, dim=dim,
                    batch=rng.randint(1, max(1, min(4, 8192 // tokens))),
                    heads=heads * 128 // max(dim, 128),
                    kv_heads=max(1, heads * 128 // max(dim, 128) // rng.choice([1, 2, 4])),
                    rotary=rng.choice([0, dim // 4, dim // 2, dim]),
                    norm=rng.choice(["rms", "l2"]), weights=rng.random() < 0.5,
                    interleaved=rng.random() < 0.5, far=rng.choice([0, 1000, 120000]))
    if op in ("delta", "delta_step"):
        heads, group = rng.choice([2, 4, 8, 16]), rng.choice([1, 2])
        case.update(heads=heads, value_heads=heads * group, key_dim=rng.choice([64, 128, 128]),
                    value_dim=rng.choice([64, 128, 128]))
    if op == "delta":
        tokens = _log(rng, 1, 8192 if group * heads <= 16 else 4096)
        ragged = rng.random() < 0.5
        case.update(mode=rng.choice(["train", "infer"]), tokens=tokens,
                    batch=1 if ragged else rng.randint(1, max(1, min(4, 4096 // tokens))),
                    sequences=_log(rng, 1, 24) if ragged else 0, split=rng.randrange(1000),
                    states=rng.random() < 0.5)
    return case


def _lengths(case):
    """Lengths of a packed batch: uneven cuts of the tokens, some of them empty or short."""
    r = random.Random(case["split"])
    total, n = case["tokens"], case["sequences"]
    cuts = sorted(int(total * r.random() ** 1.5) for _ in range(n - 1))
    edges = [0] + cuts + [total]
    return [b - a for a, b in zip(edges, edges[1:])]


def _edges(case):
    edges = [0]
    for n in _lengths(case):
        edges.append(edges[-1] + n)
    return edges


# ------------------------------- the inputs ----------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dtype):
        return (scale * torch.randn(shape, generator=gen, device="cuda")).to(dtype)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    op, train = case["op"], case.get("mode") == "train"
    s = {"case": case}
    if case.get("sequences"):
        s["cu_seqlens"] = torch.tensor(_edges(case), dtype=torch.int32, device="cuda")
        # the plain form's gather of a packed batch into a padded one, and back
        lens, edges = _lengths(case), _edges(case)
        longest = max(lens)
        at = torch.arange(longest, device="cuda")
        s["inside"] = at[None] < torch.tensor(lens, device="cuda")[:, None]
        s["rows"] = (torch.tensor(edges[:-1], device="cuda")[:, None] + at[None]).clamp_max(
            max(0, case["tokens"] - 1))
    count = case.get("sequences") or case["batch"]
    if op in ("conv", "conv_step"):
        c, k = case["channels"], case["taps"]
        s["x"] = normal(case["batch"], case["tokens"], c)
        s["w"] = normal(k, c, scale=k ** -0.5)
        s["bias"] = normal(c, scale=0.2) if case["bias"] else None
        if op == "conv_step":
            s["state"] = normal(case["slots"], k - 1, c)
        else:
            s["state"] = normal(count, k - 1, c) if case["states"] else None
            s["dy"] = normal(*s["x"].shape) if train else None
            s["dfinal"] = normal(*s["state"].shape) if train and case["states"] else None
    if op == "qk":
        b, t, h, hk, d = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "dim"))
        # one packed projection per token, as a layer's matrix product leaves it
        packed = normal(b, t, (h + 2 * hk) * d)
        s["q"] = packed[..., :h * d].view(b, t, h, d)
        s["k"] = packed[..., h * d:(h + hk) * d].view(b, t, hk, d)
        s["q_weight"] = (1 + 0.2 * normal(d)).to(dtype) if case["weights"] else None
        s["k_weight"] = (1 + 0.2 * normal(d)).to(dtype) if case["weights"] else None
        s["cos"] = s["sin"] = s["positions"] = None
        if case["rotary"]:
            half = case["rotary"] // 2
            freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
            angle = torch.arange(case["far"] + t, device="cuda", dtype=torch.float64)[:, None] * freq
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
            start = (uniform(b) * (case["far"] + 1)).long().clamp_max(case["far"])
            s["positions"] = (start[:, None] + torch.arange(t, device="cuda")).to(torch.int32)
        s["dq"] = normal(b, t, h, d) if train else None
        s["dk"] = normal(b, t, hk, d) if train else None
    if op in ("delta", "delta_step"):
        b, t, h, hv = (case[n] for n in ("batch", "tokens", "heads", "value_heads"))
        dk, dv = case["key_dim"], case["value_dim"]

        def unit(*shape):
            # neighbouring tokens' keys resemble each other: a shared direction
            x = torch.randn(shape, generator=gen, device="cuda")
            x = x + 0.5 * torch.randn((shape[0], 1) + shape[2:], generator=gen, device="cuda")
            return (x / x.norm(dim=-1, keepdim=True)).to(dtype)

        s["q"], s["k"], s["v"] = unit(b, t, h, dk), unit(b, t, h, dk), normal(b, t, hv, dv)
        # decays as layers start out: rates of 1 to 16 times a softplus around 1e-3 to 1e-1
        rate = 1 + 15 * uniform(hv)
        step = torch.exp(uniform(hv) * 4.6 - 6.9)
        raw = torch.randn((b, t, hv), generator=gen, device="cuda") + torch.log(torch.expm1(step))
        s["g"] = -rate * torch.nn.functional.softplus(raw)
        s["beta"] = torch.sigmoid(torch.randn((b, t, hv), generator=gen, device="cuda")).to(dtype)
        if op == "delta_step":
            s["state"] = normal(case["slots"], hv, dk, dv, scale=0.3, dtype=torch.float32)
        else:
            s["state"] = (normal(count, hv, dk, dv, scale=0.3, dtype=torch.float32)
                          if case["states"] else None)
            s["do"] = normal(b, t, hv, dv) if train else None
            s["dfinal"] = (normal(count, hv, dk, dv, scale=0.3, dtype=torch.float32)
                           if train and case["states"] else None)
    if op in ("conv_step", "delta_step"):
        slots = torch.randperm(case["slots"], generator=gen, device="cuda")[:case["batch"]]
        s["slots"] = slots.to(torch.int32)
    if train:
        for name in ("x", "w", "bias", "q", "k", "v", "g", "beta", "state", "q_weight",
                     "k_weight"):
            if s.get(name) is not None:
                s[name] = s[name].detach().requires_grad_()
    return s


# ------------------------------- one pass ------------------------------------

def run(s):
    return {"conv": _run_conv, "conv_step": _run_conv_step, "qk": _run_qk,
            "delta": _run_delta, "delta_step": _run_delta_step}[s["case"]["op"]](s)


def _gradients(outputs, grads, inputs):
    """{name: gradient} of the inputs that are there."""
    names = [n for n, t in inputs.items() if t is not None]
    pairs = [(o, g) for o, g in zip(outputs, grads) if g is not None]
    got = torch.autograd.grad([o for o, _ in pairs], [inputs[n] for n in names],
                              [g for _, g in pairs])
    return dict(zip(["d" + n for n in names], got))


def _run_conv(s):
    case = s["case"]
    if own:
        out = _ops().causal_conv1d(
            s["x"], s["w"], s["bias"], activation=case["act"], initial_state=s["state"],
            cu_seqlens=s.get("cu_seqlens"), output_final_state=case["states"])
    else:
        out = _plain_conv(s["x"], s["w"], s["bias"], case["act"], s["state"], s.get("rows"),
                          s.get("inside"), case["states"])
    y, final = out if case["states"] else (out, None)
    if case["mode"] == "infer":
        return {"y": y, "final": final}
    got = _gradients([y, final], [s["dy"], s["dfinal"]],
                     {"x": s["x"], "w": s["w"], "bias": s["bias"], "state": s["state"]})
    return {"y": y.detach(), "final": None if final is None else final.detach(), **got}


def _run_conv_step(s):
    case = s["case"]
    if own:
        y = _ops().causal_conv1d_step(s["x"], s["w"], s["bias"], s["state"],
                                      activation=case["act"], state_indices=s["slots"])
    else:
        slots = s["slots"].long()
        y, final = _plain_conv(s["x"], s["w"], s["bias"], case["act"], s["state"][slots], None,
                               None, True)
        s["state"][slots] = final
    return {"y": y, "state": s["state"]}


def _run_qk(s):
    case = s["case"]
    if own:
        q, k = _ops().qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"],
                                   norm=case["norm"], cos=s["cos"], sin=s["sin"],
                                   positions=s["positions"], interleaved=case["interleaved"])
    else:
        q, k = (_plain_norm_rope(s[n], s[n + "_weight"], case["norm"], s["cos"], s["sin"],
                                 s["positions"], case["interleaved"]) for n in ("q", "k"))
    if case["mode"] == "infer":
        return {"q": q, "k": k}
    got = _gradients([q, k], [s["dq"], s["dk"]], {
        n: s[n] for n in ("q", "k", "q_weight", "k_weight")})
    return {"q": q.detach(), "k": k.detach(), **got}


def _run_delta(s):
    case = s["case"]
    if own:
        out = _ops().gated_delta_rule(
            s["q"], s["k"], s["v"], s["g"], s["beta"], initial_state=s["state"],
            cu_seqlens=s.get("cu_seqlens"), output_final_state=True)
    else:
        out = _plain_delta(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], s.get("rows"),
                           s.get("inside"))
    o, final = out
    if case["mode"] == "infer":
        return {"o": o, "final": final}
    got = _gradients([o, final], [s["do"], s["dfinal"]], {
        n: s[n] for n in ("q", "k", "v", "g", "beta", "state")})
    return {"o": o.detach(), "final": final.detach(), **got}


def _run_delta_step(s):
    if own:
        o = _ops().gated_delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"],
                                    state_indices=s["slots"])
    else:
        slots = s["slots"].long()
        o, final = _plain_delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"][slots])
        s["state"][slots] = final
    return {"o": o, "state": s["state"]}


# ----------------------------- the plain forms -------------------------------

def _plain_conv(x, w, bias, act, state, rows, inside, want_final):
    """y[t] = act(sum_k w[k] x[t - (K-1) + k] + bias), earlier inputs from the state."""
    taps, dtype = w.shape[0], x.dtype
    shape = x.shape
    if rows is not None:
        x = x[0][rows] * inside[..., None]
    xf = x.float()
    past = (xf.new_zeros(xf.shape[0], taps - 1, xf.shape[2]) if state is None else state.float())
    xf = torch.cat([past, xf], 1)
    t = x.shape[1]
    wf = w.float()
    acc = sum(xf[:, i:i + t] * wf[i] for i in range(taps))
    if bias is not None:
        acc = acc + bias.float()
    y = (acc * torch.sigmoid(acc) if act == "silu" else acc).to(dtype)
    if inside is not None:
        y = y[inside].view(shape)
    if not want_final:
        return y
    if inside is None:
        final = xf[:, t:]
    else:
        last = inside.sum(1)[:, None] + torch.arange(taps - 1, device=x.device)
        final = xf.gather(1, last[..., None].expand(-1, -1, xf.shape[2]))
    return y, final.to(dtype)


def _plain_norm_rope(x, weight, norm, cos, sin, positions, interleaved, eps=1e-6):
    """x / sqrt(mean(x^2) + eps) ("rms") or x / sqrt(sum(x^2) + eps) ("l2"), times the
    weight, then the rotation of the first 2 * cos.shape[1] values of each head."""
    xf = x.float()
    square = xf.square()
    square = square.mean(-1, keepdim=True) if norm == "rms" else square.sum(-1, keepdim=True)
    y = xf * torch.rsqrt(square + eps)
    if weight is not None:
        y = y * weight.float()
    if cos is not None:
        c, s = (t[positions.long()][..., None, :] for t in (cos, sin))
        n = cos.shape[1]
        head, rest = y[..., :2 * n], y[..., 2 * n:]
        a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :n], head[..., n:])
        u, v = a * c - b * s, b * c + a * s
        head = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
        y = torch.cat([head, rest], -1)
    return y.to(x.dtype)


def _unit_lower_inverse(a):
    """(I + a)^-1 of strictly lower triangular a [..., n, n], n a power of two: diagonal
    blocks of 1, 2, 4, ... are joined, inv([[P, 0], [B, R]]) = [[P', 0], [-R' B P', R']]."""
    n = a.shape[-1]
    inv = torch.ones_like(a[..., :1, :1]).expand(*a.shape[:-2], n, 1).unsqueeze(-1)
    size = 1
    while size < n:
        m = n // (2 * size)
        blocks = a.unflatten(-1, (m, 2 * size)).unflatten(-3, (m, 2 * size))
        blocks = blocks.diagonal(dim1=-4, dim2=-2).movedim(-1, -3)
        low = blocks[..., size:, :size]
        pair = inv.unflatten(-3, (m, 2))
        p, r = pair[..., 0, :, :], pair[..., 1, :, :]
        join = -(r @ (low @ p))
        inv = torch.cat([torch.cat([p, torch.zeros_like(p)], -1), torch.cat([join, r], -1)], -2)
        size *= 2
    return inv.squeeze(-3)


def _plain_delta(q, k, v, g, beta, state, rows, inside, chunk=64):
    """S_t = e^g_t S_(t-1) + beta_t k_t (v_t - (e^g_t S_(t-1))^T k_t)^T, o_t = S_t^T q_t / sqrt(K),
    in chunks: within one, the corrections u solve a unit triangular system."""
    dtype, shape, group = v.dtype, v.shape, v.shape[2] // q.shape[2]
    scale = q.shape[-1] ** -0.5
    if rows is not None:
        q, k, v, g, beta = (t[0][rows] * inside.view(inside.shape + (1,) * (t.dim() - 2))
                            for t in (q, k, v, g, beta))
    b, t, hv, dv = v.shape
    n = max(1, -(-t // chunk))

    def chunks(x):  # [B, T, H, ...] -> [B, HV, n, chunk, ...] in 32 bits, padded with zeros
        x = x.float().movedim(2, 1)
        x = torch.cat([x, x.new_zeros(x.shape[:2] + (n * chunk - t,) + x.shape[3:])], 2)
        return x.repeat_interleave(hv // x.shape[1], 1).unflatten(2, (n, chunk))

    q, k, v, g, beta = (chunks(x) for x in (q, k, v, g, beta))
    total = g.double().cumsum(-1)
    decay = torch.tril((total[..., :, None] - total[..., None, :]).tril().exp()).float()
    from_start, to_end = total.exp().float(), (total[..., -1:] - total).exp().float()
    kk = torch.tril((k @ k.mT) * decay, -1) * beta[..., :, None]
    solve = _unit_lower_inverse(kk) * beta[..., None, :]
    mix = torch.tril((q @ k.mT) * decay) * scale
    q, kd = q * (scale * from_start)[..., None], k * from_start[..., None]
    ke = k * to_end[..., None]
    s = v.new_zeros(b, hv, k.shape[-1], dv) if state is None else state.float()
    out = []
    for i in range(n):
        u = solve[:, :, i] @ (v[:, :, i] - kd[:, :, i] @ s)
        out.append(q[:, :, i] @ s + mix[:, :, i] @ u)
        s = from_start[:, :, i, -1, None, None] * s + ke[:, :, i].mT @ u
    o = torch.stack(out, 2).flatten(2, 3)[:, :, :t].movedim(1, 2).to(dtype)
    if inside is not None:
        o = o[inside].view(shape)
    return o, s


def _plain_delta_step(q, k, v, g, beta, s):
    """The recurrence itself, token after token."""
    group, scale = v.shape[2] // q.shape[2], q.shape[-1] ** -0.5
    out = []
    for i in range(q.shape[1]):
        qi, ki = (x[:, i].float().repeat_interleave(group, 1) for x in (q, k))
        s = s * g[:, i].float().exp()[..., None, None]
        u = (v[:, i].float() - (ki[..., None, :] @ s)[..., 0, :]) * beta[:, i].float()[..., None]
        s = s + ki[..., :, None] * u[..., None, :]
        out.append((qi[..., None, :] @ s)[..., 0, :] * scale)
    return torch.stack(out, 1).to(v.dtype), s


# ------------------------- the definition in 64 bits -------------------------

def exact(case, seed):
    s = {n: t.detach().double() if isinstance(t, torch.Tensor) and t.is_floating_point() else t
         for n, t in prepare(case, seed).items()}
    with torch.no_grad():
        return {"conv": _exact_conv, "conv_step": _exact_conv_step, "qk": _exact_qk,
                "delta": _exact_delta, "delta_step": _exact_delta_step}[case["op"]](s)


def _pieces(s, count):
    """(rows of the batch, from, to) of each sequence."""
    case = s["case"]
    if case.get("sequences"):
        e = _edges(case)
        return [(0, e[i], e[i + 1]) for i in range(len(e) - 1)]
    return [(b, 0, case["tokens"]) for b in range(count)]


def _exact_conv(s):
    case = s["case"]
    x, w, bias, state = s["x"], s["w"], s["bias"], s["state"]
    taps, train = w.shape[0], case["mode"] == "train"
    y = torch.empty_like(x)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    db = torch.zeros_like(w[0])
    final = None if state is None else torch.empty_like(state)
    dstate = None if state is None else torch.zeros_like(state)
    for i, (b, lo, hi) in enumerate(_pieces(s, x.shape[0])):
        n = hi - lo
        past = x.new_zeros(taps - 1, x.shape[2]) if state is None else state[i]
        xp = torch.cat([past, x[b, lo:hi]])
        pre = torch.stack([xp[j:j + n] * w[j] for j in range(taps)]).sum(0)
        if bias is not None:
            pre = pre + bias
        gate = 1 / (1 + torch.exp(-pre))
        y[b, lo:hi] = pre * gate if case["act"] == "silu" else pre
        if final is not None:
            final[i] = xp[n:]
        if train:
            d = s["dy"][b, lo:hi]
            if case["act"] == "silu":
                d = d * gate * (1 + pre * (1 - gate))
            dxp = torch.zeros_like(xp)
            if final is not None:
                dxp[n:] = s["dfinal"][i]
            for j in range(taps):
                dxp[j:j + n] += d * w[j]
                dw[j] += (d * xp[j:j + n]).sum(0)
            db += d.sum(0)
            dx[b, lo:hi] = dxp[taps - 1:]
            if dstate is not None:
                dstate[i] = dxp[:taps - 1]
    out = {"y": y, "final": final}
    if train:
        out.update({"dx": dx, "dw": dw})
        if bias is not None:
            out["dbias"] = db
        if state is not None:
            out["dstate"] = dstate
    return out


def _exact_conv_step(s):
    x, w, state = s["x"], s["w"], s["state"]
    slots, taps = s["slots"].long(), w.shape[0]
    xp = torch.cat([state[slots], x], 1)
    y = torch.einsum("btkc,kc->btc", xp.unfold(1, taps, 1).transpose(2, 3), w)
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["case"]["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    state[slots] = xp[:, x.shape[1]:]
    return {"y": y, "state": state}


def _exact_qk(s):
    case, out = s["case"], {}
    for name in ("q", "k"):
        x, weight = s[name], s[name + "_weight"]
        d = x.shape[-1]
        inv = (x.pow(2).sum(-1, keepdim=True) / (d if case["norm"] == "rms" else 1) + 1e-6) ** -0.5
        hat = x * inv
        y = hat if weight is None else hat * weight
        n, turn = 0, None
        if s["cos"] is not None:
            n = s["cos"].shape[1]
            at = s["positions"].long()
            turn = torch.complex(s["cos"][at], s["sin"][at])[..., None, :]
        def rotate(y, turn):
            if turn is None:
                return y
            y = y.clone()
            pairs = y[..., :2 * n].unflatten(-1, (n, 2) if case["interleaved"] else (2, n))
            pairs = pairs if case["interleaved"] else pairs.transpose(-1, -2)
            z = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * turn)
            z = z if case["interleaved"] else z.transpose(-1, -2)
            y[..., :2 * n] = z.flatten(-2)
            return y
        out[name] = rotate(y, turn)
        if case["mode"] == "train":
            dy = rotate(s["d" + name], None if turn is None else turn.conj())
            if weight is not None:
                out["d" + name + "_weight"] = (dy * hat).sum((0, 1, 2))
                dy = dy * weight
            mean = (dy * hat).sum(-1, keepdim=True) / (d if case["norm"] == "rms" else 1)
            out["d" + name] = inv * (dy - hat * mean)
    return out


def _exact_delta(s):
    case, train = s["case"], s["case"]["mode"] == "train"
    pieces = _pieces(s, s["v"].shape[0])
    longest = max(hi - lo for _, lo, hi in pieces)
    group, scale = case["value_heads"] // case["heads"], case["key_dim"] ** -0.5
    count, hv, dk, dv = len(pieces), case["value_heads"], case["key_dim"], case["value_dim"]

    def padded(x, per_key_head=False):  # [longest, N, HV, ...], zeros behind each sequence's end
        y = x.new_zeros((longest, count) + x.shape[2:])
        for i, (b, lo, hi) in enumerate(pieces):
            y[:hi - lo, i] = x[b, lo:hi]
        return y.repeat_interleave(group, 2) if per_key_head else y

    def packed(y, like):
        x = torch.empty_like(like)
        for i, (b, lo, hi) in enumerate(pieces):
            x[b, lo:hi] = y[:hi - lo, i]
        return x

    q, k = padded(s["q"], True), padded(s["k"], True)
    v, g, beta = padded(s["v"]), padded(s["g"]), padded(s["beta"])
    if train and longest * count * hv * dk * dv * 8 > 70e9:
        return None
    state = v.new_zeros(count, hv, dk, dv) if s["state"] is None else s["state"].clone()
    o, before, us = torch.empty_like(v), [], torch.empty_like(v)
    for t in range(longest):
        state = state * g[t].exp()[..., None, None]
        u = v[t] - torch.einsum("nhkv,nhk->nhv", state, k[t])
        us[t] = u
        if train:
            before.append(state)
        state = state + torch.einsum("nhk,nhv->nhkv", k[t], u * beta[t][..., None])
        o[t] = scale * torch.einsum("nhkv,nhk->nhv", state, q[t])
    out = {"o": packed(o, s["v"]), "final": state}
    if train:
        do = padded(s["do"])
        dst = torch.zeros_like(state) if s["dfinal"] is None else s["dfinal"].clone()
        dq, dkey, dval = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        dg, dbeta = torch.empty_like(g), torch.empty_like(beta)
        for t in range(longest - 1, -1, -1):
            old = before.pop()
            b = beta[t][..., None]
            new = old + torch.einsum("nhk,nhv->nhkv", k[t], us[t] * b)
            dq[t] = scale * torch.einsum("nhkv,nhv->nhk", new, do[t])
            dst = dst + scale * torch.einsum("nhk,nhv->nhkv", q[t], do[t])
            down = torch.einsum("nhkv,nhk->nhv", dst, k[t])
            du = b * down
            dbeta[t] = (down * us[t]).sum(-1)
            dkey[t] = (torch.einsum("nhkv,nhv->nhk", dst, us[t] * b)
                       - torch.einsum("nhkv,nhv->nhk", old, du))
            dval[t] = du
            dst = dst - torch.einsum("nhk,nhv->nhkv", k[t], du)
            dg[t] = (dst * old).sum((-1, -2))
            dst = dst * g[t].exp()[..., None, None]
        for name, grad, like in (("dq", dq, s["q"]), ("dk", dkey, s["k"])):
            out[name] = packed(grad.unflatten(2, (case["heads"], group)).sum(3), like)
        out.update({"dv": packed(dval, s["v"]), "dg": packed(dg, s["g"]),
                    "dbeta": packed(dbeta, s["beta"])})
        if s["state"] is not None:
            out["dstate"] = dst
    return out


def _exact_delta_step(s):
    case, slots = s["case"], s["slots"].long()
    part = {**s, "state": s["state"][slots], "case": {**case, "mode": "infer"}}
    got = _exact_delta(part)
    s["state"][slots] = got["final"]
    return {"o": got["o"], "state": s["state"]}


# ------------------------------- its work ------------------------------------

def work(case):
    """Bytes with each input read and each output written once; operations of the
    recurrences themselves."""
    size, b, t = 2, case["batch"], case["tokens"]
    op, train = case["op"], case.get("mode") == "train"
    count = case.get("sequences") or b
    if op in ("conv", "conv_step"):
        c, k = case["channels"], case["taps"]
        states = 2 * (b if op == "conv_step" else count if case["states"] else 0) * (k - 1) * c
        n = b * t * c
        # x, y and in training dy, dx
        return {"bytes": size * ((4 if train else 2) * n + states * (2 if train else 1) + k * c),
                "flops": n * k * (6 if train else 2)}
    if op == "qk":
        n = b * t * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": size * n * (4 if train else 2) + b * t * case["rotary"] * 4,
                "flops": n * (25 if train else 8)}
    h, hv, dk, dv = (case[n] for n in ("heads", "value_heads", "key_dim", "value_dim"))
    state = hv * dk * dv * 4
    keys, values, gates = size * b * t * h * dk, size * b * t * hv * dv, b * t * hv * (4 + size)
    states = 2 * state * b if op == "delta_step" else state * count * (2 if case["states"] else 1)
    # q, k, v, g, beta, o and in training do, dq, dk, dv, dg, dbeta
    moved = 2 * keys + 2 * values + gates
    if train:
        moved += 2 * keys + 2 * values + gates
        states += 2 * states if case["states"] else 0
    return {"bytes": moved + states, "flops": b * t * hv * dk * dv * (20 if train else 6)}
