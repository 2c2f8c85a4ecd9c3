"""Gradients of the causal convolution where a thread's run of rows is long: nearly all rows go
through the loop that tests nothing, K rows at a time.

Tolerance: values as in test_seq_conv1d.  A weight's gradient is summed over at most 64 rows
by a thread, 32 threads of a block, then 40 blocks' sums by 8 lanes and the 8: a term
passes at most 64 + 32 + 5 + 3 roundings of 2^-24 of a partial sum.  Random terms' partial sums
stay below the sum of all magnitudes, at most 16 of the largest result here (5100 terms, a
result of the size of their root): 104 * 16 * 2^-24 < 2^-13, and the kernel's sigmoid (2^-20
a term) is far below: 2^-12 as there."""
import pytest
import torch

import seq_reference as R
import test_seq_conv1d as V

pytestmark = pytest.mark.gpu


def _want(c, act):
    """fp64, all rows of a sequence at once."""
    d = {k: t.double().requires_grad_() if isinstance(t, torch.Tensor) else t for k, t in c.items()}
    leaves = {k: d[k] for k in ("x", "w", "bias", "state") if d[k] is not None}
    taps, (B, T, C) = c["w"].shape[0], c["x"].shape
    ys, finals = [torch.zeros(0, C, dtype=torch.float64)], []
    at = 0
    for n, (b, lo, hi) in enumerate(R.pieces(B, T, c["cu"])):
        past = d["x"].new_zeros(taps - 1, C) if d["state"] is None else d["state"][n]
        xs = torch.cat([past, d["x"][b, lo:hi]])
        z = sum(xs[j:j + hi - lo] * d["w"][j] for j in range(taps))
        z = z if d["bias"] is None else z + d["bias"]
        ys += [torch.zeros(b * T + lo - at, C, dtype=torch.float64),
               z * torch.sigmoid(z) if act == "silu" else z]
        at = b * T + hi
        finals.append(xs[hi - lo:])
    ys.append(torch.zeros(B * T - at, C, dtype=torch.float64))
    y, f = torch.cat(ys).view(B, T, C), torch.stack(finals)
    grads = torch.autograd.grad([y, f], list(leaves.values()), [c["dy"].double(), c["df"].double()])
    return {"y": y, "final": f, **{"d" + k: g for k, g in zip(leaves, grads)}}


@pytest.mark.parametrize("K", [4, 5, 8])
@pytest.mark.parametrize("B,T,cu", [
    (1, 5000, None), (3, 1700, None),
    (1, 5100, [3, 3, 700, 701, 705, 1400, 2111, 2119, 4000, 5090])])   # ends inside the runs
@pytest.mark.parametrize("act,bias,state,dtype", [("silu", True, True, "bf16"),
                                                  ("none", False, False, "fp16")])
def test_gradients_of_long_runs(K, B, T, cu, act, bias, state, dtype):
    c = V._case(B, T, 1024, K, dtype, bias, state, cu, seed=K)
    V._check(V._run(c, act), _want(c, act))
