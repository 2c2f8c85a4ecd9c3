"""The fp32 outputs of the chunked gated delta rule (final states, gradients of the
decays, of fp32 betas and of the initial states) have fp32's exactness.

Tolerance, of the 2-norm of the error over that of the result in fp64.  A sum of 128
products takes 8 steps of the tensor core, each off by at most 2^-23 of the partial sum;
the steps' errors are independent, so a product of a chunk is off by sqrt(8) 2^-23 at most.
A value passes three such products in its own chunk, those of chunks before fade with the
state: sqrt(3 * 8) 2^-23 < 5 * 2^-23.  The decays' exponentials add 2^-22, products and
sums of single values 2^-23 together: 8 * 2^-23 = 2^-20.  Operands of 16 bits (2^-17)
miss it by far."""
import pytest
import torch

import tdc_sequence as S
from test_seq_delta import _case, _run, _want

TOL = 2 ** -20
FP32 = ("final", "dg", "dbeta", "dstate")


def _off(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    return ((got - want).norm() / want.norm()).item()


def _exact(name, got, want):
    assert got.dtype == torch.float32, name
    off = _off(got, want)
    assert off <= TOL, f"{name}: {off:.3g} of the norm"


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,H,HV,K,V,dtype,cu", [
    (2, 300, 2, 4, 128, 128, "bf16", None),
    (2, 300, 2, 4, 128, 128, "fp16", None),
    (1, 200, 1, 2, 64, 64, "bf16", None),
    (1, 200, 1, 2, 64, 64, "fp16", None),
    (1, 150, 2, 2, 128, 256, "bf16", [3, 20, 20, 101, 148]),
    (1, 150, 2, 2, 128, 256, "fp16", [3, 20, 20, 101, 148]),
    (1, 130, 1, 1, 64, 128, "fp16", [0, 64, 130])])
def test_fp32_outputs(B, T, H, HV, K, V, dtype, cu):
    c = _case(B, T, H, HV, K, V, dtype, state=True, cu=cu, beta_f32=True, seed=T)
    got, want = _run(c), _want(c)
    for name in FP32:
        _exact(name, got[name], want[name])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("K,V", [(64, 128), (128, 64)])
def test_final_state_of_a_sequence_in_segments(K, V, dtype):
    c = _case(1, 1700, 1, 2, K, V, dtype, state=True, seed=K)
    args = [c[k] for k in ("q", "k", "v", "g", "beta")]
    _, f = S.gated_delta_rule(*(t.cuda() for t in args), None, c["state"].cuda(), None, True)
    d = [t.double().cuda() for t in args]
    k, s = d[1].repeat_interleave(2, 2), c["state"].double().cuda()
    for t in range(1700):
        s = s * d[3][:, t].exp()[..., None, None]
        u = (d[2][:, t] - torch.einsum("bhkv,bhk->bhv", s, k[:, t])) * d[4][:, t][..., None]
        s = s + k[:, t][..., None] * u[:, :, None, :]
    _exact("final", f, s)
