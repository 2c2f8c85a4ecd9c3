"""The sequence operators without a GPU: the C ABI exports what its header
declares and refuses wrong arguments before any CUDA call, the Python functions
refuse wrong tensors, and the rotary tables are what they say."""
import ctypes as C
import math
import os
import re

import pytest
import torch

import tdc_sequence as S

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HDR = os.path.join(REPO, "include", "tdc_sequence.h")
CODES = {m.group(1): int(m.group(2))
         for h in ("tdc_dwconv.h", "tdc_sequence.h")
         for m in re.finditer(r"#define (TDC_\w+)\s+(-?\d+)",
                              open(os.path.join(REPO, "include", h)).read())}


@pytest.fixture(scope="module")
def lib():
    L = C.CDLL(os.path.join(REPO, "tma-depthwise-conv_b200", "libtdc_sm100.so"))
    for n in ("tdc_conv1d_bwd_workspace", "tdc_qk_norm_rope_bwd_workspace",
              "tdc_delta_fwd_workspace", "tdc_delta_bwd_workspace"):
        getattr(L, n).restype = C.c_int64
    return L


def _struct(name):
    """ctypes form of a struct of the header: pointers, int64 and double fields."""
    src = open(HDR).read()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), src, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = []
    for line in body.split(";"):
        line = " ".join(line.split())
        if not line:
            continue
        if "*" in line:
            fields.append((line.split("*")[-1].strip(), C.c_void_p))
        else:
            kind, names = line.split(" ", 1)
            ctype = {"int64_t": C.c_int64, "double": C.c_double}[kind]
            fields += [(n.strip(), ctype) for n in names.split(",")]
    return type(name, (C.Structure,), {"_fields_": fields})


Conv, ConvStep = _struct("tdc_conv1d_args"), _struct("tdc_conv1d_step_args")
Qk, QkGrad = _struct("tdc_qk_args"), _struct("tdc_qk_grad_args")
Delta, DeltaGrad = _struct("tdc_delta_args"), _struct("tdc_delta_grad_args")

P = 1 << 20   # an aligned address that no check reads from


def _conv(**over):
    a = dict(x=P, w=P, y=P, B=2, T=10, C=64, K=4, x_sb=640, x_st=64, dtype=CODES["TDC_BF16"], act=3)
    a.update(over)
    return Conv(**a)


def _qk(**over):
    a = dict(q=P, k=P, q_out=P, k_out=P, B=2, T=10, Hq=4, Hk=2, D=64, q_sb=2560, q_st=256, q_sh=64,
             k_sb=1280, k_st=128, k_sh=64, norm=1, eps=1e-6)
    a.update(over)
    return Qk(**a)


def _delta(**over):
    a = dict(q=P, k=P, v=P, g=P, beta=P, o=P, B=2, T=10, H=2, HV=4, K=64, V=64, q_sb=1280, q_st=128,
             q_sh=64, k_sb=1280, k_st=128, k_sh=64, v_sb=2560, v_st=256, v_sh=64, g_sb=40, g_st=4,
             b_sb=40, b_st=4, scale=0.125)
    a.update(over)
    return Delta(**a)


def test_exports_every_declared_symbol(lib):
    names = re.findall(r"TDC_API\s+[\w\s\*]+?\b(tdc_\w+)\s*\(", open(HDR).read())
    assert len(names) >= 12
    for n in names:
        assert hasattr(lib, n), n


@pytest.mark.parametrize("over,code", [
    (dict(dtype=7), "TDC_ERR_UNSUPPORTED"), (dict(act=1), "TDC_ERR_ACT"),
    (dict(B=-1), "TDC_ERR_BAD_SHAPE"), (dict(T=-1), "TDC_ERR_BAD_SHAPE"),
    (dict(K=1), "TDC_ERR_FILTER_SHAPE"), (dict(K=9), "TDC_ERR_FILTER_SHAPE"),
    (dict(C=60), "TDC_ERR_CHANNELS"), (dict(C=1 << 50), "TDC_ERR_TOO_LARGE"),
    (dict(x_st=60), "TDC_ERR_ALIGNMENT"), (dict(x=P + 2), "TDC_ERR_ALIGNMENT"),
    (dict(bias=P + 8), "TDC_ERR_ALIGNMENT"), (dict(x=None), "TDC_ERR_NULL_POINTER"),
    (dict(y=None), "TDC_ERR_NULL_POINTER"), (dict(cu_seqlens=P, num_seqs=2), "TDC_ERR_BAD_SHAPE"),
    (dict(cu_seqlens=P, num_seqs=0, B=1), "TDC_ERR_BAD_SHAPE")])
def test_conv_refusals(lib, over, code):
    assert lib.tdc_conv1d_fwd(C.byref(_conv(**over)), None) == CODES[code]


def test_conv_more_refusals(lib):
    assert lib.tdc_conv1d_fwd(None, None) == CODES["TDC_ERR_NULL_POINTER"]
    for over in (dict(B=0), dict(T=0), dict(C=0)):
        assert lib.tdc_conv1d_fwd(C.byref(_conv(x=None, w=None, y=None, **over)), None) == 0
    a = _conv()
    need = lib.tdc_conv1d_bwd_workspace(C.byref(a))
    assert need > 0
    p = C.c_void_p(P)
    args = lambda ws, n: (C.byref(a), p, C.c_int64(640), C.c_int64(64), None, p, p, None, None, ws,  # noqa: E731
                          C.c_int64(n), None)
    assert lib.tdc_conv1d_bwd(*args(p, need - 1)) == CODES["TDC_ERR_WORKSPACE"]
    assert lib.tdc_conv1d_bwd(*args(None, need)) == CODES["TDC_ERR_NULL_POINTER"]
    s = dict(x=P, w=P, state=P, y=P, B=2, T=1, C=64, K=4, x_sb=64, x_st=64, slots=4)
    step = lambda **o: lib.tdc_conv1d_step(C.byref(ConvStep(**{**s, **o})), None)  # noqa: E731
    assert step(slots=-1) == CODES["TDC_ERR_BAD_SHAPE"]
    assert step(state=None) == CODES["TDC_ERR_NULL_POINTER"]
    assert step(state=P + 4) == CODES["TDC_ERR_ALIGNMENT"]
    assert step(B=0) == 0


@pytest.mark.parametrize("over,code", [
    (dict(dtype=2), "TDC_ERR_UNSUPPORTED"), (dict(norm=3), "TDC_ERR_UNSUPPORTED"),
    (dict(Hq=-1), "TDC_ERR_BAD_SHAPE"), (dict(D=4), "TDC_ERR_CHANNELS"),
    (dict(D=264), "TDC_ERR_CHANNELS"), (dict(D=60), "TDC_ERR_CHANNELS"),
    (dict(R=80), "TDC_ERR_BAD_SHAPE"), (dict(R=24), "TDC_ERR_BAD_SHAPE"),
    (dict(R=32), "TDC_ERR_NULL_POINTER"), (dict(R=32, cos=P, sin=P + 4), "TDC_ERR_ALIGNMENT"),
    (dict(eps=-1.0), "TDC_ERR_BAD_SHAPE"), (dict(eps=float("nan")), "TDC_ERR_BAD_SHAPE"),
    (dict(q_sh=65), "TDC_ERR_ALIGNMENT"), (dict(k=P + 2), "TDC_ERR_ALIGNMENT"),
    (dict(q=None), "TDC_ERR_NULL_POINTER"), (dict(k_out=None), "TDC_ERR_NULL_POINTER"),
    (dict(B=1 << 20, T=1 << 20), "TDC_ERR_TOO_LARGE")])
def test_qk_refusals(lib, over, code):
    assert lib.tdc_qk_norm_rope(C.byref(_qk(**over)), None) == CODES[code]


def test_qk_more_refusals(lib):
    assert lib.tdc_qk_norm_rope(C.byref(_qk(T=0, q=None, k=None)), None) == 0
    a = _qk(q_weight=P)
    need = lib.tdc_qk_norm_rope_bwd_workspace(C.byref(a))
    g = dict(dq_out=P, dk_out=P, dq=P, dk=P, dq_weight=P, gq_sb=2560, gq_st=256, gq_sh=64,
             gk_sb=1280, gk_st=128, gk_sh=64)
    run = lambda n, **o: lib.tdc_qk_norm_rope_bwd(  # noqa: E731
        C.byref(a), C.byref(QkGrad(**{**g, **o})), C.c_void_p(P), C.c_int64(n), None)
    assert run(need - 1) == CODES["TDC_ERR_WORKSPACE"]
    assert run(need, dq_weight=None) == CODES["TDC_ERR_NULL_POINTER"]
    assert run(need, gk_st=4) == CODES["TDC_ERR_ALIGNMENT"]
    assert run(need, dq=None) == CODES["TDC_ERR_NULL_POINTER"]


@pytest.mark.parametrize("over,code", [
    (dict(dtype=5), "TDC_ERR_UNSUPPORTED"), (dict(HV=3), "TDC_ERR_BAD_SHAPE"),
    (dict(H=0), "TDC_ERR_BAD_SHAPE"), (dict(K=96), "TDC_ERR_CHANNELS"),
    (dict(V=32), "TDC_ERR_CHANNELS"), (dict(T=-1), "TDC_ERR_BAD_SHAPE"),
    (dict(T=1 << 40), "TDC_ERR_TOO_LARGE"), (dict(v_st=1 << 32), "TDC_ERR_TOO_LARGE"),
    (dict(q_st=100), "TDC_ERR_ALIGNMENT"), (dict(v=P + 8), "TDC_ERR_ALIGNMENT"),
    (dict(cu_seqlens=P, num_seqs=3), "TDC_ERR_BAD_SHAPE")])
def test_delta_refusals(lib, over, code):
    a = _delta(**over)
    ws = lambda n: (C.byref(a), C.c_void_p(P), C.c_int64(n), None)  # noqa: E731
    assert lib.tdc_delta_fwd_workspace(C.byref(a)) == CODES[code]
    assert lib.tdc_delta_fwd(*ws(1 << 40)) == CODES[code]
    assert lib.tdc_delta_step(C.byref(a), C.c_void_p(P), C.c_int64(4), None, C.c_int64(0), None) == \
        CODES[code]


def test_delta_more_refusals(lib):
    a = _delta()
    n, nb = (getattr(lib, f)(C.byref(a)) for f in ("tdc_delta_fwd_workspace",
                                                   "tdc_delta_bwd_workspace"))
    assert 0 < n < nb
    fwd = lambda a, ws, n: lib.tdc_delta_fwd(C.byref(a), C.c_void_p(ws), C.c_int64(n), None)  # noqa: E731
    assert fwd(a, P, n - 1) == CODES["TDC_ERR_WORKSPACE"]
    assert fwd(a, P + 16, n) == CODES["TDC_ERR_ALIGNMENT"]
    assert fwd(a, None, n) == CODES["TDC_ERR_NULL_POINTER"]
    assert fwd(_delta(g=None), P, n) == CODES["TDC_ERR_NULL_POINTER"]
    assert fwd(_delta(o=P + 2), P, n) == CODES["TDC_ERR_ALIGNMENT"]
    g = dict(d_o=P, dq=P, dk=P, dv=P, dg=P, dbeta=P, do_sb=2560, do_st=256, do_sh=64)
    bwd = lambda n, **o: lib.tdc_delta_bwd(  # noqa: E731
        C.byref(a), C.byref(DeltaGrad(**{**g, **o})), C.c_void_p(P), C.c_int64(n), None)
    assert bwd(nb - 1) == CODES["TDC_ERR_WORKSPACE"]
    assert bwd(nb, dg=None) == CODES["TDC_ERR_NULL_POINTER"]
    assert bwd(nb, do_sh=3) == CODES["TDC_ERR_ALIGNMENT"]
    step = lambda st, s: lib.tdc_delta_step(C.byref(a), C.c_void_p(st), C.c_int64(s), None,  # noqa: E731
                                            C.c_int64(0), None)
    assert step(None, 4) == CODES["TDC_ERR_NULL_POINTER"]
    assert step(P, -1) == CODES["TDC_ERR_BAD_SHAPE"]
    assert lib.tdc_delta_fwd_withhold(C.byref(a), C.c_void_p(P), C.c_int64(n), C.c_int64(-1),
                                      C.c_int64(1), None) == CODES["TDC_ERR_BAD_SHAPE"]


# ------------------------------ Python ---------------------------------------------

def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


X, W = _t(2, 10, 64), _t(4, 64)
Q, V, G = _t(2, 10, 2, 64), _t(2, 10, 4, 64), torch.zeros(2, 10, 4)
COS = torch.zeros(10, 16)
CU = torch.tensor([0, 10])


@pytest.mark.parametrize("call,text", [
    (lambda: S.causal_conv1d(X, W), "must be CUDA tensors"),
    (lambda: S.causal_conv1d(X.float(), W.float()), "fp16 or bf16"),
    (lambda: S.causal_conv1d(X, W.half()), "w must have x's dtype"),
    (lambda: S.causal_conv1d(X[0], W), r"x must be \[B,T,C\]"),
    (lambda: S.causal_conv1d(X, W[:, :32]), "agree on C"),
    (lambda: S.causal_conv1d(X[..., :12], W[:, :12]), "multiple of 8"),
    (lambda: S.causal_conv1d(X, W[:1]), "K must be 2 to 8"),
    (lambda: S.causal_conv1d(X, W, W[0, :8]), "bias must be"),
    (lambda: S.causal_conv1d(X, W, initial_state=_t(2, 4, 64)), "initial_state must be"),
    (lambda: S.causal_conv1d(X, W, cu_seqlens=CU), "batch dimension of 1"),
    (lambda: S.causal_conv1d(X[:1], W, cu_seqlens=CU.float()), "int32 or int64"),
    (lambda: S.causal_conv1d(X[:1], W, cu_seqlens=CU[:1]), "at least 2 offsets"),
    (lambda: S.causal_conv1d_step(X, W, None, _t(1, 3, 64)), "fewer slots"),
    (lambda: S.causal_conv1d_step(X, W, None, _t(3, 2, 64)), "state must be"),
    (lambda: S.causal_conv1d_step(X, W, None, _t(3, 3, 128)[..., ::2]), "contiguous"),
    (lambda: S.causal_conv1d_step(X, W, None, _t(3, 3, 64), state_indices=torch.zeros(3).int()),
     "one slot for each request"),
    (lambda: S.qk_norm_rope(Q, Q), "must be CUDA tensors"),
    (lambda: S.qk_norm_rope(Q, Q[:, :5]), "agree on B, T and D"),
    (lambda: S.qk_norm_rope(Q[..., :4], Q[..., :4]), "multiple of 8"),
    (lambda: S.qk_norm_rope(Q, Q, _t(32)), r"q_weight must be \[D\]"),
    (lambda: S.qk_norm_rope(Q, Q, cos=COS), "come together"),
    (lambda: S.qk_norm_rope(Q, Q, cos=COS[:, :12], sin=COS[:, :12]), "multiple of 16"),
    (lambda: S.qk_norm_rope(Q, Q, cos=COS[:5], sin=COS[:5]), "fewer rows"),
    (lambda: S.qk_norm_rope(Q, Q, cos=COS.double(), sin=COS.double()), "cos must be fp32"),
    (lambda: S.qk_norm_rope(Q, Q, positions=torch.zeros(10).long()), "need cos and sin"),
    (lambda: S.qk_norm_rope(Q, Q, cos=COS, sin=COS, positions=torch.zeros(9).long()),
     "positions must be"),
    (lambda: S.gated_delta_rule(Q, Q, V, G, G), "must be CUDA tensors"),
    (lambda: S.gated_delta_rule(Q, Q.half(), V, G, G), "k must have q's dtype"),
    (lambda: S.gated_delta_rule(Q, Q[:, :, :1], V, G, G), "q's shape"),
    (lambda: S.gated_delta_rule(Q, Q, V[:, :, :3], G[..., :3], G[..., :3]), "multiple of the key heads"),
    (lambda: S.gated_delta_rule(Q, Q, V, G[..., :2], G), r"g and beta must be \[B,T,HV\]"),
    (lambda: S.gated_delta_rule(Q, Q, V, G.bfloat16(), G), "g must be fp32"),
    (lambda: S.gated_delta_rule(Q, Q, V, G, G.double()), "beta must be"),
    (lambda: S.gated_delta_rule(Q[..., :32], Q[..., :32], V, G, G), "64 or 128"),
    (lambda: S.gated_delta_rule(Q, Q, V[..., :32], G, G), "64, 128 or 256"),
    (lambda: S.gated_delta_rule(Q, Q, V, G, G, initial_state=torch.zeros(2, 4, 64, 32)),
     "initial_state must be"),
    (lambda: S.gated_delta_step(Q, Q, V, G, G, torch.zeros(2, 4, 64, 64).half()), "state must be fp32"),
    (lambda: S.gated_delta_step(Q, Q, V, G, G, torch.zeros(1, 4, 64, 64)), "fewer slots"),
])
def test_python_refusals(call, text):
    with pytest.raises(RuntimeError, match=text):
        call()


def test_python_value_errors():
    for call in (lambda: S.causal_conv1d(X, W, activation="relu"),
                 lambda: S.qk_norm_rope(Q, Q, norm="layer"),
                 lambda: S.rotary_table(20, 5), lambda: S.rotary_table(16, -1),
                 lambda: S.rotary_table(16, 5, scaling="other"),
                 lambda: S.rotary_table(16, 5, scaling="linear", factor=0.5),
                 lambda: S.rotary_table(16, 5, scaling="parts", factor=2.0),
                 lambda: S.GatedDeltaMixer(64, 2, 3), lambda: S.GatedDeltaMixer(64, 2, key_dim=96),
                 lambda: S.GatedDeltaMixer(64, 2, taps=9),
                 lambda: S.GatedDeltaMixer(64, 2, rotary_dim=32),
                 lambda: S.GatedDeltaMixer(64, 2, dtype=torch.float32)):
        with pytest.raises(ValueError):
            call()


def test_steps_have_no_gradients():
    with pytest.raises(RuntimeError, match="no gradients"):
        S.causal_conv1d_step(X.clone().requires_grad_(), W, None, _t(2, 3, 64))
    with pytest.raises(RuntimeError, match="no gradients"):
        S.gated_delta_step(Q.clone().requires_grad_(), Q, V, G, G, torch.zeros(2, 4, 64, 64))


# ------------------------------ tables ----------------------------------------------

def test_rotary_table():
    cos, sin = S.rotary_table(32, 100001)
    for pos in (0, 1, 77, 100000):
        for i in (0, 3, 15):
            angle = pos * 10000.0 ** (-2 * i / 32)
            # the fp64 angle is off by pos * 2^-52, the result by half a step of fp32
            assert abs(cos[pos, i].item() - math.cos(angle)) <= 2 ** -24 + 1e-9
            assert abs(sin[pos, i].item() - math.sin(angle)) <= 2 ** -24 + 1e-9


def test_rotary_table_scaling():
    n, half = 4001, 16
    plain = S.rotary_table(2 * half, n)
    # linear: position p of the stretched table is position p / factor
    lin = S.rotary_table(2 * half, n, scaling="linear", factor=4.0)
    for a, b in zip(plain, lin):
        assert (a[:1000] - b[::4][:1000]).abs().max() <= 2 ** -23
    # base: the highest frequency as it was, the lowest divided by the factor
    base = S.rotary_table(2 * half, n, scaling="base", factor=4.0)
    assert torch.equal(base[0][:, 0], plain[0][:, 0])
    assert (base[1][:4000:4, -1] - plain[1][:1000, -1]).abs().max() <= 2 ** -20
    # parts: fast frequencies kept, slow ones divided, all times 0.1 ln(factor) + 1
    size = 0.1 * math.log(4.0) + 1
    parts = S.rotary_table(2 * half, n, scaling="parts", factor=4.0, original_length=2048)
    assert (parts[0][:, 0] - size * plain[0][:, 0]).abs().max() <= 2 ** -22
    assert (parts[1][:4000:4, -1] - size * plain[1][:1000, -1]).abs().max() <= 2 ** -22
    assert torch.equal(S.rotary_table(32, 10, scaling="parts", factor=1.0, original_length=64)[0],
                       S.rotary_table(32, 10)[0])
