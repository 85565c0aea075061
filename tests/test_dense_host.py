"""The dense layer without a GPU: its oracle against finite differences, and
the refusals of the C entry points and the Python calls, all answered before
any CUDA call."""
import numpy as np
import pytest
import torch

from cutile_b200 import B200Error, _lib, ops
from oracle import oracle as O

NP = 1 << 20  # a non-NULL pointer that no refused call may follow
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


@pytest.mark.parametrize("act", ACTS)
def test_oracle_slopes_against_differences(act):
    z = np.linspace(-6, 6, 241) + 0.013  # no kink within a step
    h = 1e-5
    d = (O.activation(z + h, act)[0] - O.activation(z - h, act)[0]) / (2 * h)
    assert np.abs(d - O.activation(z, act)[1]).max() < 1e-8  # h^2 / 6 * third derivative


@pytest.mark.parametrize("act", ACTS)
def test_oracle_gradients_against_differences(act):
    rng = np.random.default_rng(1)
    A, B, b = rng.standard_normal((4, 3)), rng.standard_normal((5, 4)), rng.standard_normal(3)
    dC = rng.standard_normal((5, 3))
    z = O.dense(A, B, b, act)[1]
    dA, dB, db, _ = O.dense_bwd(dC, A, B, act, z)
    f = lambda: (O.dense(A, B, b, act)[0] * dC).sum()  # noqa: E731
    for arr, grad in ((A, dA), (B, dB), (b, db)):
        for k in np.ndindex(arr.shape):
            v = arr[k]
            arr[k] = v + 1e-6
            up = f()
            arr[k] = v - 1e-6
            dn = f()
            arr[k] = v
            assert abs((up - dn) / 2e-6 - grad[k]) < 1e-7


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=_lib.CTB_F32), -2), (dict(M=-1), -3), (dict(N=-1), -3), (dict(K=-1), -3),
    (dict(act=5), -1), (dict(act=-1), -1), (dict(bias=NP, bd=_lib.CTB_BF16), -2),
    (dict(bias=NP, bd=_lib.CTB_F64), -2), (dict(lda=15), -4), (dict(ldb=31), -4),
    (dict(ldc=15), -4), (dict(R=NP, ldr=15), -4), (dict(Z=NP, ldz=15), -4), (dict(A=None), -1),
    (dict(B=None), -1), (dict(C=None), -1), (dict(Z=NP), -1), (dict(Z=NP + 64, R=NP + 64), -1),
    (dict(M=0, A=None, C=None), 0),
    (dict(N=0, B=None, C=None), 0),
])
def test_dense_refusals(kw, code):
    a = dict(dtype=_lib.CTB_F16, A=NP, B=NP, bias=None, bd=0, R=None, Z=None, C=NP, M=16, N=4, K=32,
             lda=16, ldb=32, ldr=16, ldz=16, ldc=16, act=0)
    a.update(kw)
    assert _lib.load().ctb_dense_fwd(
        a["dtype"], a["A"], a["B"], a["bias"], a["bd"], a["R"], a["Z"], a["C"], a["M"], a["N"],
        a["K"], a["lda"], a["ldb"], a["ldr"], a["ldz"], a["ldc"], a["act"], None, 0, None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=_lib.CTB_F64), -2), (dict(M=-1), -3), (dict(N=-1), -3), (dict(K=-1), -3),
    (dict(act=9), -1), (dict(lddc=15), -4), (dict(lda=15), -4), (dict(ldb=31), -4),
    (dict(ldz=15), -4), (dict(ldda=15), -4), (dict(lddb=31), -4), (dict(dC=None), -1),
    (dict(A=None), -1), (dict(B=None), -1), (dict(Z=None), -1), (dict(ws=None), -1),
    (dict(wsb=100), -1), (dict(ws=NP + 8), -1),
])
def test_dense_bwd_refusals(kw, code):
    a = dict(dtype=_lib.CTB_BF16, dC=NP, A=NP, B=NP, Z=NP, dA=NP, dB=NP, db=NP, M=16, N=4, K=32,
             lddc=16, lda=16, ldb=32, ldz=16, ldda=16, lddb=32, act=4, ws=NP, wsb=1 << 30)
    a.update(kw)
    assert _lib.load().ctb_dense_bwd(
        a["dtype"], a["dC"], a["A"], a["B"], a["Z"], a["dA"], a["dB"], a["db"], a["M"], a["N"],
        a["K"], a["lddc"], a["lda"], a["ldb"], a["ldz"], a["ldda"], a["lddb"], a["act"], a["ws"],
        a["wsb"], None) == code


@pytest.mark.parametrize("same", [("C", "A"), ("C", "B"), ("Z", "A"), ("Z", "B"), ("Z", "C"), ("Z", "R")])
def test_dense_refuses_outputs_over_inputs(same):
    p = {k: NP + 4096 * i for i, k in enumerate("ABCZR")}
    p[same[0]] = p[same[1]]
    assert _lib.load().ctb_dense_fwd(_lib.CTB_F16, p["A"], p["B"], None, 0, p["R"], p["Z"], p["C"], 16,
                                     4, 32, 16, 32, 16, 16, 16, 0, None, 0, None) == -1
    assert b"of their own" in _lib.load().ctb_last_error()


@pytest.mark.parametrize("same", [("dA", "A"), ("dA", "B"), ("dA", "dC"), ("dB", "B"), ("dB", "dC"),
                                  ("dB", "Z"), ("dA", "dB"), ("db", "dC")])
def test_dense_bwd_refuses_outputs_over_inputs(same):
    p = {k: NP + 4096 * i for i, k in enumerate(("dC", "A", "B", "Z", "dA", "dB", "db"))}
    p[same[0]] = p[same[1]]
    assert _lib.load().ctb_dense_bwd(_lib.CTB_F16, p["dC"], p["A"], p["B"], p["Z"], p["dA"], p["dB"],
                                     p["db"], 16, 4, 32, 16, 16, 32, 16, 16, 32, 4, NP, 1 << 30,
                                     None) == -1
    assert b"of their own" in _lib.load().ctb_last_error()


def test_workspace_sizes():
    L = _lib.load()
    assert L.ctb_dense_fwd_workspace_bytes(NP, NP, 4096, 7, 512, 4096, 512) == 0
    assert L.ctb_dense_fwd_workspace_bytes(NP, NP, -1, 7, 512, 4096, 512) in (0, -1)
    # dZ needs N rows of M elements
    assert L.ctb_dense_bwd_workspace_bytes(NP, NP, NP, 100, 10, 30, 100, 100, 30, 4, 0) >= 2 * 1000
    assert L.ctb_dense_bwd_workspace_bytes(NP, NP, NP, 104, 10, 32, 104, 104, 32, 0, 0) == 0


def test_python_calls_refuse_host_tensors():
    A, B = torch.zeros(8, 16, dtype=torch.float16), torch.zeros(2, 8, dtype=torch.float16)
    for call in (lambda: ops.dense(A, B), lambda: ops.dense_bwd(B, A, B)):
        with pytest.raises(B200Error) as e:
            call()
        assert e.value.status == "CTB_ERR_ARG"
