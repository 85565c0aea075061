"""Routing and combine without a GPU: the float64 oracles against finite
differences and hand-worked rows, and the refusals of the C entry points and
of the Python calls (all answered before any CUDA call)."""
import ctypes

import numpy as np
import pytest
import torch

from cutile_b200 import B200Error, _lib, ops
from oracle import oracle as O

NP = 1 << 20  # a non-NULL pointer that no refused call may follow


def test_oracle_route_by_hand():
    w, i = O.moe_route(np.array([[0.0, 2.0, 1.0, 2.0]]), 3)
    assert i.tolist() == [[1, 3, 2]]  # the tie goes to the lower index
    e = np.exp([0.0, 0.0, -1.0])
    np.testing.assert_allclose(w[0], e / e.sum(), rtol=1e-15)
    w, i = O.moe_route(np.array([[0.0, 2.0, 1.0, 2.0]]), 1, bias=[1.0, 0.0, 0.0, 0.1])
    assert i.tolist() == [[0]] and w[0, 0] == 1.0  # the bias chooses, the score weighs
    w, i = O.moe_route(np.array([[-np.inf] * 4, [np.nan, 1.0, -np.inf, -np.inf]]), 2, renorm=False)
    assert i.tolist() == [[-1, -1], [1, -1]] and w.tolist() == [[0, 0], [1, 0]]
    # groups by the sum of their two best: {0.9, 0} loses to {0.5, 0.5}
    x = np.log(np.array([[0.9, 1e-9, 0.5, 0.5]]))
    assert O.moe_route(x, 1, groups=2, topk_groups=1)[1].tolist() == [[2]]
    assert O.moe_route(x, 1, groups=2, topk_groups=1, group_top=1)[1].tolist() == [[0]]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_oracle_route_gradient_against_differences(score, renorm):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((3, 7))
    dw = rng.standard_normal((3, 2))
    _, ids = O.moe_route(x, 2, score, renorm=renorm, scale=1.7)
    dx = O.moe_route_bwd(dw, x, ids, score, renorm, 1.7)
    h = 1e-5
    for t in range(3):
        for e in range(7):
            up, dn = x.copy(), x.copy()
            up[t, e] += h
            dn[t, e] -= h
            wu, iu = O.moe_route(up, 2, score, renorm=renorm, scale=1.7)
            wd, idn = O.moe_route(dn, 2, score, renorm=renorm, scale=1.7)
            assert (iu == ids).all() and (idn == ids).all()
            # central difference: error h^2/6 * third derivative (< 10) + 1e-16/h
            assert abs(((wu - wd) * dw).sum() / (2 * h) - dx[t, e]) < 1e-8


def test_oracle_combine_gradient_against_differences():
    rng = np.random.default_rng(4)
    y, w, d = rng.standard_normal((6, 5)), rng.random((3, 2)), rng.standard_normal((3, 5))
    ids = np.array([[0, 1], [-1, 2], [3, 0]])
    dy, dw = O.moe_combine_bwd(d, y, 2, w, ids, 3)
    f = lambda: (O.moe_combine(y, 2, w, ids, 3) * d).sum()  # noqa: E731
    for arr, grad in ((y, dy), (w, dw)):
        for k in np.ndindex(arr.shape):
            v = arr[k]
            arr[k] = v + 1e-5
            up = f()
            arr[k] = v - 1e-5
            dn = f()
            arr[k] = v
            assert abs((up - dn) / 2e-5 - grad[k]) < 1e-8  # the function is bilinear


def route(dtype=_lib.CTB_F32, x=NP, w=NP, i=NP, T=4, E=8, topk=2, ldx=8, score=0, groups=1,
          topk_groups=1, group_top=2):
    return _lib.load().ctb_moe_route(dtype, x, None, w, i, T, E, topk, ldx, score, groups,
                                     topk_groups, group_top, 1, ctypes.c_float(1.0), None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=_lib.CTB_F64), -2), (dict(T=-1), -3), (dict(E=0, ldx=0), -3),
    (dict(E=257, ldx=257), -3), (dict(topk=0), -3), (dict(topk=9), -3),
    (dict(E=64, ldx=64, topk=33), -3), (dict(ldx=7), -4), (dict(score=2), -1),
    (dict(groups=0), -3), (dict(groups=3), -3), (dict(E=66, ldx=66, groups=33), -3),
    (dict(groups=4, topk_groups=5), -3), (dict(groups=4, topk_groups=0), -3),
    (dict(groups=4, topk_groups=1, topk=3), -3), (dict(group_top=3), -1),
    (dict(x=None), -1), (dict(w=None), -1), (dict(i=None), -1),
])
def test_route_refusals(kw, code):
    assert route(**kw) == code
    assert b"moe_route" in _lib.load().ctb_last_error()


def test_route_of_no_rows_is_a_no_op():
    assert route(T=0, x=None, w=None, i=None) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=_lib.CTB_I32), -2), (dict(T=-1), -3), (dict(topk=0), -3), (dict(E=300), -3),
    (dict(ldx=7), -4), (dict(lddx=7), -4), (dict(score=-1), -1), (dict(dw=None), -1),
    (dict(dx=None), -1), (dict(ids=None), -1), (dict(x=None), -1), (dict(T=0, x=None), 0),
])
def test_route_bwd_refusals(kw, code):
    a = dict(dtype=_lib.CTB_F32, dw=NP, x=NP, ids=NP, dx=NP, T=4, E=8, topk=2, ldx=300, lddx=300,
             score=0)
    a.update(kw)
    assert _lib.load().ctb_moe_route_bwd(a["dtype"], a["dw"], a["x"], a["ids"], a["dx"], a["T"],
                                         a["E"], a["topk"], a["ldx"], a["lddx"], a["score"], 1,
                                         ctypes.c_float(1.0), None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=_lib.CTB_F32), -2), (dict(T=-1), -3), (dict(N=-1), -3), (dict(topk=0), -3),
    (dict(T=1 << 30, topk=4), -3), (dict(ids=NP, E=0), -3), (dict(ldy=15), -4),
    (dict(ldo=15), -4), (dict(res=NP, ldr=15), -4), (dict(y=None), -1), (dict(out=None), -1),
    (dict(out=NP + 4096, y=NP + 4096), -1),
    (dict(T=0, y=None), 0), (dict(N=0, ldy=0, ldo=0, y=None), 0),
])
def test_combine_refusals(kw, code):
    a = dict(dtype=_lib.CTB_F16, y=NP, ids=None, res=None, out=NP, T=4, topk=2, N=16, E=4, ldy=16,
             ldr=16, ldo=16)
    a.update(kw)
    assert _lib.load().ctb_moe_combine(a["dtype"], a["y"], None, a["ids"], a["res"], a["out"],
                                       a["T"], a["topk"], a["N"], a["E"], a["ldy"], a["ldr"],
                                       a["ldo"], None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=_lib.CTB_F32), -2), (dict(T=-1), -3), (dict(topk=-2), -3), (dict(lddo=15), -4),
    (dict(ldy=15), -4), (dict(lddy=15), -4), (dict(d=None), -1), (dict(y=None), -1),
    (dict(dy=None), -1), (dict(dw=None), -1), (dict(dy=NP), -1), (dict(T=0, d=None), 0), (dict(ids=NP, E=-1), -3),
])
def test_combine_bwd_refusals(kw, code):
    a = dict(dtype=_lib.CTB_BF16, d=NP, y=NP, w=NP, ids=None, dy=NP, dw=NP, T=4, topk=2, N=16, E=4,
             lddo=16, ldy=16, lddy=16)
    a.update(kw)
    assert _lib.load().ctb_moe_combine_bwd(a["dtype"], a["d"], a["y"], a["w"], a["ids"], a["dy"],
                                           a["dw"], a["T"], a["topk"], a["N"], a["E"], a["lddo"],
                                           a["ldy"], a["lddy"], None) == code


def test_python_calls_refuse_host_tensors():
    x = torch.zeros(4, 8)
    for call in (lambda: ops.moe_route(x, 2),
                 lambda: ops.moe_route_bwd(x[:, :2], x, torch.zeros(4, 2, dtype=torch.int32)),
                 lambda: ops.moe_combine(x.half(), 2),
                 lambda: ops.moe_combine_bwd(x.half(), None, 2)):
        with pytest.raises(B200Error) as e:
            call()
        assert e.value.status == "CTB_ERR_ARG"
