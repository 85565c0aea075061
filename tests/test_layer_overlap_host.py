"""Layer calls whose outputs share memory with what they read, or with one
another, are refused before any CUDA call, at every offset and pair of strides;
rows that lie between one another's are not taken for overlapping ones."""
import ctypes
import itertools
import random

import pytest
import torch

from cutile_b200 import _lib

# A call that is not refused goes on to the device with pointers to nothing: this
# file is for machines without one.
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="needs a machine without a GPU")

NP = 1 << 30
F16, F32, BF16 = _lib.CTB_F16, _lib.CTB_F32, _lib.CTB_BF16


def refused(rc):
    if rc == -1:
        assert b"of its own" in _lib.load().ctb_last_error() or b"of their own" in _lib.load().ctb_last_error()
    else:
        assert rc in (-5, -6), rc  # a CUDA error, or no device: the operands were accepted
    return rc == -1


def test_refused_exactly_where_a_byte_is_shared():
    """moe_combine's out against its residual, both T x N, against the sets of
    their elements."""
    L = _lib.load()
    rng = random.Random(1)
    seen = {True: 0, False: 0}
    for _ in range(4000):
        T, N = rng.randint(1, 6), rng.randint(1, 9)
        ldo = N + rng.choice([0, 0, 1, 3, N, 20])
        ldr = rng.choice([ldo, N, N + rng.randint(0, 30)])
        at = rng.randint(-70, 70)
        out = {i * ldo + c for i in range(T) for c in range(N)}
        res = {at + i * ldr + c for i in range(T) for c in range(N)}
        want = bool(out & res) and not (at == 0 and (ldo == ldr or T == 1))
        rc = L.ctb_moe_combine(F16, NP << 1, None, None, NP + 2 * at, NP, T, 1, N, 1, N, ldr, ldo, None)
        assert refused(rc) == want, (T, N, ldo, ldr, at)
        seen[want] += 1
    assert min(seen.values()) > 500


def call(name, **kw):
    """One small call with every operand in memory of its own, `kw` put over it."""
    L, at = _lib.load(), iter(range(NP + (1 << 24), 2 * NP, 1 << 20))
    p = lambda *names: {n: next(at) for n in names}  # noqa: E731
    if name == "dense":  # M 16, N 4, K 32
        a = dict(p("A", "B", "bias", "R", "Z", "C", "ws"), lda=17, ldb=32, ldr=16, ldz=16, ldc=16)
        a.update(kw)
        return L.ctb_dense_fwd(F16, a["A"], a["B"], a["bias"], F32, a["R"], a["Z"], a["C"], 16, 4, 32,
                               a["lda"], a["ldb"], a["ldr"], a["ldz"], a["ldc"], 1, a["ws"], 1 << 16, None)
    if name == "dense_bwd":
        a = dict(p("dC", "A", "B", "Z", "dA", "dB", "db", "ws"), lddc=16, lda=16, ldb=32, ldz=16,
                 ldda=16, lddb=32)
        a.update(kw)
        return L.ctb_dense_bwd(BF16, a["dC"], a["A"], a["B"], a["Z"], a["dA"], a["dB"], a["db"], 16, 4,
                               32, a["lddc"], a["lda"], a["ldb"], a["ldz"], a["ldda"], a["lddb"], 4,
                               a["ws"], 1 << 16, None)
    if name == "moe_route":  # T 4, E 8, topk 2
        a = dict(p("x", "bias", "w", "i"), ldx=8)
        a.update(kw)
        return L.ctb_moe_route(F32, a["x"], a["bias"], a["w"], a["i"], 4, 8, 2, a["ldx"], 0, 1, 1, 2, 1,
                               ctypes.c_float(1), None)
    if name == "moe_route_bwd":
        a = dict(p("dw", "x", "i", "dx"), ldx=8, lddx=8)
        a.update(kw)
        return L.ctb_moe_route_bwd(F32, a["dw"], a["x"], a["i"], a["dx"], 4, 8, 2, a["ldx"], a["lddx"],
                                   0, 1, ctypes.c_float(1), None)
    if name == "moe_combine":  # N 16
        a = dict(p("y", "w", "i", "R", "out"), T=4, topk=2, ldy=16, ldr=16, ldo=16)
        a.update(kw)
        return L.ctb_moe_combine(F16, a["y"], a["w"], a["i"], a["R"], a["out"], a["T"], a["topk"], 16, 3,
                                 a["ldy"], a["ldr"], a["ldo"], None)
    a = dict(p("d", "y", "w", "i", "dy", "dw"), T=4, topk=2, lddo=16, ldy=16, lddy=16)
    a.update(kw)
    return L.ctb_moe_combine_bwd(F16, a["d"], a["y"], a["w"], a["i"], a["dy"], a["dw"], a["T"],
                                 a["topk"], 16, 3, a["lddo"], a["ldy"], a["lddy"], None)


PAIRS = {
    "dense": [("C", o) for o in ("A", "B", "bias", "R", "Z", "ws")] +
             [("Z", o) for o in ("A", "B", "bias", "R", "C", "ws")] +
             [("ws", o) for o in ("A", "B", "bias", "R")],
    "dense_bwd": [(o, i) for o in ("dA", "dB", "db", "ws")
                  for i in ("dC", "A", "B", "Z", "dA", "dB", "db", "ws") if o != i],
    "moe_route": [("w", "x"), ("w", "bias"), ("w", "i"), ("i", "x"), ("i", "bias")],
    "moe_route_bwd": [("dx", "dw"), ("dx", "x"), ("dx", "i")],
    "moe_combine": [("out", o) for o in ("y", "w", "i", "R")],
    "moe_combine_bwd": [("dy", o) for o in ("d", "y", "w", "i", "dw")] +
                       [("dw", o) for o in ("d", "y", "w", "i")],
}


@pytest.mark.parametrize("name", sorted(PAIRS))
def test_operands_of_their_own_are_accepted(name):
    assert not refused(call(name))


@pytest.mark.parametrize("name,out,other", [(n, *p) for n, ps in PAIRS.items() for p in ps])
def test_outputs_shifted_into_another_operand(name, out, other):
    for shift in (4, 28):  # bytes; every operand is at least 32 long
        assert refused(call(name, **{out: NP + (1 << 28) + shift, other: NP + (1 << 28)}))
        assert refused(call(name, **{out: NP + (1 << 28), other: NP + (1 << 28) + shift}))


@pytest.mark.parametrize("name,kw", [
    ("dense", dict(C=NP, R=NP, ldc=16, ldr=24)), ("dense", dict(C=NP, R=NP, ldc=24, ldr=16)),
    ("moe_route_bwd", dict(dx=NP, x=NP, ldx=8, lddx=9)),
    ("moe_combine", dict(out=NP, R=NP, ldo=24)), ("moe_combine", dict(out=NP, y=NP, topk=1, ldy=32)),
    ("moe_combine", dict(out=NP, y=NP)),
    ("moe_combine_bwd", dict(dy=NP, d=NP, topk=1, lddo=17)), ("moe_combine_bwd", dict(dy=NP, d=NP)),
    ("moe_combine_bwd", dict(dy=NP, y=NP, ldy=32)),
])
def test_in_place_needs_the_same_rows(name, kw):
    assert refused(call(name, **kw))


@pytest.mark.parametrize("name,kw", [
    ("dense", dict(C=NP, R=NP)), ("dense", dict(C=NP, R=NP, ldc=40, ldr=40)),
    ("moe_route_bwd", dict(dx=NP, x=NP)),
    ("moe_combine", dict(out=NP, R=NP)), ("moe_combine", dict(out=NP, y=NP, topk=1)),
    ("moe_combine", dict(out=NP, R=NP, T=1, ldo=24, ldr=16)),  # one row has no stride
    ("moe_combine_bwd", dict(dy=NP, d=NP, topk=1)), ("moe_combine_bwd", dict(dy=NP, y=NP)),
    ("moe_combine_bwd", dict(dw=NP, w=NP)),
    # not read: A where dB is not wanted, y without weights
    ("dense_bwd", dict(dA=NP, A=NP, dB=None)), ("moe_combine_bwd", dict(dy=NP + 2, y=NP, w=None)),
])
def test_in_place_and_operands_that_are_not_read(name, kw):
    assert not refused(call(name, **kw))


def test_columns_and_rows_of_one_buffer():
    wide = dict(ldc=64, ldr=64, ldz=64, C=NP, R=NP + 32, Z=NP + 64)
    assert not refused(call("dense", **wide))
    assert refused(call("dense", **dict(wide, Z=NP + 62)))
    for rows in itertools.permutations((NP, NP + 32, NP + 64)):  # every third row each
        kw = dict(zip("CRZ", rows), ldc=48, ldr=48, ldz=48)
        assert not refused(call("dense", **kw))
