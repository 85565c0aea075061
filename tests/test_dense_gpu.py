"""The dense layer on the GPU against float64.

Tolerances, per element. A product's Float32 sum of K terms errs by at most
K * 2^-24 of the sum of their magnitudes (tensor cores add in blocks of 16, so
by less); the activations' slopes are at most 1.13 and their own error is below
2e-6 of |z| + 1; the result is rounded to 16 bits once: half a step of its
value, or of the type's smallest step (Float16: 2^-24). In the gradients dZ is
itself rounded: half a step of each term more.
"""
import numpy as np
import pytest
import torch

from cutile_b200 import B200Error, ops
from oracle import oracle as O

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16}
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
EPS32 = 2.0 ** -24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    return 2.0 ** -25 if dt == torch.float16 else 1e-38


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def inputs(dev, dt, N, M, K, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    A = (r(K, M) / max(K, 1) ** 0.5).to(DT[dt]).to(dev)
    B = r(N, K).to(DT[dt]).to(dev)
    return A, B, r(M).to(dev), r(N, M).to(DT[dt]).to(dev)


def check_forward(dev, dt, N, M, K, act, A, B, bias, R, **kw):
    Z = torch.full((N, M), 3.0, dtype=DT[dt], device=dev)
    C = ops.dense(A, B, bias=bias, act=act, residual=R, preact=Z, **kw)
    y, z = O.dense(f64(A), f64(B), f64(bias), act, f64(R))
    mag = np.abs(f64(B)) @ np.abs(f64(A))
    if bias is not None:
        mag = mag + np.abs(f64(bias))
    h, t = half_step(DT[dt]), tiny(DT[dt])
    zerr = (K + 2) * EPS32 * mag
    assert np.all(np.abs(f64(Z) - z) <= zerr + h * np.abs(z) * (1 + 1e-5) + t)
    yerr = 1.13 * zerr + 2e-6 * (np.abs(z) + 1) + (0 if R is None else EPS32 * np.abs(f64(R)))
    assert np.all(np.abs(f64(C) - y) <= yerr * (1 + h) + h * np.abs(y) + t)
    assert torch.equal(ops.dense(A, B, bias=bias, act=act, residual=R), C)
    return C


SHAPES = [(1, 1, 1), (1, 8, 8), (1, 256, 1024), (3, 17, 33), (2, 4096, 64), (16, 128, 256),
          (17, 200, 512), (37, 513, 96), (64, 64, 4096), (65, 264, 72), (100, 1000, 1000),
          (129, 129, 257), (200, 520, 136), (300, 384, 640), (513, 1001, 77)]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("N,M,K", SHAPES)
def test_dense_shapes(dev, dt, N, M, K):
    A, B, bias, R = inputs(dev, dt, N, M, K, N + M + K)
    check_forward(dev, dt, N, M, K, "none", A, B, None, None)
    check_forward(dev, dt, N, M, K, "silu", A, B, bias, R)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("N", [5, 300])
def test_dense_epilogues(dev, dt, act, N):
    A, B, bias, R = inputs(dev, dt, N, 136, 72, N)
    for b in (None, bias, bias.to(DT[dt])):
        for r in (None, R):
            check_forward(dev, dt, N, 136, 72, act, A, B, b, r)


def exact64(A, B, bias, act, R):
    """The same formula in float64 on the device, for sizes numpy takes too long for."""
    z = B.double() @ A.double()
    if bias is not None:
        z = z + bias.double()
    y = {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "silu": lambda v: v * torch.sigmoid(v),
         "gelu": lambda v: v * torch.special.ndtr(v)}[act](z)
    return (y if R is None else y + R.double()), z


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("N,M,K,act", [(1, 4096, 4096, "silu"), (7, 14336, 1024, "gelu"),
                                       (96, 2048, 8192, "relu"), (1000, 2056, 520, "gelu"),
                                       (2049, 2304, 200, "silu"), (4096, 2560, 1024, "none"),
                                       (2304, 4099, 333, "relu"), (40000, 48, 64, "relu"),
                                       (30000, 330, 40, "gelu"), (60001, 8, 128, "silu")])
def test_dense_large(dev, dt, N, M, K, act):
    A, B, bias, R = inputs(dev, dt, N, M, K, 7)
    Z = torch.empty((N, M), dtype=DT[dt], device=dev)
    C = ops.dense(A, B, bias=bias, act=act, residual=R, preact=Z)
    ops.check_device()
    y, z = exact64(A, B, bias, act, R)
    mag = B.double().abs() @ A.double().abs() + bias.double().abs()
    h, t = half_step(DT[dt]), tiny(DT[dt])
    zerr = (K + 2) * EPS32 * mag
    assert bool(((Z.double() - z).abs() <= zerr + h * z.abs() * (1 + 1e-5) + t).all())
    yerr = 1.13 * zerr + 2e-6 * (z.abs() + 1) + EPS32 * R.double().abs()
    assert bool(((C.double() - y).abs() <= yerr * (1 + h) + h * y.abs() + t).all())
    # and far nearer on the whole: rounding alone is at most h
    assert float((C.double() - y).norm() / y.norm()) <= 1.05 * h


def check_gradients(dev, dt, N, M, K, act, A, B, dC, Z, on_device=False, **kw):
    dA, dB, db = ops.dense_bwd(dC, A, B, act=act, preact=Z, **kw)
    h, t = half_step(DT[dt]), tiny(DT[dt])
    if on_device:
        z = Z.double()
        s = torch.sigmoid(z)
        slope = {"none": lambda: torch.ones_like(z), "silu": lambda: s * (1 + z * (1 - s)),
                 "relu": lambda: (z > 0).double()}[act]()
        dz = dC.double() * slope
        a, b = A.double(), B.double()
        rA, rB, rb = b.t() @ dz, dz @ a.t(), dz.sum(0)
        mA, mB, mb = b.abs().t() @ dz.abs(), dz.abs() @ a.abs().t(), dz.abs().sum(0)
        gA, gB, gb = dA.double(), dB.double(), db.double()
        ok = lambda v: bool(v.all())  # noqa: E731
    else:
        rA, rB, rb, dz = O.dense_bwd(f64(dC), f64(A), f64(B), act, f64(Z))
        mA, mB = np.abs(f64(B)).T @ np.abs(dz), np.abs(dz) @ np.abs(f64(A)).T
        mb = np.abs(dz).sum(0)
        gA, gB, gb = f64(dA), f64(dB), f64(db)
        ok = np.all
    # each dZ: 3e-6 of |dC| for the slope (at most 2e-6 (|z| + 1) / |z| in the products
    # of this size, which |dz| bounds up to the kinks), half a step, tiny
    slack = 4e-6 * float(dC.abs().max())
    term = h * (1 + 1e-5)
    aB, aA = float(B.abs().max()) if K else 0, float(A.abs().max()) if K else 0
    assert ok(abs(gA - rA) <= ((N + 1) * EPS32 + term) * mA + h * abs(rA) + N * aB * (slack + t) + t)
    assert ok(abs(gB - rB) <= ((M + 1) * EPS32 + term) * mB + h * abs(rB) + M * aA * (slack + t) + t)
    assert ok(abs(gb - rb) <= (N + 1) * EPS32 * mb + N * slack + 1e-30)
    return dA, dB, db


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("N,M,K", SHAPES)
def test_dense_gradients(dev, dt, N, M, K):
    A, B, _, Z = inputs(dev, dt, N, M, K, N + M)
    dC = torch.randn(N, M, generator=torch.Generator().manual_seed(K)).to(DT[dt]).to(dev)
    check_gradients(dev, dt, N, M, K, "silu", A, B, dC, Z)
    check_gradients(dev, dt, N, M, K, "none", A, B, dC, None)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("act", ACTS)
def test_dense_gradients_of_each_activation(dev, dt, act):
    A, B, _, Z = inputs(dev, dt, 130, 136, 72, 3)
    Z[0, :5] = torch.tensor([0.0, -0.0, 60000.0, -60000.0, 1e-7], device=dev)
    dC = torch.randn(130, 136, generator=torch.Generator().manual_seed(4)).to(DT[dt]).to(dev)
    dA, dB, db = check_gradients(dev, dt, 130, 136, 72, act, A, B, dC, Z)
    assert bool(torch.isfinite(dA).all() & torch.isfinite(dB).all() & torch.isfinite(db).all())
    only = ops.dense_bwd(dC, A, B, act=act, preact=Z, need_dB=False, need_dbias=False)
    assert torch.equal(only[0], dA) and only[1] is None and only[2] is None
    only = ops.dense_bwd(dC, A, B, act=act, preact=Z, need_dA=False)
    assert only[0] is None and torch.equal(only[1], dB) and torch.equal(only[2], db)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("N,M,K,act", [(2049, 2304, 520, "silu"), (4096, 2560, 2048, "relu"),
                                       (1000, 2307, 1003, "none"), (8, 4096, 4096, "silu"),
                                       (50000, 72, 56, "silu")])
def test_dense_gradients_large(dev, dt, N, M, K, act):
    A, B, _, Z = inputs(dev, dt, N, M, K, 11)
    dC = torch.randn(N, M, generator=torch.Generator().manual_seed(4)).to(DT[dt]).to(dev)
    check_gradients(dev, dt, N, M, K, act, A, B, dC, Z, on_device=True)
    ops.check_device()


def test_activation_extremes(dev):
    """Values before the activation from far below to far above 0, and the
    smallest ones: z = x * 1 exactly."""
    x = torch.tensor([0.0, -0.0, 1e-7, -1e-7, 0.5, -0.5, 5.0, -5.0, 9.0, -9.0, 30.0, -30.0, 300.0,
                      -300.0, 6e4, -6e4], device=dev).half()
    B = torch.zeros(16, 16, dtype=torch.float16, device=dev)
    B[:, 0] = x
    A = torch.zeros(16, 16, dtype=torch.float16, device=dev)
    A[0] = 1
    for act in ACTS:
        C = f64(ops.dense(A, B, act=act))
        ref = O.activation(f64(x), act)[0][:, None]
        assert np.all(np.abs(C - ref) <= 2.0 ** -11 * np.abs(ref) + 2e-6 * (np.abs(f64(x)) + 1)[:, None] * (np.abs(ref) < 1e-3) + 2.0 ** -24)


@pytest.mark.parametrize("N", [16, 300])
def test_non_finite_values_through_the_activations(dev, N):
    """NaN stays NaN; +inf is +inf; and a gradient of 0 at an infinite value
    before the activation stays 0 under relu and gelu."""
    A = torch.zeros(16, 16, dtype=torch.bfloat16, device=dev)
    A[0, 0] = 1
    B = torch.zeros(N, 16, dtype=torch.bfloat16, device=dev)
    B[:3, 0] = torch.tensor([float("nan"), float("inf"), -float("inf")], device=dev)
    for act in ACTS:
        C = ops.dense(A, B, act=act)[:, 0]
        assert bool(C[0].isnan()) and C[1].item() == float("inf")
        assert C[2].item() == (-float("inf") if act == "none" else 0.0) or act in ("silu", "gelu_tanh")
        assert bool((C[3:] == 0).all())
    Z = torch.full((N, 16), float("inf"), dtype=torch.bfloat16, device=dev)
    Z[::2] = -float("inf")
    for act in ("relu", "gelu"):
        dC = torch.zeros_like(Z)
        dC[0, 0], dC[1, 1] = 2, 3  # slopes 0 at -inf, 1 at +inf
        db = ops.dense_bwd(dC, A, torch.zeros_like(B), act=act, preact=Z)[2]
        assert db.tolist() == [0.0, 3.0] + [0.0] * 14


def test_strides_alignment_and_guards(dev):
    N, M, K = 40, 144, 80
    A, B, bias, R = inputs(dev, "f16", N, M, K, 5)
    ref = ops.dense(A, B, bias=bias, act="silu", residual=R)
    dC = R
    Z = torch.empty_like(ref)
    ops.dense(A, B, bias=bias, act="silu", preact=Z)
    gref = ops.dense_bwd(dC, A, B, act="silu", preact=Z)
    for off in (0, 8, 1, 2):
        def view(t, fill=9.0):
            big = torch.full((t.shape[0], t.shape[1] + 24), fill, dtype=t.dtype, device=dev)
            v = big[:, off:off + t.shape[1]]
            v.copy_(t)
            return big, v

        _, Av = view(A)
        _, Bv = view(B, float("nan"))  # what lies between rows is not read into sums
        _, Rv = view(R, float("nan"))
        big, Cv = view(torch.zeros_like(ref))
        zbig, Zv = view(torch.zeros_like(ref))
        ops.dense(Av, Bv, bias=bias, act="silu", residual=Rv, out=Cv, preact=Zv)
        assert torch.equal(Cv, ref) and torch.equal(Zv, Z)
        for b in (big, zbig):
            assert bool((b[:, :off] == 9).all()) and bool((b[:, off + M:] == 9).all())
        abig, dAv = view(torch.zeros_like(A))
        bbig, dBv = view(torch.zeros_like(B))
        got = ops.dense_bwd(Rv, Av, Bv, act="silu", preact=Zv, dA_t=dAv, dB_t=dBv)
        for g, r in zip(got, gref):
            assert torch.equal(g, r)
        for b, n in ((abig, M), (bbig, K)):
            assert bool((b[:, :off] == 9).all()) and bool((b[:, off + n:] == 9).all())
    out = R.clone()
    ops.dense(A, B, bias=bias, act="silu", residual=out, out=out)
    assert torch.equal(out, ref)


def test_empty_dimensions(dev):
    z = lambda *s: torch.zeros(*s, dtype=torch.float16, device=dev)  # noqa: E731
    bias = torch.arange(4.0, device=dev)
    assert ops.dense(z(8, 4), z(0, 8)).shape == (0, 4)
    assert ops.dense(z(8, 0), z(3, 8)).shape == (3, 0)
    got = ops.dense(z(0, 4), z(3, 0), bias=bias, act="relu", residual=z(3, 4) + 1)
    assert torch.equal(got, (bias + 1).half().expand(3, 4))  # a product over nothing is zero
    dA, dB, db = ops.dense_bwd(z(0, 4), z(8, 4), z(0, 8))
    assert bool((dA == 0).all()) and dB.shape == (0, 8) and bool((db == 0).all())
    dA, dB, db = ops.dense_bwd(z(3, 0), z(8, 0), z(3, 8) + 1, dB_t=z(3, 8) + 5)
    assert dA.shape == (8, 0) and bool((dB == 0).all()) and db.shape == (0,)
    dA, dB, db = ops.dense_bwd(z(3, 4) + 1, z(0, 4), z(3, 0), act="relu", preact=z(3, 4) + 1)
    assert dA.shape == (0, 4) and dB.shape == (3, 0) and bool((db == 3).all())


def test_non_finite_values_stay_where_they_are(dev):
    """A NaN or an infinity in one token's row reaches that row only, in one
    weight's column that column only."""
    for N, M, K in ((3, 40, 64), (300, 520, 136), (37, 33, 21)):
        A, B, _, _ = inputs(dev, "bf16", N, M, K, 2)
        ref = ops.dense(A, B)
        Bn = B.clone()
        Bn[1, K // 2] = float("nan")
        got = ops.dense(A, Bn)
        assert bool(got[1].isnan().all()) and torch.equal(got[2:], ref[2:]) and torch.equal(got[0], ref[0])
        An = A.clone()
        An[K - 1, 5] = float("inf")
        got = ops.dense(An, B)
        assert not bool(torch.isfinite(got[:, 5]).any())
        assert torch.equal(got[:, 6:], ref[:, 6:]) and torch.equal(got[:, :5], ref[:, :5])


def test_refusals(dev):
    h = lambda *s: torch.zeros(*s, dtype=torch.float16, device=dev)  # noqa: E731
    bad = [
        lambda: ops.dense(h(8, 4), h(3, 7)), lambda: ops.dense(h(8, 4).float(), h(3, 8).float()),
        lambda: ops.dense(h(8, 4), h(3, 8).bfloat16()), lambda: ops.dense(h(8, 4)[0], h(3, 8)),
        lambda: ops.dense(h(4, 8).t(), h(3, 8)), lambda: ops.dense(h(8, 4), h(8, 3).t()),
        lambda: ops.dense(h(8, 4), h(3, 8), act="tanh"),
        lambda: ops.dense(h(8, 4), h(3, 8), bias=h(3)),
        lambda: ops.dense(h(8, 4), h(3, 8), bias=h(4).bfloat16()),
        lambda: ops.dense(h(8, 4), h(3, 8), bias=h(8)[::2]),
        lambda: ops.dense(h(8, 4), h(3, 8), residual=h(3, 5)),
        lambda: ops.dense(h(8, 4), h(3, 8), preact=h(4, 4)),
        lambda: ops.dense(h(8, 4), h(3, 8), out=h(3, 4).bfloat16()),
        lambda: ops.dense(h(8, 4), h(1, 8).expand(3, 8)),
        lambda: ops.dense(h(8, 4), torch.zeros(3, 8, dtype=torch.float16)),
        lambda: ops.dense_bwd(h(3, 5), h(8, 4), h(3, 8)),
        lambda: ops.dense_bwd(h(3, 4), h(8, 4), h(3, 8), act="silu"),
        lambda: ops.dense_bwd(h(3, 4), h(8, 4), h(3, 8), dA_t=h(4, 8)),
        lambda: ops.dense_bwd(h(3, 4), h(8, 4), h(3, 8), dbias=h(4)),
        lambda: ops.dense_bwd(h(1).expand(3, 4), h(8, 4), h(3, 8)),
    ]
    for call in bad:
        with pytest.raises(B200Error):
            call()


def test_captured_and_on_another_stream(dev):
    """One call and its gradients eagerly, on a side stream, and twice replayed
    from each of two graphs: the same bits every time."""
    cases = []
    for N, M, K in ((3, 264, 512), (300, 33, 77), (2304, 2304, 128)):
        A, B, bias, R = inputs(dev, "bf16", N, M, K, N)
        cases.append((A, B, bias, R))

    def work():
        out = []
        for A, B, bias, R in cases:
            Z = torch.empty_like(R)
            out += [ops.dense(A, B, bias=bias, act="gelu", residual=R, preact=Z), Z]
            out += ops.dense_bwd(R, A, B, act="gelu", preact=Z)
        return out

    eager = work()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = work()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, work()))
    for _ in range(2):
        for g, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for held in (other, graphs[0][1], graphs[1][1]):
        for a, b in zip(eager, held):
            assert torch.equal(a, b)
    ops.check_device()
