"""Routing and combine on the GPU against the float64 oracles.

Tolerances. Weights (Float32): expf is documented to 2 ulp, its argument is
rounded (|x| <= 24 here: 24 * 2^-24), the row's sum and the division add a few
2^-24, the fast exponentials of the sum weigh in with at most 2e-6: 1e-5
relative covers them. Route gradients: the same relative error on each term,
so 1e-5 of the row's largest term, plus the output type's half step. Combine:
topk Float32 multiply-adds, (topk + 1) * 2^-24 of the terms' magnitudes, plus
the half step eps / 2 of the result. Ids must be equal.
"""
import numpy as np
import pytest
import torch

from cutile_b200 import B200Error, ops
from oracle import oracle as O

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def half_step(dt):
    return torch.finfo(dt).eps / 2


def f64(t):
    return t.detach().double().cpu().numpy()


def logits(T, E, dt, seed, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, E, generator=g) * scale).to(DT[dt])


def check_route(dev, x, topk, **kw):
    bias = kw.pop("bias", None)
    w, i = ops.moe_route(x, topk, bias=None if bias is None else bias.to(dev), **kw)
    rw, ri = O.moe_route(f64(x), topk, bias=None if bias is None else f64(bias), **kw)
    np.testing.assert_array_equal(i.cpu().numpy(), ri)
    np.testing.assert_allclose(f64(w), rw, rtol=1e-5, atol=1e-30)
    return w, i


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,topk", [(1, 1, 1), (1, 8, 2), (5, 7, 7), (33, 16, 3), (100, 31, 4),
                                      (17, 64, 6), (9, 65, 8), (50, 128, 32), (40, 250, 9),
                                      (77, 256, 8)])
@pytest.mark.parametrize("renorm", [True, False])
def test_route(dev, dt, score, T, E, topk, renorm):
    x = logits(T, E, dt, T * 1000 + E).to(dev)
    check_route(dev, x, topk, score=score, renorm=renorm, scale=1.5)
    g = torch.Generator().manual_seed(E)
    bias = torch.randn(E, generator=g) * 0.2
    check_route(dev, x, topk, score=score, renorm=renorm, bias=bias)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("E,groups,keep,top,topk", [
    (8, 2, 1, 2, 2), (12, 4, 2, 1, 3), (64, 8, 3, 2, 8), (96, 32, 5, 2, 4), (160, 8, 3, 2, 6),
    (256, 8, 4, 2, 8), (256, 8, 1, 1, 32), (255, 5, 2, 2, 8), (32, 32, 7, 2, 7), (9, 3, 3, 2, 4)])
def test_route_groups(dev, score, biased, E, groups, keep, top, topk):
    for dt in ("bf16", "f32"):
        x = logits(70, E, dt, E + keep).to(dev)
        g = torch.Generator().manual_seed(E)
        bias = torch.randn(E, generator=g) * 0.3 if biased else None
        check_route(dev, x, topk, score=score, bias=bias, groups=groups, topk_groups=keep,
                    group_top=top)


def test_route_strides_and_alignment(dev):
    big = logits(40, 300, "bf16", 5).to(dev)
    for x in (big[:, :64], big[:, 1:65], big[::3, 7:107], big[3:4, 2:10]):
        check_route(dev, x, 4)
        w = torch.rand(x.shape[0], 4, device=dev)
        _, ids = ops.moe_route(x, 4)
        dx = torch.full((x.shape[0], x.shape[1] + 3), 7.0, dtype=x.dtype, device=dev)
        ops.moe_route_bwd(w, x, ids, dlogits=dx[:, 1:-2])
        assert bool((dx[:, 0] == 7).all()) and bool((dx[:, -2:] == 7).all())
        assert torch.equal(dx[:, 1:-2], ops.moe_route_bwd(w, x.contiguous(), ids))


def test_route_rows_that_are_masked(dev):
    inf = float("inf")
    low = torch.finfo(torch.float32).min
    rows = torch.tensor([
        [-inf] * 6,                          # nothing left
        [-inf, 1.0, -inf, -inf, -inf, 0.5],  # fewer than topk
        [float("nan")] * 5 + [2.0],          # NaN is not available
        [low] * 6,                           # the type's lowest value is a value
        [low, 3.0, low, low, 1.0, low],
        [-200.0, -210.0, -190.0, -inf, -205.0, -201.0],  # sigmoids underflow
        [90.0, 120.0, 500.0, 88.0, 3e38, -3e38],
    ], device=dev)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            w, i = ops.moe_route(rows, 3, score=score, renorm=renorm)
            rw, ri = O.moe_route(f64(rows), 3, score=score, renorm=renorm)
            np.testing.assert_array_equal(i.cpu().numpy(), ri)
            # 1e-5, and |x| = 210 rounds a difference by 210 * 2^-24 more
            np.testing.assert_allclose(f64(w), rw, rtol=3e-5, atol=1e-37)
            d = torch.ones_like(w)
            assert bool(torch.isfinite(ops.moe_route_bwd(d, rows, i, score, renorm)).all())
    assert ops.moe_route(rows[:1], 3)[1].tolist() == [[-1, -1, -1]]
    bias = torch.tensor([0.0, -inf, 0.0, float("nan"), 0.0, inf], device=dev)
    x = torch.zeros(1, 6, device=dev)
    assert ops.moe_route(x, 4, bias=bias, score="sigmoid")[1].tolist() == [[5, 0, 2, 4]]
    assert ops.moe_route(x, 5, bias=bias, score="sigmoid")[1].tolist() == [[5, 0, 2, 4, -1]]
    up = torch.tensor([[inf, 0.0, 1.0]], device=dev)
    w, i = ops.moe_route(up, 2, score="sigmoid", renorm=False)
    assert i.tolist() == [[0, 2]] and w[0, 0].item() == 1.0


def test_route_ties_and_values_closer_than_float32(dev):
    x = torch.zeros(3, 200, device=dev)
    x[1, 100:] = -0.0  # -0 and +0 are one value
    _, i = ops.moe_route(x, 8)
    assert i.tolist() == [list(range(8))] * 3
    # Biases one Float32 step apart, so that s + bias rounds to the same Float32
    # for pairs that differ in exact arithmetic.
    g = torch.Generator().manual_seed(1)
    for E, groups, keep in ((64, 1, 1), (256, 8, 3), (24, 4, 2)):
        x = torch.randn(200, E, generator=g) * 1e-6
        bias = 1000.0 + torch.randint(0, 3, (E,), generator=g) * 6.1e-5
        for score in ("sigmoid", "softmax"):
            check_route(dev, x.to(dev), min(8, E), score=score, bias=bias.float(), groups=groups,
                        topk_groups=keep)
    # A whole warp's row: a few that tie in Float32 (100 steps), more of them than
    # lanes (3 steps); and groups that are certain while the order within is not.
    for E, groups, keep, steps in ((256, 1, 1, 100), (256, 1, 1, 3), (200, 1, 1, 60),
                                   (256, 8, 2, 12), (130, 5, 2, 20)):
        x = torch.randn(300, E, generator=g) * 1e-6
        x[::7, ::3] = float("-inf")
        bias = 1000.0 + torch.randint(0, steps, (E,), generator=g) * 6.1e-5
        bias += torch.arange(E) // (E // groups) * 10.0
        for score in ("sigmoid", "softmax"):
            check_route(dev, x.to(dev), 8, score=score, bias=bias.float(), groups=groups,
                        topk_groups=keep, renorm=False)
    # group sums far below 1: softmax of a row with one dominant expert
    x = torch.randn(300, 64, generator=g) * 1e-5 - 60
    x[:, 0] = 30
    check_route(dev, x.to(dev), 4, groups=8, topk_groups=2)


def test_route_many_rows(dev):
    """More rows than the oracle's loops take: the same rows in another order,
    in one call and in two, give the same bits."""
    x = logits(20011, 256, "f32", 9, 1.5).to(dev)
    bias = torch.randn(256, generator=torch.Generator().manual_seed(2)).to(dev) * 0.1
    kw = dict(score="sigmoid", bias=bias, groups=8, topk_groups=4, scale=2.5)
    w, i = ops.moe_route(x, 8, **kw)
    perm = torch.randperm(20011, generator=torch.Generator().manual_seed(3)).to(dev)
    wp, ip = ops.moe_route(x[perm], 8, **kw)
    assert torch.equal(wp, w[perm]) and torch.equal(ip, i[perm])
    rw, ri = O.moe_route(f64(x[:500]), 8, score="sigmoid", bias=f64(bias), groups=8, topk_groups=4,
                         scale=2.5)
    np.testing.assert_array_equal(i[:500].cpu().numpy(), ri)
    np.testing.assert_allclose(f64(w[:500]), rw, rtol=1e-5)


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T,E,topk", [(1, 1, 1), (1, 8, 2), (6, 13, 5), (40, 64, 6), (21, 100, 32),
                                      (30, 256, 8)])
def test_route_gradient(dev, dt, score, renorm, T, E, topk):
    x = logits(T, E, dt, T + E).to(dev)
    _, ids = ops.moe_route(x, topk, score=score)
    ids[0, topk - 1] = -1 if T > 1 else ids[0, topk - 1]
    dw = torch.randn(T, topk, generator=torch.Generator().manual_seed(T)).to(dev)
    dx = ops.moe_route_bwd(dw, x, ids, score, renorm, 1.5)
    ref = O.moe_route_bwd(f64(dw), f64(x), ids.cpu().numpy(), score, renorm, 1.5)
    top = 1.5 * np.abs(f64(dw)).max(1, keepdims=True)  # shares are at most 1
    # f16: results below its normal range are rounded to a step of 2^-24
    tiny = 2.0 ** -25 if dt == "f16" else 0.0
    assert np.all(np.abs(f64(dx) - ref) <= 1e-5 * top + half_step(DT[dt]) * np.abs(ref) + tiny)


def test_route_gradient_same_expert_twice(dev):
    x = logits(2, 20, "f32", 1).to(dev)
    ids = torch.tensor([[3, 3], [7, 25]], dtype=torch.int32, device=dev)
    dw = torch.tensor([[1.0, 2.0], [3.0, 4.0]], device=dev)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            dx = ops.moe_route_bwd(dw, x, ids, score, renorm)
            ref = O.moe_route_bwd(f64(dw), f64(x), ids.cpu().numpy(), score, renorm)
            assert np.abs(f64(dx) - ref).max() <= 1e-5 * 4


def combine_inputs(dev, dt, T, topk, N, seed, drop):
    g = torch.Generator().manual_seed(seed)
    y = torch.randn(T * topk, N, generator=g).to(DT[dt])
    w = torch.rand(T, topk, generator=g)
    ids = torch.randint(0, 5, (T, topk), generator=g, dtype=torch.int32)
    if drop:
        lost = torch.rand(T, topk, generator=g) < 0.3
        ids[lost] = torch.where(torch.rand(int(lost.sum()), generator=g) < 0.5, -1, 5).to(torch.int32)
        y[lost.reshape(-1)] = float("nan")
        w[lost] = float("inf")
    r = torch.randn(T, N, generator=g).to(DT[dt])
    return y.to(dev), w.to(dev), ids.to(dev), r.to(dev)


SHAPES = [(1, 1, 1), (1, 8, 4096), (3, 2, 17), (64, 3, 256), (5, 40, 72), (257, 6, 1000),
          (33, 4, 520), (2, 5, 14336)]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("T,topk,N", SHAPES)
@pytest.mark.parametrize("drop", [False, True])
def test_combine(dev, dt, T, topk, N, drop):
    y, w, ids, r = combine_inputs(dev, dt, T, topk, N, T + N, drop)
    use = dict(ids=ids, num_experts=5) if drop else {}
    for weights in ((w,) if drop else (w, None)):
        for res in (None, r):
            out = ops.moe_combine(y, topk, weights, residual=res, **use)
            n = {k: (f64(v) if v is not None else None) for k, v in dict(y=y, w=weights, r=res).items()}
            i = ids.cpu().numpy() if drop else None
            ref = O.moe_combine(n["y"], topk, n["w"], i, 5, n["r"])
            mag = O.moe_combine(np.abs(n["y"]), topk, n["w"], i, 5,
                                None if n["r"] is None else np.abs(n["r"]))
            tol = (topk + 1) * 2.0 ** -24 * mag + half_step(DT[dt]) * np.abs(ref) * (1 + 1e-5) + 1e-7
            assert np.all(np.abs(f64(out) - ref) <= tol)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("T,topk,N", SHAPES)
@pytest.mark.parametrize("drop", [False, True])
def test_combine_gradients(dev, dt, T, topk, N, drop):
    y, w, ids, d = combine_inputs(dev, dt, T, topk, N, T + N, drop)
    use = dict(ids=ids, num_experts=5) if drop else {}
    i = ids.cpu().numpy() if drop else None
    dy, dw = ops.moe_combine_bwd(d, y, topk, w, **use)
    rdy, rdw = O.moe_combine_bwd(f64(d), f64(y), topk, f64(w), i, 5)
    # one product rounded to 32 bits, then to the output
    assert np.all(np.abs(f64(dy) - rdy) <= (half_step(DT[dt]) * (1 + 1e-5) + 2.0 ** -24) * np.abs(rdy) + 1e-7)
    # each of 32 lanes adds N / 32 products in turn, then 5 levels of a tree
    _, mag = O.moe_combine_bwd(np.abs(f64(d)), np.abs(f64(y)), topk, f64(w), i, 5)
    assert np.all(np.abs(f64(dw) - rdw) <= (N / 32 + 7) * 2.0 ** -24 * mag + 1e-30)
    dy, none = ops.moe_combine_bwd(d, None, topk, **use)
    assert none is None
    rdy, _ = O.moe_combine_bwd(f64(d), None, topk, None, i, 5)
    np.testing.assert_array_equal(f64(dy), rdy)


def test_combine_strides_in_place_and_guards(dev):
    y, w, ids, r = combine_inputs(dev, "f16", 19, 3, 264, 3, False)
    ref = ops.moe_combine(y, 3, w, residual=r)
    pad = torch.full((57, 300), 9.0, dtype=torch.float16, device=dev)
    for off in (0, 8, 3):  # whole 16-byte rows, and not
        ys = pad.clone()
        ys[:, off:off + 264] = y
        out = torch.full((19, 300), 5.0, dtype=torch.float16, device=dev)
        ops.moe_combine(ys[:, off:off + 264], 3, w, residual=r, out=out[:, off:off + 264])
        assert torch.equal(out[:, off:off + 264], ref)
        assert bool((out[:, :off] == 5).all()) and bool((out[:, off + 264:] == 5).all())
        dy = torch.full((57, 300), 5.0, dtype=torch.float16, device=dev)
        ops.moe_combine_bwd(r, ys[:, off:off + 264], 3, w, dy=dy[:, off:off + 264])
        full, _ = ops.moe_combine_bwd(r, y, 3, w)
        assert torch.equal(dy[:, off:off + 264], full)
        assert bool((dy[:, :off] == 5).all()) and bool((dy[:, off + 264:] == 5).all())
    ops.moe_combine(y, 3, w, residual=r, out=r)
    assert torch.equal(r, ref)


def test_empty(dev):
    x = torch.empty(0, 8, device=dev)
    w, i = ops.moe_route(x, 2)
    assert w.shape == (0, 2) and i.shape == (0, 2)
    assert ops.moe_route_bwd(w, x, i).shape == (0, 8)
    y = torch.empty(0, 16, dtype=torch.float16, device=dev)
    assert ops.moe_combine(y, 2).shape == (0, 16)
    dy, dw = ops.moe_combine_bwd(torch.empty(3, 0, dtype=torch.float16, device=dev),
                                 torch.empty(6, 0, dtype=torch.float16, device=dev), 2,
                                 torch.ones(3, 2, device=dev))
    assert dy.shape == (6, 0) and bool((dw == 0).all())


def test_refusals(dev):
    x = torch.zeros(4, 8, device=dev)
    h = torch.zeros(8, 16, dtype=torch.float16, device=dev)
    i = torch.zeros(4, 2, dtype=torch.int32, device=dev)
    bad = [
        lambda: ops.moe_route(x, 9), lambda: ops.moe_route(x, 0), lambda: ops.moe_route(x[0], 2),
        lambda: ops.moe_route(x.t(), 2), lambda: ops.moe_route(x.double(), 2),
        lambda: ops.moe_route(x, 2, score="tanh"), lambda: ops.moe_route(x, 2, bias=x[0].half()),
        lambda: ops.moe_route(x, 2, bias=x[0, :7]), lambda: ops.moe_route(x, 2, bias=torch.zeros(8)),
        lambda: ops.moe_route(x, 2, groups=3), lambda: ops.moe_route(x, 2, ids=i.long()),
        lambda: ops.moe_route(x, 2, weights=torch.zeros(4, 3, device=dev)),
        lambda: ops.moe_route(x[:1].expand(4, 8), 2),
        lambda: ops.moe_route_bwd(x[:, :2], x, i),  # dweights not contiguous
        lambda: ops.moe_route_bwd(torch.zeros(4, 3, device=dev), x, i),
        lambda: ops.moe_combine(h, 3), lambda: ops.moe_combine(h.float(), 2),
        lambda: ops.moe_combine(h, 2, ids=i), lambda: ops.moe_combine(h, 2, weights=h[:4, :2]),
        lambda: ops.moe_combine(h, 2, residual=h), lambda: ops.moe_combine(h.t(), 2),
        lambda: ops.moe_combine_bwd(h[:4], None, 2, weights=torch.ones(4, 2, device=dev)),
        lambda: ops.moe_combine_bwd(h[:4], h, 2, dweights=torch.ones(4, 2, device=dev)),
        lambda: ops.moe_combine_bwd(h[:1].sum().expand(4, 16), h, 2),
    ]
    for call in bad:
        with pytest.raises(B200Error):
            call()


def test_captured_and_on_another_stream(dev):
    x = logits(300, 64, "bf16", 3).to(dev)
    y = torch.randn(1200, 128, device=dev).half()
    r = torch.randn(300, 128, device=dev).half()

    def work():
        w, i = ops.moe_route(x, 4, groups=8, topk_groups=3)
        out = ops.moe_combine(y, 4, w, i, 64, r)
        dy, dw = ops.moe_combine_bwd(r, y, 4, w, i, 64)
        return w, i, out, dy, dw, ops.moe_route_bwd(dw, x, i)

    eager = work()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = work()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = work()
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(eager, other, held):
        assert torch.equal(a, b) and torch.equal(a, c)
