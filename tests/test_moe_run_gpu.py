"""A mixture-of-experts layer as a program runs it, from the library's calls:

    logits = dense(gate, x)                   the router's projection
    w, ids = moe_route(logits)                padded tokens go to no expert
    y      = moe_gemm(x, experts, moe_align(ids))
    out    = moe_combine(y, w, ids, residual = dense(shared, x, bias, silu, residual = x))

and back: combine, routing and both dense layers, against float64 autograd of
the same formulas on the same ids. Also the calls at sizes whose offsets pass
32 bits.

Tolerances: every step rounds to float16 once (half a step, 2^-11, of its
value); norm-wise the errors of the 4 roundings on the longest path (logits,
expert rows or shared expert, output; the gradient one more) add up to at most
6 * 2^-11 of the result's norm times the largest slope (1.13) and the share of
cancelled terms, for which a factor 2 is allowed: 7e-3.
"""
import pytest
import torch

from cutile_b200 import ops

pytestmark = pytest.mark.gpu


def rel(got, ref):
    return float((got.double() - ref).norm() / ref.norm())


@pytest.mark.parametrize("T,pad", [(1, 0), (3, 1), (300, 17)])
def test_layer_forward_and_backward(dev, T, pad):
    D, E, topk = 256, 16, 3
    g = torch.Generator(device=dev).manual_seed(T)
    r = lambda *s, k=1.0: (torch.randn(*s, generator=g, device=dev) * k).half()  # noqa: E731
    x, gate = r(T, D), r(D, E, k=2 * D ** -0.5)
    experts, shared = r(E, D, D, k=D ** -0.5), r(D, D, k=D ** -0.5)
    bias = torch.randn(D, generator=g, device=dev)
    G = r(T, D)

    logits = ops.dense(gate, x)
    if pad:
        logits[T - pad:] = float("-inf")
    w, ids = ops.moe_route(logits, topk, groups=4, topk_groups=2)
    sid, eid, ntp = ops.moe_align(ids, E)
    y = torch.full((T * topk, D), float("nan"), dtype=torch.float16, device=dev)
    ops.moe_gemm(x, experts, sid, eid, ntp, topk, out=y)
    z = torch.empty(T, D, dtype=torch.float16, device=dev)
    base = ops.dense(shared, x, bias=bias, act="silu", residual=x, preact=z)
    out = ops.moe_combine(y, topk, w, ids, E, residual=base)
    if pad:
        assert bool((ids[T - pad:] == -1).all()) and torch.equal(out[T - pad:], base[T - pad:])
        assert not bool((ids[:T - pad] == -1).any())

    live = T - pad
    gd = gate.double().requires_grad_(True)
    sd = shared.double().requires_grad_(True)
    bd = bias.double().requires_grad_(True)
    xd = x.double()
    i64 = ids[:live].long()
    lw = torch.softmax((xd @ gd)[:live].gather(1, i64), -1)
    rows = torch.einsum("td,tkod->tko", xd[:live], experts.double()[i64])
    base64 = torch.nn.functional.silu(xd @ sd + bd) + xd
    out64 = base64.clone()
    out64[:live] += (lw.unsqueeze(-1) * rows).sum(1)
    assert rel(out, out64.detach()) <= 7e-3
    (out64 * G.double()).sum().backward()

    dy, dw = ops.moe_combine_bwd(G, y, topk, w, ids, E)
    assert bool((dy.view(T, topk, D)[live:] == 0).all()) and bool((dw[live:] == 0).all())
    dlogits = ops.moe_route_bwd(dw, logits, ids)
    assert bool((dlogits[live:] == 0).all())
    dgate, dx_gate, _ = ops.dense_bwd(dlogits, gate, x, need_dbias=False)
    dshared, _, dbias = ops.dense_bwd(G, shared, x, act="silu", preact=z)
    assert rel(dgate, gd.grad) <= 2e-2  # differences of shares: the weights' rounding weighs twice
    assert rel(dshared, sd.grad) <= 7e-3 and rel(dbias, bd.grad) <= 7e-3
    assert bool(torch.isfinite(dx_gate).all())
    ops.check_device()


def test_layer_captured_once_replayed_on_new_inputs(dev):
    """The forward pass as one CUDA graph: new inputs copied in give what the
    same calls give eagerly."""
    T, D, E, topk = 64, 128, 8, 2
    g = torch.Generator(device=dev).manual_seed(0)
    r = lambda *s, k=1.0: (torch.randn(*s, generator=g, device=dev) * k).half()  # noqa: E731
    x, gate, experts = r(T, D), r(D, E), r(E, D, D, k=D ** -0.5)
    ws = ops.moe_workspace(2048, D, dev)

    def run(x):
        w, ids = ops.moe_route(ops.dense(gate, x), topk)
        sid, eid, ntp = ops.moe_align(ids, E)
        y = torch.zeros((T * topk, D), dtype=torch.float16, device=dev)
        ops.moe_gemm(x, experts, sid, eid, ntp, topk, out=y, workspace=ws)
        return ops.moe_combine(y, topk, w, ids, E, residual=x)

    run(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(x)
    for _ in range(3):
        x.copy_(r(T, D))
        graph.replay()
        assert torch.equal(held, run(x))


def test_offsets_past_32_bits(dev):
    """More than 2^31 elements in a matrix: the first and the last rows are those
    of the same rows alone."""
    T, topk, N = 70_001, 8, 4096
    y = torch.empty(T * topk, N, dtype=torch.float16, device=dev)  # 2.29e9 elements
    ops.fill_uniform(y, 3)
    w = torch.rand(T, topk, device=dev)
    out = ops.moe_combine(y, topk, w)
    d = torch.empty(T, N, dtype=torch.float16, device=dev)
    ops.fill_uniform(d, 4)
    dy, dw = ops.moe_combine_bwd(d, y, topk, w)
    for sl in (slice(0, 3), slice(T - 3, T)):
        ys = y.view(T, topk, N)[sl].reshape(-1, N)
        assert torch.equal(out[sl], ops.moe_combine(ys, topk, w[sl].contiguous()))
        a, b = ops.moe_combine_bwd(d[sl], ys, topk, w[sl].contiguous())
        assert torch.equal(dy.view(T, topk, N)[sl].reshape(-1, N), a) and torch.equal(dw[sl], b)
    del y, out, d, dy, dw

    T, E = 8_400_005, 256
    x = torch.empty(T, E, dtype=torch.bfloat16, device=dev)  # 2.15e9 elements
    ops.fill_normal(x, 5)
    w, i = ops.moe_route(x, 4)
    dx = ops.moe_route_bwd(w, x, i, renorm=False)
    for sl in (slice(0, 9), slice(T - 9, T)):
        ws, is_ = ops.moe_route(x[sl], 4)
        assert torch.equal(w[sl], ws) and torch.equal(i[sl], is_)
        assert torch.equal(dx[sl], ops.moe_route_bwd(ws, x[sl], is_, renorm=False))
    del x, w, i, dx

    N, M, K = 150_001, 14_400, 64
    A = torch.empty(K, M, dtype=torch.float16, device=dev)
    B = torch.empty(N, K, dtype=torch.float16, device=dev)
    ops.fill_uniform(A, 6)
    ops.fill_uniform(B, 7)
    C = ops.dense(A, B, act="relu", residual=None)  # 2.16e9 elements
    for sl in (slice(0, 40), slice(N - 40, N)):
        ref = (B[sl].double() @ A.double()).clamp(min=0)
        # K Float32 additions and half a step
        assert bool(((C[sl].double() - ref).abs() <= 64 * 2.0 ** -24 * 64 + 2.0 ** -11 * ref).all())
    dA, dB, db = ops.dense_bwd(C, A, B, act="relu", preact=C)
    ref = torch.zeros(K, M, dtype=torch.float64, device=dev)
    for s in range(0, N, 10_000):
        ref += B[s:s + 10_000].double().t() @ C[s:s + 10_000].double()
    assert rel(dA, ref) <= 2.0 ** -11 + 1e-4
    tail = C[N - 40:].double() @ A.double().t()
    assert rel(dB[N - 40:], tail) <= 2.0 ** -11 + 1e-4
    ops.check_device()


@pytest.mark.parametrize("T,D,hidden", [(1, 128, 512), (40, 256, 1024), (600, 520, 2304)])
def test_back_to_back_is_as_with_waits_between(dev, T, D, hidden):
    """Kernels start under the tail of the one before. A chain that reads what
    was just written, writes in place over what was just read and changes
    its weights gives the same bits whether or not each call is waited for."""
    E, topk = 8, 2
    g = torch.Generator(device=dev).manual_seed(T)
    r = lambda *s, k=1.0: (torch.randn(*s, generator=g, device=dev) * k).bfloat16()  # noqa: E731
    x0, up0, down0 = r(T, D), r(D, hidden, k=D ** -0.5), r(hidden, D, k=hidden ** -0.5)
    gate, bias = r(D, E, k=D ** -0.5), torch.randn(hidden, generator=g, device=dev)

    def chain(wait):
        x, up, down = x0.clone(), up0.clone(), down0.clone()
        h, z = torch.empty(T, hidden, dtype=x.dtype, device=dev), torch.empty(T, hidden, dtype=x.dtype, device=dev)
        y = torch.empty(T * topk, D, dtype=x.dtype, device=dev)
        steps = []

        def step(out):
            steps.append(out)
            if wait:
                torch.cuda.synchronize()
            return out

        for _ in range(12):
            step(ops.dense(up, x, bias=bias, act="gelu", out=h, preact=z))
            step(ops.dense(down, h, residual=x, out=x))
            w, i = step(ops.moe_route(ops.dense(gate, x), topk))
            dy, _ = step(ops.moe_combine_bwd(x, None, topk, dy=y))
            step(ops.moe_combine(dy, topk, w, i, E, out=x))
            dx = step(ops.dense_bwd(h, up, x, act="gelu", preact=z))
            step(ops.moe_combine(x, 1, residual=dx[1], out=x))
            up.add_(dx[0], alpha=1e-3)  # another library's kernel in between
            x.div_(x.float().norm() / (T * D) ** 0.5 + 1e-3)
        torch.cuda.synchronize()
        return [x, up, h, z, y, w, i]

    for a, b in zip(chain(True), chain(False)):
        assert torch.equal(a, b)
    assert bool(torch.isfinite(chain(False)[0]).all())
