"""The layer's calls at once on several streams, beside the library's other
tensor-core kernels: each gives the bits that it gives alone."""
import pytest
import torch

from cutile_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graphs", [False, True])
def test_calls_at_once_on_streams(dev, graphs):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).half().to(dev)  # noqa: E731
    layers = [(r(1024, 2048), r(rows, 1024), r(rows, 2048)) for rows in (1, 24, 100, 600, 2304)]
    logits, y, d = torch.randn(900, 256, generator=g).to(dev), r(1800, 512), r(900, 512)
    bias = torch.randn(256, generator=g).to(dev) * 0.1
    q = r(2, 4, 512, 128)

    def dense(i):
        A, B, R = layers[i]
        Z = torch.empty_like(R)
        C = ops.dense(A, B, act="silu", residual=R, preact=Z)
        return [C, Z, *ops.dense_bwd(R, A, B, act="silu", preact=Z)]

    def route():
        w, i = ops.moe_route(logits, 2, score="sigmoid", bias=bias, groups=8, topk_groups=3)
        out = ops.moe_combine(y, 2, w, i, 256, d)
        dy, dw = ops.moe_combine_bwd(out, y, 2, w, i, 256)
        return [w, i, out, dy, dw, ops.moe_route_bwd(dw, logits, i, "sigmoid")]

    work = [lambda: dense(0) + dense(4), lambda: dense(1) + route(), lambda: dense(2) + dense(3),
            lambda: [ops.matmul(layers[4][0], layers[4][1]), ops.fmha(q, q, q, 0.1), *route()],
            lambda: dense(4) + dense(0)]
    alone = [w() for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    held = []
    if graphs:
        for w in work:
            c = torch.cuda.CUDAGraph()
            with torch.cuda.graph(c):
                held.append((c, w()))
    for _ in range(20):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                if graphs:
                    held[i][0].replay()
                    got.append(held[i][1])
                else:
                    got.append(work[i]())
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(x, z) for x, z in zip(a, b))
    ops.check_device()
