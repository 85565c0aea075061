"""The layer calls on operands that share a buffer: the pairs that may be one and
the same matrix, and matrices that lie between one another's rows, give the
bits that separate buffers give."""
import pytest
import torch

from cutile_b200 import B200Error, ops

pytestmark = pytest.mark.gpu


def rand(dev, seed, *shape, dt=torch.float16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dt).to(dev)


@pytest.mark.parametrize("T,N", [(1, 264), (70, 264), (70, 261), (600, 2304)])
def test_same_matrix(dev, T, N):
    """Of one matrix each, with columns to spare so that rows have a stride."""
    def held(t):
        big = torch.full((t.shape[0], t.shape[1] + 16), 9.0, dtype=t.dtype, device=dev)
        big[:, :t.shape[1]] = t
        return big, big[:, :t.shape[1]]

    y, d, w = rand(dev, 1, T, N), rand(dev, 2, T, N), rand(dev, 3, T, 1, dt=torch.float32)
    A, B = rand(dev, 4, 72, N), rand(dev, 5, T, 72)
    dy, dw = ops.moe_combine_bwd(d, y, 1, w)
    cases = [
        (ops.dense(A, B, act="silu", residual=y), y, lambda v: ops.dense(A, B, act="silu", residual=v, out=v)),
        (ops.moe_combine(d, 1, w, residual=y), y, lambda v: ops.moe_combine(d, 1, w, residual=v, out=v)),
        (ops.moe_combine(y, 1, w, residual=d), y, lambda v: ops.moe_combine(v, 1, w, residual=d, out=v)),
        (ops.moe_combine(y, 1, w, residual=y), y, lambda v: ops.moe_combine(v, 1, w, residual=v, out=v)),
        (dy, d, lambda v: ops.moe_combine_bwd(v, y, 1, w, dy=v)[0]),
        (dy, y, lambda v: ops.moe_combine_bwd(d, v, 1, w, dy=v)[0]),
    ]
    for ref, start, run in cases:
        big, v = held(start)
        run(v)
        assert torch.equal(v, ref) and bool((big[:, N:] == 9).all())
    w2 = w.clone()
    assert torch.equal(ops.moe_combine_bwd(d, y, 1, w2, dweights=w2)[1], dw)
    for dt in (torch.float32, torch.bfloat16):
        for E, topk in ((8, 2), (100, 4), (256, 8)):
            x = rand(dev, E, T, E, dt=dt)
            for score in ("softmax", "sigmoid"):
                for renorm in (True, False):
                    g, ids = ops.moe_route(x, topk, score=score, renorm=renorm)
                    ref = ops.moe_route_bwd(g, x, ids, score, renorm)
                    big, v = held(x)
                    ops.moe_route_bwd(g, v, ids, score, renorm, dlogits=v)
                    assert torch.equal(v, ref) and bool((big[:, E:] == 9).all())
    ops.check_device()


@pytest.mark.parametrize("N,M", [(1, 40), (37, 264), (300, 520)])
def test_columns_and_rows_of_one_buffer(dev, N, M):
    A, B, R = rand(dev, 1, 72, M), rand(dev, 2, N, 72), rand(dev, 3, N, M)
    Z = torch.empty_like(R)
    C = ops.dense(A, B, act="gelu", residual=R, preact=Z)
    side = torch.zeros(N, 3 * M, dtype=torch.float16, device=dev)
    parts = [side[:, i * M:(i + 1) * M] for i in range(3)]
    rows = torch.zeros(3 * N, M, dtype=torch.float16, device=dev)
    for c, r, z in (parts, [rows[i::3] for i in range(3)], [parts[2], rows[1::3], parts[0]]):
        r.copy_(R)
        ops.dense(A, B, act="gelu", residual=r, out=c, preact=z)
        assert torch.equal(c, C) and torch.equal(r, R) and torch.equal(z, Z)


def test_views_that_overlap_are_refused(dev):
    T, N = 6, 32
    buf = torch.zeros(4 * T, N, dtype=torch.float16, device=dev)
    A, B = torch.zeros(8, N, dtype=torch.float16, device=dev), torch.zeros(T, 8, dtype=torch.float16, device=dev)
    w, x = torch.zeros(T, 2, device=dev), torch.zeros(2 * T, 8, device=dev)
    ids = torch.zeros(T, 2, dtype=torch.int32, device=dev)
    bad = [
        lambda: ops.dense(A, B, residual=buf[:T], out=buf[1:T + 1]),
        lambda: ops.dense(A, B, residual=buf[:2 * T:2], out=buf[:T]),
        lambda: ops.dense(A, B, out=buf[:T], preact=buf[T - 1:2 * T - 1]),
        lambda: ops.moe_combine(buf[:2 * T], 2, w, out=buf[2 * T - 1:3 * T - 1]),
        lambda: ops.moe_combine(buf[:2 * T], 2, w, residual=buf[2 * T:4 * T:2], out=buf[2 * T:3 * T]),
        lambda: ops.moe_combine_bwd(buf[:T], buf[T:3 * T], 2, w, dy=buf[T + 1:3 * T + 1]),
        lambda: ops.moe_combine_bwd(buf[:T], buf[T:3 * T], 2, w, dy=buf[:2 * T]),
        lambda: ops.moe_route_bwd(w, x[:T], ids, dlogits=x[1:T + 1]),
        lambda: ops.moe_route_bwd(w, x[:2 * T:2], ids, dlogits=x[:T]),
    ]
    for call in bad:
        with pytest.raises(B200Error) as e:
            call()
        assert e.value.status == "CTB_ERR_ARG"
