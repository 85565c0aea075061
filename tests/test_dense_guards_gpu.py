"""What lies between the rows of the dense layer's outputs stays as it was: rows
of every length modulo 8 in 16-byte-aligned lines, as a program has them that
pads its leading dimensions or writes a slice of a wider buffer."""
import pytest
import torch

from cutile_b200 import ops

pytestmark = pytest.mark.gpu


def holder(rows, cols, dt, dev):
    """A buffer of nines and its first columns, with at least eight left over."""
    big = torch.full((rows, (cols + 15) // 8 * 8), 9.0, dtype=dt, device=dev)
    return big, big[:, :cols]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,M", [(1, 1), (1, 7), (2, 33), (5, 1001), (300, 62), (300, 290), (257, 1003),
                                 (40, 516), (300, 133), (33, 1006), (260, 527), (2304, 2309)])
def test_between_output_rows(dev, dt, N, M):
    K = 72
    g = torch.Generator().manual_seed(N + M)
    r = lambda *s: torch.randn(*s, generator=g).to(dt).to(dev)  # noqa: E731
    A, B, R, bias = r(K, M), r(N, K), r(N, M), torch.randn(M, generator=g).to(dev)
    cb, C = holder(N, M, dt, dev)
    zb, Z = holder(N, M, dt, dev)
    rb, Rp = holder(N, M, dt, dev)
    Rp.copy_(R)
    ops.dense(A, B, bias=bias, act="relu", residual=Rp, out=C, preact=Z)
    ab, dA = holder(K, M, dt, dev)
    A2, B2, dC = r(M, K), r(N, M), r(N, K)  # the transposed layer: its dB has rows of M
    bb, dB = holder(N, M, dt, dev)
    ops.dense_bwd(R, A, B, dA_t=dA, need_dB=False, need_dbias=False)
    ops.dense_bwd(dC, A2, B2, dB_t=dB, need_dA=False, need_dbias=False)
    ops.check_device()
    for big in (cb, zb, rb, ab, bb):
        assert bool((big[:, M:] == 9).all())
    z = torch.empty_like(R)
    assert torch.equal(C, ops.dense(A, B, bias=bias, act="relu", residual=R, preact=z)) and torch.equal(Z, z)
    assert torch.equal(dA, ops.dense_bwd(R, A, B, need_dB=False, need_dbias=False)[0])
    assert torch.equal(dB, ops.dense_bwd(dC, A2, B2, need_dA=False, need_dbias=False)[1])


def test_after_the_only_row(dev):
    """One row of any length ends where the matrix ends: the elements after it
    belong to someone else."""
    for M in (1, 31, 257, 1001, 4099):
        A = torch.ones(8, M, dtype=torch.float16, device=dev)
        B = torch.ones(1, 8, dtype=torch.float16, device=dev)
        buf = torch.full((M + 32,), 9.0, dtype=torch.float16, device=dev)
        ops.dense(A, B, out=buf[:M].view(1, M))
        assert bool((buf[:M] == 8).all()) and bool((buf[M:] == 9).all())
