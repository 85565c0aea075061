"""The layer calls at the longest rows they accept: columns near 2^31, where the
step past the end of a row does not fit 31 bits.

Every checked value is one product (or the sum of a few exact ones), so it is
the rounded product and can be compared for equality with torch's.
"""
import pytest
import torch

from cutile_b200 import ops

pytestmark = pytest.mark.gpu

CHUNK = 1 << 28


def uniform(n, dev, seed):
    t = torch.empty(n, dtype=torch.float16, device=dev)
    ops.fill_uniform(t, seed)
    return t


def assert_same(a, piece):
    """Equality of a long vector with one that is given piece by piece."""
    for at in range(0, a.numel(), CHUNK):
        assert torch.equal(a[at:at + CHUNK], piece(slice(at, min(at + CHUNK, a.numel())))), at


def test_combine_gradients_of_the_longest_rows(dev):
    N = 2 ** 31 - 8  # whole 16-byte runs; a warp's last step ends above 2^31
    d, y = uniform(N, dev, 1), torch.zeros(N, dtype=torch.float16, device=dev)
    at = torch.tensor([0, N // 2, N - 1025, N - 1], device=dev)
    y[at] = torch.tensor([1.0, 2.0, 4.0, 8.0], dtype=torch.float16, device=dev)
    guard = torch.full((N + 4096,), 9.0, dtype=torch.float16, device=dev)
    dy = guard[2048:2048 + N].view(1, N)
    w = torch.tensor([[0.75]], device=dev)
    _, dw = ops.moe_combine_bwd(d.view(1, N), y.view(1, N), 1, w, dy=dy)
    assert_same(dy[0], lambda s: (d[s].float() * 0.75).half())
    # four exact products, three additions of Float32
    terms = (d[at].double() * y[at].double())
    assert abs(float(dw) - float(terms.sum())) <= 3 * 2.0 ** -24 * float(terms.abs().sum())
    skipped = torch.tensor([[-1]], dtype=torch.int32, device=dev)
    _, dw = ops.moe_combine_bwd(d.view(1, N), y.view(1, N), 1, w, skipped, 1, dy=dy)
    assert_same(dy[0], lambda s: torch.zeros_like(d[s]))
    assert float(dw) == 0
    assert bool((guard[:2048] == 9).all()) and bool((guard[2048 + N:] == 9).all())


def test_dense_copies_the_longest_lines(dev):
    """One line of 2^31 - 1 weights off a 16-byte boundary, which is copied to the
    workspace; one token of one input, so that each output is one product."""
    M = 2 ** 31 - 1
    A = uniform(M + 1, dev, 3)[1:].view(1, M)
    B = torch.full((1, 1), 0.75, dtype=torch.float16, device=dev)
    guard = torch.full((M + 4097,), 9.0, dtype=torch.float16, device=dev)
    C = guard[2048:2048 + M].view(1, M)
    ops.dense(A, B, out=C)
    ops.check_device()
    assert_same(C[0], lambda s: (A[0, s].float() * 0.75).half())
    assert bool((guard[:2048] == 9).all()) and bool((guard[2048 + M:] == 9).all())
