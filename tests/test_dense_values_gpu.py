"""The dense layer's activations and slopes at values as large as BFloat16 holds,
where a square or a cube of the value passes the range of Float32.

Far from 0 every activation is max(z, 0) and every slope 0 or 1 (the tails are
below 1e-300), so results are exact: z is a power of two.
"""
import pytest
import torch

from cutile_b200 import ops

pytestmark = pytest.mark.gpu

LARGE = [2.0 ** e for e in (10, 40, 62, 63, 64, 65, 100, 127)]


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("M", [16, 21])  # 16-byte rows, and not
def test_large_values_and_slopes(dev, act, M):
    z = torch.zeros(M, device=dev)
    z[:16] = torch.tensor(LARGE + [-v for v in LARGE], device=dev)
    A = torch.zeros(8, M, dtype=torch.bfloat16, device=dev)
    A[0] = z
    B = torch.zeros(5, 8, dtype=torch.bfloat16, device=dev)
    B[:, 0] = 1
    Z = torch.empty(5, M, dtype=torch.bfloat16, device=dev)
    C = ops.dense(A, B, act=act, preact=Z)
    assert torch.equal(Z, z.bfloat16().expand(5, M))
    assert torch.equal(C[:, :16].float(), (z if act == "none" else z.clamp(min=0))[:16].expand(5, 16))
    dC = torch.full((5, M), 3.0, dtype=torch.bfloat16, device=dev)
    _, _, db = ops.dense_bwd(dC, A, B, act=act, preact=Z)
    slope = torch.ones_like(z) if act == "none" else (z > 0).float()
    assert torch.equal(db[:16], 15 * slope[:16])
