"""moe_combine for every number of slots that has code of its own, and some that
share the loop, against float64.

Tolerance: topk + 1 Float32 multiply-adds, 2^-24 each of the terms' magnitudes,
and half a step of the result.
"""
import numpy as np
import pytest
import torch

from cutile_b200 import ops
from oracle import oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N", [72, 61])  # 16-byte rows, and not
@pytest.mark.parametrize("topk", [1, 2, 3, 4, 5, 6, 7, 8, 9, 16])
def test_slots(dev, dt, N, topk):
    T, E = 37, 6
    g = torch.Generator().manual_seed(topk)
    y = torch.randn(T * topk, N, generator=g).to(dt)
    w, r = torch.rand(T, topk, generator=g), torch.randn(T, N, generator=g).to(dt)
    ids = torch.randint(-2, E + 2, (T, topk), generator=g, dtype=torch.int32)
    lost = (ids < 0) | (ids >= E)
    y[lost.reshape(-1)] = float("nan")  # never written, so not read
    w[lost] = float("nan")
    for residual in (None, r):
        out = ops.moe_combine(y.to(dev), topk, w.to(dev), ids.to(dev), E,
                              None if residual is None else residual.to(dev))
        res = None if residual is None else residual.double().numpy()
        ref = O.moe_combine(y.double().numpy(), topk, w.double().numpy(), ids.numpy(), E, res)
        mag = O.moe_combine(y.double().abs().numpy(), topk, w.double().numpy(), ids.numpy(), E,
                            None if res is None else np.abs(res))
        tol = (topk + 1) * 2.0 ** -24 * mag + torch.finfo(dt).eps / 2 * np.abs(ref) * (1 + 1e-5) + 2.0 ** -25
        assert np.all(np.abs(out.double().cpu().numpy() - ref) <= tol)
