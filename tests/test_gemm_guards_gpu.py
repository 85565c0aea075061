"""What lies between the columns of a padded C stays as it was, for matmul and
its batched form on both tensor-core kernels (CTB_GEMM_PAIR is read once per
process, hence the subprocesses)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = r"""
import sys
sys.path.insert(0, "cutile-triton_b200"); sys.path.insert(0, ".")
import torch
from cutile_b200 import ops
dev = torch.device("cuda", 0)
for batch, M, N, K in [(1, 1, 1, 8), (1, 7, 3, 64), (1, 1001, 40, 72), (1, 300, 260, 200),
                       (1, 513, 300, 64), (3, 203, 70, 72), (2, 262, 33, 136), (1, 512, 64, 64)]:
    pad = lambda n: (n + 15) // 8 * 8
    A = torch.zeros(batch, K, pad(M), dtype=torch.float16, device=dev)[:, :, :M]
    B = torch.zeros(batch, N, pad(K), dtype=torch.float16, device=dev)[:, :, :K]
    A.copy_(ops.fill_uniform(torch.empty(batch, K, M, dtype=torch.float16, device=dev), 1))
    B.copy_(ops.fill_uniform(torch.empty(batch, N, K, dtype=torch.float16, device=dev), 2))
    big = torch.full((batch, N, pad(M)), 9.0, dtype=torch.float16, device=dev)
    C = big[:, :, :M]
    if batch == 1:
        ops.matmul(A[0], B[0], C[0])
    else:
        ops.bmm(A, B, C)
    ops.check_device()
    assert bool((big[:, :, M:] == 9).all()), (batch, M, N, K)
    ref = B.double() @ A.double()
    # K Float32 additions of products below 1, and half a step
    assert bool(((C.double() - ref).abs() <= K * K * 2.0 ** -24 + 2.0 ** -11 * ref.abs() + 2.0 ** -25).all())
"""


@pytest.mark.parametrize("pair", ["1", "0"])
def test_between_columns(pair):
    r = subprocess.run([sys.executable, "-c", SCRIPT], cwd=ROOT, env=dict(os.environ, CTB_GEMM_PAIR=pair),
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
