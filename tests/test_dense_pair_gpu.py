"""Both tensor-core kernels of the dense layer on every shape of its tests: the
CTA-pair kernel (256 x 256 tiles over two SMs) forced for all, and the split
kernel forced for all (CTB_DENSE_PAIR, read once per process, hence the
subprocesses)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("pair", ["1", "0"])
def test_forced_kernel(pair):
    env = dict(os.environ, CTB_DENSE_PAIR=pair)
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu",
                        os.path.join("tests", "test_dense_gpu.py")], cwd=ROOT, env=env,
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-1000:]
