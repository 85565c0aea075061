"""The dense layer's two kernels on shapes for which the model of their times
takes the other one: each forced for all (CTB_DENSE_PAIR, read once per process,
hence the subprocesses)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("pair", ["1", "0"])
@pytest.mark.parametrize("tests", ["test_dense_guards_gpu.py test_dense_values_gpu.py",
                                   "test_layer_limits_gpu.py -k longest_lines"])
def test_forced_kernel(pair, tests):
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu", *tests.split(),
                        "--rootdir", ROOT], cwd=os.path.join(ROOT, "tests"),
                       env=dict(os.environ, CTB_DENSE_PAIR=pair), capture_output=True, text=True,
                       timeout=600)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-1000:]
