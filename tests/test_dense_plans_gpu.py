"""Every tile, split and operand order of the dense layer's kernels against
float64, whatever the model of their times would take: rows that fill no tile
(29 and 150), whose number no split divides, in whole 16-byte rows and not.

Tolerances as in test_dense_gpu.py: a sum of K terms errs by at most (K + 2) *
2^-24 of their magnitudes, silu's slope is at most 1.13 and its own error below
2e-6 of |z| + 1, each result is rounded by half a step.
"""
import pytest
import torch

from cutile_b200 import B200Error, _lib, ops

pytestmark = pytest.mark.gpu

DEPTH = 1100  # 18 k-blocks, the last one short: two at least for each of 8 CTAs
PLANS = [(rows, split) for rows in (16, 32, 64, 128) for split in range(1, 9)] + [(256, 1)]
EPS32 = 2.0 ** -24


@pytest.fixture(params=PLANS, ids=lambda p: "%dx%d" % p)
def plan(request, dev):
    _lib.call("ctb_selftest_dense_plan", *request.param)
    yield request.param
    _lib.call("ctb_selftest_dense_plan", 0, 0)


@pytest.fixture(autouse=True)
def as_before():
    yield
    _lib.call("ctb_selftest_dense_plan", 0, 0)


def rand(dev, dt, seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dt).to(dev)


def half_step(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    return 2.0 ** -25 if dt == torch.float16 else 1e-38


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [29, 150])
@pytest.mark.parametrize("cols", [200, 333])
def test_forward(dev, plan, dt, rows, cols):
    A, B = rand(dev, dt, 1, DEPTH, cols) / DEPTH ** 0.5, rand(dev, dt, 2, rows, DEPTH)
    bias, R = rand(dev, torch.float32, 3, cols), rand(dev, dt, 4, rows, cols)
    Z = torch.empty_like(R)
    C = ops.dense(A, B, bias=bias, act="silu", residual=R, preact=Z)
    plain = ops.dense(A, B)
    ops.check_device()
    s = B.double() @ A.double()
    z = s + bias.double()
    y = z * torch.sigmoid(z) + R.double()
    mag = B.double().abs() @ A.double().abs() + bias.double().abs()
    h, t, err = half_step(dt), tiny(dt), (DEPTH + 2) * EPS32 * mag
    assert bool(((plain.double() - s).abs() <= err + h * s.abs() * (1 + 1e-5) + t).all())
    assert bool(((Z.double() - z).abs() <= err + h * z.abs() * (1 + 1e-5) + t).all())
    yerr = 1.13 * err + 2e-6 * (z.abs() + 1) + EPS32 * R.double().abs()
    assert bool(((C.double() - y).abs() <= yerr * (1 + h) + h * y.abs() + t).all())


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [29, 150])
@pytest.mark.parametrize("cols", [200, 333])
def test_gradients(dev, plan, dt, rows, cols):
    """dB (rows x cols over DEPTH: both operands k-major) and dA (neither)."""
    h, t = half_step(dt), tiny(dt)
    A, B = rand(dev, dt, 1, cols, DEPTH), rand(dev, dt, 2, rows, cols)
    dC = rand(dev, dt, 3, rows, DEPTH)
    dB = ops.dense_bwd(dC, A, B, need_dA=False, need_dbias=False)[1]
    ref, mag = dC.double() @ A.double().t(), dC.double().abs() @ A.double().abs().t()
    assert bool(((dB.double() - ref).abs() <= (DEPTH + 2) * EPS32 * mag + h * ref.abs() * (1 + 1e-5) + t).all())
    A, B = rand(dev, dt, 4, rows, cols), rand(dev, dt, 5, DEPTH, rows)
    dC = rand(dev, dt, 6, DEPTH, cols)
    dA = ops.dense_bwd(dC, A, B, need_dB=False, need_dbias=False)[0]
    ref, mag = B.double().t() @ dC.double(), B.double().abs().t() @ dC.double().abs()
    assert bool(((dA.double() - ref).abs() <= (DEPTH + 2) * EPS32 * mag + h * ref.abs() * (1 + 1e-5) + t).all())
    ops.check_device()


@pytest.mark.parametrize("rows", range(1, 34))
def test_owners_of_few_rows(dev, rows):
    """Every number of rows of the tiles whose sums are sent to owners, with
    every split: some CTAs own fewer rows than others, some none."""
    A, B = rand(dev, torch.float16, 1, DEPTH, 136) / DEPTH ** 0.5, rand(dev, torch.float16, 2, rows, DEPTH)
    s = B.double() @ A.double()
    tol = (DEPTH + 2) * EPS32 * (B.double().abs() @ A.double().abs()) + 2.0 ** -11 * s.abs() * (1 + 1e-5) + 2.0 ** -25
    for tile in (16, 32):
        for split in range(1, 9):
            _lib.call("ctb_selftest_dense_plan", tile, split)
            for out in (torch.empty_like(s, dtype=torch.float16),
                        torch.empty(rows, 139, dtype=torch.float16, device=dev)[:, 1:137]):
                ops.dense(A, B, out=out)
                assert bool(((out.double() - s).abs() <= tol).all()), (tile, split)
    ops.check_device()


def test_bad_plans_are_refused(dev):
    for rows, split in ((8, 1), (48, 2), (512, 1), (16, 0), (16, 9), (-16, 1)):
        with pytest.raises(B200Error):
            _lib.call("ctb_selftest_dense_plan", rows, split)
