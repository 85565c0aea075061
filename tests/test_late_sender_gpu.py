"""A CTA that waits for what another CTA of its cluster sends into its shared
memory (the dense layer's few-token tiles): where the wait gives up, the host
is told, and the CTA stays until the sends have landed."""
import pytest
import torch

from cutile_b200 import _lib

pytestmark = pytest.mark.gpu

MS = 1_000_000


@pytest.mark.parametrize("limit,delay,late", [(500 * MS, 1 * MS, 0), (1 * MS, 20 * MS, 1)])
def test_sends_that_come_late(dev, limit, delay, late):
    st = torch.cuda.current_stream().cuda_stream
    L = _lib.load()
    assert L.ctb_check_device(st) == 0
    for _ in range(2):
        status = torch.full((2,), -1, dtype=torch.int32, device=dev)
        _lib.call("ctb_selftest_late_sender", limit, delay, status.data_ptr(), st)
        assert L.ctb_check_device(st) == (-7 if late else 0)
        assert status.tolist() == [32, late]
        assert L.ctb_check_device(st) == 0


def test_bad_limits_are_refused(dev):
    status = torch.zeros(2, dtype=torch.int32, device=dev)
    st = torch.cuda.current_stream().cuda_stream
    for limit, delay in ((0, MS), (MS, 0), (-1, MS), (MS, 2_000_000_000), (2_000_000_000, MS)):
        with pytest.raises(_lib.B200Error):
            _lib.call("ctb_selftest_late_sender", limit, delay, status.data_ptr(), st)
