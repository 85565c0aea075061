"""Flags of the layer calls that have no truth value are refused like any other
bad argument."""
import pytest
import torch

from cutile_b200 import B200Error, ops

pytestmark = pytest.mark.gpu


def test_flags_without_a_truth_value(dev):
    both = torch.tensor([True, False])
    x = torch.randn(4, 8, device=dev)
    w, ids = ops.moe_route(x, 2)
    A, B = torch.zeros(8, 16, dtype=torch.float16, device=dev), torch.zeros(4, 8, dtype=torch.float16, device=dev)
    dC = torch.zeros(4, 16, dtype=torch.float16, device=dev)
    bad = [lambda: ops.moe_route(x, 2, renorm=both), lambda: ops.moe_route_bwd(w, x, ids, renorm=both)]
    bad += [lambda k=k: ops.dense_bwd(dC, A, B, **{k: both}) for k in ("need_dA", "need_dB", "need_dbias")]
    for call in bad:
        with pytest.raises(B200Error) as e:
            call()
        assert e.value.status == "CTB_ERR_ARG" and "truth" in str(e.value)
    assert torch.equal(ops.moe_route(x, 2, renorm=torch.tensor(True))[0], w)
