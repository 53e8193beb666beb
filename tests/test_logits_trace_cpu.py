"""The logits operators on fake CUDA tensors: no kernel runs, the dispatch is
the real one."""
import pytest
import torch
import torch.autograd.forward_ad as fw
from torch._subclasses.fake_tensor import FakeTensorMode

from vllm_sm70_b200 import _ext, ops

pytestmark = pytest.mark.skipif(not _ext.load(), reason="native library not built")


def _inputs():
    x = torch.empty(3, 64, device="cuda")
    return (x, torch.zeros(3, dtype=torch.int64, device="cuda"),
            torch.zeros(3, 4, dtype=torch.int32, device="cuda"), torch.zeros(3, 4, device="cuda"))


@pytest.fixture
def fake():
    ops.register()
    with FakeTensorMode():
        yield


def test_tangents_are_refused(fake):
    x, y, ids, lp = _inputs()
    t = torch.ones_like(x)
    calls = [lambda z: ops.token_logprobs(z, y).logprobs,
             lambda z: ops.token_logprobs(z, y, top_n=3).entropy,
             *(lambda z, r=r: ops.distill_loss(z, ids, lp, reduction=r)
               for r in ("none", "sum", "mean"))]
    for f in calls:
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(f, (x,), (t,))
        with fw.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            f(fw.make_dual(x, t))
        f(x)  # none: no objection
    with fw.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        ops.distill_loss(x, ids, fw.make_dual(lp, lp))
    with fw.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        ops.distill_loss(x, ids, lp, fw.make_dual(lp[:, 0].contiguous(), lp[:, 0].contiguous()))
