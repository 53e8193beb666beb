"""Edges of the logits operators' CPU forms, which are the kernels' oracles."""
import pytest
import torch

from vllm_sm70_b200 import ops

INF = float("inf")


@pytest.mark.parametrize("tail", [True, False])
def test_nan_of_the_teacher_reaches_loss_and_gradient(tail):
    x = torch.randn(3, 9, generator=torch.Generator().manual_seed(1)).requires_grad_(True)
    ids = torch.arange(3).expand(3, 3).contiguous()
    lp = torch.full((3, 3), -2.0)
    lp[1, 2] = float("nan")
    lp[2] = -INF
    rows = ops.distill_loss(x, ids, lp, tail=tail, reduction="none")
    assert torch.isnan(rows).tolist() == [False, True, False]
    g, = torch.autograd.grad(rows.sum(), x)
    assert torch.isnan(g).any(1).tolist() == [False, True, False]
    assert tail or (float(rows[2].detach()) == 0 and bool((g[2] == 0).all()))
    assert bool(torch.isnan(ops.distill_loss(x, ids, lp, tail=tail)))
    # an absent id's value is not read
    ids[1, 2] = -1
    assert bool(torch.isfinite(ops.distill_loss(x, ids, lp, tail=tail)))
