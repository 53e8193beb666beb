"""GPU: the training forms of the logits operators traced into a graph of the
ops that they call, forward and backward; and the launch counter's reset."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from vllm_sm70_b200 import ops
from vllm_sm70_b200.utils import launch_count

pytestmark = pytest.mark.gpu


def _inputs(dtype):
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(5, 777, device="cuda", generator=g).to(dtype)
    ids = torch.arange(4, device="cuda", dtype=torch.int32).expand(5, 4).contiguous()
    lp = torch.log_softmax(torch.randn(5, 4, device="cuda", generator=g), 1) - 0.2
    return x, torch.arange(5, device="cuda"), ids, lp


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mode", ["real", "fake"])
def test_training_forms_trace(b200_ops, mode, dtype):
    ops.register()
    args = _inputs(dtype)

    def step_of(f):
        def step(z, y, ids, lp):
            z = z.detach().requires_grad_(True)
            loss = f(z, y, ids, lp).sum() * 0.5
            return loss, *torch.autograd.grad(loss, z)
        return step

    for name, f in {"scores": lambda z, y, ids, lp: ops.token_logprobs(z, y).logprobs,
                    "rows": lambda z, y, ids, lp: ops.distill_loss(z, ids, lp, reduction="none"),
                    "mean": lambda z, y, ids, lp: ops.distill_loss(z, ids, lp)}.items():
        step = step_of(f)
        graph = make_fx(step, tracing_mode=mode)(*args)
        called = [str(n.target) for n in graph.graph.nodes if n.op == "call_function"]
        assert sum("_b200_C" in c for c in called) == 2, (name, called)
        assert not any("_train" in c for c in called)
        for a, b in zip(graph(*args), step(*args)):
            assert torch.equal(a, b), name


def test_counter_after_reset(b200_ops):
    x, _, ids, lp = _inputs(torch.bfloat16)
    x.requires_grad_(True)
    ops.distill_loss(x, ids, lp).backward()  # launches of before do not count
    launch_count.reset()
    assert launch_count.total() == 0
    loss = ops.distill_loss(x, ids, lp)
    assert launch_count.total() == 2
    loss.backward()
    assert launch_count.total() == 3
    launch_count.reset()
    assert launch_count.total() == 0
