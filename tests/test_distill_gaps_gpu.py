"""GPU: distill_loss where the teacher's tokens and the others lie far apart
in the student, against the 64-bit oracle.

Tolerances. A row's loss is p_t times the gap, and more: fp32 holds the gap
to 2^-23 of itself, the teacher's p to 2^-22, their sum and p_t to 2^-21, and
p_t is 0.05 or more: relative errors below 2^-16 < TOL. The gradient outside
is p_t times a softmax over the others alone, inside it is q - p: the bound of
the logits tests (5e-5, and half a unit of 2^-8 in bf16) holds for both.
"""
import math

import pytest
import torch

from vllm_sm70_b200 import ops
from vllm_sm70_b200.ops import logits as L

pytestmark = pytest.mark.gpu
TOL = 5e-5
DTYPES = [torch.bfloat16, torch.float32]
# (rows, V): a CTA and a cluster a row, many rows, a row that no cluster holds
SHAPES = [(3, 64), (3, 32003), (2, 151936), (700, 8195), (2, 2 ** 21 + 5)]


def _assert_grad(got, want, dtype):
    rel = (2.0 ** -8 if dtype == torch.bfloat16 else 0.0) + TOL
    err = (got.double() - want).abs()
    lim = rel * want.abs() + TOL * want.abs().amax(1, keepdim=True) + 1e-30
    assert bool((err <= lim).all()), float((err - lim).max())


def _check(x, ids, lp, t, tail=True):
    xd = x.detach().double().requires_grad_(True)
    want = L.distill_rows_ref(xd, ids, lp, None, t, tail, dtype=torch.float64)
    e, = torch.autograd.grad(want.sum(), xd)
    want = want.detach()
    assert bool(torch.isfinite(want).all()) and bool(torch.isfinite(e).all())
    with torch.no_grad():
        rows = ops.distill_loss(x, ids, lp, None, t, tail, reduction="none")
    torch.testing.assert_close(rows.double(), want, atol=2 * TOL, rtol=TOL)
    xg = x.detach().requires_grad_(True)
    for red, scale in (("none", 1.0), ("sum", 1.0), ("mean", 1.0 / x.shape[0])):
        loss = ops.distill_loss(xg, ids, lp, None, t, tail, reduction=red).sum()
        g, = torch.autograd.grad(loss, xg, retain_graph=True)
        _assert_grad(g, e * scale, x.dtype)
        g, = torch.autograd.grad(loss, xg)  # from the saved numbers
        _assert_grad(g, e * scale, x.dtype)


def _rows(rows, V, K, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, V, device="cuda", generator=g)
    ids = (torch.randint(0, V, (rows, 1), device="cuda", generator=g)
           + (V // K) * torch.arange(K, device="cuda")) % V
    lp = torch.log_softmax(torch.randn(rows, K, device="cuda", generator=g), 1) + math.log(0.9)
    return x.to(dtype), ids, lp


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", SHAPES)
@pytest.mark.parametrize("gap,t", [(80, 1.0), (90, 1.0), (130, 1.0), (1000, 1.0), (1e4, 1.0),
                                   (12, 0.1), (100, 0.1), (12, 0.01), (-100, 1.0), (-100, 0.1)])
def test_gaps(b200_ops, rows, V, gap, t, dtype):
    x, ids, lp = _rows(rows, V, 5, dtype, V)
    x.scatter_add_(1, ids, torch.full_like(ids, 1).to(dtype) * gap)
    _check(x, ids, lp, t)
    if gap < 0:
        _check(x, ids, lp, t, tail=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", SHAPES)
@pytest.mark.parametrize("value", [-1e4, -1e9, -1e20, None])
def test_only_the_teachers_tokens_are_allowed(b200_ops, rows, V, value, dtype):
    """All others at a finite mask."""
    x, ids, lp = _rows(rows, V, 5, dtype, V)
    m = torch.full_like(x, torch.finfo(dtype).min if value is None else value)
    m.scatter_(1, ids, x.gather(1, ids))
    _check(m, ids, lp, 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [5003, 2 ** 21 + 5])
@pytest.mark.parametrize("tail", [True, False])
def test_teacher_rows_without_a_distribution(b200_ops, V, tail, dtype):
    """What token_logprobs says of a row whose mask leaves nothing: ids with
    log-probs of -inf, which are no mass."""
    x, _, _ = _rows(4, V, 5, dtype, 1)
    teacher = x.roll(1, 0).clone()
    teacher[1] = -float("inf")
    s = ops.token_logprobs(teacher, torch.zeros(4, dtype=torch.int64, device="cuda"), top_n=6)
    assert bool((s.top_logprobs[1] == -float("inf")).all())
    _check(x, s.top_ids, s.top_logprobs, 1.0, tail)
    xg = x.detach().requires_grad_(True)
    for red in ("none", "sum"):
        loss = ops.distill_loss(xg, s.top_ids, s.top_logprobs, tail=tail, reduction=red)
        g, = torch.autograd.grad(loss.sum(), xg)
        if not tail:
            assert bool((g[1] == 0).all())
            if red == "none":
                assert float(loss[1].detach()) == 0


@pytest.mark.parametrize("V", [5003, 2 ** 21 + 5])
@pytest.mark.parametrize("tail", [True, False])
def test_nan_of_the_teacher_reaches_loss_and_gradient(b200_ops, V, tail):
    x, ids, lp = _rows(3, V, 5, torch.float32, 1)
    lp[1, 2] = float("nan")
    xg = x.requires_grad_(True)
    for red in ("none", "sum"):
        loss = ops.distill_loss(xg, ids, lp, tail=tail, reduction=red)
        assert torch.isnan(loss).tolist() == ([False, True, False] if red == "none" else True)
        g, = torch.autograd.grad(loss.sum(), xg)
        assert torch.isnan(g).any(1).tolist() == [False, True, False]
    ids[1, 2] = -1  # an absent id's value is not read
    assert bool(torch.isfinite(ops.distill_loss(xg, ids, lp, tail=tail)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", [(5, 3001), (700, 8195), (2, 2 ** 21 + 5)])
@pytest.mark.parametrize("up", [0.37, -3.0, 1.0, 1e-3])
def test_gradient_is_rounded_once_for_any_upstream(b200_ops, up, rows, V, dtype):
    """Half a unit of the type, once; and the graph gives the same bits again."""
    x, ids, lp = _rows(rows, V, 5, dtype, 3)
    ids[0, 4] = ids[0, 1]
    w = 0.5 + torch.rand(rows, device="cuda")
    xd = x.double().requires_grad_(True)
    e, = torch.autograd.grad(
        L.distill_rows_ref(xd, ids, lp, w.double(), 1.0, True, dtype=torch.float64).mean() * up, xd)
    loss = ops.distill_loss(x.requires_grad_(True), ids, lp, w) * up
    g1, = torch.autograd.grad(loss, x, retain_graph=True)
    g2, = torch.autograd.grad(loss, x)
    assert torch.equal(g1, g2)
    # a bf16 value's unit is 2^-7 of the power of two below it: half of it is
    # between 2^-9 and 2^-8 of the value. Twice rounded is up to 1.5 halves.
    half = torch.exp2(torch.floor(torch.log2(e.abs().clamp(min=1e-300)))) * 2.0 ** -8 \
        if dtype == torch.bfloat16 else 0.0
    err = (g1.double() - e).abs()
    assert bool((err <= 1.001 * half + TOL * e.abs() + TOL * 0.01 * e.abs().amax(1, keepdim=True)
                 + 1e-30).all())


def test_upstream_of_zero(b200_ops):
    """Nothing comes back: no gradient, whatever a row holds."""
    x, ids, lp = _rows(5, 3001, 5, torch.bfloat16, 3)
    x[2] = float("nan")
    loss = ops.distill_loss(x.requires_grad_(True), ids, lp) * 0.0
    g, = torch.autograd.grad(loss, x)
    assert bool((g == 0).all())


@pytest.mark.parametrize("V", [64, 5003, 2 ** 21 + 5])
def test_no_token_and_no_distribution(b200_ops, V):
    """No id of the teacher's is there: nothing to learn, from a row whose
    mask leaves nothing neither."""
    x, ids, lp = _rows(4, V, 5, torch.float32, 1)
    x[1] = -float("inf")
    ids[:2] = -1
    ids[1, 0] = V
    x[2] = -float("inf")
    want = L.distill_rows_ref(x, ids, lp, dtype=torch.float64)
    assert want[:3].tolist() == [0, 0, float("inf")]
    xg = x.requires_grad_(True)
    for reduction in ("none", "sum"):
        rows = ops.distill_loss(xg, ids, lp, reduction=reduction)
        g, = torch.autograd.grad(rows.sum(), xg)
        assert bool((g[:3] == 0).all()) and bool((g[3] != 0).any())
    rows = ops.distill_loss(xg.detach(), ids, lp, reduction="none")
    torch.testing.assert_close(rows.double(), want, atol=2 * TOL, rtol=TOL)
