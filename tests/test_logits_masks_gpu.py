"""GPU: token_logprobs and distill_loss on rows with finite masks, against the
64-bit oracle.

Tolerances. Elements that are masked by more than 150 T below a row's largest
add less than 2^-126 of it, so a row's values come from the others alone, and
the bound of the logits tests holds: with |x / T| up to 45 an exponent carries
45 * 1.45 * 2 * 2^-24, an exponential 2^-22, a sum of a few hundred terms 600 *
2^-24 at the most, in all less than 5e-5. Where every element of a row is at
the mask, the exponents are 0 but for the rounding of one product, which is
taken out again.
"""
import pytest
import torch

from vllm_sm70_b200 import ops
from vllm_sm70_b200.ops import logits as L

pytestmark = pytest.mark.gpu
TOL = 5e-5
DTYPES = [torch.bfloat16, torch.float32]


def _check_scores(x, y, n, t=1.0):
    r = ops.token_logprobs(x, y, top_n=n, temperature=t)
    e = L.token_logprobs_ref(x, y, n, t, dtype=torch.float64)
    assert torch.equal(r.ranks, e.ranks) and torch.equal(r.top_ids, e.top_ids)
    for a, b in ((r.logprobs, e.logprobs), (r.entropy, e.entropy), (r.lse, e.lse),
                 (r.top_logprobs, e.top_logprobs)):
        torch.testing.assert_close(a, b.float(), atol=TOL, rtol=TOL)


def _assert_grad(got, want, dtype):
    rel = (2.0 ** -8 if dtype == torch.bfloat16 else 0.0) + TOL
    err = (got.double() - want).abs()
    lim = rel * want.abs() + TOL * want.abs().amax(1, keepdim=True) + 1e-30
    assert bool((err <= lim).all()), float((err - lim).max())


def _check_distill(x, ids, lp, t=1.0, tail=True):
    """Losses and gradients of every form."""
    xd = x.detach().double().requires_grad_(True)
    want = L.distill_rows_ref(xd, ids, lp, None, t, tail, dtype=torch.float64)
    e, = torch.autograd.grad(want.sum(), xd)
    want = want.detach()
    xg = x.detach().requires_grad_(True)
    with torch.no_grad():
        rows = ops.distill_loss(x, ids, lp, None, t, tail, reduction="none")
    torch.testing.assert_close(rows.double(), want, atol=2 * TOL, rtol=TOL)
    for red in ("none", "sum"):
        loss = ops.distill_loss(xg, ids, lp, None, t, tail, reduction=red).sum()
        assert abs(float(loss.detach()) - float(want.sum())) <= \
            2 * TOL * float((1 + want.abs()).sum())
        g, = torch.autograd.grad(loss, xg)
        _assert_grad(g, e, x.dtype)


MASKS = [-1e6, -1e9, -1e10, -1e15, -1e20, -1e29, None]  # None: the type's lowest value


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t", [1.0, 0.9, 0.1])
@pytest.mark.parametrize("value", MASKS)
def test_scores_of_masked_rows(b200_ops, value, t, dtype):
    """Masks of any size, in CTAs that see the mask first and in slices that
    hold nothing else."""
    value = torch.finfo(dtype).min if value is None else value
    for rows, V in ((600, 32000), (3, 200000)):
        x = torch.empty(rows, V, device="cuda").normal_(
            generator=torch.Generator(device="cuda").manual_seed(V)).to(dtype)
        x[:, : V * 2 // 3] = value
        x[1] = value
        x[2] = value
        x[2, V - 100] = 2.0
        y = torch.full((rows,), V - 5, device="cuda")
        _check_scores(x, y, 5, t)
        xg = x.detach().requires_grad_(True)
        r = ops.token_logprobs(xg, y, temperature=t)
        g, = torch.autograd.grad((r.logprobs + r.entropy).sum(), xg)
        xd = x.double().requires_grad_(True)
        e = L.token_logprobs_ref(xd, y, 0, t, dtype=torch.float64)
        w, = torch.autograd.grad((e.logprobs + e.entropy).sum(), xd)
        _assert_grad(g, w, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t", [1.0, 0.9, 0.1])
@pytest.mark.parametrize("value", MASKS)
def test_distillation_of_masked_rows(b200_ops, value, t, dtype):
    value = torch.finfo(dtype).min if value is None else value
    for rows, V in ((400, 16000), (3, 200000), (2, 2 ** 21)):
        g = torch.Generator(device="cuda").manual_seed(V)
        x = torch.empty(rows, V, device="cuda").normal_(generator=g).to(dtype)
        x[:, : V * 2 // 3] = value
        x[1] = value
        ids = (V - 9 + torch.arange(8, device="cuda")).expand(rows, 8).contiguous()
        lp = torch.log_softmax(torch.randn(rows, 8, device="cuda", generator=g), 1) - 0.2
        for tail in (True, False):
            _check_distill(x, ids, lp, t, tail)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", [(400, 20011), (3, 200003)])
def test_one_token_left_at_the_lowest_value(b200_ops, rows, V, dtype):
    """All but two elements at the type's lowest value, in rows at every
    alignment: warps that hold nothing else sum their own vectors again, the
    same ones."""
    E = 128 // torch.finfo(dtype).bits
    x = torch.full((rows, V), torch.finfo(dtype).min, device="cuda", dtype=dtype)
    r = torch.arange(rows, device="cuda")
    # the last lane of a warp, where a row begins inside a 16-byte vector
    p = 32 * E * (1 + r % 70)
    x[r, p] = 1.5
    x[:, 5] = 0.5
    _check_scores(x, p, 2)
    ids = torch.full((rows, 1), 5, device="cuda")
    lp = torch.full((rows, 1), -0.25, device="cuda")
    _check_distill(x, ids, lp)


@pytest.mark.parametrize("dtype", DTYPES)
def test_lowest_value_in_rows_that_no_cluster_holds(b200_ops, dtype):
    E = 128 // torch.finfo(dtype).bits
    V = 2 ** 22 - 3
    x = torch.full((2, V), torch.finfo(dtype).min, device="cuda", dtype=dtype)
    x[:, 5] = 0.5
    x[0, 32 * E * 3] = 1.5
    x[1, 32 * E * 9] = 1.5
    ids = torch.full((2, 1), 5, device="cuda")
    _check_distill(x, ids, torch.full((2, 1), -0.25, device="cuda"))
