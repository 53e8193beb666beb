"""Oracles of the logits operators against direct sums in Python floats, the
gradients they carry against differences, and the refusals."""
import math

import pytest
import torch

from vllm_sm70_b200 import ops
from vllm_sm70_b200.ops import logits as L

INF = float("inf")


def _row_direct(x, y, n, t):
    z = [v / t for v in x]
    m = max(z)
    s = sum(math.exp(v - m) for v in z)
    lse = m + math.log(s)
    lp = [v - lse for v in z]
    ent = -sum(math.exp(v) * v for v in lp if v > -INF)
    order = sorted(range(len(x)), key=lambda j: (-x[j], j))
    return lp[y], order.index(y) + 1, ent, lse, order[:n], [lp[j] for j in order[:n]]


@pytest.mark.parametrize("t", [1.0, 0.5])
def test_token_logprobs_direct(t):
    g = torch.Generator().manual_seed(3)
    x = torch.randint(-6, 7, (9, 23), generator=g).double() / 2  # ties
    x[2, 5:20] = -INF
    y = torch.randint(0, 5, (9,), generator=g)
    r = L.token_logprobs_ref(x, y, 4, t, dtype=torch.float64)
    for i in range(9):
        lp, rank, ent, lse, ids, top = _row_direct(x[i].tolist(), int(y[i]), 4, t)
        assert int(r.ranks[i]) == rank and r.top_ids[i].tolist() == ids
        for got, want in ((r.logprobs[i], lp), (r.entropy[i], ent), (r.lse[i], lse)):
            assert abs(float(got) - want) < 1e-12
        assert torch.allclose(r.top_logprobs[i], torch.tensor(top, dtype=torch.float64))


def test_token_logprobs_edges():
    x = torch.full((4, 6), -INF)
    x[1, 3] = 2.0
    x[2] = torch.tensor([1.0, float("nan"), 3.0, -INF, 0.0, 3.0])
    x[3] = 5.0
    r = ops.token_logprobs(x, torch.tensor([2, -1, 0, 6]), top_n=5)
    assert r.lse[0] == -INF and r.logprobs[0] == -INF and r.entropy[0] == 0
    assert r.top_ids[0].tolist() == [0, 1, 2, 3, 4]
    assert r.logprobs[1] == 0 and r.ranks[1] == 0 and r.entropy[1] == 0
    assert r.top_ids[1].tolist() == [3, 0, 1, 2, 4] and r.top_logprobs[1, 0] == 0
    assert torch.isnan(r.logprobs[2]) and torch.isnan(r.entropy[2]) and r.ranks[2] == 3
    assert r.top_ids[2].tolist() == [2, 5, 0, 4, 3]
    assert r.logprobs[3] == 0 and r.ranks[3] == 0 and abs(float(r.entropy[3]) - math.log(6)) < 1e-6
    y = torch.tensor([[float("nan"), 1.0]])
    assert ops.token_logprobs(y, torch.tensor([1]), top_n=2).top_ids.tolist() == [[1, -1]]


@pytest.mark.parametrize("tail", [True, False])
def test_distill_direct(tail):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(5, 17, generator=g, dtype=torch.float64)
    ids = torch.stack([torch.randperm(17, generator=g)[:4] for _ in range(5)])
    ids[2, 1] = -1
    ids[3, 2] = 99
    lp = torch.log_softmax(torch.randn(5, 4, generator=g), 1) - 0.2
    w = torch.tensor([1.0, 0.0, 2.0, 0.5, 1.0])
    got = L.distill_rows_ref(x, ids, lp, w, 0.7, tail, dtype=torch.float64)
    for i in range(5):
        z = [v / 0.7 for v in x[i].tolist()]
        s = sum(math.exp(v) for v in z)
        q = [math.exp(v) / s for v in z]
        pairs = [(int(a), float(b)) for a, b in zip(ids[i], lp[i]) if 0 <= a < 17]
        p = [math.exp(b) for _, b in pairs]
        if not tail:
            p = [v / sum(p) for v in p]
        loss = sum(a * (math.log(a) - math.log(q[j])) for a, (j, _) in zip(p, pairs))
        if tail:
            pt = 1 - sum(p)
            qt = sum(v for j, v in enumerate(q) if j not in {a for a, _ in pairs})
            loss += pt * (math.log(pt) - math.log(qt))
        assert abs(float(got[i]) - loss * float(w[i])) < 1e-6


@pytest.mark.parametrize("tail", [True, False])
def test_gradients_by_differences(tail):
    """The oracles' gradients (which the kernels are held to) agree with
    central differences in 64 bits: error O(h^2) + 2^-52 / h."""
    g = torch.Generator().manual_seed(7)
    x = torch.randn(3, 11, generator=g, dtype=torch.float64).requires_grad_(True)
    y = torch.tensor([4, 0, -1])
    ids = torch.tensor([[1, 5, 7], [2, 2, 9], [0, -1, 3]])
    lp = torch.log_softmax(torch.randn(3, 3, generator=g), 1) - 0.3
    a, b = torch.randn(3, generator=g).double(), torch.randn(3, generator=g).double()

    def f(z):
        r = L.token_logprobs_ref(z, y, 0, 1.3, dtype=torch.float64)
        d = L.distill_rows_ref(z, ids, lp, None, 1.3, tail, dtype=torch.float64)
        return (a * r.logprobs + b * r.entropy + a * d).sum()

    grad, = torch.autograd.grad(f(x), x)
    with torch.no_grad():
        for i in range(3):
            for j in range(11):
                e = torch.zeros_like(x)
                e[i, j] = 1e-5
                assert abs(float((f(x + e) - f(x - e)) / 2e-5 - grad[i, j])) < 1e-8


def test_distill_edges():
    x = torch.full((3, 5), -INF)
    x[1] = torch.tensor([float("nan"), INF, 0.0, 1.0, 2.0])
    x[2] = torch.tensor([0.0, 1.0, 2.0, 3.0, 4.0])
    ids = torch.tensor([[0, 1], [0, 1], [-1, 7]])
    lp = torch.log(torch.tensor([[0.5, 0.25]] * 3))
    w = torch.tensor([1.0, 0.0, 1.0])
    r = ops.distill_loss(x, ids, lp, weights=w, reduction="none")
    assert r[0] == INF and r[1] == 0
    assert abs(float(r[2])) < 1e-6  # no token of the teacher's is there: 1 against 1
    assert ops.distill_loss(x[2:], ids[2:], lp[2:], tail=False, reduction="sum") == 0
    assert ops.distill_loss(x[:0], ids[:0], lp[:0]) == 0


def test_refusals():
    x = torch.zeros(2, 8)
    y = torch.zeros(2, dtype=torch.int64)
    ids, lp = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3)
    for call in (
        lambda: ops.token_logprobs(x.half(), y),
        lambda: ops.token_logprobs(x[0], y),
        lambda: ops.token_logprobs(x.t().contiguous().t(), y),
        lambda: ops.token_logprobs(x, y[:1]),
        lambda: ops.token_logprobs(x, y.float()),
        lambda: ops.token_logprobs(x, y, top_n=9),
        lambda: ops.token_logprobs(x, y, top_n=-1),
        lambda: ops.token_logprobs(x, y, temperature=0.0),
        lambda: ops.distill_loss(x, ids, lp[:, :2]),
        lambda: ops.distill_loss(x, ids.float(), lp),
        lambda: ops.distill_loss(x, ids, lp.double()),
        lambda: ops.distill_loss(x, ids[:, :0], lp[:, :0]),
        lambda: ops.distill_loss(x, ids[:1], lp[:1]),
        lambda: ops.distill_loss(x, ids, lp, weights=torch.ones(3)),
        lambda: ops.distill_loss(x, ids, lp, reduction="batchmean"),
        lambda: ops.distill_loss(x, ids, lp.clone().requires_grad_(True)),
        lambda: ops.distill_loss(x, ids, lp, temperature=float("nan")),
    ):
        with pytest.raises(ValueError):
            call()
