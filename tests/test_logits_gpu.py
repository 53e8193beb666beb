"""GPU: log-probabilities of given tokens and top-logit distillation against
the 64-bit oracle.

Tolerances. The base-2 exponents x * log2(e) / T - r are one fused product,
so an exponent of size D carries D * 2^-24; each e_j has the 2^-22 of the
hardware exponential; a thread adds at most a few hundred terms one after
the other (2^-24 each). With |x / T| up to 40 that bounds the relative error
of a probability, and the absolute error of a log-probability, by 60 * 2^-24
+ 2^-22 + 600 * 2^-24 < 5e-5. bf16 gradients add half a unit of 2^-8.
"""
import pytest
import torch

from vllm_sm70_b200 import ops
from vllm_sm70_b200.ops import logits as L

pytestmark = pytest.mark.gpu
INF = float("inf")
TOL = 5e-5


def _rows(T, V, dtype, seed, pad=0, offset=0):
    """Peaked rows; with pad / offset a view into a wider, misaligned buffer
    whose other columns are poisoned."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty(T, V, device="cuda").normal_(0, 2.5, generator=g)
    x[:, :: max(1, V // 5)] += 7.0
    x = x.to(dtype)
    if pad or offset:
        buf = torch.full((T, V + pad + offset), float("nan"), device="cuda", dtype=dtype)
        buf[:, offset:offset + V] = x
        x = buf[:, offset:offset + V]
    return x


def _check_scores(x, y, n, t=1.0):
    r = ops.token_logprobs(x, y, top_n=n, temperature=t)
    e = L.token_logprobs_ref(x, y, n, t, dtype=torch.float64)
    assert torch.equal(r.ranks, e.ranks)
    assert torch.equal(r.top_ids, e.top_ids)
    for a, b in ((r.logprobs, e.logprobs), (r.entropy, e.entropy), (r.lse, e.lse),
                 (r.top_logprobs, e.top_logprobs)):
        # (rounded to the output's type: 64 bits hold log-probs that fp32 has as -inf)
        torch.testing.assert_close(a, b.float(), atol=TOL, rtol=TOL, equal_nan=True)


SHAPES = [(1, 1), (3, 7), (5, 1000), (2, 32003), (17, 4099), (9, 151936), (700, 1031),
          (300, 8195), (160, 70001)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V", SHAPES)
def test_scores(b200_ops, T, V, dtype):
    x = _rows(T, V, dtype, T + V)
    g = torch.Generator(device="cuda").manual_seed(1)
    y = torch.randint(0, V, (T,), device="cuda", generator=g)
    y[:: 3] = x[:: 3].float().argmax(1)
    for n in sorted({0, 1, min(5, V), min(64, V)}):
        _check_scores(x, y, n)
    _check_scores(x, y.to(torch.int32), min(20, V), 0.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad,offset", [(1, 0), (3, 1), (0, 5), (8, 8)])
def test_scores_strided(b200_ops, dtype, pad, offset):
    x = _rows(11, 5003, dtype, 4, pad, offset)
    _check_scores(x, torch.arange(11, device="cuda") * 400, 20)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [13, 400])  # a cluster a row, a CTA a row
def test_scores_masks_and_ties(b200_ops, dtype, rows):
    V = 20011
    x = _rows(rows, V, dtype, 9)
    low = torch.finfo(dtype).min
    x[0] = -INF                       # nothing left
    x[1] = -INF
    x[1, 777] = 1.5                   # one token left
    x[2] = -INF
    x[2, 100:130] = 2.0               # fewer than 64, all equal
    x[3] = low                        # the type's lowest value everywhere
    x[4] = low
    x[4, 3:9] = torch.arange(6, device="cuda").to(dtype)
    x[5] = 1.25                       # all equal
    x[6] = torch.linspace(-9, 9, V, device="cuda").to(dtype)   # ascending, ties in bf16
    x[7] = torch.linspace(9, -9, V, device="cuda").to(dtype)
    x[8, 4096:8192] = 30.0            # thousands of ties at the top
    x[9] = 0.0
    x[9, 1::2] = -0.0                 # the two zeros are equal
    x[10] = -5.0
    x[10, 512 * 8 * 2: 512 * 8 * 2 + 8] = 5.0   # the top in one thread's vector
    x[11, :] = -1e4
    x[11, 19000:] = torch.linspace(0, 20, V - 19000, device="cuda").to(dtype)
    y = torch.randint(0, V, (rows,), device="cuda",
                      generator=torch.Generator(device="cuda").manual_seed(2))
    y[0], y[1], y[2], y[8], y[9] = 17, 777, 129, 5000, 19999
    for n in (0, 5, 20, 64):
        _check_scores(x, y, n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scores_far_out_and_forbidden(b200_ops, dtype):
    """Rows whose maximum lies far below or above, and given tokens whose own
    logit is -inf, in rows at every alignment."""
    x = _rows(40, 4099, dtype, 3, pad=2, offset=3)
    x[0], x[1, :] = -3e37, 2e37
    x[1, 7] = 2.5e37
    x[2] = -5e29
    x[2, 9:12] = -4e29
    x[3, ::2] = -2e30
    x[4, 1:] = -INF
    x[4, 0] = torch.finfo(dtype).min
    x[5:] = torch.where(torch.rand(35, 4099, device="cuda") < 0.5, -INF, x[5:].float()).to(dtype)
    x[5:, 2000] = -INF
    _check_scores(x, torch.full((40,), 2000, device="cuda"), 20)
    _check_scores(x, torch.arange(40, device="cuda") % 9, 5, 0.01)


def test_scores_clustered_top(b200_ops):
    """More than 512 elements of few threads above every other thread's: the
    bound is raised to the exact one."""
    V = 512 * 8 * 40
    x = torch.full((3, V), -3.0, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    v = x.view(3, 40, 512, 8)
    v[:, :, :20] = torch.randn(3, 40, 20, 8, device="cuda", generator=g) + 10
    xf = x.repeat(110, 1)
    y = torch.randint(0, V, (330,), device="cuda", generator=g)
    _check_scores(xf.bfloat16(), y, 64)
    _check_scores(xf.view(330, V), y, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scores_largest_vocabulary(b200_ops, dtype):
    """Where a thread has more groups of vectors than places for their maxima."""
    x = _rows(2, 2 ** 22 - 3, dtype, 6, pad=3, offset=1)
    _check_scores(x, torch.tensor([2 ** 22 - 4, 0], device="cuda"), 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [3, 600])
def test_scores_top_in_every_warp(b200_ops, dtype, rows):
    """Some 1500 elements above every other, in few groups of every warp."""
    x = torch.full((rows, 65536), -3.0, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    x.view(rows, 1024, 64)[:, ::2, :3] = torch.randn(rows, 512, 3, device="cuda", generator=g) + 10
    y = torch.randint(0, 65536, (rows,), device="cuda", generator=g)
    _check_scores(x.to(dtype), y, 64)
    _check_scores(x.to(dtype), y, 9)


def test_scores_nan_inf_and_no_token(b200_ops):
    x = _rows(6, 9001, torch.float32, 21)
    x[1, 4000] = float("nan")
    x[2, 8000] = INF
    x[3] = float("nan")
    y = torch.tensor([-1, 5, 6, 7, 9001, 2 ** 40], device="cuda")
    r = ops.token_logprobs(x, y, top_n=3)
    e = L.token_logprobs_ref(x, y, 3)
    assert torch.equal(r.ranks, e.ranks)
    assert torch.equal(r.top_ids[[0, 1, 2, 4, 5]], e.top_ids[[0, 1, 2, 4, 5]])
    assert r.top_ids[3].tolist() == [-1, -1, -1]
    torch.testing.assert_close(r.logprobs, e.logprobs, atol=TOL, rtol=TOL, equal_nan=True)
    assert torch.isnan(r.entropy[1:4]).all() and torch.isnan(r.lse[1:4]).all()
    assert not torch.isnan(r.entropy[[0, 4, 5]]).any()


def _assert_grad(got, want, dtype):
    # half a unit in the last place of the type, and the bound of the head of this file
    rel = (2.0 ** -8 if dtype == torch.bfloat16 else 0.0) + TOL
    err = (got.double() - want).abs()
    lim = rel * want.abs() + TOL * want.abs().amax(1, keepdim=True) + 1e-30
    assert bool((err <= lim).all()), float((err - lim).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V", SHAPES)
@pytest.mark.parametrize("which", ["logprob", "entropy", "both"])
def test_score_gradient(b200_ops, T, V, dtype, which):
    x = _rows(T, V, dtype, T * 3 + V).requires_grad_(True)
    g = torch.Generator(device="cuda").manual_seed(8)
    y = torch.randint(-1, V, (T,), device="cuda", generator=g)
    a, b = (torch.randn(T, device="cuda", generator=g) for _ in range(2))
    a[:: 4] = 0
    r = ops.token_logprobs(x, y, temperature=0.8)
    xd = x.detach().double().requires_grad_(True)
    e = L.token_logprobs_ref(xd, y, 0, 0.8, dtype=torch.float64)
    f = {"logprob": lambda q, u, v: (q.logprobs * u).sum(),
         "entropy": lambda q, u, v: (q.entropy * v).sum(),
         "both": lambda q, u, v: (q.logprobs * u + q.entropy * v).sum()}[which]
    got, = torch.autograd.grad(f(r, a, b), x)
    want, = torch.autograd.grad(f(e, a.double(), b.double()), xd)
    assert got.dtype == dtype
    _assert_grad(got, want, dtype)


def test_score_gradient_rows_without_one(b200_ops):
    x = _rows(4, 3001, torch.bfloat16, 2)
    x[0] = -INF
    x[1, 5] = float("nan")
    x = x.requires_grad_(True)
    r = ops.token_logprobs(x, torch.tensor([3, 4, -1, 9], device="cuda"))
    g, = torch.autograd.grad((r.logprobs, r.entropy), x, (
        torch.tensor([1.0, 0.0, 1.0, 0.0], device="cuda"), torch.zeros(4, device="cuda")))
    assert bool((g == 0).all())


def _teacher(T, V, K, seed, spread=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    step = max(1, V // max(K, 1))
    ids = (torch.randint(0, V, (T, 1), device="cuda", generator=g)
           + step * torch.arange(K, device="cuda")) % V
    rest = 0.02 + 0.3 * torch.rand(T, 1, device="cuda", generator=g)
    lp = torch.log_softmax(torch.randn(T, K, device="cuda", generator=g), 1) + torch.log1p(-rest)
    return ids, lp


def _check_distill(x, ids, lp, w, t, tail, dtype):
    want = L.distill_rows_ref(x, ids, lp, w, t, tail, dtype=torch.float64)
    rows = ops.distill_loss(x, ids, lp, w, t, tail, reduction="none")
    torch.testing.assert_close(rows.double(), want, atol=2 * TOL, rtol=TOL)
    xg = x.detach().requires_grad_(True)
    xd = x.detach().double().requires_grad_(True)
    up = torch.rand(x.shape[0], device="cuda") + 0.5
    g1, = torch.autograd.grad(ops.distill_loss(xg, ids, lp, w, t, tail, reduction="none"), xg, up)
    e1, = torch.autograd.grad(L.distill_rows_ref(xd, ids, lp, w, t, tail, dtype=torch.float64), xd,
                              up.double())
    _assert_grad(g1, e1, dtype)
    loss = ops.distill_loss(xg, ids, lp, w, t, tail)
    assert abs(float(loss) - float(want.mean())) <= 2 * TOL * (1 + float(want.abs().mean()))
    g2, = torch.autograd.grad(loss, xg)
    e2, = torch.autograd.grad(
        L.distill_rows_ref(xd, ids, lp, w, t, tail, dtype=torch.float64).mean(), xd)
    _assert_grad(g2, e2, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("T,V,K", [(1, 1, 1), (3, 7, 3), (5, 1000, 8), (2, 32003, 128),
                                   (17, 4099, 20), (6, 151936, 64), (700, 1031, 5),
                                   (330, 40001, 33), (3, 300007, 16)])
def test_distill(b200_ops, T, V, K, tail, dtype):
    x = _rows(T, V, dtype, T + V)
    ids, lp = _teacher(T, V, K, T + K)
    w = (torch.arange(T, device="cuda") % 4 != 1).float() * 1.5
    if V > K:  # the student's mass outside the teacher's tokens is not zero
        _check_distill(x, ids, lp, w, 1.0, tail, dtype)
    _check_distill(x, ids.int(), lp, None, 2.0, tail and V > K, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V", [(3, 1000003), (2, 2 ** 22 - 3)])
def test_distill_rows_that_no_cluster_holds(b200_ops, T, V, dtype):
    x = _rows(T, V, dtype, 5, pad=3, offset=1)
    ids, lp = _teacher(T, V, 20, 7)
    ids[0, 5] = ids[0, 3]
    _check_distill(x, ids, lp, torch.tensor([1.5, 0.5, 0.0], device="cuda")[:T], 1.0, True, dtype)
    _check_distill(x, ids, lp, None, 2.0, False, dtype)
    xg = x.detach().requires_grad_(True)
    g, = torch.autograd.grad(ops.distill_loss(xg, ids, lp), xg)
    assert bool((g != 0).all())  # every element has its own, however small


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V", [(500, 30011), (40, 128257), (7, 5003), (330, 70001)])
def test_every_element_has_its_gradient(b200_ops, T, V, dtype):
    """None is left out or written over, however small it is."""
    x = _rows(T, V, dtype, 5, pad=3, offset=1).requires_grad_(True)
    ids, lp = _teacher(T, V, 20, 7)
    y = ids[:, 0].contiguous()
    for loss in (ops.distill_loss(x, ids, lp), ops.distill_loss(x, ids, lp, reduction="none").sum(),
                 ops.token_logprobs(x, y).logprobs.sum()):
        g, = torch.autograd.grad(loss, x)
        assert bool((g != 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distill_graph(b200_ops, dtype):
    """More rows than clusters (the rows come from a counter), replayed."""
    x = _rows(500, 30011, dtype, 3).requires_grad_(True)
    ids, lp = _teacher(500, 30011, 9, 2)
    g, = torch.autograd.grad(ops.distill_loss(x, ids, lp), x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.distill_loss(x, ids, lp), x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got, = torch.autograd.grad(ops.distill_loss(x, ids, lp), x)
    torch.cuda.synchronize()
    for _ in range(3):
        got.zero_()
        graph.replay()
        assert torch.equal(got, g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad,offset", [(1, 0), (3, 1), (0, 5)])
def test_distill_strided(b200_ops, dtype, pad, offset):
    x = _rows(7, 5003, dtype, 4, pad, offset)
    ids, lp = _teacher(7, 5003, 12, 3)
    _check_distill(x, ids, lp, None, 1.0, True, dtype)


def test_distill_repeated_and_absent_ids(b200_ops):
    V = 70001
    x = _rows(9, V, torch.float32, 31)
    ids, lp = _teacher(9, V, 10, 5)
    ids[1, 3] = ids[1, 7]
    ids[2, :] = 12345           # one token, ten times
    ids[3, 2:5] = -1
    ids[4, :] = V + 5
    ids[5, 9] = 2 ** 40
    for tail in (True, False):
        _check_distill(x, ids, lp, None, 1.0, tail, torch.float32)


def test_distill_sharp_student(b200_ops):
    """A student whose mass outside the teacher's tokens is 1e-7 and less: the
    mass is summed, not taken from 1."""
    x = torch.randn(4, 9000, device="cuda")
    ids, lp = _teacher(4, 9000, 4, 5)
    x.scatter_(1, ids, torch.tensor([[24.0], [30.0], [35.0], [40.0]], device="cuda").expand(4, 4))
    want = L.distill_rows_ref(x, ids, lp, dtype=torch.float64)
    got = ops.distill_loss(x, ids, lp, reduction="none")
    torch.testing.assert_close(got.double(), want, atol=2 * TOL, rtol=TOL)


def test_distill_rows_that_do_not_count(b200_ops):
    x = _rows(5, 8000, torch.bfloat16, 6)
    x[0] = float("nan")
    x[2] = INF
    ids, lp = _teacher(5, 8000, 6, 5)
    lp[2] = float("nan")
    w = torch.tensor([0.0, 1.0, 0.0, 0.0, 2.0], device="cuda")
    xg = x.requires_grad_(True)
    for red in ("none", "sum", "mean"):
        loss = ops.distill_loss(xg, ids, lp, w, reduction=red).sum()
        assert bool(torch.isfinite(loss))
        g, = torch.autograd.grad(loss, xg)
        assert bool(torch.isfinite(g).all()) and bool((g[[0, 2, 3]] == 0).all())
        assert bool((g[[1, 4]] != 0).any(1).all())


def test_distill_empty_row_and_masked_token(b200_ops):
    x = _rows(3, 5000, torch.float32, 6)
    ids, lp = _teacher(3, 5000, 6, 5)
    x[0] = -INF
    x[1, ids[1, 2]] = -INF
    x[2] = -INF
    x[2, ids[2]] = 1.0          # no mass outside
    xg = x.requires_grad_(True)
    loss = ops.distill_loss(xg, ids, lp, reduction="none")
    assert bool((loss == INF).all())
    g, = torch.autograd.grad(ops.distill_loss(xg, ids, lp, reduction="sum"), xg)
    assert bool((g[0] == 0).all()) and bool(torch.isfinite(g).all())
    r = ops.distill_loss(xg, ids, lp, tail=False, reduction="none")
    assert bool(torch.isfinite(r[2])) and r[0] == INF and r[1] == INF


def test_scalar_upstream_and_second_backward(b200_ops):
    """The scalar's gradient is scaled by what comes back, and a graph that is
    kept gives the same gradient again."""
    x = _rows(6, 3001, torch.float32, 6).requires_grad_(True)
    ids, lp = _teacher(6, 3001, 6, 5)
    base, = torch.autograd.grad(ops.distill_loss(x, ids, lp), x)
    loss = ops.distill_loss(x, ids, lp) * 0.37
    g1, = torch.autograd.grad(loss, x, retain_graph=True)
    keep = g1.clone()
    g2, = torch.autograd.grad(loss, x)
    torch.testing.assert_close(g1, base * 0.37, atol=1e-9, rtol=1e-6)
    assert torch.equal(g1, keep)
    torch.testing.assert_close(g2, g1, atol=1e-9, rtol=1e-5)


@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_differentiable_once(b200_ops, reduction):
    x = _rows(5, 777, torch.float32, 8).requires_grad_(True)
    ids, lp = _teacher(5, 777, 4, 1)
    y = torch.arange(5, device="cuda")
    for loss in (ops.distill_loss(x, ids, lp, reduction=reduction).sum(),
                 ops.token_logprobs(x, y).logprobs.sum()):
        g, = torch.autograd.grad(loss, x, create_graph=True)
        assert torch.isfinite(g).all()
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            g.sum().backward()


def test_launches_are_counted(b200_ops):
    from vllm_sm70_b200.utils import launch_count
    x = _rows(5, 777, torch.bfloat16, 8).requires_grad_(True)
    ids, lp = _teacher(5, 777, 4, 1)
    ops.distill_loss(x, ids, lp)  # (the first call adds the native counter)
    before = launch_count.total()
    loss = ops.distill_loss(x, ids, lp)
    assert launch_count.total() - before == 2
    loss.backward()
    assert launch_count.total() - before == 3
    with torch.no_grad():
        ops.token_logprobs(x, torch.arange(5, device="cuda"))
    assert launch_count.total() - before == 4


def test_same_bits_twice_and_other_stream(b200_ops):
    x = _rows(40, 70001, torch.bfloat16, 12)
    y = torch.arange(40, device="cuda") * 31
    ids, lp = _teacher(40, 70001, 50, 5)
    a = ops.token_logprobs(x, y, 20)
    xg = x.requires_grad_(True)
    ga, = torch.autograd.grad(ops.distill_loss(xg, ids, lp), xg)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = ops.token_logprobs(x.detach(), y, 20)
        gb, = torch.autograd.grad(ops.distill_loss(xg, ids, lp), xg)
    torch.cuda.current_stream().wait_stream(s)
    for p, q in zip(a, b):
        assert torch.equal(p.view(torch.int32), q.view(torch.int32))
    assert torch.equal(ga, gb)


def test_no_rows(b200_ops):
    x = torch.empty(0, 100, device="cuda")
    r = ops.token_logprobs(x, torch.empty(0, dtype=torch.int64, device="cuda"), 5)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 5)
    e = torch.empty(0, 3, device="cuda")
    assert float(ops.distill_loss(x, e.int(), e)) == 0
    assert ops.distill_loss(x, e.int(), e, reduction="none").shape == (0,)


def test_refusals_cuda(b200_ops):
    x = torch.zeros(2, 8, device="cuda")
    y = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError):
        ops.token_logprobs(x, y)  # ids on another device
    with pytest.raises(RuntimeError):
        ops.distill_loss(x, torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3))
    with pytest.raises(RuntimeError):
        b200_ops.token_logprobs(x.half(), y.cuda(), 0, 1.0)
    with pytest.raises(RuntimeError):
        b200_ops.token_logprobs(x, y.cuda(), 65, 1.0)
