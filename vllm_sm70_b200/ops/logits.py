"""Operators over rows of logits: log-probabilities of given tokens with
their rank, entropy and top alternatives, and distillation from a teacher's
top log-probabilities. Both have a backward pass (reverse mode, once; on CUDA
tensors forward-mode derivatives raise ``NotImplementedError``).

Rows of logits are ``[rows, V]``, bf16 or fp32, with a unit inner stride and
any row stride (a slice of a wider buffer is read in place). Sums are held in
fp32; gradients have the logits' dtype, rounded once.

Reference parity: the reference leaves log-probabilities to vLLM's sampler
(``sm70/vllm_sm70/sample_greedy.py:74-328`` covers the greedy fast path only)
and has no training operators.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _ext
from ..utils import launch_count

MAX_TOP_N = 64
MAX_TEACHER_K = 128


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # [rows] fp32, log softmax(logits / T) at the token
    ranks: torch.Tensor         # [rows] int32, 1 = first by (logit descending, id ascending)
    entropy: torch.Tensor       # [rows] fp32, nats
    lse: torch.Tensor           # [rows] fp32, logsumexp(logits / T)
    top_ids: torch.Tensor       # [rows, top_n] int32, in that order; -1 where there is none
    top_logprobs: torch.Tensor  # [rows, top_n] fp32


# ------------------------------------------------------------------ references
def _sums(z: torch.Tensor):
    """(lse, log-probs, probs) of rows; a row without an element above -inf
    has lse -inf, log-probs -inf and probs 0."""
    m = torch.where(torch.isnan(z), float("-inf"), z.detach()).amax(1, keepdim=True)
    empty = (m == float("-inf")) & ~torch.isnan(z.detach()).any(1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    s = torch.exp(z - m).sum(1, keepdim=True)
    ls = torch.log(torch.where(empty, torch.ones_like(s), s))
    lp = torch.where(empty, torch.full_like(z, float("-inf")), z - m - ls)
    lse = torch.where(empty, torch.full_like(m, float("-inf")), m + ls)[:, 0]
    return lse, lp, torch.exp(lp)


def token_logprobs_ref(logits: torch.Tensor, token_ids: torch.Tensor, top_n: int = 0,
                       temperature: float = 1.0, dtype=torch.float32) -> TokenLogprobs:
    """Oracle of :func:`token_logprobs` (differentiable torch operations)."""
    x = logits.to(dtype)
    T, V = x.shape
    lse, lp, p = _sums(x / temperature)
    finite = lp > float("-inf")
    ent = -torch.where(finite | torch.isnan(lp), p * torch.where(finite, lp, lp.nan_to_num(0.0)),
                       torch.zeros_like(p)).sum(1)
    ent = torch.where(torch.isnan(lp.detach()).any(1), torch.full_like(ent, float("nan")), ent)
    ids = token_ids.to(torch.int64)
    ok = (ids >= 0) & (ids < V)
    at = torch.where(ok, ids, torch.zeros_like(ids))[:, None]
    xd = x.detach()
    xy, col = xd.gather(1, at), torch.arange(V, device=x.device)
    rank = 1 + ((xd > xy) | ((xd == xy) & (col < at))).sum(1)
    rank = torch.where(ok & ~torch.isnan(xy[:, 0]), rank, torch.zeros_like(rank))
    got = torch.where(ok, lp.gather(1, at)[:, 0], torch.zeros_like(ent))
    # NaN elements are nobody's alternative: they sort behind -inf
    nan = torch.isnan(xd)
    order = torch.sort(torch.where(nan, float("-inf"), xd), dim=1, descending=True, stable=True)[1]
    order = order.gather(1, torch.sort(nan.gather(1, order).to(torch.int8), dim=1,
                                       stable=True)[1])[:, :top_n]
    absent = nan.gather(1, order)
    top_ids = torch.where(absent, -1, order).to(torch.int32)
    top_lp = torch.where(absent, float("-inf"), lp.detach().gather(1, order))
    return TokenLogprobs(got, rank.to(torch.int32), ent, lse.detach(), top_ids, top_lp)


def distill_rows_ref(logits: torch.Tensor, teacher_ids: torch.Tensor,
                     teacher_logprobs: torch.Tensor, weights: torch.Tensor | None = None,
                     temperature: float = 1.0, tail: bool = True,
                     dtype=torch.float32) -> torch.Tensor:
    """Oracle of :func:`distill_loss` with ``reduction="none"``."""
    w = None if weights is None else weights.to(dtype)
    x = logits.to(dtype)
    if w is not None:  # rows that do not count may hold anything
        x = torch.where((w == 0)[:, None], torch.zeros_like(x), x)
    V = x.shape[1]
    _, lq, _ = _sums(x / temperature)
    ids = teacher_ids.to(torch.int64)
    ok = (ids >= 0) & (ids < V)
    at = torch.where(ok, ids, torch.zeros_like(ids))
    lp = torch.where(ok, teacher_logprobs.to(dtype), float("-inf"))
    if not tail:
        norm = torch.logsumexp(lp, 1, keepdim=True)
        lp = torch.where(ok, lp - torch.where(norm == float("-inf"), torch.zeros_like(norm), norm),
                         float("-inf"))
    p = torch.exp(lp)
    on = ~(p <= 0)  # a NaN counts
    zero = torch.zeros_like(p)
    rows = torch.where(on, p * (torch.where(on, lp, zero) - torch.where(on, lq.gather(1, at), zero)),
                       zero).sum(1)
    if tail:
        pt = (1 - p.sum(1)).clamp(min=0)
        inside = torch.zeros_like(x, dtype=torch.int32).scatter_add_(1, at, ok.int()) > 0
        lqt = _sums(torch.where(inside, torch.full_like(lq, float("-inf")), lq))[0]
        on = (pt > 0) & ok.any(1)  # no token at all: p_t = q_t = 1, nothing to learn
        rows = rows + torch.where(on, pt * (torch.log(torch.where(on, pt, torch.ones_like(pt)))
                                            - torch.where(on, lqt, torch.zeros_like(lqt))),
                                  torch.zeros_like(pt))
    return rows if w is None else torch.where(w == 0, torch.zeros_like(rows), rows * w)


# ------------------------------------------------------------------ checks
def _check_rows(logits: torch.Tensor, what: str) -> None:
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"{what}: logits must be [rows, V] in bf16 or fp32, got "
                         f"{list(logits.shape)} {logits.dtype}")
    if logits.shape[1] < 1 or logits.shape[1] > 1 and logits.stride(1) != 1:
        raise ValueError(f"{what}: logits need V >= 1 and a unit inner stride")


def _check_temperature(temperature: float, what: str) -> float:
    t = float(temperature)
    if not 1e-3 <= t <= 1e3:
        raise ValueError(f"{what}: temperature must be in [1e-3, 1e3], got {temperature}")
    return t


def _count_backward() -> None:
    """The native backward passes count their launches themselves."""
    launch_count.also(torch.ops._b200_C.backward_launches)


# ------------------------------------------------------------------ token log-probs
def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor, top_n: int = 0,
                   temperature: float = 1.0) -> TokenLogprobs:
    """Log-probability, rank and alternatives of one given token a row.

    ``logits [rows, V]`` (bf16 / fp32), ``token_ids [rows]`` (int32 / int64);
    the distribution is ``softmax(logits / temperature)``. ``top_n`` (at most
    64, and at most V) alternatives come in the order of the ranks: larger
    logit first, lower id first among equals. ``logprobs`` and ``entropy`` are
    differentiable with respect to the logits; the other outputs are not.

    * a token id outside ``[0, V)`` stands for "no token": log-prob 0, rank 0,
      no gradient through it (the entropy's still flows);
    * a row whose logits are all ``-inf`` has no distribution: log-probs
      ``-inf``, entropy 0, gradient 0;
    * a row with NaN or ``+inf`` has NaN log-probs and entropy (as
      ``log_softmax`` has); a NaN is not counted in ranks and never listed.
    """
    _check_rows(logits, "token_logprobs")
    rows, V = logits.shape
    if token_ids.dtype not in (torch.int32, torch.int64) or tuple(token_ids.shape) != (rows,):
        raise ValueError(f"token_logprobs: token_ids must be int32 or int64 [{rows}], got "
                         f"{list(token_ids.shape)} {token_ids.dtype}")
    if not 0 <= top_n <= min(MAX_TOP_N, V):
        raise ValueError(f"token_logprobs: top_n must be in [0, {min(MAX_TOP_N, V)}], got {top_n}")
    t = _check_temperature(temperature, "token_logprobs")
    if not logits.is_cuda:
        return token_logprobs_ref(logits, token_ids, top_n, t)
    _ext.require()
    ids = token_ids.contiguous()
    launch_count.add(1)
    if logits.requires_grad and torch.is_grad_enabled():
        _count_backward()
        return TokenLogprobs(*torch.ops._b200_C.token_logprobs_train(logits, ids, top_n, t))
    return TokenLogprobs(*torch.ops._b200_C.token_logprobs(logits, ids, top_n, t)[:6])


# ------------------------------------------------------------------ distillation
def distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor,
                 weights: torch.Tensor | None = None, temperature: float = 1.0,
                 tail: bool = True, reduction: str = "mean") -> torch.Tensor:
    """Forward KL of a student from a teacher's top log-probabilities.

    ``logits [rows, V]`` (bf16 / fp32) are the student's; ``teacher_ids``
    (integer) and ``teacher_logprobs`` (fp32) ``[rows, K]``, K at most 128,
    are tokens and log-probs of the teacher at the same temperature (such as
    :func:`token_logprobs` returns with ``top_n``). With ``p_k =
    exp(teacher_logprobs)`` and ``q = softmax(logits / temperature)`` the loss
    of a row is

    * ``tail=True``: ``sum_k p_k (log p_k - log q_k) + p_t (log p_t - log
      q_t)``, where ``p_t`` and ``q_t`` are the masses outside the K tokens
      (``p_t = max(0, 1 - sum p_k)``);
    * ``tail=False``: the sum over the K alone, ``p`` renormalised over them
      (loss and gradient 0 where none of them has any).

    ``weights [rows]`` multiply the rows' losses; a row of weight 0 counts
    nothing, whatever it holds, and is not read. ``reduction``: ``"none"``
    (``[rows]``), ``"sum"``, or ``"mean"`` (the sum over the number of rows).
    The gradient with respect to the logits does not include the customary
    factor ``temperature ** 2``; the teacher is a constant. ``"sum"`` and
    ``"mean"`` compute the gradient in the forward pass (one read of the
    logits, one write of the gradient).

    Ids outside ``[0, V)`` are absent (their mass joins the tail); a repeated
    id's values are both held against that token. A student that gives a
    teacher's token no probability, or one that fp32 has no logarithm for (a
    mask of the lowest value over a temperature below 1), has loss ``inf``. So
    has one with no mass outside the tokens where ``p_t`` is not 0: log-probs
    that hold all of the teacher's mass still sum to 1 only within their
    rounding, and want ``tail=False`` if the student is masked outside them.
    """
    what = "distill_loss"
    _check_rows(logits, what)
    rows = logits.shape[0]
    if teacher_ids.dim() != 2 or teacher_ids.shape != teacher_logprobs.shape or \
            teacher_ids.shape[0] != rows or not 1 <= teacher_ids.shape[1] <= MAX_TEACHER_K:
        raise ValueError(f"{what}: teacher_ids and teacher_logprobs must be [{rows}, K] with K in "
                         f"[1, {MAX_TEACHER_K}], got {list(teacher_ids.shape)} and "
                         f"{list(teacher_logprobs.shape)}")
    if teacher_ids.dtype not in (torch.int32, torch.int64) or \
            teacher_logprobs.dtype != torch.float32:
        raise ValueError(f"{what}: teacher_ids must be int32 or int64 and teacher_logprobs fp32, "
                         f"got {teacher_ids.dtype} and {teacher_logprobs.dtype}")
    if teacher_logprobs.requires_grad or weights is not None and weights.requires_grad:
        raise ValueError(f"{what}: the teacher's values and the weights are constants (detach them)")
    if weights is not None and (tuple(weights.shape) != (rows,) or weights.dtype != torch.float32):
        raise ValueError(f"{what}: weights must be fp32 [{rows}], got {list(weights.shape)} "
                         f"{weights.dtype}")
    if reduction not in ("none", "sum", "mean"):
        raise ValueError(f"{what}: reduction must be none, sum or mean, got {reduction!r}")
    t = _check_temperature(temperature, what)
    scale = 1.0 / max(rows, 1) if reduction == "mean" else 1.0
    if not logits.is_cuda:
        r = distill_rows_ref(logits, teacher_ids, teacher_logprobs, weights, t, tail)
        return r if reduction == "none" else r.sum() * scale
    _ext.require()
    # an id that does not fit 32 bits is outside every vocabulary
    ids = teacher_ids if teacher_ids.dtype == torch.int32 else \
        teacher_ids.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    ids, lp = ids.contiguous(), teacher_logprobs.contiguous()
    w = None if weights is None else weights.contiguous()
    train = logits.requires_grad and torch.is_grad_enabled()
    if train:
        _count_backward()
    launch_count.add(1 if reduction == "none" else 2)
    if reduction == "none":
        if train:
            return torch.ops._b200_C.distill_rows_train(logits, ids, lp, w, t, tail)
        return torch.ops._b200_C.distill_loss(logits, ids, lp, w, t, tail, 1.0, False, False)[0]
    if train:
        return torch.ops._b200_C.distill_scalar_train(logits, ids, lp, w, t, tail, scale)
    return torch.ops._b200_C.distill_loss(logits, ids, lp, w, t, tail, scale, True, False)[3]
