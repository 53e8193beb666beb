"""Attention of a tree of drafted tokens over the paged cache, and the masks
of such trees.

Speculative decoding verifies several drafts at once: the drafted tokens form
a tree under the last accepted token, the target runs over all nodes in one
step, and each node attends to the context and to its own ancestors. The
nodes' keys and values sit in the last ``q_len`` slots of their sequence's
cache (written by :func:`~vllm_sm70_b200.ops.rope_kv_write` with positions
``prefix + depth``), so the cache layout and the block table are those of
:func:`~vllm_sm70_b200.ops.paged_attention`.

Reference parity: the reference verifies a chain of drafts
(``sm70/csrc/flash_v100/verify_decode.cu:133-368``); a chain is the tree whose
node j has the parent j - 1.
"""
from __future__ import annotations

import torch

from .. import _ext
from ..utils import launch_count
from .attention import gather_paged


def tree_mask(parents: torch.Tensor, cu_q: torch.Tensor, words: int | None = None) -> torch.Tensor:
    """Ancestor masks ``[T, words]`` int32 of trees given by their parents.

    ``parents [T]`` (int): the index of a node's parent within its own tree,
    smaller than the node's own (anything else: a root); ``cu_q [B + 1]``: the trees'
    bounds. Bit ``i % 32`` of word ``i // 32`` of a node's row is set for the
    node itself and its ancestors. ``words``: row width (default: the widest
    tree's need; the default reads ``cu_q`` on the host)."""
    if parents.dim() != 1 or cu_q.dim() != 1 or cu_q.numel() < 1:
        raise ValueError("tree_mask: parents [T] and cu_q [B + 1]")
    T, dev = parents.numel(), parents.device
    if words is None:
        widest = int((cu_q[1:] - cu_q[:-1]).max()) if cu_q.numel() > 1 else 1
        words = max(1, -(-widest // 32))
    tok = torch.arange(T, device=dev)
    seq = torch.searchsorted(cu_q.to(torch.int64), tok, right=True) - 1
    start = cu_q.to(torch.int64)[seq.clamp(min=0)]
    node = tok - start
    rows = torch.arange(words * 32, device=dev) == node[:, None]
    up = parents.to(torch.int64)
    jump = torch.where((up >= 0) & (up < node), start + up, torch.full_like(up, -1))
    for _ in range((words * 32 - 1).bit_length()):  # 1, 2, 4, ... ancestors
        on = jump >= 0
        to = jump.clamp(min=0)
        rows = rows | (on[:, None] & rows[to])
        jump = torch.where(on, jump[to], jump)
    bit = torch.ones(32, dtype=torch.int64, device=dev) << torch.arange(32, device=dev)
    w = (rows.view(T, words, 32).to(torch.int64) * bit).sum(2)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def tree_attention_ref(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       block_table: torch.Tensor, seq_lens: torch.Tensor, cu_q: torch.Tensor,
                       mask: torch.Tensor, scale: float, window: int = 0,
                       sinks: torch.Tensor | None = None, dtype=torch.float32) -> torch.Tensor:
    """Oracle of :func:`tree_attention` (``[T, Hq, D]`` in ``dtype``)."""
    T, hq, d = q.shape
    hkv = k_cache.shape[1]
    out = torch.zeros(T, hq, d, dtype=dtype, device=q.device)
    bits = ((mask.to(torch.int64)[:, :, None] >> torch.arange(32, device=q.device)) & 1).bool()
    bits = bits.reshape(T, -1)
    for s in range(seq_lens.numel()):
        a, b = max(0, int(cu_q[s])), min(int(cu_q[s + 1]), T)
        L = max(0, min(int(seq_lens[s]), block_table.shape[1] * k_cache.shape[2]))
        if b <= a or L == 0:
            continue
        n = min(b - a, L)  # nodes whose keys exist
        k = gather_paged(k_cache, block_table[s], L).to(dtype)  # [L, Hkv, D]
        v = gather_paged(v_cache, block_table[s], L).to(dtype)
        seen = torch.zeros(b - a, L, dtype=torch.bool, device=q.device)
        seen[:, : L - n] = True
        m = min(n, bits.shape[1])
        tree = bits[a:b, :m]
        if window > 0:
            pos = L - n + tree.sum(1).clamp(min=1) - 1
            seen &= torch.arange(L, device=q.device) > (pos - window)[:, None]
        seen[:, L - n: L - n + m] = tree
        k = k.repeat_interleave(hq // hkv, 1)
        # keys that no node sees may hold anything
        some = seen.any(0)
        v = torch.where(some[:, None, None], v, torch.zeros_like(v)).repeat_interleave(hq // hkv, 1)
        sc = torch.einsum("nhd,lhd->nhl", q[a:b].to(dtype), k) * scale
        sc = torch.where(seen[:, None], sc, torch.full_like(sc, float("-inf")))
        mx = sc.amax(2, keepdim=True)
        if sinks is not None:
            mx = torch.maximum(mx, sinks.to(dtype)[None, :, None])
        mx = torch.where(mx == float("-inf"), torch.zeros_like(mx), mx)
        p = torch.exp(sc - mx)
        den = p.sum(2, keepdim=True)
        if sinks is not None:
            den = den + torch.exp(sinks.to(dtype)[None, :, None] - mx)
        p = p / torch.where(den == 0, torch.ones_like(den), den)
        out[a:b] = torch.einsum("nhl,lhd->nhd", p, v)
    return out


def tree_attention_workspace(head_dim: int, device) -> torch.Tensor:
    """A workspace for :func:`tree_attention` calls on ``device`` (kept by a
    caller that captures graphs; calls that may overlap on different streams
    need one each)."""
    _ext.require()
    dev = torch.device(device)
    index = dev.index if dev.index is not None else torch.cuda.current_device()
    n = torch.ops._b200_C.tree_attention_workspace(head_dim, index)
    return torch.empty(n, dtype=torch.uint8, device=dev)


def tree_attention(out: torch.Tensor, q: torch.Tensor, k_cache: torch.Tensor,
                   v_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                   cu_q: torch.Tensor, mask: torch.Tensor, scale: float, window: int = 0,
                   sinks: torch.Tensor | None = None,
                   workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``out [T, Hq, D]`` <- attention of tree nodes ``q [T, Hq, D]`` over the
    paged cache (``q`` may be a strided view into the QKV projection).

    Sequence s has the nodes ``cu_q[s] .. cu_q[s + 1]``; their keys are the
    last of its ``seq_lens[s]`` cache entries. A node sees every key of the
    prefix and the nodes set in its row of ``mask [T, words]`` (int32 bits, see
    :func:`tree_mask`; its own bit included, or it does not see itself). A
    node that sees nothing (no prefix, no bits) gets 0. ``window > 0`` limits
    the prefix to the positions ``> prefix + depth - window`` (depth: the bits
    of the row minus one); it has to hold the whole tree (``32 * words``).
    ``sinks [Hq]`` join the denominators. Weights are rounded to bf16 before
    they meet V, as in :func:`~vllm_sm70_b200.ops.paged_attention`; scores and
    sums are fp32. Cache entries that no node sees may
    hold anything, NaN too: those from ``seq_lens[s]`` on, before the window of
    a node of depth 0, and the slots of nodes whose bit no row sets. What one
    node sees has to be finite for the others too. Head sizes 64, 128 and 256, any
    number of query heads a key head, block sizes of a power of two from 8.
    Lengths are read on the device (keys beyond the block table and nodes
    beyond ``T`` do not exist): a captured graph replays with new ones,
    and with fewer nodes than ``T`` (rows of ``out`` that belong to no tree,
    from ``cu_q[B]`` on, are left as they are).
    """
    if q.dim() != 3 or out.shape != q.shape or mask.dim() != 2 or mask.shape[0] != q.shape[0]:
        raise ValueError(f"tree_attention: out and q [T, Hq, D] and mask [T, words], got "
                         f"{list(out.shape)}, {list(q.shape)}, {list(mask.shape)}")
    if window < 0 or 0 < window < 32 * mask.shape[1]:
        raise ValueError("tree_attention: a sliding window must be 0 (none) or hold the whole "
                         f"tree ({32 * mask.shape[1]}), got {window}")
    if not scale > 0:
        raise ValueError(f"tree_attention: scale must be positive, got {scale}")
    if q.is_cuda:
        _ext.require()
        if q.stride(2) != 1 or q.shape[1] > 1 and q.stride(1) != q.shape[2] or \
                q.stride(0) % 8 or q.data_ptr() % 16:
            q = q.contiguous()
        torch.ops._b200_C.tree_attention(out, q, k_cache, v_cache, block_table, seq_lens, cu_q,
                                         mask, scale, window, sinks, workspace)
        launch_count.add(2)
        return out
    r = tree_attention_ref(q, k_cache, v_cache, block_table, seq_lens, cu_q, mask, scale, window,
                           sinks)
    first, last = max(0, int(cu_q[0])), min(int(cu_q[-1]), q.shape[0])
    out[first:last] = r[first:last].to(out.dtype)
    return out
