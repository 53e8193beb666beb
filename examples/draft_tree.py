"""Draft a tree, verify it in one step, train the draft heads on the way.

A small random one-layer target decodes greedily. Two draft heads guess the
next two tokens after the newest one from its hidden state; their best guesses form a tree
per sequence, which the target verifies in one step:

* ``ops.tree_mask`` / ``ops.tree_attention``: every node attends to the
  sequence's paged cache and to its own ancestors;
* ``ops.token_logprobs``: the target's rank of every drafted token (1: it is
  accepted) and its top alternatives at the accepted nodes;
* ``ops.distill_loss``: the draft heads learn from those alternatives.

    python examples/draft_tree.py                  # CUDA where there is a GPU
    python examples/draft_tree.py --device cpu --rounds 8

The mean number of tokens a step grows from 1 as the heads learn.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from vllm_sm70_b200 import ops  # noqa: E402

BRANCH = (3, 2)  # guesses of head 1, and of head 2 under each of them
HEADS, KV_HEADS, DIM, BLOCK = 4, 2, 64, 16
NODES = 1 + BRANCH[0] + BRANCH[0] * BRANCH[1]
PARENTS = [-1] + [0] * BRANCH[0] + [1 + i for i in range(BRANCH[0]) for _ in range(BRANCH[1])]
TOP = 16  # the target's alternatives that the heads learn from


class Target:
    """Embedding, one attention layer over a paged cache, output projection."""

    def __init__(self, vocab: int, batch: int, max_len: int, device, seed: int = 0):
        g = torch.Generator().manual_seed(seed)
        hidden = HEADS * DIM
        dtype = torch.bfloat16 if torch.device(device).type == "cuda" else torch.float32

        def weight(*shape):
            return (torch.randn(*shape, generator=g) / shape[0] ** 0.5).to(device, dtype)

        self.embed = weight(vocab, hidden) * vocab ** 0.5
        self.qkv = weight(hidden, (HEADS + 2 * KV_HEADS) * DIM)
        self.out = weight(hidden, hidden)
        self.head = weight(hidden, vocab) * 2
        blocks = -(-max_len // BLOCK)
        self.k = torch.zeros(batch * blocks, KV_HEADS, BLOCK, DIM, device=device, dtype=dtype)
        self.v = torch.zeros_like(self.k)
        # sequences share the pool, their blocks in no order
        order = torch.randperm(batch * blocks, generator=g).to(device, torch.int32)
        self.table = order.view(batch, blocks)

    def _slots(self, seq, pos):
        """(block, offset) of positions ``pos`` of sequences ``seq``."""
        return self.table[seq, pos // BLOCK].long(), pos % BLOCK

    def step(self, tokens, seq, pos, cu, mask, lens):
        """Hidden states and logits of the nodes; their keys and values go to
        the slots ``pos`` of their sequences."""
        x = self.embed[tokens]
        y = x @ self.qkv
        q, k, v = y.split([HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM], 1)
        b, o = self._slots(seq, pos)
        self.k[b, :, o] = k.reshape(-1, KV_HEADS, DIM)
        self.v[b, :, o] = v.reshape(-1, KV_HEADS, DIM)
        q = q.unflatten(1, (HEADS, DIM))
        att = torch.empty(q.shape, device=q.device, dtype=q.dtype)
        ops.tree_attention(att, q, self.k, self.v, self.table, lens, cu, mask, DIM ** -0.5)
        h = x + att.flatten(1) @ self.out
        return h, h @ self.head

    def move(self, seq, src, dst):
        """Keys and values of accepted nodes to their places in the sequence."""
        (b0, o0), (b1, o1) = self._slots(seq, src), self._slots(seq, dst)
        self.k[b1, :, o1], self.v[b1, :, o1] = self.k[b0, :, o0], self.v[b0, :, o0]


def run(device="cpu", vocab=211, batch=4, rounds=20, lr=1.0, seed=0):
    """(tokens a step of each round, loss of each round, the sequences)."""
    target = Target(vocab, batch, (len(BRANCH) + 1) * rounds + NODES, device, seed)
    heads = [torch.zeros(HEADS * DIM, vocab, device=device, requires_grad=True)
             for _ in BRANCH]
    idx = {"device": device, "dtype": torch.int32}
    cu = torch.arange(0, batch * NODES + 1, NODES, **idx)
    parents = torch.tensor(PARENTS * batch, **idx)
    mask = ops.tree_mask(parents, cu)
    seq = torch.arange(batch, device=device).repeat_interleave(NODES)
    drafted = parents >= 0
    up = (seq * NODES + parents)[drafted]  # rows of the drafted nodes' parents

    newest = [s % vocab for s in range(batch)]
    hidden = torch.zeros(batch, HEADS * DIM, device=device, dtype=target.embed.dtype)
    length = [0] * batch
    texts = [[t] for t in newest]
    speed, losses = [], []
    for _ in range(rounds):
        # The tree: the newest token, head 1's guesses, head 2's under each.
        with torch.no_grad():
            guess = [(hidden.float() @ w).topk(n, 1).indices for w, n in zip(heads, BRANCH)]
        tokens = torch.cat([torch.tensor(newest, device=device)[:, None], guess[0],
                            guess[1].repeat(1, BRANCH[0])], 1).flatten()
        start = torch.tensor(length, device=device)
        pos = (start[:, None] + torch.arange(NODES, device=device)).flatten()
        h, logits = target.step(tokens, seq, pos, cu, mask, (start + NODES).to(torch.int32))

        # A drafted token is what the target would have chosen if it ranks
        # first after its parent. Where does each path of such tokens end?
        first = torch.zeros_like(drafted)
        first[drafted] = ops.token_logprobs(logits[up], tokens[drafted]).ranks == 1
        choice = ops.token_logprobs(logits, tokens, top_n=1).top_ids[:, 0].tolist()
        first = first.tolist()
        paths, made = [], 0
        for s in range(batch):
            path = [0]
            while True:
                nxt = [j for j in range(1, NODES)
                       if PARENTS[j] == path[-1] and first[s * NODES + j]]
                if not nxt:
                    break
                path.append(nxt[0])
            paths.append([s * NODES + j for j in path])
            texts[s] += [int(tokens[r]) for r in paths[s][1:]] + [choice[paths[s][-1]]]
            newest[s] = choice[paths[s][-1]]
            at = torch.tensor(path, device=device)
            target.move(torch.full_like(at, s), length[s] + at,
                        length[s] + torch.arange(len(path), device=device))
            length[s] += len(path)
            made += len(path)
        speed.append(made / batch)

        # Head d learns at every state what the target says d + 1 nodes on;
        # the state before a path's root is that of the step before.
        rows = [r for p in paths for r in p]
        teacher = ops.token_logprobs(logits[rows], tokens[rows], top_n=TOP)
        where = {r: i for i, r in enumerate(rows)}
        states = torch.cat([h, hidden])
        total = 0.0
        for d, w in enumerate(heads):
            pairs = [(([len(h) + s] + p)[i], where[p[i + d]])
                     for s, p in enumerate(paths) for i in range(len(p) - d)]
            if not pairs:
                continue
            src, to = [a for a, _ in pairs], [b for _, b in pairs]
            loss = ops.distill_loss(states[src].float() @ w, teacher.top_ids[to],
                                    teacher.top_logprobs[to], reduction="sum")
            loss.backward()
            with torch.no_grad():
                w -= lr / w.shape[0] * w.grad
            w.grad = None
            total += loss.item() / len(pairs)
        losses.append(total)
        hidden = h[[p[-1] for p in paths]]
    return speed, losses, texts


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    ap.add_argument("--vocab", type=int, default=211)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--rounds", type=int, default=40)
    a = ap.parse_args(argv)
    speed, losses, _ = run(a.device, a.vocab, a.batch, a.rounds)
    for i in range(0, a.rounds, max(1, a.rounds // 8)):
        print(f"round {i:3d}: {speed[i]:.2f} tokens a step, loss {losses[i]:.3f}")
    n = max(1, a.rounds // 4)
    print(f"first {n} rounds: {sum(speed[:n]) / n:.2f} tokens a step, "
          f"last {n}: {sum(speed[-n:]) / n:.2f}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
