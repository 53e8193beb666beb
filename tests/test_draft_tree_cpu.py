"""CPU: the draft-tree example against decoding one token at a time."""
import importlib.util
from pathlib import Path

import torch

from vllm_sm70_b200 import ops


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "draft_tree.py"
    spec = importlib.util.spec_from_file_location("draft_tree", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _one_at_a_time(m, n, vocab, batch):
    t = m.Target(vocab, batch, n + m.NODES, "cpu")
    tokens = torch.arange(batch) % vocab
    seq, cu = torch.arange(batch), torch.arange(batch + 1, dtype=torch.int32)
    mask = ops.tree_mask(torch.full((batch,), -1), cu)
    out = [tokens.tolist()]
    for i in range(n):
        at = torch.full((batch,), i)
        _, logits = t.step(tokens, seq, at, cu, mask, (at + 1).to(torch.int32))
        tokens = logits.argmax(1)
        out.append(tokens.tolist())
    return [list(x) for x in zip(*out)]


def test_same_tokens_as_one_at_a_time():
    m = _example()
    speed, losses, texts = m.run("cpu", vocab=61, batch=3, rounds=24)
    want = _one_at_a_time(m, max(len(t) for t in texts) - 1, 61, 3)
    for got, w in zip(texts, want):
        assert got == w[:len(got)]
    assert sum(speed[-6:]) > sum(speed[:6])  # the heads learn
    assert all(x > -1e-4 for x in losses)
    assert sum(len(t) for t in texts) == 3 + round(3 * sum(speed))


def test_command(capsys):
    assert _example().main(["--device", "cpu", "--rounds", "4", "--vocab", "31"]) == 0
    assert "tokens a step" in capsys.readouterr().out
