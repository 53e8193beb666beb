"""GPU: the draft-tree example on the kernels."""
import importlib.util
import math
from pathlib import Path

import pytest

from vllm_sm70_b200.utils import launch_count

pytestmark = pytest.mark.gpu


def test_heads_learn_on_the_kernels(b200_ops):
    path = Path(__file__).resolve().parents[1] / "examples" / "draft_tree.py"
    spec = importlib.util.spec_from_file_location("draft_tree", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    before = launch_count.total()
    speed, losses, texts = m.run("cuda", vocab=211, batch=4, rounds=48)
    assert launch_count.total() - before >= 48 * 8
    assert sum(speed[-12:]) > sum(speed[:12])
    assert all(math.isfinite(x) and x > -1e-4 for x in losses)
    assert sum(len(t) for t in texts) == 4 + round(4 * sum(speed))
    assert all(0 <= x < 211 for t in texts for x in t)
