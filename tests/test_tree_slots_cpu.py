"""Tree attention on the CPU: rows that belong to no tree."""
import torch

from vllm_sm70_b200 import ops
from vllm_sm70_b200.ops.attention import build_paged_kv


def test_rows_of_no_tree_are_left_as_they_are():
    g = torch.Generator().manual_seed(0)
    k = [torch.randn(n, 2, 64, generator=g) for n in (20, 7)]
    kc, vc, bt, sl = build_paged_kv(k, [t + 1 for t in k], 16, generator=g)
    cu = torch.tensor([1, 4, 6], dtype=torch.int32)
    q = torch.randn(9, 4, 64, generator=g)
    m = ops.tree_mask(torch.tensor([-1, -1, 0, 1, -1, 0, -1, -1, -1]), cu, 1)
    out = torch.full_like(q, 7.0)
    ops.tree_attention(out, q, kc, vc, bt, sl, cu, m, 0.125)
    assert bool((out[[0, 6, 7, 8]] == 7).all()) and not bool((out[1:6] == 7).any())
    exact = ops.tree_attention(torch.empty_like(q[1:6]), q[1:6], kc, vc, bt, sl, cu - 1, m[1:6],
                               0.125)
    assert torch.equal(out[1:6], exact)


def test_lengths_beyond_the_tensors():
    g = torch.Generator().manual_seed(0)
    k = [torch.randn(32, 2, 64, generator=g)]
    kc, vc, bt, sl = build_paged_kv(k, k, 16, generator=g)
    q, cu = torch.randn(3, 4, 64, generator=g), torch.tensor([0, 3], dtype=torch.int32)
    m = ops.tree_mask(torch.tensor([-1, 0, 0]), cu)
    want = ops.tree_attention(torch.empty_like(q), q, kc, vc, bt, sl, cu, m, 0.125)
    for lens, c in ((40, [0, 3]), (2 ** 31 - 1, [0, 3]), (32, [-4, 3]), (32, [0, 9])):
        got = ops.tree_attention(torch.empty_like(q), q, kc, vc, bt,
                                 torch.tensor([lens], dtype=torch.int32),
                                 torch.tensor(c, dtype=torch.int32), m, 0.125)
        assert torch.equal(got, want)
