"""Tree attention's oracle and masks on CPU, and the refusals."""
import pytest
import torch

from vllm_sm70_b200 import ops
from vllm_sm70_b200.ops.attention import build_paged_kv, paged_attention_ref


def test_mask_of_parents():
    parents = torch.tensor([-1, 0, 0, 1, 3, -1, 5, -1, 0, 1, 7])
    cu = torch.tensor([0, 7, 7, 11], dtype=torch.int32)
    m = ops.tree_mask(parents, cu)
    # the last tree's node 3 names a parent that is not before it: a root
    want = [1, 0b11, 0b101, 0b1011, 0b11011, 1 << 5, 0b1100000, 1, 0b11, 0b111, 1 << 3]
    assert m.dtype == torch.int32 and m[:, 0].tolist() == want


def test_mask_wide_and_deep():
    n = 70
    m = ops.tree_mask(torch.arange(n) - 1, torch.tensor([0, n]))
    assert m.shape == (n, 3)
    for j in (0, 31, 32, 63, 69):
        full = (1 << (j + 1)) - 1
        got = sum((int(w) & 0xFFFFFFFF) << (32 * i) for i, w in enumerate(m[j]))
        assert got == full
    assert ops.tree_mask(torch.empty(0, dtype=torch.int64), torch.tensor([0]), 2).shape == (0, 2)


def _setup(lens, nodes, hq=6, hkv=2, d=64, bs=16, seed=0):
    g = torch.Generator().manual_seed(seed)
    k = [torch.randn(n, hkv, d, generator=g) for n in lens]
    v = [torch.randn(n, hkv, d, generator=g) for n in lens]
    kc, vc, bt, sl = build_paged_kv(k, v, bs, generator=g)
    cu = torch.tensor([0] + list(torch.tensor(nodes).cumsum(0)), dtype=torch.int32)
    q = torch.randn(int(cu[-1]), hq, d, generator=g)
    return q, kc, vc, bt, sl, cu


@pytest.mark.parametrize("window", [0, 64])
def test_chain_is_causal_attention(window):
    q, kc, vc, bt, sl, cu = _setup([40, 150, 5], [4, 1, 5])
    m = ops.tree_mask(torch.cat([torch.arange(n) - 1 for n in (4, 1, 5)]), cu, 2)
    sinks = torch.randn(6)
    got = ops.tree_attention(torch.empty_like(q), q, kc, vc, bt, sl, cu, m, 0.125, window, sinks)
    want = paged_attention_ref(q, kc, vc, bt, sl, cu, 0.125, window, sinks)
    assert torch.allclose(got, want, atol=1e-5)


def test_siblings_do_not_see_each_other():
    q, kc, vc, bt, sl, cu = _setup([20], [3])
    m = ops.tree_mask(torch.tensor([-1, 0, 0]), cu)
    full = ops.tree_attention(torch.empty_like(q), q, kc, vc, bt, sl, cu, m, 0.125)
    # the third node alone, with the second one's cache entry gone
    blk = int(bt[0, 1])
    kc[blk, :, 18 - 16] = 99.0
    vc[blk, :, 18 - 16] = 99.0
    again = ops.tree_attention(torch.empty_like(q), q, kc, vc, bt, sl, cu, m, 0.125)
    assert torch.equal(full[[0, 2]], again[[0, 2]]) and not torch.equal(full[1], again[1])


def test_nothing_visible_is_zero():
    q, kc, vc, bt, sl, cu = _setup([2, 0], [2, 1])
    m = torch.tensor([[0], [0b10], [1]], dtype=torch.int32)
    o = ops.tree_attention(torch.empty_like(q), q, kc, vc, bt, sl, cu, m, 0.125)
    assert bool((o[0] == 0).all()) and bool((o[2] == 0).all()) and bool((o[1] != 0).any())


def test_refusals():
    q, kc, vc, bt, sl, cu = _setup([20], [3])
    m = ops.tree_mask(torch.tensor([-1, 0, 0]), cu)
    o = torch.empty_like(q)
    for bad in (dict(window=-1), dict(window=31), dict(scale=0.0), dict(scale=float("nan")),
                dict(mask=m[:2]), dict(mask=m[:, 0]), dict(q=q[0]), dict(out=o[:2])):
        a = dict(out=o, q=q, k_cache=kc, v_cache=vc, block_table=bt, seq_lens=sl, cu_q=cu, mask=m,
                 scale=0.125)
        a.update(bad)
        with pytest.raises(ValueError):
            ops.tree_attention(**a)
    with pytest.raises(ValueError):
        ops.tree_mask(torch.zeros(2, 2, dtype=torch.int64), cu)
