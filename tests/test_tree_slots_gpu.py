"""GPU: tree attention where slots of the cache hold nothing of use, against
the 64-bit oracle.

Tolerance: P is rounded to bf16 (relative 2^-8 a term) and so is the output:
|error| <= 2^-8 (sum p |v| + |o|), and 2^-12 of sum p |v| for the exponentials
and the fp32 sums.
"""
import math

import pytest
import torch

from vllm_sm70_b200 import ops
from vllm_sm70_b200.ops.attention import build_paged_kv
from vllm_sm70_b200.ops.tree import tree_attention_ref

pytestmark = pytest.mark.gpu
HEADS = [(32, 8, 128), (16, 2, 256), (24, 8, 64), (6, 6, 64)]


def _setup(lens, nodes, heads, bs, seed=0, words=None):
    hq, hkv, d = heads
    g = torch.Generator(device="cuda").manual_seed(seed)
    gc = torch.Generator().manual_seed(seed)

    def rnd(*s):
        return torch.randn(*s, device="cuda", generator=g).bfloat16()

    kc, vc, bt, sl = build_paged_kv([rnd(n, hkv, d) for n in lens], [rnd(n, hkv, d) for n in lens],
                                    bs, generator=gc)
    cu = torch.tensor([0] + list(torch.tensor(nodes).cumsum(0)), dtype=torch.int32, device="cuda")
    parents = torch.cat([(torch.rand(n, generator=gc) * torch.arange(n)).long()
                         - (torch.arange(n) == 0).long() for n in nodes])
    return rnd(int(cu[-1]), hq, d), kc, vc, bt, sl, cu, ops.tree_mask(parents.cuda(), cu, words)


def _check(q, kc, vc, bt, sl, cu, m, window=0, sinks=None):
    scale = 1 / math.sqrt(q.shape[2])
    out = ops.tree_attention(torch.full_like(q, float("nan")), q, kc, vc, bt, sl, cu, m, scale,
                             window, sinks)
    d = torch.float64
    want = tree_attention_ref(q, kc, vc, bt, sl, cu, m, scale, window, sinks, d)
    size = tree_attention_ref(q, kc, vc.abs(), bt, sl, cu, m, scale, window, sinks, d)
    assert not bool(torch.isnan(want).any())
    err = (out.double() - want).abs()
    bad = ~(err <= 2.0 ** -8 * (size + want.abs()) + 2.0 ** -12 * size + 1e-30)
    assert not bool(bad.any()), (int(bad.sum()), float(err[bad].max()), bad.nonzero()[:4].tolist())


def _forget(m, kc, vc, bt, lens, nodes, gone, value):
    """No row sees the nodes in gone[s] of sequence s; their slots hold value."""
    bs, at = kc.shape[2], 0
    m = m.clone()
    for s, (n, w) in enumerate(zip(lens, nodes)):
        for i in gone[s]:
            if i // 32 < m.shape[1]:
                m[at:at + w, i // 32] &= ~(1 << i % 32) if i % 32 < 31 else 2 ** 31 - 1
            pos = n - w + i
            b = int(bt[s, pos // bs])
            kc[b, :, pos % bs] = value
            vc[b, :, pos % bs] = value
        at += w
    return m


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens,nodes", [
    ([700, 90], [9, 5]), ([128, 256, 640], [8, 16, 64]),   # ends on a tile's edge
    ([1000, 330, 260], [200, 256, 129]), ([8], [8]), ([5000], [130])])
def test_slots_that_no_node_sees(b200_ops, heads, lens, nodes, value):
    q, kc, vc, bt, sl, cu, m = _setup(lens, nodes, heads, 16, seed=sum(lens))
    gone = [sorted({n - 1, n // 2, *range(3, n, 7)} - {0}) for n in nodes]
    m = _forget(m, kc, vc, bt, lens, nodes, gone, value)
    _check(q, kc, vc, bt, sl, cu, m)
    window = 32 * m.shape[1] + 40
    _check(q, kc, vc, bt, sl, cu, m, window=window, sinks=torch.randn(heads[0], device="cuda"))


@pytest.mark.parametrize("heads", HEADS)
def test_nodes_past_the_mask(b200_ops, heads):
    """More nodes than the mask's row has bits: nobody sees the rest."""
    lens, nodes = [500, 300], [70, 40]
    q, kc, vc, bt, sl, cu, m = _setup(lens, nodes, heads, 16, words=1)
    m = _forget(m, kc, vc, bt, lens, nodes, [list(range(32, 70)), list(range(32, 40))],
                float("nan"))
    _check(q, kc, vc, bt, sl, cu, m)


@pytest.mark.parametrize("heads", HEADS)
def test_a_tree_that_sees_none_of_itself(b200_ops, heads):
    """Every slot of the tree unwritten: the nodes see the prefix alone, and
    nothing where there is none."""
    lens, nodes = [300, 24, 129], [24, 24, 1]
    q, kc, vc, bt, sl, cu, m = _setup(lens, nodes, heads, 16)
    m = _forget(m, kc, vc, bt, lens, nodes, [range(24), range(24), range(1)], float("nan"))
    _check(q, kc, vc, bt, sl, cu, m)


def test_rows_of_no_tree_are_left_as_they_are(b200_ops):
    """Also where a captured graph is replayed with fewer nodes."""
    lens, nodes = [700, 90], [9, 5]
    q, kc, vc, bt, sl, cu, m = _setup(lens, nodes, (32, 8, 128), 16)
    more = torch.cat([q, q[:3]])
    mm = torch.cat([m, m[:3]])
    out = torch.full_like(more, 7.0)
    ops.tree_attention(out, more, kc, vc, bt, sl, cu, mm, 0.09)
    want = ops.tree_attention(torch.empty_like(q), q, kc, vc, bt, sl, cu, m, 0.09)
    assert bool((out[14:] == 7).all()) and torch.equal(out[:14], want)
    ws, now = ops.tree_attention_workspace(128, "cuda"), cu.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.tree_attention(out, more, kc, vc, bt, sl, now, mm, 0.09, workspace=ws)
    for n in (17, 14, 11):
        now.copy_(torch.tensor([0, 9, n]))
        out.fill_(7.0)
        graph.replay()
        want = ops.tree_attention(torch.empty_like(more[:n]), more[:n], kc, vc, bt, sl, now.clone(),
                                  mm[:n], 0.09)
        assert bool((out[n:] == 7).all()) and torch.equal(out[:n], want)


@pytest.mark.parametrize("heads", HEADS[:3])
def test_lengths_beyond_the_tensors(b200_ops, heads):
    """Keys beyond the block table and nodes beyond q do not exist."""
    lens, nodes = [160, 90], [9, 5]
    q, kc, vc, bt, sl, cu, m = _setup(lens, nodes, heads, 16)
    kc, vc = kc.nan_to_num(0.5), vc.nan_to_num(0.5)
    for n in (161, 300, 2 ** 31 - 1):
        _check(q, kc, vc, bt, torch.tensor([n, 90], dtype=torch.int32, device="cuda"), cu, m)
    _check(q, kc, vc, bt, sl, torch.tensor([-7, 9, 2 ** 31 - 1], dtype=torch.int32, device="cuda"),
           m)
