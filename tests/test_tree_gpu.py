"""GPU: tree attention against the 64-bit oracle.

Tolerance: P is rounded to bf16 (8 significant bits: relative 2^-8 a term) and
so is the output, so |error| <= 2^-8 (sum p |v| + |o|); the exponentials (2^-22), their
exponents (a score of size s log2(e) carries s 2^-24; |s| < 64 here) and the
fp32 sums stay below 2^-12 of sum p |v| more.
"""
import math

import pytest
import torch

from vllm_sm70_b200 import ops
from vllm_sm70_b200.ops.attention import build_paged_kv
from vllm_sm70_b200.ops.tree import tree_attention_ref

pytestmark = pytest.mark.gpu


def _setup(lens, nodes, heads, bs, seed=0, words=None, extra_blocks=3):
    hq, hkv, d = heads
    g = torch.Generator(device="cuda").manual_seed(seed)
    gc = torch.Generator().manual_seed(seed)

    def rnd(*s):
        return torch.randn(*s, device="cuda", generator=g).bfloat16()

    k, v = [rnd(n, hkv, d) for n in lens], [rnd(n, hkv, d) for n in lens]
    total = sum(max(1, -(-n // bs)) for n in lens)
    kc, vc, bt, sl = build_paged_kv(k, v, bs, num_blocks=total + extra_blocks, generator=gc)
    cu = torch.tensor([0] + list(torch.tensor(nodes).cumsum(0)), dtype=torch.int32, device="cuda")
    T = int(cu[-1])
    parents = torch.cat([(torch.rand(n, generator=gc) * torch.arange(n)).long() - (torch.arange(n) == 0).long()
                         for n in nodes]) if T else torch.empty(0, dtype=torch.int64)
    m = ops.tree_mask(parents.cuda(), cu, words)
    return rnd(T, hq, d), kc, vc, bt, sl, cu, m


def _check(q, kc, vc, bt, sl, cu, m, window=0, sinks=None, scale=None, out=None, workspace=None):
    scale = scale or 1 / math.sqrt(q.shape[2])
    out = torch.full_like(q, float("nan")) if out is None else out
    ops.tree_attention(out, q, kc, vc, bt, sl, cu, m, scale, window, sinks, workspace)
    d = torch.float64
    want = tree_attention_ref(q, kc, vc, bt, sl, cu, m, scale, window, sinks, d)
    size = tree_attention_ref(q, kc, vc.abs(), bt, sl, cu, m, scale, window, sinks, d)
    err = (out.double() - want).abs()
    lim = 2.0 ** -8 * (size + want.abs()) + 2.0 ** -12 * size + 1e-30
    bad = ~(err <= lim)
    assert not bool(bad.any()), (int(bad.sum()), float(err[bad].max()), bad.nonzero()[:4].tolist())
    return out


HEADS = [(32, 8, 128), (16, 2, 256), (6, 6, 64), (21, 3, 128), (24, 8, 64), (40, 1, 128)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens,nodes", [
    ([1], [1]), ([1000], [8]), ([17, 300, 64, 129, 5], [1, 7, 33, 2, 5]),
    ([2048, 31, 700], [64, 16, 3]), ([64], [64]), ([5000], [1])])
def test_shapes(b200_ops, heads, lens, nodes):
    _check(*_setup(lens, nodes, heads, 16))


@pytest.mark.parametrize("bs", [8, 32, 64, 128, 256])
@pytest.mark.parametrize("heads", [(32, 8, 128), (16, 2, 256), (24, 8, 64)])
def test_block_sizes(b200_ops, heads, bs):
    _check(*_setup([1027, 130, 9, 256], [12, 1, 9, 20], heads, bs, seed=bs))


@pytest.mark.parametrize("heads", [(32, 8, 128), (16, 2, 256), (24, 8, 64)])
@pytest.mark.parametrize("window", [32, 100, 1000])
def test_window_and_sinks(b200_ops, heads, window):
    a = _setup([2000, 333, 31, 64, 1030], [20, 32, 31, 1, 3], heads, 16, seed=window)
    _check(*a, window=window)
    _check(*a, window=window, sinks=torch.randn(heads[0], device="cuda") * 3)
    _check(*a, sinks=torch.full((heads[0],), -1e30, device="cuda"))


@pytest.mark.parametrize("heads", [(16, 2, 128), (16, 2, 256)])
def test_window_starts_row_by_row(b200_ops, heads):
    """Long windowed contexts, several units a share: a window starts inside a
    tile, at another key for each depth, so that the exponent reference of
    some rows rises in a unit's second tile."""
    lens = [8000 - 217 * i for i in range(16)]
    nodes = [24 - i for i in range(16)]
    _check(*_setup(lens, nodes, heads, 32), window=4096)


def test_window_hides_stale_blocks(b200_ops):
    """Cache entries before every node's window may have been given away: what
    they hold (NaN here) does not reach the output."""
    q, kc, vc, bt, sl, cu, m = _setup([700, 555], [9, 4], (32, 8, 128), 16)
    for s, (n, w) in enumerate(((700, 9), (555, 4))):
        first = n - w - 64 + 1
        for b in range(first // 16):
            kc[bt[s, b].long()] = float("nan")
            vc[bt[s, b].long()] = float("nan")
        blk = int(bt[s, first // 16])
        kc[blk, :, : first % 16] = float("nan")
        vc[blk, :, : first % 16] = float("nan")
    kz, vz = kc.nan_to_num(0.0), vc.nan_to_num(0.0)
    a = ops.tree_attention(torch.empty_like(q), q, kc, vc, bt, sl, cu, m, 0.09, 64)
    b = ops.tree_attention(torch.empty_like(q), q, kz, vz, bt, sl, cu, m, 0.09, 64)
    assert torch.equal(a, b) and not bool(torch.isnan(a).any())


def test_wide_trees(b200_ops):
    _check(*_setup([900, 257, 200], [200, 256, 129], (32, 8, 128), 16))
    _check(*_setup([300, 131], [100, 131], (16, 2, 256), 16))


@pytest.mark.parametrize("heads", [(32, 8, 128), (16, 2, 256), (8, 2, 64)])
@pytest.mark.parametrize("lens,nodes", [
    ([5000, 300, 64], [64, 64, 64]),        # two tiles of rows at 4 heads a key head
    ([9000], [96]), ([4000, 700], [128, 64]), ([900, 5, 3000], [64, 0, 128]),
    ([1500] * 9, [256] * 9), ([2000, 2100], [300, 290])])
def test_row_tiles_over_the_same_keys(b200_ops, heads, lens, nodes):
    _check(*_setup(lens, nodes, heads, 16, seed=len(lens)))


def test_ragged_batch_and_long_context(b200_ops):
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(1, 900, (300,), generator=g).tolist()
    nodes = [min(n, int(k)) for n, k in zip(lens, torch.randint(1, 9, (300,), generator=g))]
    _check(*_setup(lens, nodes, (8, 2, 128), 16))
    _check(*_setup([100003, 40], [5, 40], (8, 2, 128), 64))
    _check(*_setup([30001], [64], (16, 2, 256), 16))


@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128), (16, 2, 256)])
def test_many_short_sequences(b200_ops, heads):
    """Units of a few tiles, whose edges fall anywhere in a share."""
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(1, 400, (450,), generator=g).tolist()
    nodes = [min(n, int(k)) for n, k in zip(lens, torch.randint(1, 7, (450,), generator=g))]
    _check(*_setup(lens, nodes, heads, 16))
    _check(*_setup([130] * 160, [4] * 160, heads, 16))


def test_sequences_without_nodes_or_keys(b200_ops):
    q, kc, vc, bt, sl, cu, m = _setup([50, 60, 70, 300], [3, 0, 0, 2], (32, 8, 128), 16)
    _check(q, kc, vc, bt, sl, cu, m)
    sl = sl.clone()
    sl[0] = 0       # no key at all: zeros
    sl[3] = 1       # fewer keys than nodes: the second node's own is not there
    out = _check(q, kc, vc, bt, sl, cu, m)
    assert bool((out[:3] == 0).all())


def test_arbitrary_masks(b200_ops):
    q, kc, vc, bt, sl, cu, m = _setup([40, 500, 24], [24, 40, 24], (32, 8, 128), 16, words=3)
    g = torch.Generator(device="cuda").manual_seed(1)
    m = torch.randint(-2 ** 31, 2 ** 31 - 1, m.shape, device="cuda", generator=g,
                      dtype=torch.int64).to(torch.int32)
    m[66:] = 0      # nothing of the tree; the last sequence has no prefix either
    out = _check(q, kc, vc, bt, sl, cu, m)
    assert bool((out[66:] == 0).all())


def test_large_scores(b200_ops):
    """Running maxima that rise by more than 2^8 on the way: O is rescaled."""
    q, kc, vc, bt, sl, cu, m = _setup([3000, 1500], [20, 64], (32, 8, 128), 16)
    for s in range(2):
        for b in range(0, int(sl[s]) // 16):
            kc[bt[s, b].long()] *= 0.25 + 2.0 * b / 188
    _check(q, kc, vc, bt, sl, cu, m)


def test_strides_workspace_stream(b200_ops):
    _, kc, vc, bt, sl, cu, m = _setup([700, 90], [9, 5], (32, 8, 128), 16)
    qkv = torch.randn(14, 48, 128, device="cuda").bfloat16()
    q = qkv[:, :32]
    ws = ops.tree_attention_workspace(128, "cuda")
    a = _check(q, kc, vc, bt, sl, cu, m, workspace=ws)
    buf = torch.zeros(14, 40, 128, device="cuda", dtype=torch.bfloat16)
    b = _check(q, kc, vc, bt, sl, cu, m, out=buf[:, 4:36], workspace=ws)
    assert torch.equal(a, b) and bool((buf[:, :4] == 0).all()) and bool((buf[:, 36:] == 0).all())
    odd = torch.randn(14, 32 * 128 + 3, device="cuda").bfloat16()[:, 3:].view(14, 32, 128)
    _check(odd, kc, vc, bt, sl, cu, m)
    # K and V interleaved in one allocation
    both = torch.stack([kc, vc], 1)
    c = _check(q, both[:, 0], both[:, 1], bt, sl, cu, m)
    assert torch.equal(a, c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        d = ops.tree_attention(torch.empty_like(q), q, kc, vc, bt, sl, cu, m, 128 ** -0.5)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a, d)


def test_graph_replays_with_new_lengths(b200_ops):
    q, kc, vc, bt, sl, cu, m = _setup([900, 500], [6, 6], (32, 8, 128), 16)
    ws = ops.tree_attention_workspace(128, "cuda")
    out, lens = torch.empty_like(q), sl.clone()
    ops.tree_attention(out, q, kc, vc, bt, lens, cu, m, 0.09, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.tree_attention(out, q, kc, vc, bt, lens, cu, m, 0.09, workspace=ws)
    for new in ([900, 500], [300, 37], [6, 499]):
        lens.copy_(torch.tensor(new))
        g.replay()
        want = ops.tree_attention(torch.empty_like(q), q, kc, vc, bt, lens.clone(), cu, m, 0.09)
        assert torch.equal(out, want)


def test_chain_agrees_with_paged_attention(b200_ops):
    q, kc, vc, bt, sl, cu, _ = _setup([800, 77], [5, 3], (32, 8, 128), 16)
    m = ops.tree_mask(torch.tensor([-1, 0, 1, 2, 3, -1, 0, 1], device="cuda"), cu)
    a = ops.tree_attention(torch.empty_like(q), q, kc, vc, bt, sl, cu, m, 0.09)
    b = ops.paged_attention(torch.empty_like(q), q, kc, vc, bt, sl, cu, 5, 0.09, decode=True)
    # both round P and the output to bf16: 2^-8 each of sum p |v| and |o|
    assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -8 * 4 * float(
        vc.nan_to_num(0.0).abs().max())


def test_refusals_cuda(b200_ops):
    q, kc, vc, bt, sl, cu, m = _setup([40], [3], (32, 8, 128), 16)
    o = torch.empty_like(q)
    ok = dict(out=o, q=q, k_cache=kc, v_cache=vc, block_table=bt, seq_lens=sl, cu_q=cu, mask=m,
              scale=0.1)
    for bad in (dict(q=q.half()), dict(k_cache=kc[:, :3]), dict(v_cache=vc[:-1]),
                dict(k_cache=kc[:, :, ::2], v_cache=vc[:, :, ::2]), dict(mask=m.long()),
                dict(block_table=bt.long()), dict(cu_q=cu[:1]), dict(seq_lens=sl.cpu()),
                dict(sinks=torch.zeros(8, device="cuda")),
                dict(workspace=torch.empty(16, dtype=torch.uint8, device="cuda")),
                dict(out=o.float()), dict(out=torch.empty(3, 32, 130, device="cuda",
                                                          dtype=torch.bfloat16)[:, :, :128])):
        with pytest.raises(RuntimeError):
            ops.tree_attention(**{**ok, **bad})
