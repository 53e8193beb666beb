"""Measured cases of the draft-and-verify operators: tree attention over the
paged cache, log-probabilities of given tokens, and distillation from a
teacher's top log-probabilities.

Each pass has two forms. ``own`` False: elementary torch operations in 32
bits, rounded once at the end. ``own`` True: the calls a user makes of
``vllm_sm70_b200.ops``. ``exact`` gives the same outputs from the definitions
in 64 bits.
"""
import math

import torch

own = False

_DEV = "cuda"
_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # One interactive user: a small draft tree over a short chat, where
        # the launch and the joins cost more than the bytes.
        _tree("tree one user", batch=1, nodes=8, ctx=1000, heads=(32, 8, 128), block=16),
        # A serving batch of the 8B configuration: ragged contexts and trees.
        _tree("tree batch", batch=64, nodes=16, ctx=4096, heads=(32, 8, 128), block=16),
        # Two long documents with the widest tree a step verifies (64 nodes,
        # 256 query rows a key head).
        _tree("tree long context", batch=2, nodes=64, ctx=60001, heads=(32, 8, 128), block=16),
        # Full-attention layers with wide heads (16 query heads on 2, 256
        # wide), sinks, and a sliding window inside the context.
        _tree("tree wide heads", batch=16, nodes=24, ctx=8000, heads=(16, 2, 256), block=32,
              window=4096, sinks=True),
        # The tokens one decode step produced, with the server's usual five
        # alternatives: latency.
        _score("score decode step", rows=8, vocab=128256, dtype="bf16", top_n=5),
        # Teacher-forced scoring of a prompt chunk with the server's largest
        # number of alternatives.
        _score("score prompt", rows=4096, vocab=128256, dtype="bf16", top_n=20),
        # fp32 logits, an odd number of rows, teacher values for distillation
        # (64 alternatives).
        _score("score teacher f32", rows=509, vocab=151936, dtype="f32", top_n=64),
        # A policy step on given tokens: log-probabilities and entropies
        # forward, the logits' gradient backward.
        _score("score policy step", rows=2048, vocab=151936, dtype="bf16", top_n=0, train=True),
        # Draft head against stored teacher values, forward only, a loss a row.
        _distill("distill eval", rows=61, vocab=128256, dtype="bf16", k=20, tail=True),
        # A short fp32 step over a smaller vocabulary of odd size, K
        # renormalised teacher values.
        _distill("distill small step", rows=33, vocab=32003, dtype="f32", k=8, tail=False,
                 train=True),
        # The training step of a draft head: weighted mean, loss and gradient.
        _distill("distill step", rows=2048, vocab=128256, dtype="bf16", k=64, tail=True,
                 train=True, temperature=2.0),
        # A loss a row, whose gradient comes from what the caller does with
        # the rows.
        _distill("distill rows", rows=1024, vocab=151936, dtype="bf16", k=128, tail=True,
                 train=True, rowwise=True),
    ]


def _tree(name, batch, nodes, ctx, heads, block, window=0, sinks=False):
    c = {"op": "tree", "batch": batch, "nodes": nodes, "ctx": ctx, "hq": heads[0],
         "hkv": heads[1], "d": heads[2], "block": block, "window": window, "sinks": sinks}
    return {"name": name, **c} if name else c


def _score(name, rows, vocab, dtype, top_n, train=False, temperature=1.0):
    c = {"op": "score", "rows": rows, "vocab": vocab, "dtype": dtype, "top_n": top_n,
         "train": train, "temperature": temperature}
    return {"name": name, **c} if name else c


def _distill(name, rows, vocab, dtype, k, tail, train=False, rowwise=False, temperature=1.0):
    c = {"op": "distill", "rows": rows, "vocab": vocab, "dtype": dtype, "k": k, "tail": tail,
         "train": train, "rowwise": rowwise, "temperature": temperature}
    return {"name": name, **c} if name else c


def _log_between(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree", "score", "distill"])
    if op == "tree":
        heads = rng.choice([(32, 8, 128), (64, 8, 128), (32, 4, 128), (16, 2, 256), (21, 3, 128),
                            (16, 16, 64), (24, 8, 64)])
        ctx = _log_between(rng, 16, 60001)
        # keys x key heads x width stay within the serving batch's; so do the
        # query rows times keys
        most = 64 * 4096 * 8 * 128 // (ctx * heads[1] * heads[2])
        batch = _log_between(rng, 1, max(1, min(128, most)))
        rows = 2 * 60001 * 64 * 32 * 128 // (ctx * batch * heads[0] * heads[2])
        nodes = _log_between(rng, 1, max(1, min(64, rows)))
        return _tree(None, batch, nodes, ctx, heads, rng.choice([16, 32, 64]),
                     rng.choice([0, 0, 1024]), rng.random() < 0.3)
    dtype = rng.choice(["bf16", "bf16", "f32"])
    vocab = _log_between(rng, 1000, 200000)
    most = 4096 * 128256 * 2 // (vocab * (2 if dtype == "bf16" else 4))
    t = rng.choice([1.0, 1.0, 0.7, 2.0])
    if op == "score":
        train = rng.random() < 0.35
        rows = _log_between(rng, 1, min(16384, most // 2 if train else most))
        return _score(None, rows, vocab, dtype, rng.choice([0, 1, 5, 20, 64]), train, t)
    train = rng.random() < 0.7
    rows = _log_between(rng, 1, min(16384, most // 2))
    return _distill(None, rows, vocab, dtype, _log_between(rng, 1, 128), rng.random() < 0.6, train,
                    rng.random() < 0.3, t)


# ------------------------------------------------------------- sizes of a batch
def _lens(c):
    """Context and tree sizes of each sequence: the first has the largest,
    the others spread between a quarter (half) of it and all of it."""
    lens, nodes = [], []
    for i in range(c["batch"]):
        n = c["nodes"] if i == 0 else max(1, int(c["nodes"] * (0.5 + 0.5 * (i * 0.4142135 % 1))))
        x = c["ctx"] if i == 0 else int(c["ctx"] * (0.25 + 0.75 * (i * 0.6180339 % 1)))
        nodes.append(n)
        lens.append(max(x, n))
    return lens, nodes


# --------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(seed * 7919 + 17)
    return _prepare_tree(case, g, seed) if case["op"] == "tree" else _prepare_rows(case, g)


def _prepare_tree(c, g, seed):
    lens, nodes = _lens(c)
    bs, hq, hkv, d = c["block"], c["hq"], c["hkv"], c["d"]
    blocks = [-(-n // bs) for n in lens]
    total = sum(blocks) + 8
    bf = torch.bfloat16
    kc = torch.empty(total, hkv, bs, d, device=_DEV, dtype=bf).normal_(generator=g)
    vc = torch.empty(total, hkv, bs, d, device=_DEV, dtype=bf).normal_(generator=g)
    perm = torch.randperm(total, generator=g, device=_DEV).to(torch.int32)
    bt = torch.zeros(c["batch"], max(blocks), dtype=torch.int32, device=_DEV)
    at = 0
    for i, n in enumerate(blocks):
        bt[i, :n] = perm[at:at + n]
        at += n
    cu = [0]
    for n in nodes:
        cu.append(cu[-1] + n)
    T = cu[-1]
    # the query and the key projection share one buffer, as the model's do
    qkv = torch.empty(T, (hq + 2 * hkv) * d, device=_DEV, dtype=bf).normal_(generator=g)
    words = max(1, -(-c["nodes"] // 32))
    # random trees: a node hangs on any earlier one; bit i of a row is node i
    r = torch.Generator().manual_seed(seed * 31 + 5)
    pick = torch.rand(T, generator=r).tolist()
    rows = []
    for i, n in enumerate(nodes):
        seen = []
        for j in range(n):
            m = 1 << j
            if j:
                m |= seen[int(pick[cu[i] + j] * j)]
            seen.append(m)
        rows += [[(m >> (32 * w)) & 0xFFFFFFFF for w in range(words)] for m in seen]
    mask = torch.tensor(rows, dtype=torch.int64)
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(torch.int32).to(_DEV)
    return {"op": "tree", "q": qkv.view(T, hq + 2 * hkv, d)[:, :hq], "kc": kc, "vc": vc, "bt": bt,
            "lens": torch.tensor(lens, dtype=torch.int32, device=_DEV),
            "cu": torch.tensor(cu, dtype=torch.int32, device=_DEV), "mask": mask,
            "scale": 1.0 / math.sqrt(d), "window": c["window"],
            "sinks": torch.randn(hq, generator=g, device=_DEV) if c["sinks"] else None,
            "max_nodes": c["nodes"], "max_len": max(lens), "out_dtype": bf}


def _prepare_rows(c, g):
    T, V, dt = c["rows"], c["vocab"], _DTYPES[c["dtype"]]
    x = torch.empty(T, V, device=_DEV, dtype=dt).normal_(0.0, 2.0, generator=g)
    # a model's rows are peaked: a few tokens far above the rest
    peaks = torch.randint(0, V, (T, 4), generator=g, device=_DEV)
    lift = 6.0 + 6.0 * torch.rand(T, 4, generator=g, device=_DEV)
    x.scatter_(1, peaks, lift.to(dt))
    # some rows carry an allow-list: a stretch of the vocabulary is forbidden
    lo = V // 3
    x[::16, lo:lo + V // 4] = float("-inf")
    s = {"op": c["op"], "temperature": c["temperature"], "train": c["train"]}
    if c["op"] == "score":
        ids = torch.randint(0, V, (T,), generator=g, device=_DEV)
        s["ids"] = torch.where(torch.rand(T, generator=g, device=_DEV) < 0.6, peaks[:, 0], ids)
        # forbidden tokens are not the ones that were given
        inside = (s["ids"] >= lo) & (s["ids"] < lo + V // 4)
        inside &= torch.arange(T, device=_DEV) % 16 == 0
        s["ids"] = torch.where(inside, s["ids"] % lo, s["ids"])
        s["top_n"] = c["top_n"]
        if c["train"]:
            # what a policy loss sends back: advantages, and a small weight
            # on the entropy
            s["g_lp"] = torch.randn(T, generator=g, device=_DEV) / T
            s["g_ent"] = torch.full((T,), -0.01 / T, device=_DEV)
    else:
        K = c["k"]
        first = torch.randint(0, V, (T, 1), generator=g, device=_DEV)
        step = 1 + torch.randint(0, max(1, V // K - 1), (T, 1), generator=g, device=_DEV)
        ids = (first + step * torch.arange(K, device=_DEV)) % V  # K distinct tokens
        tl = (1.5 * torch.randn(T, K, generator=g, device=_DEV) + 6.0).sort(1, descending=True)[0]
        # the teacher keeps 1 to 20 % of its mass outside the K
        rest = 0.01 + 0.19 * torch.rand(T, 1, generator=g, device=_DEV)
        s["t_ids"] = ids.to(torch.int32)
        s["t_lp"] = torch.log_softmax(tl, 1) + torch.log1p(-rest)
        near = tl + 0.7 * torch.randn(T, K, generator=g, device=_DEV)
        x.scatter_(1, ids, near.to(dt))
        s["tail"] = c["tail"]
        s["rowwise"] = c["rowwise"]
        # prompt positions do not count
        s["w"] = (torch.rand(T, generator=g, device=_DEV) < 0.9).float()
        if c["rowwise"]:
            s["g_rows"] = torch.rand(T, generator=g, device=_DEV) / T
    s["x"] = x.requires_grad_(bool(c["train"]))
    return s


# ------------------------------------------------------------------- one pass
def run(s):
    if s["op"] == "tree":
        return _own_tree(s) if own else _plain_tree(s)
    if s["op"] == "score":
        return _own_score(s) if own else _plain_score(s)
    return _own_distill(s) if own else _plain_distill(s)


def _own_tree(s):
    from vllm_sm70_b200 import ops
    out = torch.empty(s["q"].shape, dtype=s["out_dtype"], device=s["q"].device)
    return ops.tree_attention(out, s["q"], s["kc"], s["vc"], s["bt"], s["lens"], s["cu"],
                              s["mask"], s["scale"], window=s["window"], sinks=s["sinks"])


def _own_score(s):
    from vllm_sm70_b200 import ops
    r = ops.token_logprobs(s["x"], s["ids"], top_n=s["top_n"], temperature=s["temperature"])
    out = {"logprobs": r.logprobs.detach(), "ranks": r.ranks, "entropy": r.entropy.detach(),
           "lse": r.lse, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs}
    if s["train"]:
        out["grad"], = torch.autograd.grad((r.logprobs, r.entropy), s["x"],
                                           (s["g_lp"], s["g_ent"]))
    return out


def _own_distill(s):
    from vllm_sm70_b200 import ops
    loss = ops.distill_loss(s["x"], s["t_ids"], s["t_lp"], weights=s["w"],
                            temperature=s["temperature"], tail=s["tail"],
                            reduction="mean" if s["train"] and not s["rowwise"] else "none")
    out = {"loss": loss.detach()}
    if s["train"]:
        out["grad"], = torch.autograd.grad(loss, s["x"], s["g_rows"] if s["rowwise"] else None)
    return out


# ------------------------------------------------------------------ plain forms
def _plain_tree(s):
    q, kc, bt, lens, cu = s["q"], s["kc"], s["bt"].long(), s["lens"].long(), s["cu"].long()
    B, N = lens.numel(), s["max_nodes"]
    hkv, bs, d = kc.shape[1:]
    hq = q.shape[1]
    grp = hq // hkv
    L = bt.shape[1] * bs
    k = kc[bt].float().permute(0, 2, 1, 3, 4).reshape(B, hkv, L, d)
    v = s["vc"][bt].float().permute(0, 2, 1, 3, 4).reshape(B, hkv, L, d)
    n = cu[1:] - cu[:-1]
    node = torch.arange(N, device=q.device)
    tok = (cu[:-1, None] + node).clamp(max=q.shape[0] - 1)
    qf = q[tok].float().view(B, N, hkv, grp, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, grp * N, d)
    sc = (qf @ k.transpose(2, 3)) * s["scale"]
    bits = (s["mask"][tok][..., None] >> torch.arange(32, device=q.device)) & 1
    bits = bits.reshape(B, N, -1).bool() & (torch.arange(bits.shape[2] * 32, device=q.device)
                                            < n[:, None, None])
    key = torch.arange(L, device=q.device)
    prefix = lens - n
    at = key - prefix[:, None]
    seen = bits.gather(2, at.clamp(0, bits.shape[2] - 1)[:, None].expand(B, N, L))
    vis = torch.where(at[:, None] >= 0, seen, True) & (key < lens[:, None])[:, None]
    if s["window"]:
        pos = prefix[:, None] + bits.sum(2).clamp(min=1) - 1
        vis &= (at[:, None] >= 0) | (key > pos[..., None] - s["window"])
    vis = vis[:, None, None].expand(B, 1, grp, N, L).reshape(B, 1, grp * N, L)
    sc = torch.where(vis, sc, torch.full_like(sc, float("-inf")))
    m = sc.amax(3, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, hkv, grp, 1).expand(B, hkv, grp, N).reshape(B, hkv, -1, 1)
        m = torch.maximum(m, sink)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = torch.exp(sc - m)
    den = p.sum(3, keepdim=True)
    if s["sinks"] is not None:
        den = den + torch.exp(sink - m)
    o = (p @ v) / torch.where(den == 0, torch.ones_like(den), den)
    o = o.view(B, hkv, grp, N, d).permute(0, 3, 1, 2, 4).reshape(B, N, hq, d)
    own_seq = torch.searchsorted(cu, torch.arange(q.shape[0], device=q.device), right=True) - 1
    own_node = torch.arange(q.shape[0], device=q.device) - cu[own_seq]
    return o[own_seq, own_node].to(s["out_dtype"])


def _plain_score(s):
    x = s["x"].detach().float()
    T, V = x.shape
    ids = s["ids"].long()
    z = x / s["temperature"]
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    den = e.sum(1, keepdim=True)
    lse = m + torch.log(den)
    p = e / den
    lp = z - lse
    plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    ent = -plp.sum(1)
    xy = x.gather(1, ids[:, None])
    col = torch.arange(V, device=x.device)
    rank = 1 + ((x > xy) | ((x == xy) & (col < ids[:, None]))).sum(1)
    # order: larger value first, lower id first among equals
    b = x.view(torch.int32)
    key = torch.where(b < 0, b ^ 0x7FFFFFFF, b).long() * (1 << 20) + (V - 1 - col)
    top = torch.topk(key, s["top_n"], dim=1)[1] if s["top_n"] else ids.new_zeros(T, 0)
    out = {"logprobs": lp.gather(1, ids[:, None])[:, 0], "ranks": rank.to(torch.int32),
           "entropy": ent, "lse": lse[:, 0], "top_ids": top.to(torch.int32),
           "top_logprobs": lp.gather(1, top)}
    if s["train"]:
        gr = -s["g_lp"][:, None] * p - s["g_ent"][:, None] * (plp + p * ent[:, None])
        gr.scatter_add_(1, ids[:, None], s["g_lp"][:, None])
        out["grad"] = (gr / s["temperature"]).to(s["x"].dtype)
    return out


def _plain_distill(s):
    z = s["x"].detach().float() / s["temperature"]
    T, V = z.shape
    ids = s["t_ids"].long()
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    den = e.sum(1, keepdim=True)
    q = e / den
    lq = (z - m - torch.log(den)).gather(1, ids)
    tl = s["t_lp"]
    if s["tail"]:
        p = torch.exp(tl)
        pt = (1 - p.sum(1)).clamp(min=0)
    else:
        p = torch.exp(tl - tl.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
        tl = torch.log(p)
        pt = torch.zeros_like(den[:, 0])
    mass = p.sum(1) + pt
    loss = (p * (tl - lq)).sum(1)
    ratio = torch.zeros_like(pt)
    if s["tail"]:
        qt = q.scatter(1, ids, 0.0).sum(1)
        ratio = pt / qt
        loss = loss + torch.where(pt > 0, pt * (torch.log(pt) - torch.log(qt)), pt)
    rows = loss * s["w"]
    mean = s["train"] and not s["rowwise"]
    out = {"loss": rows.sum() / T if mean else rows}
    if s["train"]:
        gr = q * (mass - ratio)[:, None]
        gr.scatter_(1, ids, q.gather(1, ids) * mass[:, None])
        gr.scatter_add_(1, ids, -p)
        up = s["w"] * (s["g_rows"] if s["rowwise"] else 1.0 / T) / s["temperature"]
        out["grad"] = (gr * up[:, None]).to(s["x"].dtype)
    return out


# ------------------------------------------------------------- least work of a pass
def work(case):
    c = case
    if c["op"] == "tree":
        lens, nodes = _lens(c)
        w = c["window"]
        # a window leaves the keys that some node of the tree can reach
        keys = sum(min(n, w + q) if w else n for n, q in zip(lens, nodes))
        pairs = sum((min(n, w + q) if w else n) * q for n, q in zip(lens, nodes))
        T = sum(nodes)
        return {"bytes": 4 * keys * c["hkv"] * c["d"] + 4 * T * c["hq"] * c["d"],
                "flops": 4 * pairs * c["hq"] * c["d"]}
    T, V = c["rows"], c["vocab"]
    size = 2 if c["dtype"] == "bf16" else 4
    small = 28 * T + 8 * T * c.get("top_n", 0) + 8 * T * c.get("k", 0)
    passes = 2 if c["train"] else 1  # logits in, gradient out
    return {"bytes": passes * size * T * V + small, "flops": (12 if c["train"] else 6) * T * V}


# ------------------------------------------------------------- values in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "tree":
            return _exact_tree(s)
        if case["op"] == "score":
            return _exact_score(s)
        return _exact_distill(s)


def _exact_tree(s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    hq, hkv, bs = s["q"].shape[1], s["kc"].shape[1], s["kc"].shape[2]
    for i, n in enumerate(lens):
        a, b = cu[i], cu[i + 1]
        blocks = s["bt"][i, : -(-n // bs)].long()
        k = s["kc"][blocks].transpose(0, 1).reshape(hkv, -1, s["kc"].shape[3])[:, :n].double()
        v = s["vc"][blocks].transpose(0, 1).reshape(hkv, -1, s["kc"].shape[3])[:, :n].double()
        words = s["mask"][a:b].tolist()
        vis = torch.zeros(b - a, n, dtype=torch.bool)
        for j in range(b - a):
            anc = [t for t in range(b - a) if (words[j][t // 32] >> (t % 32)) & 1]
            first = 0
            if s["window"]:
                first = max(0, n - (b - a) + max(len(anc), 1) - 1 - s["window"] + 1)
            vis[j, first:n - (b - a)] = True
            vis[j, [n - (b - a) + t for t in anc]] = True
        vis = vis.to(k.device)
        for h in range(hq):
            sc = s["q"][a:b, h].double() @ k[h * hkv // hq].T * s["scale"]
            sc = sc.masked_fill(~vis, float("-inf"))
            if s["sinks"] is not None:
                extra = s["sinks"][h].double().expand(b - a, 1)
                w = torch.softmax(torch.cat([sc, extra], 1), 1)[:, :-1]
            else:
                w = torch.softmax(sc, 1)
            out[a:b, h] = w @ v[h * hkv // hq]
    return out


def _exact_score(s):
    ids = s["ids"].long()[:, None]
    out = {"logprobs": [], "ranks": None, "entropy": [], "lse": [], "top_ids": None,
           "top_logprobs": []}
    if s["train"]:
        out["grad"] = []
    T = ids.shape[0]
    for a in range(0, T, 256):  # rows at a time: 64 bits of every logit are large
        i = ids[a:a + 256]
        z = s["x"][a:a + 256].detach().double() / s["temperature"]
        lse = torch.logsumexp(z, 1)
        lp = z - lse[:, None]
        p = torch.exp(lp)
        h = torch.special.entr(p).sum(1)
        out["logprobs"].append(lp.gather(1, i)[:, 0])
        out["entropy"].append(h)
        out["lse"].append(lse)
        out["top_logprobs"].append(torch.topk(lp, s["top_n"], dim=1)[0])
        if s["train"]:
            # d log p_y / dz = [y] - p; d H / dz = -p (log p + H)
            gl, ge = s["g_lp"][a:a + 256].double(), s["g_ent"][a:a + 256].double()
            hot = torch.zeros_like(z).scatter_(1, i, 1.0)
            ds = (hot - p) * gl[:, None]
            ds += (torch.special.entr(p) - p * h[:, None]) * ge[:, None]
            out["grad"].append((ds / s["temperature"]).to(torch.float64))
    return {k: torch.cat(v) if isinstance(v, list) else v for k, v in out.items()}


def _exact_distill(s):
    loss, grad = [], []
    T, V = s["x"].shape
    for a in range(0, T, 256):
        z = s["x"][a:a + 256].detach().double() / s["temperature"]
        ids, tl = s["t_ids"][a:a + 256].long(), s["t_lp"][a:a + 256].double()
        logq = torch.log_softmax(z, 1)
        dense = torch.zeros_like(z)
        if s["tail"]:
            dense.scatter_(1, ids, tl.exp())
            rest = (1 - tl.exp().sum(1)).clamp(min=0)
            out_logq = torch.logsumexp(z.scatter(1, ids, float("-inf")), 1) - torch.logsumexp(z, 1)
            row = torch.special.xlogy(rest, rest) - rest * out_logq
        else:
            dense.scatter_(1, ids, torch.softmax(tl, 1))
            rest, out_logq, row = None, None, 0
        p = dense.gather(1, ids)
        row = row + (torch.special.xlogy(p, p) - p * logq.gather(1, ids)).sum(1)
        w = s["w"][a:a + 256].double()
        loss.append(row * w)
        if s["train"]:
            q = logq.exp()
            target = dense
            if s["tail"]:
                # the rest of the teacher's mass, spread as the student spreads it
                inside = torch.zeros_like(z).scatter_(1, ids, 1.0)
                target = dense + (1 - inside) * q * (rest / out_logq.exp())[:, None]
            up = s["g_rows"][a:a + 256].double() if s["rowwise"] else 1.0 / T
            mass = target.sum(1, keepdim=True)
            grad.append((q * mass - target) * (w * up / s["temperature"])[:, None])
    loss = torch.cat(loss)
    mean = s["train"] and not s["rowwise"]
    out = {"loss": loss.sum() / T if mean else loss}
    if s["train"]:
        out["grad"] = torch.cat(grad)
    return out
