"""Operators of speculative decoding over a tree of drafted tokens, each case one pass through the public entry points.

A step of it: queries and keys are normed for each head and rotated, keys and values go to a paged cache; the tree's
tokens attend to the cached positions and to their ancestors; a path through the tree is accepted; its keys and
values are moved together in the cache. Head layouts and vocabularies are those of the benchmark models (32 heads of
64 or 128 over 8 KV heads, 16 layers, vocabulary 128256 and 151936) or generic.

`own` False computes the plain forms in elementary torch operations, True calls the framework.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # decode: the new token of one chat, norms and rotation on its way to the cache: pure latency
        dict(name="norm_one", kind="append", seqs=1, new=1, heads=32, kv=8, hd=128, rot=128, neox=True, dtype="f32",
             cache="f16", page=16, longest=1000, tree=False),
        # a batch's trees: rotary positions by depth, cache positions by node
        dict(name="norm_trees", kind="append", seqs=48, new=32, heads=32, kv=8, hd=128, rot=128, neox=True,
             dtype="bf16", cache="bf16", page=16, longest=6000, tree=True),
        # queries of a long document, no cache, an odd number of heads, three quarters of each rotated
        dict(name="norm_long", kind="norm", tokens=16381, heads=33, hd=128, rot=96, neox=False, dtype="f16",
             far=1000000),
        # one chat's tree over its first thousand positions, where launches and joins count
        dict(name="tree_one", kind="attend", seqs=1, new=8, heads=32, kv=8, hd=64, dtype="f32", cache="f16", page=16,
             longest=1001, window=0, ragged=False),
        # a batch of chats of very different lengths, trees of 32
        dict(name="tree_batch", kind="attend", seqs=24, new=32, heads=32, kv=8, hd=128, dtype="bf16", cache="bf16",
             page=16, longest=6000, window=0, ragged=False),
        # two long documents, trees of 64: all the products of a prompt over all the keys of a decode step
        dict(name="tree_long", kind="attend", seqs=2, new=64, heads=32, kv=8, hd=128, dtype="f16", cache="f16",
             page=64, longest=131072, window=0, ragged=False),
        # a sliding window, f32 queries, pages that end inside a tile, an odd number of nodes
        dict(name="tree_window", kind="attend", seqs=13, new=25, heads=32, kv=8, hd=128, dtype="f32", cache="f16",
             page=24, longest=9000, window=4096, ragged=False),
        # one chat's tree
        dict(name="verify_one", kind="verify", seqs=1, new=16, vocab=128256),
        # a batch's trees over the larger vocabulary
        dict(name="verify_batch", kind="verify", seqs=48, new=32, vocab=151936),
        # what one chat accepted, all layers
        dict(name="keep_one", kind="keep", layers=16, seqs=1, new=16, kv=8, hd=64, cache="f16", page=16, longest=300),
        # what a batch accepted, all layers
        dict(name="keep_batch", kind="keep", layers=16, seqs=48, new=48, kv=8, hd=128, cache="bf16", page=16,
             longest=200),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "append", "append", "attend", "attend", "attend", "verify", "keep"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    cache = dtype if dtype != "f32" else rng.choice(["f16", "bf16"])
    hd = rng.choice([64, 96, 128, 128, 256])
    rot = rng.choice([hd, hd, hd // 2, 2 * rng.randint(1, hd // 2)])
    if kind == "norm":
        heads = rng.choice([1, 3, 8, 20, 32, 40])
        return dict(kind=kind, tokens=_log(rng, 1, 60000000 // (heads * hd)), heads=heads, hd=hd, rot=rot,
                    neox=rng.random() < 0.5, dtype=dtype, far=_log(rng, 1000, 1000000))
    if kind == "append":
        seqs, kv, tree = _log(rng, 1, 64), rng.choice([1, 2, 8]), rng.random() < 0.5
        new = rng.randint(2, 64) if tree else rng.choice([1, 1, _log(rng, 1, max(2, 4096 // seqs))])
        return dict(kind=kind, seqs=seqs, new=new, heads=kv * rng.choice([1, 4, 5]), kv=kv, hd=hd, rot=rot,
                    neox=rng.random() < 0.5, dtype=dtype, cache=cache, page=rng.choice([16, 32, 64, 24]),
                    longest=max(new, _log(rng, 16, 8192)), tree=tree)
    if kind == "attend":
        kv, group, new = rng.choice([1, 2, 4, 8, 8]), rng.choice([1, 4, 4, 5, 8]), rng.randint(2, 64)
        # positions that cost no more than the longest listed case
        room = min(400000000 // (kv * hd * 4), 100000000000 // (4 * kv * group * new * hd))
        seqs = _log(rng, 1, 64)
        return dict(kind=kind, seqs=seqs, new=new, heads=kv * group, kv=kv, hd=hd, dtype=dtype, cache=cache,
                    page=rng.choice([16, 32, 64, 128, 24, 1]),
                    longest=max(new, _log(rng, 16, max(32, min(131072, room // seqs)))),
                    window=rng.choice([0, 0, 0, _log(rng, 16, 8192)]), ragged=rng.random() < 0.3)
    if kind == "verify":
        return dict(kind=kind, seqs=_log(rng, 1, 48), new=rng.randint(2, 32), vocab=_log(rng, 1000, 151936))
    new = rng.randint(2, 64)
    return dict(kind=kind, layers=rng.choice([1, 16, 16, 28]), seqs=_log(rng, 1, 48), new=new, kv=rng.choice([1, 8]),
                hd=rng.choice([64, 128]), cache=cache, page=rng.choice([16, 32, 24, 1]),
                longest=max(new, _log(rng, 16, 200)))


# ---- inputs -------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, dtype="f32", scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(DTYPES[dtype])


def _spread(case):
    """Ragged lengths: evenly spread up to the longest, each with room for its new tokens."""
    n, new = case["seqs"], case["new"]
    return [max(new, case["longest"] * (i + 1) // n) for i in range(n)]


def _lengths(case, g):
    lens = torch.tensor(_spread(case), dtype=torch.int32, device="cuda")
    return lens[torch.randperm(case["seqs"], device="cuda", generator=g)]


def _freqs(case):
    i = torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda")
    return (1000000.0 ** (-i / case["rot"])).float()


def _pages(case, g, *layers):
    """Key and value pages in one pool (one of each layer), a table of its pages in random order."""
    width = -(-max(case["longest"], case["new"]) // case["page"])
    n = case["seqs"] * width + 3
    table = torch.randperm(n, device="cuda", generator=g)[:case["seqs"] * width].to(torch.int32).view(-1, width)
    shape = (*layers, n, case["kv"], case["page"], case["hd"])
    k = torch.empty(shape, dtype=DTYPES[case["cache"]], device="cuda").normal_(generator=g)
    v = torch.empty(shape, dtype=DTYPES[case["cache"]], device="cuda").normal_(generator=g)
    return k, v, table.contiguous()


def _tree(seqs, new, g):
    """A tree for each sequence: a node hangs on one of those before it, mostly on the early ones as the best
    continuations are drafted first."""
    j = torch.arange(new, device="cuda")
    u = torch.rand(seqs, new, device="cuda", generator=g) ** 1.5
    return torch.minimum((u * j).floor().long(), j - 1).to(torch.int32)  # the first on none: -1


def _depths(parents):
    """How many nodes are above each."""
    return _above(parents).sum(-1).to(torch.int32) - 1


def _above(parents):
    """[seqs, new, new]: whether node a is node j or above it."""
    seqs, new = parents.shape
    m = torch.zeros(seqs, new, new, dtype=torch.bool, device=parents.device)
    b = torch.arange(seqs, device=parents.device)
    for j in range(new):
        p = parents[:, j].long()
        m[:, j] = m[b, p.clamp(min=0)] & (p >= 0)[:, None]
        m[:, j, j] = True
    return m


def prepare(case, seed):
    g = _gen(seed)
    kind, st = case["kind"], {"case": case}
    if kind == "norm":
        st["x"] = _normal(g, case["tokens"], case["heads"], case["hd"], dtype=case["dtype"], scale=3.0)
        st["w"] = 1.0 + 0.2 * _normal(g, case["hd"])
        st["pos"] = torch.randint(0, case["far"], (case["tokens"],), device="cuda", generator=g, dtype=torch.int32)
        st["freqs"] = _freqs(case)
    elif kind == "append":
        seqs, new = case["seqs"], case["new"]
        st["k_pages"], st["v_pages"], st["table"] = _pages(case, g)
        base = _lengths(case, g)[:, None] - new
        at = base + torch.arange(new, device="cuda", dtype=torch.int32)
        st["at"], st["pos"] = None, at.reshape(-1).to(torch.int32).contiguous()
        if case["tree"]:
            st["at"] = st["pos"]
            st["pos"] = (base + _depths(_tree(seqs, new, g))).reshape(-1).to(torch.int32).contiguous()
        st["seq"] = torch.arange(seqs, device="cuda", dtype=torch.int32).repeat_interleave(new)
        # one projection's rows: q, k and v are slices of it
        qkv = _normal(g, seqs * new, case["heads"] + 2 * case["kv"], case["hd"], dtype=case["dtype"], scale=3.0)
        st["q"], st["k"], st["v"] = qkv.split([case["heads"], case["kv"], case["kv"]], 1)
        st["wq"], st["wk"] = (1.0 + 0.2 * _normal(g, case["hd"]) for _ in range(2))
        st["freqs"] = _freqs(case)
    elif kind == "attend":
        seqs, new = case["seqs"], case["new"]
        st["k_pages"], st["v_pages"], st["table"] = _pages(case, g)
        st["lens"] = _lengths(case, g)
        st["parents"] = _tree(seqs, new, g)
        st["counts"] = None
        if case["ragged"]:
            st["counts"] = torch.randint(0, new + 1, (seqs,), device="cuda", generator=g, dtype=torch.int32)
        st["q"] = _normal(g, seqs, new, case["heads"], case["hd"], dtype=case["dtype"], scale=1.5)
    elif kind == "verify":
        seqs, new, vocab = case["seqs"], case["new"], case["vocab"]
        st["parents"] = _tree(seqs, new, g)
        # some rows nearly certain, some open; the draft's best tokens are about the target's
        logits = torch.randn(seqs, new, vocab, device="cuda", generator=g)
        logits *= 2.5 + 5.0 * torch.rand(seqs, new, 1, device="cuda", generator=g)
        st["target"] = torch.softmax(logits, -1)
        logits += 0.5 * torch.randn(seqs, new, vocab, device="cuda", generator=g)
        best = logits.topk(min(16, vocab), -1).indices
        # the k-th child of a node is its k-th best token
        p = st["parents"].long()
        j = torch.arange(new, device="cuda")
        rank = ((p[:, None, :] == p[:, :, None]) & (j < j[:, None])).sum(-1).clamp(max=best.shape[-1] - 1)
        b = torch.arange(seqs, device="cuda")[:, None]
        st["drafted"] = best[b, p.clamp(min=0), rank].to(torch.int32)
        st["uniforms"] = torch.rand(seqs, new, device="cuda", generator=g)
    else:
        seqs, new = case["seqs"], case["new"]
        st["k_pages"], st["v_pages"], st["table"] = _pages(case, g, case["layers"])
        st["lens"] = _lengths(case, g)
        # the way to a random node of a tree, from the root
        above = _above(_tree(seqs, new, g))
        node = torch.randint(0, new, (seqs,), device="cuda", generator=g)
        on = above[torch.arange(seqs, device="cuda"), node]
        j = torch.arange(new, device="cuda")
        st["path"] = torch.where(on, j, new).sort(-1).values
        st["path"] = torch.where(st["path"] < new, st["path"], -1).to(torch.int32).contiguous()
    return st


# ---- one pass -----------------------------------------------------------------------------


def _norm_rotate(x, w, pos, freqs, neox):
    """x [tokens, heads, hd] in 32 bits, the angles in 64."""
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
    a = pos.double()[:, None] * freqs.double()
    c, s = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    r = 2 * freqs.numel()
    h, rest = x[..., :r], x[..., r:]
    x0, x1 = (h[..., :r // 2], h[..., r // 2:]) if neox else (h[..., 0::2], h[..., 1::2])
    y0, y1 = x0 * c - x1 * s, x0 * s + x1 * c
    y = torch.cat((y0, y1), -1) if neox else torch.stack((y0, y1), -1).flatten(-2)
    return torch.cat((y, rest), -1)


def _seen(st, width):
    """[seqs, new, width]: which positions each node attends to."""
    case, parents, lens = st["case"], st["parents"], st["lens"].long()
    seqs, new = parents.shape
    n = st["counts"].long() if st["counts"] is not None else torch.full((seqs,), new, device="cuda")
    above, base = _above(parents), (lens - n)[:, None]
    depth = above.sum(-1) - 1
    t = torch.arange(width, device="cuda")
    ok = (t < base)[:, None].expand(seqs, new, width)
    if case["window"]:
        ok = ok & (t > (base + depth - case["window"])[..., None])
        above = above & (depth[:, :, None] - depth[:, None, :] < case["window"])
    j = torch.arange(new, device="cuda")
    at = (base + j).clamp(max=width - 1)[:, None].expand(seqs, new, new)
    live = (j < n[:, None])[:, None].expand(seqs, new, new)
    tail = torch.zeros(seqs, new, width, dtype=torch.int32, device="cuda")
    tail.scatter_add_(2, at, (above & live).int())
    return (ok | (tail > 0)) & (j < n[:, None])[..., None]


def _attend(st):
    case, q = st["case"], st["q"]
    n, new, heads, hd = q.shape
    kv, page = case["kv"], case["page"]
    width = st["table"].shape[1] * page
    idx = st["table"].long()
    k = st["k_pages"][idx].float().transpose(1, 2).reshape(n, kv, width, hd)
    v = st["v_pages"][idx].float().transpose(1, 2).reshape(n, kv, width, hd)
    rows = q.float().reshape(n, new, kv, heads // kv, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, hd)
    s = torch.matmul(rows, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(hd))
    ok = _seen(st, width)
    ok = ok[:, None, :, None].expand(n, kv, new, heads // kv, width).reshape(n, kv, -1, width)
    s = torch.where(ok, s, torch.full((), -math.inf, device="cuda"))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(s - m)
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(l > 0, l, torch.ones_like(l))
    return o.reshape(n, kv, new, heads // kv, hd).permute(0, 2, 1, 3, 4).reshape(q.shape).to(q.dtype)


def _verify(st):
    target, drafted, parents = st["target"], st["drafted"].long(), st["parents"].long()
    u = st["uniforms"].double()
    seqs, new, vocab = target.shape
    b = torch.arange(seqs, device="cuda")
    p = target[b[:, None], parents.clamp(min=0), drafted].double()
    at = torch.zeros(seqs, dtype=torch.long, device="cuda")
    left = torch.ones(seqs, dtype=torch.float64, device="cuda")
    refused = torch.zeros(seqs, new, dtype=torch.bool, device="cuda")
    path = torch.full((seqs, new + 1), -1, dtype=torch.long, device="cuda")
    path[:, 0] = 0
    count = torch.zeros(seqs, dtype=torch.long, device="cuda")
    for j in range(1, new):
        child = parents[:, j] == at
        again = (refused & (drafted == drafted[:, j:j + 1])).any(1)
        pj = torch.where(again, 0.0, p[:, j])
        take = child & (pj > 0) & (u[:, j] * left < pj)
        drop = child & ~take
        left = torch.where(take, 1.0, torch.where(drop, left - pj, left))
        refused = refused & ~take[:, None]
        refused[:, j] = drop
        at = torch.where(take, j, at)
        count = count + take
        path.scatter_(1, torch.where(take, count, new)[:, None], torch.full_like(at, j)[:, None])
    path = torch.where(torch.arange(new, device="cuda") <= count[:, None], path[:, :new], -1)
    row = target[b, at].double()
    keep = torch.ones(seqs, vocab, dtype=torch.int32, device="cuda")
    keep.scatter_add_(1, drafted, -refused.int())
    r = torch.where(keep == 1, row, torch.zeros_like(row))
    r = torch.where(r.sum(1, keepdim=True) > 0, r, row)
    c = r.cumsum(1)
    v = torch.arange(vocab, device="cuda")
    last = torch.where(r > 0, v, -1).amax(1)
    token = torch.minimum((c <= u[:, :1] * c[:, -1:]).sum(1), last)
    i = torch.arange(new, device="cuda")
    nodes = torch.nn.functional.pad(path[:, 1:], (0, 1), value=0).clamp(min=0)
    tokens = drafted.gather(1, nodes)
    tokens = torch.where(i < count[:, None], tokens, torch.where(i == count[:, None], token[:, None], -1))
    return tokens.to(torch.int32), path.to(torch.int32), count.to(torch.int32)


def _keep(st):
    case, path = st["case"], st["path"].long()
    new, page = case["new"], case["page"]
    base = st["lens"].long()[:, None] - new
    i = torch.arange(new, device="cuda")
    kept = path >= 0
    src, dst = base + torch.where(kept, path, 0), base + torch.where(kept, i, 0)
    b = torch.arange(case["seqs"], device="cuda")[:, None]
    table = st["table"].long()
    sp, dp = table[b, src // page], table[b, dst // page]
    for pages in (st["k_pages"], st["v_pages"]):
        rows = pages.transpose(2, 3)  # [layers, pages, positions, heads, hd]
        rows[:, dp, dst % page] = rows[:, sp, src % page]
    return (base[:, 0] + kept.sum(1)).to(torch.int32), st["k_pages"], st["v_pages"]


def _plain(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "norm":
        return _norm_rotate(st["x"], st["w"], st["pos"], st["freqs"], case["neox"]).to(st["x"].dtype)
    if kind == "append":
        q = _norm_rotate(st["q"], st["wq"], st["pos"], st["freqs"], case["neox"]).to(st["q"].dtype)
        k = _norm_rotate(st["k"], st["wk"], st["pos"], st["freqs"], case["neox"])
        place = (st["pos"] if st["at"] is None else st["at"]).long()
        page = st["table"][st["seq"].long(), place // case["page"]].long()
        st["k_pages"][page, :, place % case["page"]] = k.to(st["k_pages"].dtype)
        st["v_pages"][page, :, place % case["page"]] = st["v"].to(st["v_pages"].dtype)
        return q, st["k_pages"], st["v_pages"]
    if kind == "attend":
        return _attend(st)
    return _verify(st) if kind == "verify" else _keep(st)


def _own(st):
    from nightrun_amd import serve

    case = st["case"]
    kind = case["kind"]
    if kind == "norm":
        y = torch.empty_like(st["x"])
        serve.norm_rope(y, st["x"], st["w"], st["pos"], st["freqs"], eps=1e-6, neox=case["neox"])
        return y
    if kind == "append":
        y = torch.empty(st["q"].shape, dtype=st["q"].dtype, device="cuda")
        serve.norm_rope_append(y, st["q"], st["k"], st["v"], st["wq"], st["wk"], st["pos"], st["seq"], st["freqs"],
                               st["k_pages"], st["v_pages"], st["table"], eps=1e-6, neox=case["neox"], at=st["at"])
        return y, st["k_pages"], st["v_pages"]
    if kind == "attend":
        # rows behind a sequence's last node are left as they were
        y = torch.empty_like(st["q"]) if st["counts"] is None else torch.zeros_like(st["q"])
        serve.tree_attention(y, st["q"], st["k_pages"], st["v_pages"], st["table"], st["lens"], st["parents"],
                             scale=1.0 / math.sqrt(case["hd"]), window=case["window"], counts=st["counts"])
        return y
    if kind == "verify":
        seqs, new = st["drafted"].shape
        tokens, path = (torch.empty(seqs, new, dtype=torch.int32, device="cuda") for _ in range(2))
        count = torch.empty(seqs, dtype=torch.int32, device="cuda")
        serve.verify_tree(tokens, path, count, st["target"], st["drafted"], st["parents"], st["uniforms"])
        return tokens, path, count
    lens = torch.empty_like(st["lens"])
    serve.keep_path(lens, st["k_pages"], st["v_pages"], st["table"], st["lens"], st["path"])
    return lens, st["k_pages"], st["v_pages"]


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without -----------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "norm":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["hd"] * BYTES[case["dtype"]] + 4 * case["tokens"] + 2 * case["rot"] + 4 * case["hd"],
                "flops": n * (4 * case["hd"] + 3 * case["rot"])}
    if kind == "append":
        n, hd = case["seqs"] * case["new"], case["hd"]
        read = (case["heads"] + 2 * case["kv"]) * hd * BYTES[case["dtype"]]
        wrote = case["heads"] * hd * BYTES[case["dtype"]] + 2 * case["kv"] * hd * 2
        return {"bytes": n * (read + wrote + (16 if case["tree"] else 12)) + 2 * case["rot"] + 8 * hd,
                "flops": n * (case["heads"] + case["kv"]) * (4 * hd + 3 * case["rot"])}
    if kind == "attend":
        new, window, heads, hd = case["new"], case["window"], case["heads"], case["hd"]
        part = 0.5 if case["ragged"] else 1.0  # of the nodes, on average
        lens = [min(n, window + new - 1) if window else n for n in _spread(case)]
        rows = case["seqs"] * new * heads * part
        return {"bytes": sum(lens) * case["kv"] * hd * 4 + 2 * rows * hd * BYTES[case["dtype"]],
                "flops": 4 * sum(n - new + 1 for n in lens) * new * part * heads * hd}
    if kind == "verify":
        seqs, new = case["seqs"], case["new"]
        return {"bytes": seqs * (case["vocab"] * 4 + 24 * new), "flops": 2 * seqs * case["vocab"]}
    # two moves of three nodes or so a sequence: the nodes of a path that are not in their place already
    moved = case["layers"] * case["seqs"] * 2 * case["kv"] * case["hd"] * 2 * min(case["new"] - 1, 3)
    return {"bytes": 2 * moved + 4 * case["seqs"] * (case["new"] + 2), "flops": 0}


# ---- the definitions in 64 bits ----------------------------------------------------------------


def _exact_rows(x, w, pos, freqs, neox):
    """Each row by its root mean square, each pair as a complex number, times e^(i * pos * freq)."""
    x = x.double()
    x = x / torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / x.shape[-1] + 1e-6) * w.double()
    n = freqs.numel()
    pairs = torch.arange(n, device="cuda")
    re, im = (pairs, pairs + n) if neox else (2 * pairs, 2 * pairs + 1)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda").expand(pos.numel(), n).contiguous(),
                       torch.outer(pos.double(), freqs.double()))
    z = torch.complex(x[..., re], x[..., im]) * turn[:, None]
    x[..., re], x[..., im] = z.real, z.imag
    return x


def _walk(parents, j):
    """Node j and what is above it, from the root."""
    way = []
    while j >= 0:
        way.append(j)
        j = parents[j]
    return way[::-1]


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        return _exact_rows(st["x"], st["w"], st["pos"], st["freqs"], case["neox"])
    if kind == "append":
        q = _exact_rows(st["q"], st["wq"], st["pos"], st["freqs"], case["neox"])
        k = _exact_rows(st["k"], st["wk"], st["pos"], st["freqs"], case["neox"])
        kp, vp = st["k_pages"].double(), st["v_pages"].double()
        place = (st["pos"] if st["at"] is None else st["at"]).long()
        pages = st["table"].long().flatten()[st["seq"].long() * st["table"].shape[1] + place // case["page"]]
        slots = pages * case["page"] + place % case["page"]
        for pool, rows in ((kp, k), (vp, st["v"].double())):
            flat = pool.transpose(1, 2).clone(memory_format=torch.contiguous_format).view(-1, case["kv"], case["hd"])
            flat[slots] = rows
            pool.copy_(flat.view(pool.shape[0], case["page"], case["kv"], case["hd"]).transpose(1, 2))
        return q, kp, vp
    if kind == "attend":
        y = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        group, new = case["heads"] // case["kv"], case["new"]
        counts = st["counts"].tolist() if case["ragged"] else [new] * case["seqs"]
        trees = st["parents"].tolist()
        for b, (n, m) in enumerate(zip(st["lens"].tolist(), counts)):
            if m == 0:
                continue
            pages = st["table"][b, :-(-n // case["page"])].long()
            sees = torch.zeros(m, n, dtype=torch.bool)
            for j in range(m):
                way = _walk(trees[b], j)
                low = max(0, n - m + len(way) - case["window"]) if case["window"] else 0
                sees[j, low:n - m] = True
                if case["window"]:
                    way = way[-case["window"]:]
                sees[j, [n - m + a for a in way]] = True
            sees = sees.cuda()
            for h in range(case["kv"]):
                k = st["k_pages"][pages, h].double().reshape(-1, case["hd"])[:n]
                v = st["v_pages"][pages, h].double().reshape(-1, case["hd"])[:n]
                for i in range(h * group, (h + 1) * group):
                    s = torch.mm(st["q"][b, :m, i].double() / math.sqrt(case["hd"]), k.t())
                    y[b, :m, i] = torch.mm(torch.softmax(s.masked_fill_(~sees, -math.inf), -1), v)
        return y
    if kind == "verify":
        tokens, paths, counts = [], [], []
        trees, drafts, points = st["parents"].tolist(), st["drafted"].tolist(), st["uniforms"].tolist()
        for b in range(case["seqs"]):
            at, row, path, gone, left = 0, [], [0], [], 1.0
            for j in range(1, case["new"]):
                if trees[b][j] != at:
                    continue
                x = drafts[b][j]
                p = 0.0 if x in gone else float(st["target"][b, at, x])
                if p > 0 and points[b][j] * left < p:
                    at, gone, left = j, [], 1.0
                    row.append(x)
                    path.append(j)
                else:
                    gone.append(x)
                    left -= p
            r = st["target"][b, at].double()
            if gone:
                less = r.clone()
                less[gone] = 0
                r = less if float(less.sum()) > 0 else r
            c = r.cumsum(0)
            v = int(torch.searchsorted(c, c[-1:] * points[b][0], right=True))
            row.append(min(v, int(r.nonzero().max())))
            counts.append(len(path) - 1)
            tokens.append(row + [-1] * (case["new"] - len(row)))
            paths.append(path + [-1] * (case["new"] - len(path)))
        return tuple(torch.tensor(x, dtype=torch.int32) for x in (tokens, paths, counts))
    kp, vp = st["k_pages"].double(), st["v_pages"].double()
    lens, size = [], case["page"]
    table = st["table"].tolist()
    for b, n in enumerate(st["lens"].tolist()):
        way = [j for j in st["path"][b].tolist() if j >= 0]
        base = n - case["new"]
        for i, j in enumerate(way):  # a node never comes from before its place
            to, of = base + i, base + j
            for pool in (kp, vp):
                pool[:, table[b][to // size], :, to % size] = pool[:, table[b][of // size], :, of % size]
        lens.append(base + len(way))
    return torch.tensor(lens, dtype=torch.int32), kp, vp
