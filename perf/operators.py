"""The serving operators whose speed is tracked, each case one pass through the public entry points.

A serving step over several sequences: 4-bit projections (quantization of the activation and the
product), rotary positions with the append to a paged cache, attention of the new tokens over that
cache, and the verification of drafted tokens. Head layouts, widths and vocabularies are those of the
benchmark models (32 heads of 64 or 128 over 8 KV heads, dim 2048 and 2560, ffn 8192 and 9728, vocabulary
128256 and 151936) or generic.

`own` False computes the plain forms in elementary torch operations, True calls the framework.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # decode: the new token of one chat, heads of 128 in the half layout: pure latency
        dict(name="append_one", kind="append", seqs=1, new=1, heads=32, kv=8, hd=128, rot=128, neox=True, scaled=False,
             dtype="f32", cache="f16", page=16, longest=1000),
        # prefill: a long prompt's rows go into the cache, heads of 64 in the interleaved layout
        dict(name="append_prompt", kind="append", seqs=1, new=4096, heads=32, kv=8, hd=64, rot=64, neox=False,
             scaled=True, dtype="f32", cache="f16", page=64, longest=4096),
        # positions of a long document, half of each head rotated, frequencies scaled for the longer context
        dict(name="rope_long", kind="rope", tokens=4111, heads=40, hd=128, rot=64, neox=True, scaled=True, dtype="bf16",
             far=1000000),
        # decode: one chat in its first thousand positions, where launches and joins count
        dict(name="attend_one", kind="attend", seqs=1, new=1, heads=32, kv=8, hd=64, dtype="f32", cache="f16", page=16,
             longest=1001, window=0),
        # decode: a full batch of chats of very different lengths
        dict(name="attend_batch", kind="attend", seqs=48, new=1, heads=32, kv=8, hd=128, dtype="bf16", cache="bf16",
             page=16, longest=6000, window=0),
        # decode: two long documents, where only a split over the length fills the card
        dict(name="attend_long", kind="attend", seqs=2, new=1, heads=32, kv=8, hd=128, dtype="f16", cache="f16",
             page=64, longest=131072, window=0),
        # four drafted tokens and the one before them, over a sliding window, pages that end inside a tile
        dict(name="attend_drafts", kind="attend", seqs=13, new=5, heads=32, kv=8, hd=128, dtype="f32", cache="f16",
             page=24, longest=9000, window=4096),
        # one chat's drafts
        dict(name="verify_one", kind="verify", seqs=1, new=4, vocab=128256, drafts=True),
        # a full batch's drafts over the larger vocabulary
        dict(name="verify_batch", kind="verify", seqs=64, new=7, vocab=151936, drafts=True),
        # weights brought to 4 bits at load time, and back
        dict(name="mx_weights", kind="mxquant", rows=9728, cols=2560, dtype="bf16"),
        # decode: gate|up of one token, activation quantized on the way
        dict(name="mx_decode", kind="mxlinear", batch=1, rows=19456, cols=2560, dtype="f32", out="f32"),
        # prefill: gate|up of a long prompt
        dict(name="mx_prompt", kind="mxlinear", batch=2048, rows=16384, cols=2048, dtype="f32", out="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attend", "attend", "attend", "verify", "mxquant", "mxlinear", "mxlinear"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    cache = dtype if dtype != "f32" else rng.choice(["f16", "bf16"])
    hd = rng.choice([64, 96, 128, 128, 256])
    rot = rng.choice([hd, hd, hd // 2, 2 * rng.randint(1, hd // 2)])
    if kind == "rope":
        heads = rng.choice([1, 3, 8, 20, 32, 40])
        return dict(kind=kind, tokens=_log(rng, 1, min(65536, 50000000 // (heads * hd))), heads=heads, hd=hd, rot=rot,
                    neox=rng.random() < 0.5, scaled=rng.random() < 0.5, dtype=dtype, far=_log(rng, 1000, 1000000))
    if kind == "append":
        seqs, kv = _log(rng, 1, 64), rng.choice([1, 2, 8])
        new = rng.choice([1, 1, _log(rng, 1, max(2, 8192 // seqs))])
        return dict(kind=kind, seqs=seqs, new=new, heads=kv * rng.choice([1, 4, 5]), kv=kv, hd=hd, rot=rot,
                    neox=rng.random() < 0.5, scaled=rng.random() < 0.5, dtype=dtype, cache=cache,
                    page=rng.choice([16, 32, 64, 24]), longest=max(new, _log(rng, 16, 8192)))
    if kind == "attend":
        kv = rng.choice([1, 2, 4, 8, 8])
        room = 500000000 // (kv * hd * 4)  # positions that cost about as much as the longest listed case
        seqs = _log(rng, 1, 128)
        longest = _log(rng, 1, max(2, min(131072, room // seqs)))
        return dict(kind=kind, seqs=seqs, new=rng.choice([1, 1, 1, 2, 4, 7]), heads=kv * rng.choice([1, 4, 4, 5, 8]),
                    kv=kv, hd=hd, dtype=dtype, cache=cache, page=rng.choice([16, 32, 64, 128, 24, 1]), longest=longest,
                    window=rng.choice([0, 0, 0, _log(rng, 16, 8192)]))
    if kind == "verify":
        return dict(kind=kind, seqs=_log(rng, 1, 64), new=rng.randint(1, 8), vocab=_log(rng, 1000, 151936),
                    drafts=rng.random() < 0.7)
    cols = 32 * _log(rng, 4, 320)
    if kind == "mxquant":
        return dict(kind=kind, rows=_log(rng, 1, 16384), cols=cols, dtype=dtype)
    rows = _log(rng, 16, 20000)
    return dict(kind=kind, batch=_log(rng, 1, max(2, min(4096, 60000000000 // (rows * cols)))), rows=rows, cols=cols,
                dtype=dtype, out=rng.choice(["f32", dtype]))


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
    """theta^(-2i/rot); scaled: the low frequencies divided by 8, the ones between blended."""
    i = torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda")
    f = 500000.0 ** (-i / case["rot"])
    if case["scaled"]:
        turns = 8192 * f / (2 * math.pi)  # of the context that the model was trained on
        smooth = torch.clamp((turns - 1.0) / 3.0, 0, 1)
        f = (1 - smooth) * f / 8 + smooth * f
    return f.float()


def _pages(case, g):
    """Key and value pages in one pool, a table of its pages in random order."""
    width = -(-max(case["longest"], case["new"]) // case["page"])
    n = case["seqs"] * width + 3
    table = torch.randperm(n, device="cuda", generator=g)[:case["seqs"] * width].to(torch.int32).view(-1, width)
    shape = (n, case["kv"], case["page"], case["hd"])
    cache = DTYPES[case["cache"]]
    k = torch.empty(shape, dtype=cache, device="cuda").normal_(generator=g)
    v = torch.empty(shape, dtype=cache, device="cuda").normal_(generator=g)
    return k, v, table.contiguous()


def _probabilities(g, *shape, like=None):
    x = torch.randn(*shape, device="cuda", generator=g) * 2.5
    if like is not None:
        x = like + 0.3 * x
    return torch.softmax(x, -1), x


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _mx_quantize(x):
    """Blocks of 32: scale exponent floor(log2(max)) - 2, values to the nearest of 0 .5 1 1.5 2 3 4 6, ties to the
    even one of them. Returns (nibbles two to a byte, scale bytes)."""
    b = x.float().reshape(*x.shape[:-1], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    e = (torch.frexp(amax).exponent - 3).clamp(-127, 127)
    e = torch.where(amax > 0, e, torch.full_like(e, -127))
    a = torch.ldexp(b.abs(), -e)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp(max=6.0)
    code = torch.bucketize(a, torch.tensor(_E2M1, device=x.device)).to(torch.uint8)
    code = code | (torch.signbit(b).to(torch.uint8) << 3)
    code = code.reshape(*x.shape[:-1], -1, 2)
    return (code[..., 0] | code[..., 1] << 4).contiguous(), (e + 127).to(torch.uint8).squeeze(-1).contiguous()


def _mx_values(q, s):
    v = torch.tensor(_E2M1 + tuple(-x for x in _E2M1), device=q.device)
    c = torch.stack((q & 15, q >> 4), -1).flatten(-2)
    x = v[c.int()].reshape(*s.shape, 32)
    return torch.ldexp(x, (s.int() - 127)[..., None]).flatten(-2)


def prepare(case, seed):
    g = _gen(seed)
    kind, st = case["kind"], {"case": case}
    if kind == "rope":
        st["x"] = _normal(g, case["tokens"], case["heads"], case["hd"], dtype=case["dtype"])
        st["pos"] = torch.randint(0, case["far"], (case["tokens"],), device="cuda", generator=g, dtype=torch.int32)
        st["freqs"] = _freqs(case)
    elif kind == "append":
        n = case["seqs"] * case["new"]
        st["k_pages"], st["v_pages"], st["table"] = _pages(case, g)
        lens = _lengths(case, g)
        j = torch.arange(case["new"], device="cuda", dtype=torch.int32)
        st["pos"] = (lens[:, None] - case["new"] + j).reshape(-1).to(torch.int32).contiguous()
        st["seq"] = torch.arange(case["seqs"], device="cuda", dtype=torch.int32).repeat_interleave(case["new"])
        # one projection's rows: q, k and v are slices of it
        qkv = _normal(g, n, case["heads"] + 2 * case["kv"], case["hd"], dtype=case["dtype"])
        st["q"], st["k"], st["v"] = qkv.split([case["heads"], case["kv"], case["kv"]], 1)
        st["freqs"] = _freqs(case)
    elif kind == "attend":
        st["k_pages"], st["v_pages"], st["table"] = _pages(case, g)
        st["lens"] = _lengths(case, g)
        st["q"] = _normal(g, case["seqs"], case["new"], case["heads"], case["hd"], dtype=case["dtype"], scale=1.5)
    elif kind == "verify":
        n, new, vocab = case["seqs"], case["new"], case["vocab"]
        st["target"], logits = _probabilities(g, n, new + 1, vocab)
        st["draft"] = _probabilities(g, n, new, vocab, like=logits[:, :new])[0] if case["drafts"] else None
        source = st["draft"] if case["drafts"] else st["target"][:, :new]
        at = torch.rand(n, new, 1, device="cuda", generator=g) * 0.999
        st["drafted"] = torch.searchsorted(source.cumsum(-1), at).clamp(max=vocab - 1).squeeze(-1).to(torch.int32)
        st["uniforms"] = torch.rand(n, new + 1, device="cuda", generator=g)
    elif kind == "mxquant":
        st["x"] = _normal(g, case["rows"], case["cols"], dtype=case["dtype"], scale=0.05)
    else:
        w = _normal(g, case["rows"], case["cols"], scale=0.05)
        st["w"], st["w_scales"] = _mx_quantize(w)
        st["x"] = _normal(g, case["batch"], case["cols"], dtype=case["dtype"])
    return st


# ---- one pass -----------------------------------------------------------------------------


def _rotate(x, pos, freqs, neox, scale):
    """x [tokens, heads, hd] in 32 bits, the angles in 64."""
    a = pos.double()[:, None] * freqs.double()
    c, s = (torch.cos(a) * scale).float()[:, None], (torch.sin(a) * scale).float()[:, None]
    r = 2 * freqs.numel()
    x = x.float()
    h, rest = x[..., :r], x[..., r:]
    x0, x1 = (h[..., :r // 2], h[..., r // 2:]) if neox else (h[..., 0::2], h[..., 1::2])
    y0, y1 = x0 * c - x1 * s, x0 * s + x1 * c
    y = torch.cat((y0, y1), -1) if neox else torch.stack((y0, y1), -1).flatten(-2)
    return torch.cat((y, rest), -1)


def _amplitude(case):
    return 1.2079 if case["scaled"] else 1.0


def _seen(lens, new, width, window):
    """[seqs, new, width]: which positions each new token attends to."""
    t = torch.arange(width, device="cuda", dtype=torch.int32)
    at = lens[:, None] - new + torch.arange(new, device="cuda", dtype=torch.int32)
    ok = t <= at[..., None]
    return ok & (t > at[..., None] - window) if window else ok


def _attend(st):
    case, q = st["case"], st["q"]
    n, new, heads, hd = q.shape
    kv, page = case["kv"], case["page"]
    width = st["table"].shape[1] * page
    idx = st["table"].long()
    k = st["k_pages"][idx].float().transpose(1, 2).reshape(n, kv, width, hd)
    v = st["v_pages"][idx].float().transpose(1, 2).reshape(n, kv, width, hd)
    live = torch.arange(width, device="cuda") < st["lens"][:, None]
    v = torch.where(live[:, None, :, None], v, torch.zeros((), device="cuda"))
    rows = q.float().reshape(n, new, kv, heads // kv, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, hd)
    s = torch.matmul(rows, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(hd))
    ok = _seen(st["lens"], new, width, case["window"])
    ok = ok[:, None, :, None].expand(n, kv, new, heads // kv, width).reshape(n, kv, -1, width)
    s = torch.where(ok, s, torch.full((), -math.inf, device="cuda"))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(s - m)
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(l > 0, l, torch.ones_like(l))
    return o.reshape(n, kv, new, heads // kv, hd).permute(0, 2, 1, 3, 4).reshape(q.shape).to(q.dtype)


def _verify(st):
    target, draft, drafted, u = st["target"], st["draft"], st["drafted"].long(), st["uniforms"].double()
    n, new = drafted.shape
    p = target[:, :new].gather(2, drafted[..., None]).squeeze(-1).double()
    q = draft.gather(2, drafted[..., None]).squeeze(-1).double() if draft is not None else torch.ones_like(p)
    took = torch.cumprod((u[:, :new] * q < p).int(), 1)
    count = took.sum(1)
    b = torch.arange(n, device="cuda")
    row = target[b, count].double()
    at = count.clamp(max=new - 1)
    if draft is not None:
        less = draft[b, at].double()
    else:
        less = torch.zeros_like(row).scatter_(1, drafted[b, at][:, None], math.inf)
    r = torch.where((count < new)[:, None], torch.clamp(row - less, min=0), row)
    r = torch.where(r.sum(1, keepdim=True) > 0, r, row)
    c = r.cumsum(1)
    v = torch.arange(r.shape[1], device="cuda")
    last = torch.where(r > 0, v, torch.full_like(v, -1)).amax(1)
    token = torch.minimum((c <= u[:, new:] * c[:, -1:]).sum(1), last)
    j = torch.arange(new + 1, device="cuda")
    tokens = torch.nn.functional.pad(drafted, (0, 1))
    tokens = torch.where(j < count[:, None], tokens, torch.where(j == count[:, None], token[:, None], -1))
    return tokens.to(torch.int32), count.to(torch.int32)


def _plain(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "rope":
        return _rotate(st["x"], st["pos"], st["freqs"], case["neox"], _amplitude(case)).to(st["x"].dtype)
    if kind == "append":
        q = _rotate(st["q"], st["pos"], st["freqs"], case["neox"], _amplitude(case)).to(st["q"].dtype)
        k = _rotate(st["k"], st["pos"], st["freqs"], case["neox"], _amplitude(case))
        pos = st["pos"].long()
        at = st["table"][st["seq"].long(), pos // case["page"]].long()
        st["k_pages"][at, :, pos % case["page"]] = k.to(st["k_pages"].dtype)
        st["v_pages"][at, :, pos % case["page"]] = st["v"].to(st["v_pages"].dtype)
        return q, st["k_pages"], st["v_pages"]
    if kind == "attend":
        return _attend(st)
    if kind == "verify":
        return _verify(st)
    if kind == "mxquant":
        return _mx_values(*_mx_quantize(st["x"])).to(st["x"].dtype)
    x = _mx_values(*_mx_quantize(st["x"]))
    y = torch.matmul(x, _mx_values(st["w"], st["w_scales"]).t())
    return y.to(DTYPES[case["out"]])


def _own(st):
    from nightrun_amd import serve

    case = st["case"]
    kind = case["kind"]
    if kind == "rope":
        y = torch.empty_like(st["x"])
        serve.rope(y, st["x"], st["pos"], st["freqs"], neox=case["neox"], scale=_amplitude(case))
        return y
    if kind == "append":
        y = torch.empty(st["q"].shape, dtype=st["q"].dtype, device="cuda")
        serve.rope_append(y, st["q"], st["k"], st["v"], st["pos"], st["seq"], st["freqs"], st["k_pages"],
                          st["v_pages"], st["table"], neox=case["neox"], scale=_amplitude(case))
        return y, st["k_pages"], st["v_pages"]
    if kind == "attend":
        y = torch.empty_like(st["q"])
        serve.paged_attention(y, st["q"], st["k_pages"], st["v_pages"], st["table"], st["lens"],
                              scale=1.0 / math.sqrt(case["hd"]), window=case["window"])
        return y
    if kind == "verify":
        n, new = st["drafted"].shape
        tokens = torch.empty(n, new + 1, dtype=torch.int32, device="cuda")
        count = torch.empty(n, dtype=torch.int32, device="cuda")
        serve.verify_drafts(tokens, count, st["target"], st["draft"], st["drafted"], st["uniforms"])
        return tokens, count
    if kind == "mxquant":
        x = st["x"]
        q = torch.empty(case["rows"], case["cols"] // 2, dtype=torch.uint8, device="cuda")
        s = torch.empty(case["rows"], case["cols"] // 32, dtype=torch.uint8, device="cuda")
        serve.quantize_mxfp4(x, q, s)
        y = torch.empty_like(x)
        serve.dequantize_mxfp4(q, s, y)
        return y
    y = torch.empty(case["batch"], case["rows"], dtype=DTYPES[case["out"]], device="cuda")
    serve.linear_mxfp4(y, st["w"], st["w_scales"], st["x"])
    return y


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without -----------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["hd"] * BYTES[case["dtype"]] + 4 * case["tokens"] + 2 * case["rot"],
                "flops": 3 * n * case["rot"]}
    if kind == "append":
        n, hd = case["seqs"] * case["new"], case["hd"]
        read = (case["heads"] + 2 * case["kv"]) * hd * BYTES[case["dtype"]]
        wrote = case["heads"] * hd * BYTES[case["dtype"]] + 2 * case["kv"] * hd * 2
        return {"bytes": n * (read + wrote + 12) + 2 * case["rot"],
                "flops": 3 * n * (case["heads"] + case["kv"]) * case["rot"]}
    if kind == "attend":
        new, window = case["new"], case["window"]
        lens = _spread(case)
        total = sum(min(n, window + new - 1) if window else n for n in lens)
        pairs = sum(min(n - j, window) if window else n - j for n in lens for j in range(new))
        rows = case["seqs"] * case["new"] * case["heads"]
        return {"bytes": total * case["kv"] * case["hd"] * 4 + 2 * rows * case["hd"] * BYTES[case["dtype"]],
                "flops": 4 * pairs * case["heads"] * case["hd"]}
    if kind == "verify":
        n, new, vocab = case["seqs"], case["new"], case["vocab"]
        return {"bytes": n * (vocab * (8 if case["drafts"] else 4) + 20 * new + 12), "flops": 3 * n * vocab}
    if kind == "mxquant":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * BYTES[case["dtype"]] + n * 17 // 32, "flops": 4 * n}
    n = case["rows"] * case["cols"]
    return {"bytes": n * 17 // 32 + case["batch"] * (case["cols"] * BYTES[case["dtype"]] +
                                                     case["rows"] * BYTES[case["out"]]),
            "flops": 2 * n * case["batch"]}


# ---- the definitions in 64 bits ----------------------------------------------------------------


def _exact_rotate(x, pos, freqs, neox, scale):
    """Each pair as a complex number, times scale * e^(i * pos * freq)."""
    x = x.double()
    n = freqs.numel()
    pairs = torch.arange(n, device="cuda")
    re, im = (pairs, pairs + n) if neox else (2 * pairs, 2 * pairs + 1)
    turn = torch.polar(torch.full((), scale, dtype=torch.float64, device="cuda").expand(pos.numel(), n).contiguous(),
                       torch.outer(pos.double(), freqs.double()))
    z = torch.complex(x[..., re], x[..., im]) * turn[:, None]
    y = x.clone()
    y[..., re], y[..., im] = z.real, z.imag
    return y


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "rope":
        return _exact_rotate(st["x"], st["pos"], st["freqs"], case["neox"], _amplitude(case))
    if kind == "append":
        q = _exact_rotate(st["q"], st["pos"], st["freqs"], case["neox"], _amplitude(case))
        k = _exact_rotate(st["k"], st["pos"], st["freqs"], case["neox"], _amplitude(case))
        kp, vp = st["k_pages"].double(), st["v_pages"].double()
        pages = st["table"].long().flatten()[st["seq"].long() * st["table"].shape[1] + st["pos"].long() // case["page"]]
        slots = pages * case["page"] + st["pos"].long() % case["page"]
        for pool, rows in ((kp, k), (vp, st["v"].double())):
            flat = pool.transpose(1, 2).contiguous().view(-1, case["kv"], case["hd"])
            flat[slots] = rows
            pool.copy_(flat.view(pool.shape[0], case["page"], case["kv"], case["hd"]).transpose(1, 2))
        return q, kp, vp
    if kind == "attend":
        q = st["q"].double()
        y = torch.zeros_like(q)
        group = case["heads"] // case["kv"]
        for b, n in enumerate(st["lens"].tolist()):
            pages = st["table"][b, :-(-n // case["page"])].long()
            k = st["k_pages"][pages].double().transpose(0, 1).reshape(case["kv"], -1, case["hd"])[:, :n]
            v = st["v_pages"][pages].double().transpose(0, 1).reshape(case["kv"], -1, case["hd"])[:, :n]
            for j in range(case["new"]):
                end = n - case["new"] + j + 1
                at = slice(max(0, end - case["window"]) if case["window"] else 0, end)
                rows = q[b, j].view(case["kv"], group, case["hd"]) / math.sqrt(case["hd"])
                w = torch.softmax(torch.bmm(rows, k[:, at].transpose(1, 2).contiguous()), -1)
                y[b, j] = torch.bmm(w, v[:, at].contiguous()).reshape(case["heads"], case["hd"])
        return y
    if kind == "verify":
        tokens, counts = [], []
        for b in range(case["seqs"]):
            row, u, n = [], st["uniforms"][b].tolist(), 0
            while n < case["new"]:
                d = int(st["drafted"][b, n])
                q = float(st["draft"][b, n, d]) if case["drafts"] else 1.0
                if not u[n] * q < float(st["target"][b, n, d]):
                    break
                row.append(d)
                n += 1
            r = st["target"][b, n].double()
            if n < case["new"]:
                if case["drafts"]:
                    left = (r - st["draft"][b, n].double()).clamp(min=0)
                else:
                    left = r.clone()
                    left[int(st["drafted"][b, n])] = 0
                r = left if float(left.sum()) > 0 else r
            c = r.cumsum(0)
            at = int(torch.searchsorted(c, c[-1:] * u[case["new"]], right=True))
            row.append(min(at, int(r.nonzero().max())))
            tokens.append(row + [-1] * (case["new"] - n))
            counts.append(n)
        return torch.tensor(tokens, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32)
    grid = torch.tensor(_E2M1, dtype=torch.float64, device="cuda")

    def nearest(x):
        """The values that blocks of 32 of x stand for: the nearest of the grid, the even code of two as near."""
        b = x.double().reshape(-1, 32)
        top = b.abs().amax(1, keepdim=True)
        scale = 2.0 ** (torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top)))) - 2)
        a = b.abs() / scale
        up = torch.searchsorted(grid, a.clamp(max=6.0)).clamp(max=7)
        down = (up - 1).clamp(min=0)
        over, under = grid[up] - a, a - grid[down]
        pick = torch.where(over < under, up, torch.where(over > under, down, torch.where(up % 2 == 0, up, down)))
        pick = torch.where(a >= 6, torch.full_like(pick, 7), pick)
        return (grid[pick] * torch.sign(b) * scale).reshape(x.shape)

    if kind == "mxquant":
        return nearest(st["x"])
    w = torch.stack((st["w"] & 15, st["w"] >> 4), -1).reshape(case["rows"], -1)
    w = torch.where(w >= 8, -1.0, 1.0).double() * grid[(w & 7).long()]
    w = w * (2.0 ** (st["w_scales"].double() - 127)).repeat_interleave(32, 1)
    return torch.mm(nearest(st["x"]), w.t())
