"""The serving operators (include/nrq_serve.h, nightrun_amd.serve) against their
definitions in 64 bits.

Tolerances are bounds on the arithmetic: u = 2^-24 is the most that one f32
rounding changes a value by, relative to it, half an eps that of a 16-bit output. What
is whole (tokens, counts, 4-bit codes, scale bytes) is compared for equality.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def dt(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def half_step(name):
    import torch

    return torch.finfo(dt(name)).eps / 2


def gen(seed):
    import torch

    return torch.Generator().manual_seed(seed)


def normal(g, *shape, kind="f32", scale=1.0):
    import torch

    return (torch.randn(*shape, generator=g) * scale).to(dt(kind)).cuda()


def f64(t):
    return t.detach().double().cpu().numpy()


# ---- rotary positions -------------------------------------------------------------------------


def turn(x, pos, freqs, neox, scale):
    """(rotated, magnitude): x [tokens, heads, hd] in 64 bits; the magnitude is |x0| + |x1| of each pair, times scale."""
    n = len(freqs)
    a = np.asarray(pos, np.float64)[:, None] * np.asarray(freqs, np.float64)
    c, s = np.cos(a)[:, None] * scale, np.sin(a)[:, None] * scale
    i0, i1 = (np.arange(n), np.arange(n) + n) if neox else (2 * np.arange(n), 2 * np.arange(n) + 1)
    y, m = x.copy(), np.zeros_like(x)
    x0, x1 = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    m[..., i0] = m[..., i1] = (np.abs(x0) + np.abs(x1)) * abs(scale)
    return y, m


def rope_tolerance(y, m, kind, far):
    """Sine and cosine are off by at most: the turn's 64-bit rounding, 3 * 2^-53 of far radians; 3 u in the quarter
    turn's conversion, constant and product (an angle below 1); 3 u in the sums (each step's rounding weighs less
    than the one after it, the dropped terms are below u / 32); u in times scale. Then one product and one fused
    product-sum, 2 u, and the output's rounding."""
    return m * (9 * U + 3 * 2.0 ** -53 * far) + np.abs(y) * half_step(kind) + 1e-30


FREQS = {}


def freqs(n, base=10000.0):
    return (base ** (-np.arange(n) / n)).astype(np.float32)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("tokens,heads,hd,nf", [(1, 1, 2, 1), (1, 40, 128, 64), (3, 5, 64, 32), (7, 3, 96, 48),
                                                (130, 8, 128, 32), (5, 2, 66, 33), (9, 3, 80, 11), (2, 1, 1024, 512),
                                                (700, 2, 64, 3), (33, 4, 256, 128)])
def test_rope(gpu, kind, neox, tokens, heads, hd, nf):
    import torch

    from nightrun_amd import serve

    g = gen(tokens * 1000 + hd + nf)
    x = normal(g, tokens, heads, hd, kind=kind)
    far = 2 ** 20
    pos = torch.randint(0, far, (tokens,), generator=g, dtype=torch.int32).cuda()
    pos[0] = 0
    f = freqs(nf)
    fd = torch.from_numpy(f).cuda()
    y = torch.full_like(x, 7.0)
    serve.rope(y, x, pos, fd, neox=neox, scale=1.25)
    want, m = turn(f64(x), pos.cpu().numpy(), f, neox, 1.25)
    got = f64(y)
    assert np.all(np.abs(got - want) <= rope_tolerance(want, m, kind, far))
    assert np.array_equal(got[..., 2 * nf:], f64(x)[..., 2 * nf:])  # copied to the bit
    z = x.clone()
    serve.rope(z, z, pos, fd, neox=neox, scale=1.25)  # in place
    assert torch.equal(z, y)


def test_rope_far_positions_and_strides(gpu):
    """The largest and negative positions; slices of a wider projection, not 16-byte aligned; a broadcast input."""
    import torch

    from nightrun_amd import serve

    g = gen(5)
    wide = normal(g, 6, 9, 67)
    x = wide[:, 2:5, 1:65]
    out = torch.full((6, 4, 70), 3.0, device="cuda")
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31, -1, 2 ** 30 + 1, 123456789, 0], dtype=torch.int32).cuda()
    f = freqs(32, 1e6)
    fd = torch.from_numpy(f).cuda()
    for neox in (False, True):
        out.fill_(3.0)
        serve.rope(out[:, 1:, 3:67], x, pos, fd, neox=neox)
        want, m = turn(f64(x), pos.cpu().numpy(), f, neox, 1.0)
        got = f64(out)
        assert np.all(np.abs(got[:, 1:, 3:67] - want) <= rope_tolerance(want, m, "f32", 2.0 ** 31))
        assert np.all(got[:, 0] == 3) and np.all(got[..., :3] == 3) and np.all(got[..., 67:] == 3)
        one = normal(g, 1, 1, 64)
        serve.rope(out[:, 1:, 3:67], one.expand(6, 3, 64), pos, fd, neox=neox)
        want, m = turn(f64(one.expand(6, 3, 64)), pos.cpu().numpy(), f, neox, 1.0)
        assert np.all(np.abs(f64(out)[:, 1:, 3:67] - want) <= rope_tolerance(want, m, "f32", 2.0 ** 31))


# ---- the append to the cache ----------------------------------------------------------------


def pool(pages, kv, size, hd, cache, fill, layout="heads"):
    """A pool of `fill`: [pages][kv][size][hd], or a view of [pages][size][kv][hd]."""
    import torch

    if layout == "heads":
        return torch.full((pages, kv, size, hd), fill, dtype=dt(cache), device="cuda")
    return torch.full((pages, size, kv, hd), fill, dtype=dt(cache), device="cuda").transpose(1, 2)


@pytest.mark.parametrize("kind,cache", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"),
                                        ("f16", "bf16"), ("bf16", "f16")])
@pytest.mark.parametrize("neox,hd,nf,size,layout,heads,kv", [(True, 128, 64, 16, "heads", 32, 8), (False, 64, 32, 24, "rows", 5, 5),
                                                             (True, 96, 20, 1, "heads", 6, 2), (False, 256, 127, 7, "rows", 4, 1)])
def test_rope_append(gpu, kind, cache, neox, hd, nf, size, layout, heads, kv):
    """Slices of one projection; padding rows, positions behind the table, entries that are no page: left alone."""
    import torch

    from nightrun_amd import serve

    seqs, width = 3, 5
    g = gen(hd + size)
    pages = seqs * width + 2
    table = torch.randperm(pages, generator=g)[:seqs * width].to(torch.int32).view(seqs, width)
    table[1, 2], table[2, 0] = -1, pages
    rows = []  # (seq, pos)
    for s in range(seqs):
        rows += [(s, p) for p in range(0, width * size, max(1, size // 3))] + [(s, width * size), (s, width * size + 9)]
    rows += [(-1, 3), (seqs, 3), (0, -1), (2 ** 31 - 1, 0), (0, 2 ** 31 - 1)]
    order = torch.randperm(len(rows), generator=g).tolist()
    rows = [rows[i] for i in order]
    n = len(rows)
    seq = torch.tensor([r[0] for r in rows], dtype=torch.int32)
    pos = torch.tensor([r[1] for r in rows], dtype=torch.int32)
    qkv = normal(g, n, heads + 2 * kv, hd, kind=kind)
    q, k, v = qkv.split([heads, kv, kv], 1)
    f = freqs(nf)
    kp, vp = pool(pages, kv, size, hd, cache, 5.0, layout), pool(pages, kv, size, hd, cache, 6.0, layout)
    y = torch.full((n, heads, hd), 9.0, dtype=dt(kind), device="cuda")
    serve.rope_append(y, q, k, v, pos.cuda(), seq.cuda(), torch.from_numpy(f).cuda(), kp, vp, table.cuda(), neox=neox,
                      scale=0.75)
    far = 2.0 ** 31
    wq, mq = turn(f64(q), pos.numpy(), f, neox, 0.75)
    wk, mk = turn(f64(k), pos.numpy(), f, neox, 0.75)
    tq, tk = rope_tolerance(wq, mq, kind, far), rope_tolerance(wk, mk, cache, far)
    want_k, tol_k = np.full(kp.shape, 5.0), np.zeros(kp.shape)
    want_v = torch.full(vp.shape, 6.0, dtype=dt(cache))
    gy = f64(y)
    for i, (s, p) in enumerate(rows):
        if not (0 <= s < seqs and p >= 0):
            assert np.all(gy[i] == 9.0), (s, p)
            continue
        assert np.all(np.abs(gy[i] - wq[i]) <= tq[i]), (s, p)
        page = int(table[s, p // size]) if p < width * size else -1
        if 0 <= page < pages:
            want_k[page, :, p % size], tol_k[page, :, p % size] = wk[i], tk[i]
            want_v[page, :, p % size] = v[i].cpu().to(dt(cache))
    assert np.all(np.abs(f64(kp) - want_k) <= tol_k)
    assert torch.equal(vp.cpu(), want_v)
    p2, v2 = kp.clone(), vp.clone()
    q2 = qkv.clone().split([heads, kv, kv], 1)[0]
    serve.rope_append(q2, q2, k, v, pos.cuda(), seq.cuda(), torch.from_numpy(f).cuda(), p2, v2, table.cuda(),
                      neox=neox, scale=0.75)  # q in place
    good = (seq >= 0) & (seq < seqs) & (pos >= 0)
    assert torch.equal(q2.cpu()[good], y.cpu()[good]) and torch.equal(q2.cpu()[~good], q.cpu()[~good])
    assert torch.equal(p2, kp) and torch.equal(v2, vp)


# ---- attention ---------------------------------------------------------------------------------


class Cache:
    """A paged cache of random values, garbage where nothing was written."""

    def __init__(self, g, lens, kv, hd, size, cache, width=None, layout="heads", garbage=float("nan")):
        import torch

        self.lens, self.size, self.kv, self.hd = list(lens), size, kv, hd
        need = max([1] + [-(-max(n, 0) // size) for n in lens])
        self.width = width or need
        seqs = len(lens)
        pages = seqs * self.width + 2
        self.kp, self.vp = (pool(pages, kv, size, hd, cache, garbage, layout) for _ in range(2))
        self.table = torch.randperm(pages, generator=g)[:seqs * self.width].to(torch.int32).view(seqs, self.width)
        self.k, self.v = [], []
        for b, n in enumerate(lens):
            n = min(max(n, 0), self.width * size)
            k, v = (torch.randn(n, kv, hd, generator=g).to(dt(cache)) for _ in range(2))
            self.k.append(k)
            self.v.append(v)
            for rows, pages_ in ((k, self.kp), (v, self.vp)):
                t = torch.arange(n)
                pages_[self.table[b].long()[t // size].cuda(), :, (t % size).cuda()] = rows.cuda()

    def dev(self):
        import torch

        return self.kp, self.vp, self.table.cuda(), torch.tensor(self.lens, dtype=torch.int32, device="cuda")


def attention(q, c, counts, scale, window, gone=()):
    """(out, bound per value, lse) in 64 bits. q [seqs, new, heads, hd]; gone: (sequence, table column) without a page.

    The bound: a score is off by at most (hd + 2^2) u A with A the largest sum of |q_d k_d| scale (its sum's
    roundings and the pieces', 2^-22 relative), and 3 u of itself times the largest score for the changes of unit; so a weight is off
    by 2 e^(2d) - 2 relative, its pieces by 2^-15 (two bf16) at worst, and sums of T weights by (T + 8) u."""
    seqs, new, heads, hd = q.shape
    group = heads // c.kv
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    lse = np.full(q.shape[:3], -np.inf)
    for b in range(seqs):
        k, v = c.k[b].double().numpy(), c.v[b].double().numpy()
        n = len(k)
        m = counts[b]
        for j in range(m):
            p = n - m + j
            at = [t for t in range(max(0, p - window + 1) if window else 0, p + 1) if (b, t // c.size) not in gone]
            if not at:
                continue
            kk, vv = k[at], v[at]
            for h in range(heads):
                s = kk[:, h // group] @ q[b, j, h] * scale
                size = float((np.abs(kk[:, h // group]) @ np.abs(q[b, j, h])).max()) * abs(scale)
                d = (hd + 4) * U * size + 3 * U * float(np.abs(s).max())
                top = s.max()
                w = np.exp(s - top)
                out[b, j, h] = w @ vv[:, h // group] / w.sum()
                lse[b, j, h] = top + math.log(w.sum())
                weight = w @ np.abs(vv[:, h // group]) / w.sum()
                tol[b, j, h] = weight * (2 * math.expm1(2 * d) + 2 * (len(at) + 8) * U)
    return out, tol, lse


PIECES = {("f32", "f16"): 2.0 ** -21, ("f32", "bf16"): 2.0 ** -22, ("f16", "f16"): 2.0 ** -21,
          ("bf16", "bf16"): 2.0 ** -15, ("bf16", "f16"): 2.0 ** -21, ("f16", "bf16"): 2.0 ** -22}


def check_attention(c, kind, cache, new, heads, window=0, counts=None, q=None, scale=None, seed=1, gone=(), lse=True,
                    stream=None):
    import torch

    from nightrun_amd import serve

    g = gen(seed)
    seqs = len(c.lens)
    q = normal(g, seqs, new, heads, c.hd, kind=kind, scale=1.5) if q is None else q
    scale = c.hd ** -0.5 if scale is None else scale
    y = torch.full(q.shape, 11.0, dtype=q.dtype, device="cuda")
    ls = torch.full(q.shape[:3], 12.0, device="cuda") if lse else None
    kp, vp, table, lens = c.dev()
    cnt = torch.tensor(counts, dtype=torch.int32, device="cuda") if counts is not None else None
    serve.paged_attention(y, q, kp, vp, table, lens, scale, window=window, counts=cnt, lse=ls)
    use = [min(max(x, 0), new) for x in counts] if counts is not None else [new] * seqs
    want, tol, wl = attention(f64(q), c, use, scale, window, gone)
    got = f64(y)
    # every |v| behind an output weighs at most max |v|: the pieces of the weights
    for b in range(seqs):
        top = float(c.v[b].abs().max()) if len(c.v[b]) else 0.0
        tol[b] += PIECES[kind, cache] * top
    tol += half_step(kind) * np.abs(want)
    for b in range(seqs):
        assert np.all(got[b, use[b]:] == 11.0)
        assert np.all(np.abs(got[b, :use[b]] - want[b, :use[b]]) <= tol[b, :use[b]] + 1e-30), \
            (b, float(np.abs(got[b, :use[b]] - want[b, :use[b]]).max()))
        if lse:
            gl, w = f64(ls)[b, :use[b]], wl[b, :use[b]]
            none = np.isneginf(w)
            assert np.all(np.isneginf(gl[none]))
            # off by what the scores and the sum are, as the outputs: their relative bound over |v|, and rounding
            assert np.all(np.abs(gl[~none] - w[~none]) <= 1e-4 + 4 * U * np.abs(w[~none]))
            assert np.all(f64(ls)[b, use[b]:] == 12.0)
    return y


@pytest.mark.parametrize("kind,cache", sorted(PIECES))
@pytest.mark.parametrize("hd,heads,kv,size", [(32, 4, 4, 16), (64, 32, 8, 16), (96, 5, 1, 24), (128, 32, 8, 16),
                                              (256, 8, 2, 7), (64, 24, 1, 1)])
def test_attention_types_and_heads(gpu, kind, cache, hd, heads, kv, size):
    c = Cache(gen(hd + size), [1, 2, 31, 200, 0, 129], kv, hd, size, cache, layout="rows" if hd == 64 else "heads")
    check_attention(c, kind, cache, 1, heads)


@pytest.mark.parametrize("new,heads,kv,window,counts", [(5, 32, 8, 0, None), (4, 4, 4, 0, None), (7, 8, 1, 50, None),
                                                        (17, 8, 2, 0, None), (3, 6, 2, 1, None), (5, 32, 8, 33, [5, 0, 1, 9, -2, 4, 3]),
                                                        (40, 4, 2, 16, [40, 0, 1, 39, 12, 17, 33])])
@pytest.mark.parametrize("kind,cache", [("f32", "f16"), ("bf16", "bf16")])
def test_attention_drafts_and_windows(gpu, kind, cache, new, heads, kv, window, counts):
    """Several new tokens, some of them before the first position (an empty row), windows that cut tiles, padding."""
    lens = [300, 5, 1, 128, 64, 0, 257]
    c = Cache(gen(new), lens, kv, 128, 24, cache, width=13)
    check_attention(c, kind, cache, new, heads, window=window, counts=counts)


@pytest.mark.parametrize("lens,kv", [([5000], 1), ([3000, 1, 7000, 0, 130], 2), ([20000], 8), (list(range(0, 700, 5)), 1)])
def test_attention_long(gpu, lens, kv):
    """Sequences that many workgroups share, beside short and empty ones; more than 64 and 128 sequences."""
    c = Cache(gen(len(lens)), lens, kv, 64, 16, "f16")
    y = check_attention(c, "f32", "f16", 1, 4 * kv)
    import torch

    assert torch.equal(y, check_attention(c, "f32", "f16", 1, 4 * kv))  # the same bits again


def test_attention_masked_garbage(gpu):
    """NaN and infinities in the cache behind the length (in the same page and the same tile), before the window, and at
    positions that only later rows see do not reach the others."""
    import torch

    for new, window in ((1, 0), (1, 20), (6, 0), (6, 20)):
        c = Cache(gen(new), [150, 40, 33], 2, 128, 16, "f16", garbage=float("inf"))
        check_attention(c, "f32", "f16", new, 4, window=window, seed=3)
        clean = check_attention(c, "f16", "f16", new, 4, window=window, seed=3)
        if new > 1:  # the last two positions hold infinities: only the last two rows see them
            for b, n in enumerate(c.lens):
                for t in (n - 2, n - 1):
                    page = int(c.table[b, t // 16])
                    c.vp[page, :, t % 16] = float("inf")
                    c.kp[page, :, t % 16, 3] = float("nan") if t == n - 1 else 0.25
            from nightrun_amd import serve

            q = normal(gen(3), 3, new, 4, 128, kind="f16", scale=1.5)
            y = torch.empty_like(q)
            kp, vp, table, lens = c.dev()
            serve.paged_attention(y, q, kp, vp, table, lens, 128 ** -0.5, window=window)
            # the rows before keep their values (the order of additions may be another one)
            want, tol, _ = attention(f64(q), c, [new] * 3, 128 ** -0.5, window)
            tol += PIECES["f16", "f16"] * max(float(v.abs().max()) for v in c.v) + half_step("f16") * np.abs(want)
            assert np.all(np.abs(f64(y) - want)[:, :new - 2] <= tol[:, :new - 2])
            assert torch.isinf(y[:, new - 2]).all() and torch.isnan(y[:, new - 1]).all()
        if window:  # before every row's window
            for b, n in enumerate(c.lens):
                for t in range(0, max(0, n - new + 1 - window)):
                    page = int(c.table[b, t // 16])
                    c.vp[page, :, t % 16] = float("nan")
                    c.kp[page, :, t % 16] = float("nan")
            if new == 1:
                assert torch.equal(clean, check_attention(c, "f16", "f16", new, 4, window=window, seed=3))


def test_attention_bad_pages_and_lengths(gpu):
    """Table entries that are no page, lengths below zero and past the table."""
    import torch

    c = Cache(gen(9), [100, 80, 64, 1000, -7], 2, 64, 16, "bf16", width=7)
    pages = c.kp.shape[0]
    c.table[0, 2], c.table[1, 0], c.table[1, 4] = -1, pages, 2 ** 31 - 1
    c.table[2, :4] = -5  # nothing left of it
    gone = {(0, 2), (1, 0), (1, 4)} | {(2, i) for i in range(4)}
    check_attention(c, "bf16", "bf16", 3, 8, gone=gone)
    check_attention(c, "f32", "bf16", 1, 2, window=20, gone=gone)
    y = torch.full((5, 0, 4, 64), 1.0, device="cuda")  # no rows, no sequences
    from nightrun_amd import serve

    kp, vp, table, lens = c.dev()
    serve.paged_attention(y, y, kp, vp, table, lens, 1.0)
    serve.paged_attention(y[:0], y[:0], kp, vp, table[:0], lens[:0], 1.0)
    z = torch.full((2, 1, 4, 64), 1.0, device="cuda")  # a table without columns, a pool without pages
    serve.paged_attention(z, z.clone(), kp[:0], vp[:0], table[:2, :0].contiguous(), lens[:2], 1.0)
    assert torch.equal(z, torch.zeros_like(z))


@pytest.mark.parametrize("window", [167, 168, 169, 2 ** 30, 2 ** 31 - 1])
def test_attention_window_past_everything(gpu, window):
    """Windows as long as the table and longer, with rows before the first position: as without one."""
    import torch

    c = Cache(gen(11), [3, 160, 0], 2, 64, 24, "f16", width=7)  # holds 168
    y = check_attention(c, "f32", "f16", 6, 4, window=window)
    assert torch.equal(y, check_attention(c, "f32", "f16", 6, 4))


def test_two_threads(gpu):
    """Calls from two host threads, each on a stream of its own, with errors in one of them."""
    import threading

    import torch

    from nightrun_amd import NrPanic, serve

    steps, out = [Step(5), Step(6)], [None, None]
    for s in steps:
        s.run()
    torch.cuda.synchronize()
    want = [s.results() for s in steps]

    def work(i):
        st = torch.cuda.Stream()
        for _ in range(20):
            steps[i].run(stream=st)
            if i:
                with pytest.raises(NrPanic):
                    serve.rope(steps[i].x.view(-1, 4, 64), steps[i].x.view(-1, 4, 64), steps[i].pos,
                               torch.ones(33, device="cuda"), stream=st)
        st.synchronize()
        out[i] = steps[i].results()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for o, w in zip(out, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))


def test_attention_extreme_scores(gpu):
    """Rows of very different sizes (weights that underflow, f32 queries past f16's range, zeros), a scale of zero."""
    import torch

    c = Cache(gen(4), [333, 70], 2, 128, 16, "f16")
    q = normal(gen(4), 2, 4, 8, 128)
    for i, f in enumerate((1e-30, 1.0, 40.0, 0.0)):
        q[:, i] *= f
    check_attention(c, "f32", "f16", 4, 8, q=q)
    check_attention(c, "f32", "f16", 4, 8, q=q * 2.0 ** 40, scale=128 ** -0.5 * 2.0 ** -40)
    check_attention(c, "f32", "f16", 4, 8, q=q * 2.0 ** -60, scale=128 ** -0.5 * 2.0 ** 60)
    check_attention(c, "f32", "f16", 4, 8, scale=0.0)
    # weights of 2^-17 to 2^-30 of the largest, many of them, all of one sign
    c.vp[...] = c.vp.abs()
    c.v = [v.abs() for v in c.v]
    q = torch.zeros(2, 1, 2, 128, device="cuda")
    for b in range(2):
        q[b, 0] = c.k[b][0].float().cuda() * 1.2
    check_attention(c, "f32", "f16", 1, 2, q=q)


def test_attention_strides_and_far_offsets(gpu):
    """q and out as slices; pools of more than 2^32 elements, whose last pages are used."""
    import torch

    from nightrun_amd import serve

    hd, kv, size = 128, 2, 16
    pages = 2 ** 32 // (hd * kv * size) + 40
    kp = torch.empty(pages, kv, size, hd, dtype=torch.float16, device="cuda")
    vp = torch.empty(pages, kv, size, hd, dtype=torch.float16, device="cuda")
    g = gen(8)
    lens = [70, 33]
    table = torch.tensor([[pages - 1 - 3 * i - b for i in range(5)] for b in range(2)], dtype=torch.int32)
    c = Cache.__new__(Cache)
    c.lens, c.size, c.kv, c.hd, c.width, c.kp, c.vp, c.table = lens, size, kv, hd, 5, kp, vp, table
    c.k, c.v = [], []
    seqs = torch.tensor(sum([[b] * n for b, n in enumerate(lens)], []), dtype=torch.int32)
    pos = torch.cat([torch.arange(n) for n in lens]).to(torch.int32)
    k, v = (torch.randn(len(seqs), kv, hd, generator=g) for _ in range(2))
    f = torch.zeros(1, device="cuda")  # no turn
    qq = torch.zeros(len(seqs), 1, hd, device="cuda")
    serve.rope_append(qq, qq, k.cuda(), v.cuda(), pos.cuda(), seqs.cuda(), f, kp, vp, table.cuda())
    for b in range(2):
        c.k.append(k[seqs == b].half())
        c.v.append(v[seqs == b].half())
    wide = normal(g, 2, 3, 6, 200)
    q = wide[:, 1:, 1:5, 9:137]
    out = torch.full((2, 2, 5, 140), 4.0, device="cuda")
    serve.paged_attention(out[:, :, 1:, 5:133], q, kp, vp, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), 0.1)
    want, tol, _ = attention(f64(q), c, [2, 2], 0.1, 0)
    got = f64(out)
    assert np.all(np.abs(got[:, :, 1:, 5:133] - want) <= tol + 2.0 ** -21 * 6)
    assert np.all(got[:, :, 0] == 4) and np.all(got[..., :5] == 4) and np.all(got[..., 133:] == 4)


# ---- verification of drafts -----------------------------------------------------------------------


def verify(target, draft, drafted, u, n):
    """One sequence in 64 bits: (tokens, accepted)."""
    target = target.astype(np.float64)
    vocab = target.shape[1]
    for i in range(n):
        d = int(drafted[i])
        q = (float(draft[i, d]) if draft is not None else 1.0) if 0 <= d < vocab else 0.0
        if not (0 <= d < vocab and float(u[i]) * q < target[i, d]):
            break
    else:
        i = n
    row = np.where(target[i] > 0, target[i], 0.0)
    r = row
    if i < n:
        if draft is not None:
            with np.errstate(invalid="ignore"):
                r = target[i] - draft[i].astype(np.float64)
            r = np.where(r > 0, r, 0.0)
        else:
            r = row.copy()
            if 0 <= int(drafted[i]) < vocab:
                r[int(drafted[i])] = 0.0
        if not r.sum() > 0:
            r = row
    c = np.cumsum(r)
    above = np.nonzero(c > float(u[-1]) * c[-1])[0]
    weight = np.nonzero(r > 0)[0]
    token = int(above[0]) if len(above) else (int(weight[-1]) if len(weight) else -1)
    return [int(x) for x in drafted[:i]] + [token] + [-1] * (target.shape[0] - 1 - i), i


def check_verify(target, draft, drafted, u, counts=None):
    import torch

    from nightrun_amd import serve

    b, rows, _ = target.shape
    tokens = torch.full((b, rows), 99, dtype=torch.int32, device="cuda")
    acc = torch.full((b,), 99, dtype=torch.int32, device="cuda")
    cnt = torch.tensor(counts, dtype=torch.int32, device="cuda") if counts is not None else None
    serve.verify_drafts(tokens, acc, target, draft, drafted, u, counts=cnt)
    t, d, x, uu = target.cpu().numpy(), draft.cpu().numpy() if draft is not None else None, drafted.cpu().numpy(), \
        u.cpu().numpy()
    for i in range(b):
        n = min(max(counts[i], 0), rows - 1) if counts is not None else rows - 1
        want, k = verify(t[i], d[i] if d is not None else None, x[i], uu[i], n)
        assert (tokens[i].tolist(), int(acc[i])) == (want, k), i
    return tokens, acc


@pytest.mark.parametrize("b,n,vocab", [(1, 4, 128256), (5, 1, 1), (3, 3, 2), (4, 7, 2047), (4, 5, 2048), (3, 2, 2049),
                                       (9, 64, 300), (2, 0, 5000), (3, 4, 600001)])
@pytest.mark.parametrize("certain", [False, True])
def test_verify(gpu, b, n, vocab, certain):
    import torch

    g = gen(vocab + n)
    logits = torch.randn(b, n + 1, vocab, generator=g) * 2
    target = torch.softmax(logits, -1)
    other = torch.softmax(logits[:, :n] + 0.3 * torch.randn(b, n, vocab, generator=g), -1)
    drafted = torch.multinomial((target[:, :n] if certain else other).reshape(-1, vocab)[:, :2 ** 24], 1,
                                generator=g).view(b, n).to(torch.int32) if n else torch.zeros(b, 0, dtype=torch.int32)
    u = torch.rand(b, n + 1, generator=g)
    if certain:
        u[:, :n] *= 0.02  # so that some are accepted
    check_verify(target.cuda(), None if certain else other.cuda(), drafted.cuda(), u.cuda())
    counts = [int(x) for x in torch.randint(-1, n + 2, (b,), generator=g)]
    check_verify(target.cuda(), None if certain else other.cuda(), drafted.cuda(), u.cuda(), counts)


def test_verify_edges(gpu):
    """Uniforms of 0, 1 and on the borders, one-hot rows, equal rows, rows without weight, NaN, tokens out of range."""
    import torch

    vocab = 5000
    t = torch.zeros(12, 3, vocab)
    d = torch.zeros(12, 2, vocab)
    u = torch.full((12, 3), 0.5)
    x = torch.zeros(12, 2, dtype=torch.int32)
    t[:, :, 17] = 0.5
    t[:, :, 4000] = 0.5
    d[:, :, 17] = 0.5
    d[:, :, 30] = 0.5
    x[:] = 17
    u[0, 0] = 1.0            # 1 * .5 < .5: refused, left is token 4000
    u[1, :2] = 0.0
    u[1, 2] = 0.0            # the first with weight
    u[2, 2] = 0.5            # cumulative .5 is not above .5: the second
    u[3, 2] = 1.0            # nothing above: the last with weight
    x[4, 0] = 30             # no target weight: refused
    t[5, 0] = d[5, 0]
    u[5, 0] = 1.0            # refused, nothing left: drawn from the target itself
    t[6] = 0.0               # no weight at all
    t[7, 0, 17] = float("nan")
    t[8, 1, 3:9] = float("nan")
    u[8, 1] = 1.0
    x[9, 0], x[9, 1] = -1, 5
    x[10, 1] = vocab
    d[11, 0] = 0.0           # certain of nothing: u * 0 < .5 accepts
    for draft in (d.cuda(), None):
        check_verify(t.cuda(), draft, x.cuda(), u.cuda())
    # rows of another layout, not 16-byte aligned
    wide = torch.zeros(12, 4, vocab + 3)
    wide[:, 1:, 1:-2] = t
    check_verify(wide.cuda()[:, 1:, 1:-2], d.cuda(), x.cuda(), u.cuda())
    # one-hot target: verification of greedy drafts
    hot = torch.zeros(3, 3, vocab)
    for i, a in enumerate(((7, 8, 9), (7, 4, 9), (1, 8, 9))):
        for j, v in enumerate(a):
            hot[i, j, v] = 1.0
    dd = torch.tensor([[7, 8]] * 3, dtype=torch.int32).cuda()
    tokens, acc = check_verify(hot.cuda(), None, dd, torch.rand(3, 3, generator=gen(1)).cuda())
    assert tokens.tolist() == [[7, 8, 9], [7, 4, -1], [1, -1, -1]] and acc.tolist() == [2, 1, 0]


def test_verify_uniforms_below_0_and_nan(gpu):
    """Drawn with 0 and with nothing above: the first and the last token with weight."""
    import torch

    from nightrun_amd import serve

    t = torch.zeros(2, 1, 3000, device="cuda")
    t[:, 0, 11], t[:, 0, 2500] = 0.25, 0.75
    u = torch.tensor([[-0.5], [float("nan")]], device="cuda")
    tokens, accepted = (torch.full(n, 9, dtype=torch.int32, device="cuda") for n in ((2, 1), (2,)))
    serve.verify_drafts(tokens, accepted, t, None, torch.zeros(2, 0, dtype=torch.int32, device="cuda"), u)
    assert tokens.tolist() == [[11], [2500]] and accepted.tolist() == [0, 0]


# ---- MXFP4 -----------------------------------------------------------------------------------------

GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])


def mx_quantize(x):
    """(codes, scale bytes) of x [rows, cols] in 64 bits."""
    rows, cols = x.shape
    b = x.reshape(rows, cols // 32, 32)
    top = np.abs(b).max(-1)
    bad = ~np.isfinite(b).all(-1)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.where(top > 0, np.floor(np.log2(np.where(top > 0, top, 1.0))), -200) - 2
    # log2 may round up to a power of two that is not reached
    e = np.where((top > 0) & (2.0 ** (e + 2) > top), e - 1, e)
    e = np.where(bad, 128, np.clip(e, -127, 127))
    a = np.where(bad[..., None], 0.0, np.abs(np.where(np.isfinite(b), b, 0.0)) / 2.0 ** e[..., None])
    dist = np.abs(a[..., None] - GRID)
    near = dist.min(-1, keepdims=True)
    tie = dist == near
    even = np.where(tie & (np.arange(8) % 2 == 0), True, False).any(-1, keepdims=True)
    pick = np.where(even, tie & (np.arange(8) % 2 == 0), tie).argmax(-1)
    pick = np.where(a > 6, 7, pick)
    sign = np.where(bad[..., None], 0, np.signbit(b))
    return (pick | sign.astype(int) << 3).reshape(rows, cols), (e + 127).astype(int)


def mx_values(codes, scales):
    s = np.where(scales == 255, np.nan, 2.0 ** (np.minimum(scales, 254).astype(np.float64) - 127))
    v = np.where(codes >= 8, -1.0, 1.0) * GRID[codes & 7]
    return v * np.repeat(s, 32, 1)


def mx_random(g, rows, cols, spread=6):
    import torch

    q = torch.randint(0, 256, (rows, cols // 2), generator=g, dtype=torch.uint8)
    s = torch.randint(127 - spread, 128 + spread, (rows, cols // 32), generator=g, dtype=torch.uint8)
    return q, s


def unpack(q):
    q = q.cpu().numpy()
    return np.stack((q & 15, q >> 4), -1).reshape(q.shape[0], -1).astype(int)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 64), (17, 2560), (5, 96), (300, 1024)])
def test_mx_quantize(gpu, kind, rows, cols):
    import torch

    from nightrun_amd import serve

    g = gen(rows + cols)
    x = torch.randn(rows, cols, generator=g)
    x *= 2.0 ** torch.randint(-8, 8, (rows, cols // 32), generator=g).repeat_interleave(32, 1)
    x = x.to(dt(kind))
    for src in (x.cuda(), torch.nn.functional.pad(x, (1, 2)).cuda()[:, 1:-2]):  # aligned, and not
        q = torch.full((rows, cols // 2), 77, dtype=torch.uint8, device="cuda")
        s = torch.full((rows, cols // 32), 77, dtype=torch.uint8, device="cuda")
        serve.quantize_mxfp4(src, q, s)
        codes, scales = mx_quantize(x.double().numpy())
        assert np.array_equal(unpack(q), codes) and np.array_equal(s.cpu().numpy(), scales)
        for out in ("f32", "f16", "bf16"):
            wide = torch.full((rows, cols + 3), 5.0, dtype=dt(out), device="cuda")
            for y in (torch.empty(rows, cols, dtype=dt(out), device="cuda"), wide[:, 1:-2]):
                serve.dequantize_mxfp4(q, s, y)
                want = torch.from_numpy(mx_values(codes, scales)).float().to(dt(out))
                assert torch.equal(y.cpu(), want)
            assert torch.all(wide[:, 0] == 5) and torch.all(wide[:, -2:] == 5)


def test_mx_every_code_and_scale(gpu):
    """All 16 codes at all 256 scales back to values, and the values to codes again; ties, signs of zeros,
    the smallest numbers, infinities and NaN."""
    import torch

    from nightrun_amd import serve

    q = torch.arange(16, dtype=torch.uint8).repeat(256, 2)
    packed = (q[:, 0::2] | q[:, 1::2] << 4).contiguous().cuda()
    s = torch.arange(256, dtype=torch.uint8).view(256, 1).cuda()
    y = torch.empty(256, 32, device="cuda")
    serve.dequantize_mxfp4(packed, s, y)
    with np.errstate(over="ignore", invalid="ignore"):
        want = mx_values(q.numpy().astype(int), s.cpu().numpy()).astype(np.float32)
    got = y.cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[:255], want[:255])
    assert np.array_equal(np.signbit(got[:255]), np.signbit(want[:255]))
    fine = want[2:253]  # 6 * 2^125 is the largest that is finite; below 2^-126 the scale stays at its least
    q2, s2 = torch.empty_like(packed[2:253]), torch.empty_like(s[2:253])
    serve.quantize_mxfp4(y[2:253].contiguous(), q2, s2)
    assert torch.equal(q2, packed[2:253]) and torch.equal(s2, s[2:253])
    rows = []
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5, 7.0, 7.99]
    ties += [np.nextafter(np.float32(t), np.float32(d)) for t in ties for d in (0, 9)]
    ties = (ties + [4.0, -0.0])
    assert len(ties) == 32
    for scale in (1.0, 2.0 ** -100, 2.0 ** 100, -1.0, 2.0 ** -125, 2.0 ** -126, 2.0 ** -127, 2.0 ** -130, 2.0 ** -149):
        rows.append(np.array(ties, np.float32) * np.float32(scale))
    for bad in (np.nan, np.inf, -np.inf):
        r = np.ones(32, np.float32)
        r[13] = bad
        rows.append(r)
    rows.append(np.zeros(32, np.float32))
    rows.append(np.full(32, np.finfo(np.float32).max, np.float32))
    rows.append(np.full(32, np.float32(2.0 ** -149)))
    x = np.stack(rows)
    q3 = torch.empty(len(x), 16, dtype=torch.uint8, device="cuda")
    s3 = torch.empty(len(x), 1, dtype=torch.uint8, device="cuda")
    serve.quantize_mxfp4(torch.from_numpy(x).cuda(), q3, s3)
    codes, scales = mx_quantize(x.astype(np.float64))
    assert np.array_equal(s3.cpu().numpy(), scales)
    assert np.array_equal(unpack(q3), codes)
    assert np.all(fine == fine)


def check_product(y, xc, xs, wc, ws, kind):
    """Blocks are exact; their scaled sums and the sum over blocks round: (blocks + 2) u of the sum of magnitudes."""
    x, w = mx_values(xc, xs), mx_values(wc, ws)
    want, size = x @ w.T, np.abs(x) @ np.abs(w).T
    tol = (xs.shape[1] + 2) * U * size + half_step(kind) * np.abs(want)
    got = f64(y)
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(got - want) <= tol)
    if kind == "f16":  # 65520 and more round to infinity
        over = np.isinf(got) & (got * want > 0) & (np.abs(want) + tol >= 65520)
        bad = (bad & ~over) | (~over & (np.abs(want) - tol >= 65520))
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3].tolist())


@pytest.mark.parametrize("batch,rows,cols", [(1, 1, 32), (1, 40, 64), (1, 4100, 2560), (3, 16, 96), (16, 33, 512),
                                             (17, 70, 160), (64, 300, 1024), (65, 129, 352), (130, 257, 288),
                                             (300, 512, 2048), (257, 1000, 128), (512, 24, 4128), (1000, 515, 256), (300, 700, 640),
                                             (200, 150, 416), (513, 130, 480), (129, 1030, 1312), (1100, 600, 544),
                                             (70, 3000, 2080), (2100, 8300, 512), (4200, 4100, 544)])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_mx_matmul(gpu, kind, batch, rows, cols):
    import torch

    from nightrun_amd import serve

    g = gen(batch * 7 + rows + cols)
    w, ws = mx_random(g, rows, cols)
    x, xs = mx_random(g, batch, cols)
    wide = torch.full((batch, rows + 5), 3.0, dtype=dt(kind), device="cuda")
    y = wide[:, 2:2 + rows]
    serve.matmul_mxfp4(y, w.cuda(), ws.cuda(), x.cuda(), xs.cuda())
    check_product(y, unpack(x), xs.numpy(), unpack(w), ws.numpy(), kind)
    assert torch.all(wide[:, :2] == 3) and torch.all(wide[:, 2 + rows:] == 3)
    z = torch.empty(batch, rows, dtype=dt(kind), device="cuda")
    serve.matmul_mxfp4(z, w.cuda(), ws.cuda(), x.cuda(), xs.cuda())
    assert torch.equal(z, y)


@pytest.mark.parametrize("batch,rows,cols", [(65, 1, 2048), (70, 131, 9728), (130, 700, 2080), (200, 1000, 3136), (129, 515, 8192),
                                             (500, 2500, 4096), (80, 8200, 1088), (17, 2561, 5120), (64, 40, 20032)])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_mx_matmul_in_parts(gpu, kind, batch, rows, cols):
    """Few tiles behind long rows, which several workgroups share: into odd rows and aligned ones, the same bits."""
    import torch

    from nightrun_amd import serve

    g = gen(batch + rows + cols)
    w, ws = mx_random(g, rows, cols)
    x, xs = mx_random(g, batch, cols)
    wide = torch.full((batch, rows + 6), 3.0, dtype=dt(kind), device="cuda")
    y, z = wide[:, 1:1 + rows], torch.empty(batch, rows, dtype=dt(kind), device="cuda")
    args = [t.cuda() for t in (w, ws, x, xs)]
    serve.matmul_mxfp4(y, *args)
    check_product(y, unpack(x), xs.numpy(), unpack(w), ws.numpy(), kind)
    assert torch.all(wide[:, :1] == 3) and torch.all(wide[:, 1 + rows:] == 3)
    serve.matmul_mxfp4(z, *args)
    assert torch.equal(z, y)


def test_mx_parts_in_graphs_on_two_streams(gpu):
    """Products whose sums go through a workspace, captured, replayed at once: each has its own."""
    import torch

    from nightrun_amd import serve

    sizes = [(70, 2560, 9728), (130, 700, 8192)]
    calls = []
    for batch, rows, cols in sizes:
        g = gen(rows)
        w, ws = (t.cuda() for t in mx_random(g, rows, cols))
        x = torch.randn(batch, cols, generator=g).cuda()
        y = torch.empty(batch, rows, device="cuda")
        serve.linear_mxfp4(y, w, ws, x)
        graph = torch.cuda.CUDAGraph()
        want = y.clone()
        with torch.cuda.graph(graph):
            serve.linear_mxfp4(y, w, ws, x)
        calls.append((graph, y, want, (w, ws, x), torch.cuda.Stream()))
    for _ in range(4):
        for _, y, *_ in calls:
            y.fill_(float("nan"))
        torch.cuda.synchronize()
        for graph, *_, stream in calls:
            with torch.cuda.stream(stream):
                graph.replay()
        (w, ws, x) = calls[0][3]
        z = torch.empty_like(calls[0][1])
        serve.linear_mxfp4(z, w, ws, x)  # eager work beside them
        torch.cuda.synchronize()
        assert torch.equal(z, calls[0][2]) and all(torch.equal(y, want) for _, y, want, *_ in calls)


@pytest.mark.parametrize("kind,cols", [("f32", 2080), ("bf16", 2560), ("f16", 4032)])
def test_mx_matmul_tiles_of_256(gpu, kind, cols):
    """Sizes for which the larger tiles are taken, with rows and tokens that end inside one; odd output rows."""
    import torch

    from nightrun_amd import serve

    batch, rows = 1030, 8201
    g = gen(cols)
    w, ws = mx_random(g, rows, cols)
    x, xs = mx_random(g, batch, cols)
    wide = torch.full((batch, rows + 6), 3.0, dtype=dt(kind), device="cuda")
    y = wide[:, 1:1 + rows]
    serve.matmul_mxfp4(y, w.cuda(), ws.cuda(), x.cuda(), xs.cuda())
    check_product(y, unpack(x), xs.numpy(), unpack(w), ws.numpy(), kind)
    assert torch.all(wide[:, :1] == 3) and torch.all(wide[:, 1 + rows:] == 3)
    few = torch.empty(520, rows, dtype=dt(kind), device="cuda")  # the same sums in the same order on the smaller ones
    serve.matmul_mxfp4(few, w.cuda(), ws.cuda(), x[:520].cuda(), xs[:520].cuda())
    assert torch.equal(few, y[:520])


@pytest.mark.parametrize("batch,rows,cols", [(1, 20, 96), (3, 40, 160), (70, 200, 96), (70, 200, 416), (70, 200, 480), (130, 130, 544),
                                             (70, 300, 2080), (1030, 8201, 2080), (90, 131, 9728)])
def test_mx_matmul_nan_rows_stay_alone(gpu, batch, rows, cols):
    """A row of w, or a token, whose scales are all NaN: its outputs are NaN, no other changes."""
    import torch

    from nightrun_amd import serve

    g = gen(cols + rows)
    (w, ws), (x, xs) = ([t.cuda() for t in mx_random(g, n, cols)] for n in (rows, batch))
    y, z = (torch.empty(batch, rows, device="cuda") for _ in range(2))
    serve.matmul_mxfp4(y, w, ws, x, xs)
    ws[5], xs[batch // 2] = 255, 255
    serve.matmul_mxfp4(z, w, ws, x, xs)
    lost = torch.zeros_like(y, dtype=torch.bool)
    lost[:, 5] = lost[batch // 2] = True
    assert torch.all(torch.isnan(z[lost])) and torch.equal(z[~lost], y[~lost])


@pytest.mark.parametrize("batch,rows,cols", [(1, 512, 2560), (1, 100, 10016), (2, 300, 96), (13, 1531, 2048), (5, 8, 32),
                                             (100, 300, 1056), (300, 260, 512)])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_mx_linear(gpu, kind, batch, rows, cols):
    """As quantization and product after one another, to the bit; aligned rows and others."""
    import torch

    from nightrun_amd import serve

    g = gen(rows)
    w, ws = mx_random(g, rows, cols)
    x = torch.randn(batch, cols, generator=g).to(dt(kind))
    for src in (x.cuda(), torch.nn.functional.pad(x, (1, 2)).cuda()[:, 1:-2]):
        y = torch.empty(batch, rows, dtype=dt(kind), device="cuda")
        serve.linear_mxfp4(y, w.cuda(), ws.cuda(), src)
        codes, scales = mx_quantize(x.double().numpy())
        check_product(y, codes, scales, unpack(w), ws.numpy(), kind)
        q = torch.empty(batch, cols // 2, dtype=torch.uint8, device="cuda")
        s = torch.empty(batch, cols // 32, dtype=torch.uint8, device="cuda")
        serve.quantize_mxfp4(src, q, s)
        z = torch.empty_like(y)
        serve.matmul_mxfp4(z, w.cuda(), ws.cuda(), q, s)
        assert torch.equal(y, z)


def test_mx_extreme_scales_and_nan(gpu):
    """Scales far apart, products that leave f32's range, and NaN scales, which stay in their rows and columns."""
    import torch

    from nightrun_amd import serve

    for batch, rows in ((1, 20), (20, 40), (300, 300)):
        g = gen(rows)
        w, ws = mx_random(g, rows, 256, spread=60)
        x, xs = mx_random(g, batch, 256, spread=50)
        y = torch.empty(batch, rows, device="cuda")
        serve.matmul_mxfp4(y, w.cuda(), ws.cuda(), x.cuda(), xs.cuda())
        check_product(y, unpack(x), xs.numpy(), unpack(w), ws.numpy(), "f32")
        ws[3, 5] = 255
        xs[batch - 1, 2] = 255
        serve.matmul_mxfp4(y, w.cuda(), ws.cuda(), x.cuda(), xs.cuda())
        nan = torch.isnan(y).cpu()
        assert nan[:, 3].all() and nan[batch - 1].all()
        nan[:, 3] = False
        nan[batch - 1] = False
        assert not nan.any()


def test_mx_empty(gpu):
    import torch

    from nightrun_amd import serve

    u8 = dict(dtype=torch.uint8, device="cuda")
    y = torch.full((3, 5), 2.0, device="cuda")
    serve.matmul_mxfp4(y, torch.empty(5, 0, **u8), torch.empty(5, 0, **u8), torch.empty(3, 0, **u8),
                       torch.empty(3, 0, **u8))
    assert torch.equal(y, torch.zeros_like(y))
    serve.linear_mxfp4(y[:0], torch.empty(5, 16, **u8), torch.empty(5, 1, **u8), torch.empty(0, 32, device="cuda"))
    serve.quantize_mxfp4(torch.empty(0, 32, device="cuda"), torch.empty(0, 16, **u8), torch.empty(0, 1, **u8))


# ---- refusals of the Python side -------------------------------------------------------------------


def test_refusals(gpu):
    import torch

    from nightrun_amd import NrPanic, serve

    x = torch.zeros(3, 4, 64, device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    f = torch.ones(32, device="cuda")
    for bad in (dict(pos=pos.long()), dict(pos=pos[:2]), dict(freqs=f.double()), dict(y=x.half()), dict(y=x[:2]),
                dict(x=x.transpose(1, 2)), dict(pos=pos.cpu()), dict(freqs=f[::2]), dict(x=x.cpu()),
                dict(x=x.double(), y=x.double())):
        with pytest.raises(ValueError):
            serve.rope(**{**dict(y=x, x=x, pos=pos, freqs=f), **bad})
    with pytest.raises(NrPanic):
        serve.rope(x, x, pos, torch.ones(33, device="cuda"))
    k = torch.zeros(3, 2, 64, device="cuda")
    kp = torch.zeros(9, 2, 16, 64, dtype=torch.float16, device="cuda")
    tab = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    good = dict(y=x, q=x, k=k, v=k, pos=pos, seq=pos, freqs=f, k_pages=kp, v_pages=kp, table=tab)
    for bad in (dict(k=k[:, :1]), dict(v=k.half()), dict(k_pages=kp[..., :32]), dict(v_pages=kp.bfloat16()),
                dict(table=tab.long()), dict(seq=pos[:1]), dict(v_pages=kp.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            serve.rope_append(**{**good, **bad})
    q = torch.zeros(2, 1, 4, 64, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    good = dict(y=q, q=q, k_pages=kp, v_pages=kp, table=tab, lens=lens, scale=1.0)
    for bad in (dict(q=q[:1], y=q[:1]), dict(lens=lens.long()), dict(lens=lens[:1]), dict(k_pages=kp.float(), v_pages=kp.float()),
                dict(counts=lens[:1]), dict(lse=torch.zeros(2, 4, device="cuda")), dict(q=q[..., :32], y=q[..., :32])):
        with pytest.raises(ValueError):
            serve.paged_attention(**{**good, **bad})
    with pytest.raises(NrPanic):
        serve.paged_attention(**{**good, "q": q[:, :, :3].contiguous(), "y": q[:, :, :3].contiguous()})
    t, d = torch.zeros(2, 3, 50, device="cuda"), torch.zeros(2, 2, 50, device="cuda")
    tok, acc = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    good = dict(tokens=tok, accepted=acc, target=t, draft=d, drafted=tok[:, :2].contiguous(),
                uniforms=torch.zeros(2, 3, device="cuda"))
    for bad in (dict(target=t.half()), dict(draft=t), dict(drafted=tok), dict(uniforms=d[:, :, 0]), dict(tokens=tok.long()),
                dict(accepted=tok), dict(counts=tok)):
        with pytest.raises(ValueError):
            serve.verify_drafts(**{**good, **bad})
    u8 = dict(dtype=torch.uint8, device="cuda")
    w, s = torch.zeros(5, 32, **u8), torch.zeros(5, 2, **u8)
    for bad in (dict(w=w[:, :16]), dict(w_scales=s[:4]), dict(x=torch.zeros(3, 32, device="cuda")), dict(w=w.int()),
                dict(y=torch.zeros(3, 6, device="cuda")), dict(x=torch.zeros(3, 64, dtype=torch.float64, device="cuda"))):
        with pytest.raises(ValueError):
            serve.linear_mxfp4(**{**dict(y=torch.zeros(3, 5, device="cuda"), w=w, w_scales=s,
                                         x=torch.zeros(3, 64, device="cuda")), **bad})


# ---- a serving step ----------------------------------------------------------------------------------


class Step:
    """One layer's step of three sequences with drafted tokens: projections, rotary positions with the append,
    attention, output projection, and the drafts' verification over a small vocabulary."""

    def __init__(self, seed):
        import torch

        g = gen(seed)
        self.dim, self.heads, self.kv, self.hd, self.new, self.vocab = 256, 8, 2, 64, 3, 777
        self.seqs, self.size, self.width = 3, 16, 6
        n = self.seqs * self.new
        self.x = normal(g, n, self.dim)
        rows = (self.heads + 2 * self.kv) * self.hd
        self.w = {k: tuple(t.cuda() for t in mx_random(g, *shape, spread=1))
                  for k, shape in (("qkv", (rows, self.dim)), ("o", (self.dim, self.heads * self.hd)),
                                   ("head", (self.vocab, self.dim)))}
        self.w = {k: (q, (s - 6)) for k, (q, s) in self.w.items()}  # weights around 2^-6
        self.lens = torch.tensor([3, 50, 90], dtype=torch.int32).cuda()
        j = torch.arange(self.new, dtype=torch.int32).cuda()
        self.pos = (self.lens[:, None] - self.new + j).reshape(-1).to(torch.int32).contiguous()
        self.seq = torch.arange(self.seqs, dtype=torch.int32).repeat_interleave(self.new).cuda()
        self.table = torch.randperm(20, generator=g)[:18].to(torch.int32).view(3, 6).cuda()
        shape = (20, self.kv, self.size, self.hd)
        self.kp, self.vp = (torch.randn(shape, generator=g).half().cuda() for _ in range(2))
        self.freqs = torch.from_numpy(freqs(self.hd // 2)).cuda()
        self.draft = torch.softmax(torch.randn(self.seqs, self.new - 1, self.vocab, generator=g), -1).cuda()
        self.drafted = torch.randint(0, self.vocab, (self.seqs, self.new - 1), generator=g, dtype=torch.int32).cuda()
        self.u = torch.rand(self.seqs, self.new, generator=g).cuda()
        self.qkv = torch.empty(n, rows, device="cuda")
        self.att = torch.empty(self.seqs, self.new, self.heads, self.hd, device="cuda")
        self.o = torch.empty(n, self.dim, device="cuda")
        self.logits = torch.empty(n, self.vocab, device="cuda")
        self.tokens = torch.empty(self.seqs, self.new, dtype=torch.int32, device="cuda")
        self.accepted = torch.empty(self.seqs, dtype=torch.int32, device="cuda")

    def run(self, stream=None):
        import torch

        from nightrun_amd import serve

        serve.linear_mxfp4(self.qkv, *self.w["qkv"], self.x, stream=stream)
        q, k, v = self.qkv.view(-1, self.heads + 2 * self.kv, self.hd).split([self.heads, self.kv, self.kv], 1)
        serve.rope_append(q, q, k, v, self.pos, self.seq, self.freqs, self.kp, self.vp, self.table, neox=True,
                          stream=stream)
        serve.paged_attention(self.att, q.view(self.seqs, self.new, -1, self.hd) if q.is_contiguous() else
                              q.unflatten(0, (self.seqs, self.new)), self.kp, self.vp, self.table, self.lens,
                              self.hd ** -0.5, stream=stream)
        serve.linear_mxfp4(self.o, *self.w["o"], self.att.view(-1, self.heads * self.hd), stream=stream)
        serve.linear_mxfp4(self.logits, *self.w["head"], self.o, stream=stream)
        with torch.cuda.stream(stream) if stream is not None else torch.cuda.stream(torch.cuda.current_stream()):
            self.probs = torch.softmax(self.logits, -1).view(self.seqs, self.new, self.vocab)
        serve.verify_drafts(self.tokens, self.accepted, self.probs, self.draft, self.drafted, self.u, stream=stream)

    def results(self):
        return [t.clone() for t in (self.qkv, self.kp, self.vp, self.att, self.o, self.logits, self.tokens,
                                    self.accepted)]

    def reference(self):
        """Each step in 64 bits from what the step before it gave."""
        n = self.seqs * self.new

        def linear(x, w):
            codes, scales = mx_quantize(x)
            return mx_values(codes, scales), mx_values(unpack(w[0]), w[1].cpu().numpy())

        x, w = linear(f64(self.x), self.w["qkv"])
        qkv, size = x @ w.T, np.abs(x) @ np.abs(w).T
        h = self.heads
        raw = qkv.reshape(n, h + 2 * self.kv, self.hd)
        got = f64(self.qkv).reshape(raw.shape)
        slack = ((self.dim // 32 + 2) * U * size).reshape(raw.shape)
        pos = self.pos.cpu().numpy()
        f = self.freqs.cpu().numpy()
        rq, m = turn(raw[:, :h], pos, f, True, 1.0)
        _, ms = turn(slack[:, :h], pos, f, True, 1.0)
        assert np.all(np.abs(got[:, :h] - rq) <= rope_tolerance(rq, m, "f32", 100) + ms)
        assert np.all(np.abs(got[:, h:] - raw[:, h:]) <= slack[:, h:])
        c = Cache.__new__(Cache)
        c.lens, c.size, c.kv, c.hd = self.lens.tolist(), self.size, self.kv, self.hd
        c.k, c.v = [], []
        for b, ln in enumerate(c.lens):
            t = np.arange(ln)
            pages = self.table.cpu().numpy()[b, t // self.size]
            c.k.append(self.kp.cpu()[pages, :, t % self.size])
            c.v.append(self.vp.cpu()[pages, :, t % self.size])
            want = turn(raw[b * self.new:(b + 1) * self.new, h:h + self.kv], pos[b * self.new:(b + 1) * self.new], f,
                        True, 1.0)[0]
            assert np.allclose(c.k[b].double().numpy()[-self.new:], want, rtol=2.0 ** -11, atol=1e-4)
            assert np.array_equal(c.v[b].numpy()[-self.new:],
                                  self.qkv.cpu().view(n, -1, self.hd)[b * self.new:(b + 1) * self.new, h + self.kv:].half().numpy())
        q = got[:, :h].reshape(self.seqs, self.new, h, self.hd)
        want, tol, _ = attention(q, c, [self.new] * self.seqs, self.hd ** -0.5, 0)
        assert np.all(np.abs(f64(self.att) - want) <= tol + 2.0 ** -21 * 60)
        for src, dst, w in ((f64(self.att).reshape(n, -1), self.o, self.w["o"]),
                            (f64(self.o), self.logits, self.w["head"])):
            codes, scales = mx_quantize(src)
            check_product(dst, codes, scales, unpack(w[0]), w[1].cpu().numpy(), "f32")
        p, d = self.probs.cpu().numpy(), self.draft.cpu().numpy()
        for b in range(self.seqs):
            t, k = verify(p[b], d[b], self.drafted.cpu().numpy()[b], self.u.cpu().numpy()[b], self.new - 1)
            assert (self.tokens[b].tolist(), int(self.accepted[b])) == (t, k)


def test_serving_step(gpu):
    import torch

    s = Step(1)
    s.run()
    torch.cuda.synchronize()
    s.reference()


def test_serving_step_in_graphs(gpu):
    """Two captured graphs of two steps, replayed in turn and at once on two streams with eager work between; each
    replay gives the eager results to the bit."""
    import torch

    steps = [Step(1), Step(2)]
    want = []
    for s in steps:
        s.run()
        torch.cuda.synchronize()
        want.append(s.results())
    graphs = []
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.run()
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in steps]
    for replay in range(4):
        for s in steps:
            for t in (s.qkv, s.att, s.o, s.logits):
                t.fill_(float("nan"))
            s.tokens.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st) if replay % 2 else torch.cuda.stream(torch.cuda.current_stream()):
                g.replay()
        torch.cuda.synchronize()
        for s, w in zip(steps, want):
            assert all(torch.equal(a, b) for a, b in zip(s.results(), w))
        Step(3).run()  # eager work beside them


def test_serving_step_on_a_stream(gpu):
    """The stream argument: work queued on that stream, after what it waits for and in order with it."""
    import torch

    s = Step(4)
    s.run()
    torch.cuda.synchronize()
    want = s.results()
    st = torch.cuda.Stream()
    x = s.x.clone()
    s.x.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        torch.cuda._sleep(20_000_000)
        s.x.copy_(x)
    s.run(stream=st)
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(s.results(), want))


# ---- draws at the end of the sum and at its borders ---------------------------------------------------


@pytest.mark.parametrize("vocab,rows", [(32000, 300), (50257, 300), (151936, 200), (300001, 80)])
def test_verify_draw_of_1_takes_the_last_weight(gpu, vocab, rows):
    """Dense rows, whose sums round: a last uniform of 1 has no cumulative sum above it in any order of adding up."""
    import torch

    from nightrun_amd import serve

    g = torch.Generator(device="cuda").manual_seed(vocab)
    t = torch.softmax(2.5 * torch.randn(rows, 1, vocab, device="cuda", generator=g), -1)
    t[::3, 0, -vocab // 3:] = 0.0  # whole spans without weight at the end
    u = torch.full((rows, 1), 1.0, device="cuda")
    u[1::5] = 1.5
    tokens, accepted = (torch.full(n, 99, dtype=torch.int32, device="cuda") for n in ((rows, 1), (rows,)))
    serve.verify_drafts(tokens, accepted, t, None, torch.zeros(rows, 0, dtype=torch.int32, device="cuda"), u)
    v = torch.arange(vocab, device="cuda")
    assert torch.equal(tokens[:, 0].long(), torch.where(t[:, 0] > 0, v, -1).amax(1))


@pytest.mark.parametrize("vocab,some", [(32000, None), (151936, None), (600001, None), (600001, 40), (262145, 3), (5000, 7)])
def test_verify_draws_lie_between_their_sums(gpu, vocab, some):
    """Any uniform: the token drawn has weight, and the point lies between the sums before and through it, within the
    rounding of three sums (the point's, theirs, the definition's) of up to 2^20 terms in 64 bits, each off by at most 2^20 * 2^-53 of the
    whole. Rows of `some` tokens only have most of their spans empty."""
    import torch

    from nightrun_amd import serve

    rows = 64
    g = torch.Generator(device="cuda").manual_seed(vocab + (some or 0))
    t = torch.softmax(2.5 * torch.randn(rows, 1, vocab, device="cuda", generator=g), -1)
    if some:
        keep = torch.zeros(rows, 1, vocab, device="cuda")
        keep.scatter_(2, torch.randint(0, vocab, (rows, 1, some), device="cuda", generator=g), 1.0)
        t = t * keep
    u = torch.rand(rows, 1, device="cuda", generator=g)
    u[:6, 0] = torch.tensor([0.0, 2.0 ** -149, 2.0 ** -24, 1 - 2.0 ** -24, 1 - 2.0 ** -23, 0.5])
    tokens, accepted = (torch.full(n, 99, dtype=torch.int32, device="cuda") for n in ((rows, 1), (rows,)))
    serve.verify_drafts(tokens, accepted, t, None, torch.zeros(rows, 0, dtype=torch.int32, device="cuda"), u)
    p = f64(t)[:, 0]
    c = np.cumsum(p, 1)
    at, i = tokens[:, 0].cpu().numpy(), np.arange(rows)
    assert np.all(at >= 0) and np.all(p[i, at] > 0)
    point, slack = f64(u)[:, 0] * c[:, -1], 3 * 2.0 ** -33 * c[:, -1]
    assert np.all(c[i, at] > point - slack) and np.all(c[i, at] - p[i, at] <= point + slack)


# ---- outputs over inputs ------------------------------------------------------------------------------


def test_mx_outputs_over_inputs_are_refused(gpu):
    """Workgroups read what others have written by then. Columns of one matrix beside each other are no overlap."""
    import torch

    from nightrun_amd import NrqError, serve

    def f16(t, rows, cols):  # the first bytes of t as another matrix
        return t.view(-1).view(torch.uint8)[:rows * cols * 2].view(torch.float16).view(rows, cols)

    g = gen(11)
    n = 512
    w, ws = (t.cuda() for t in mx_random(g, n, n))
    kept = w.clone()
    for batch in (1, 5, 70):  # in one launch, in two
        both = normal(g, batch, 2 * n)
        x, y = both[:, :n], both[:, n:]
        before = both.clone()
        for out in (x, both[:, n // 2:n // 2 + n], both[:, n - 1:2 * n - 1], f16(both, batch, n), f16(w, 1, n).expand(batch, n)):
            if out.stride(0) == 0 and batch > 1:
                continue
            with pytest.raises(NrqError, match="overlap"):
                serve.linear_mxfp4(out, w, ws, x)
        assert torch.equal(both, before) and torch.equal(w, kept)
        serve.linear_mxfp4(y, w, ws, x)
        alone = torch.empty(batch, n, device="cuda")
        serve.linear_mxfp4(alone, w, ws, x.contiguous())
        assert torch.equal(y, alone) and torch.equal(x, before[:, :n])
    x, xs = (t.cuda() for t in mx_random(g, 3, n))
    for t in (w, ws, x, xs):
        with pytest.raises(NrqError, match="overlap"):
            serve.matmul_mxfp4(f16(t, 3, 8), w[:8], ws[:8], x, xs)
    src, s = normal(g, 8, n), torch.empty(8, n // 32, dtype=torch.uint8, device="cuda")
    q = torch.empty(8, n // 2, dtype=torch.uint8, device="cuda")
    for out, scales in ((src.view(torch.uint8).view(-1)[:q.numel()].view(q.shape), s), (q, q.view(-1)[:s.numel()].view(s.shape))):
        with pytest.raises(NrqError, match="overlap"):
            serve.quantize_mxfp4(src, out, scales)
    serve.quantize_mxfp4(src, q, s)
    for t in (q, s):
        with pytest.raises(NrqError, match="overlap"):
            serve.dequantize_mxfp4(q[:1, :32], s[:1, :2], f16(t, 1, 64))


# ---- sizes past one launch ------------------------------------------------------------------------------


@pytest.mark.parametrize("append", [False, True])
def test_rope_more_tokens_than_a_grid_has_threads_for(gpu, append):
    """2^31 - 1 tokens (the most) of one head of two, of which a launch takes at most 64 * 2^23: all tokens share one
    input row; the positions run through a page of outputs that are checked at the launches' borders and at random."""
    import torch

    from nightrun_amd import serve

    n, span = 2 ** 31 - 1, 1 << 20
    x = torch.tensor([[[1.0, 0.5]]], dtype=torch.float16, device="cuda").expand(n, 1, 2)
    y = torch.full((n, 1, 2), 9.0, dtype=torch.float16, device="cuda")
    pos = torch.arange(span, dtype=torch.int32, device="cuda").repeat(n // span + 1)[:n]
    f = torch.tensor([0.25], device="cuda")
    if append:
        seq = torch.full((n,), -1, dtype=torch.int32, device="cuda")  # padding but for two, which lie in two launches
        at = torch.tensor([5, n - 1], device="cuda")
        seq[at] = 0
        table = torch.arange(span // 2 ** 14, dtype=torch.int32, device="cuda").view(1, -1)
        kp, vp = (torch.zeros(span // 2 ** 14, 1, 2 ** 14, 8, dtype=torch.float16, device="cuda")[..., :2] for _ in range(2))
        serve.rope_append(y, x, x, x, pos, seq, f, kp, vp, table)
    else:
        at = torch.cat([torch.tensor([0, 1, n - 1]), torch.arange(1, 4) * 2 ** 29, torch.arange(1, 4) * 2 ** 29 - 1,
                        torch.randint(0, n, (100000,), generator=gen(3))]).cuda()
        serve.rope(y, x, pos, f)
        assert int((y[:, 0, 0] == 9).sum()) == 0
    p = pos[at].double().cpu().numpy()
    want, m = turn(np.tile([[[1.0, 0.5]]], (len(p), 1, 1)), p, [0.25], False, 1.0)
    tol = rope_tolerance(want, m, "f16", span)
    assert np.all(np.abs(f64(y[at]) - want) <= tol)
    if append:
        assert bool((y[6:n - 1] == 9).all())
        got = f64(kp)[:, 0].reshape(-1, 2)[p.astype(int)]
        assert np.all(np.abs(got - want[:, 0]) <= tol[:, 0])
        assert np.array_equal(f64(vp)[:, 0].reshape(-1, 2)[p.astype(int)], np.tile([1.0, 0.5], (2, 1)))
        assert int((vp != 0).any(-1).sum()) == 2


# ---- weights of the softmax in 32 bits ----------------------------------------------------------------


@pytest.mark.parametrize("new", [1, 3])
def test_attention_weights_keep_32_bits(gpu, new):
    """bf16 throughout. Three positions weigh 1, a fourth p = exp(-c s); in dimension h the values are minus the first two
    bf16 pieces of head h's p, and 1: what is left is the third piece. Values whose third piece is 2^-18.5 and more.

    The numerator is off by: 3 u of the exponent (at most 1 in units of log2) in its unit and product, 2 u in the exponential,
    and 12 products of at most 2 added up, each sum rounded or cut: 24 u for rounding. In all 29 u, below 2^-18.5 / 1.4."""
    import torch

    from nightrun_amd import serve

    def bf(x):
        return torch.tensor(x, dtype=torch.float64).bfloat16().double().numpy()

    seqs, heads, hd, s = 16, 8, 64, 0.69
    scale = float(np.float32(s))
    c = np.concatenate([(128 + np.arange(128)) / 256, 1 - np.arange(1, 100) / 256.0])
    c = c[c >= 0.5]
    p = np.exp(-c * scale)
    third = p - bf(p) - bf(p - bf(p))
    c = c[np.abs(third) >= 2.0 ** -18.5]
    assert len(c) >= 5
    pick = np.random.default_rng(2).integers(0, len(c), (seqs, heads))
    cc = c[pick]
    p = np.exp(-cc * scale)
    one, two = bf(p), bf(p - bf(p))
    q = np.zeros((seqs, new, heads, hd))
    q[..., 0] = cc[:, None]
    k, v = np.zeros((seqs, 1, 16, hd)), np.zeros((seqs, 1, 16, hd))
    k[:, 0, 3, 0] = -1.0
    v[:, 0, 0, :heads], v[:, 0, 1, :heads], v[:, 0, 3, :heads] = -one, -two, 1.0
    qd, kd, vd = (torch.from_numpy(x).to(torch.bfloat16).cuda() for x in (q, k, v))
    y = torch.empty_like(qd)
    table = torch.arange(seqs, dtype=torch.int32, device="cuda").view(-1, 1)
    serve.paged_attention(y, qd, kd, vd, table, torch.full((seqs,), 4, dtype=torch.int32, device="cuda"), scale)
    got = f64(y)[:, -1][:, np.arange(heads), np.arange(heads)]
    want = (p - one - two) / (3 + p)
    assert np.all(np.abs(want) >= 2.0 ** -18.5 / 4)
    assert np.all(np.abs(got - want) <= 29 * U / (3 + p) + half_step("bf16") * np.abs(want))


# ---- prompts: hundreds and thousands of new tokens ------------------------------------------------------


def dense_attention(q, k, v, lens, counts, scale, window):
    """(out, bound, lse, bound of lse) in 64 bits on the device: k, v [seqs, kv, width, hd]. The bound is that of
    attention(); the logarithm of the sum is off by the scores' d, by (T + 8) u of the sum, and by 4 u of itself for the
    maximum's and the logarithm's changes of unit, each at most the larger of the maximum and the result."""
    import torch

    seqs, new, heads, hd = q.shape
    kv, width = k.shape[1], k.shape[2]
    group = heads // kv
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    ltol = torch.zeros_like(lse)
    t = torch.arange(width, device="cuda")
    for b in range(seqs):
        n = counts[b]
        p = lens[b] - n + torch.arange(n, device="cuda")
        ok = (t <= p[:, None]) & (t < lens[b])
        if window:
            ok &= t > p[:, None] - window
        seen = ok.any(1)
        for h in range(heads):
            qq, kk, vv = q[b, :n, h], k[b, h // group], v[b, h // group]
            s = (qq @ kk.t()) * scale
            size = torch.where(ok, (qq.abs() @ kk.t().abs()) * abs(scale), 0.0).amax(1)
            big = torch.where(ok, s.abs(), 0.0).amax(1)
            d = (hd + 4) * U * size + 3 * U * big
            s = torch.where(ok, s, -math.inf)
            top = torch.where(seen, s.amax(1), 0.0)
            w = torch.exp(s - top[:, None])
            total = torch.where(seen, w.sum(1), 1.0)
            terms = ok.sum(1)
            out[b, :n, h] = (w @ vv) / total[:, None]
            weight = (w @ vv.abs()) / total[:, None]
            tol[b, :n, h] = weight * (2 * torch.expm1(2 * d) + 2 * (terms + 8) * U)[:, None]
            lse[b, :n, h] = torch.where(seen, top + torch.log(total), -math.inf)
            ltol[b, :n, h] = 2 * d + (terms + 8) * U + 4 * U * (1 + torch.maximum(top.abs(), torch.log(total)))
    return out, tol, lse, ltol


@pytest.mark.parametrize("hd,heads,kv,new,lens,window,counts", [
    (256, 8, 2, 37, [300, 37, 20], 0, None), (256, 4, 4, 300, [311, 129], 100, [300, 17]), (96, 10, 2, 130, [400, 131, 7], 0, None),
    (96, 3, 1, 515, [515], 64, None), (32, 8, 1, 260, [600, 260], 0, [260, 0]), (32, 4, 4, 33, [33, 4000], 1000, None),
    (64, 32, 8, 513, [513, 1030], 0, None), (128, 16, 4, 700, [701, 699, 1500], 333, [700, 512, 1]), (64, 8, 2, 4096, [4096], 0, None),
    (128, 4, 1, 2000, [5000], 1024, None)])
@pytest.mark.parametrize("kind,cache", [("f32", "f16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16")])
def test_attention_prompts(gpu, hd, heads, kv, new, lens, window, counts, kind, cache):
    """Many row tiles a head, more rows than positions, positions that only later rows see."""
    import torch

    from nightrun_amd import serve

    size, seqs = 24, len(lens)
    g = torch.Generator(device="cuda").manual_seed(hd + new)
    width = -(-max(lens) // size) + 1
    table = torch.randperm(seqs * width + 3, device="cuda", generator=g)[:seqs * width].to(torch.int32).view(seqs, width)
    kp, vp = (torch.full((seqs * width + 3, kv, size, hd), math.inf, dtype=dt(cache), device="cuda") for _ in range(2))
    k, v = (torch.randn(seqs, kv, width * size, hd, device="cuda", generator=g).to(dt(cache)) for _ in range(2))
    for b in range(seqs):  # behind the length there are infinities
        t = torch.arange(lens[b], device="cuda")
        for rows, pages in ((k, kp), (v, vp)):
            pages[table[b].long()[t // size], :, t % size] = rows[b, :, :lens[b]].transpose(0, 1)
    q = (1.5 * torch.randn(seqs, new, heads, hd, device="cuda", generator=g)).to(dt(kind))
    y = torch.full_like(q, 11.0)
    lse = torch.full((seqs, new, heads), 12.0, device="cuda")
    serve.paged_attention(y, q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), hd ** -0.5, window=window,
                          counts=None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda"), lse=lse)
    use = counts or [new] * seqs
    want, tol, wl, ltol = dense_attention(q.double(), k.double(), v.double(), lens, use, hd ** -0.5, window)
    # the weights' pieces (within 2^-23) and the queries' (counted in hd + 4), the output's rounding
    tol += 2.0 ** -22 * v.double().abs().max() + half_step(kind) * want.abs()
    for b in range(seqs):
        n = use[b]
        assert torch.all((y[b, :n].double() - want[b, :n]).abs() <= tol[b, :n])
        assert torch.all(y[b, n:] == 11) and torch.all(lse[b, n:] == 12)
        none = torch.isneginf(wl[b, :n])
        assert torch.equal(torch.isneginf(lse[b, :n]), none) and torch.all(y[b, :n][none] == 0)
        assert torch.all(((lse[b, :n].double() - wl[b, :n]).abs() <= ltol[b, :n]) | none)


@pytest.mark.parametrize("kind,cache", sorted(PIECES))
@pytest.mark.parametrize("hd,lens,heads,kv", [(128, [1, 3, 200, 1000, 5000], 8, 2), (64, [20000], 4, 1), (256, [700, 64], 2, 1)])
def test_attention_log_sums(gpu, kind, cache, hd, lens, heads, kv):
    """The logarithm of the sum of exponentials to its rounding, with scores of a few units and of hundreds."""
    import torch

    from nightrun_amd import serve

    for scale in (hd ** -0.5, 1.0):
        c = Cache(gen(hd), lens, kv, hd, 16, cache)
        kp, vp, table, ln = c.dev()
        q = normal(gen(hd + 1), len(lens), 1, heads, hd, kind=kind, scale=1.5)
        y, lse = torch.empty_like(q), torch.empty(len(lens), 1, heads, device="cuda")
        serve.paged_attention(y, q, kp, vp, table, ln, scale, lse=lse)
        k, v = (torch.zeros(len(lens), kv, max(lens), hd, dtype=torch.float64, device="cuda") for _ in range(2))
        for b, n in enumerate(lens):
            k[b, :, :n], v[b, :, :n] = c.k[b].double().cuda().transpose(0, 1), c.v[b].double().cuda().transpose(0, 1)
        want, tol, wl, ltol = dense_attention(q.double(), k, v, lens, [1] * len(lens), scale, 0)
        assert torch.all((lse.double() - wl).abs() <= ltol)
        tol += 2.0 ** -22 * v.abs().max() + half_step(kind) * want.abs()
        assert torch.all((y.double() - want).abs() <= tol)


# ---- MXFP4 at the ends of the scales -------------------------------------------------------------------


@pytest.mark.parametrize("batch,rows,cols", [(1, 40, 2560), (5, 20, 96), (40, 70, 640), (70, 200, 96), (70, 200, 512), (70, 131, 9728), (300, 260, 2080)])
def test_mx_products_of_least_and_largest_scales(gpu, batch, rows, cols):
    """Scale bytes from 0 and up to 254: the scale of a product is the sum of both, whatever each is. Bytes past 255 start
    again at 0, so that some products are below all that 32 bits hold: there each block's sum and each addition is off by at
    most half of 2^-149, the step of the subnormal numbers, beside what check_product() allows."""
    import torch

    from nightrun_amd import serve

    g = gen(rows + cols)
    (w, ws), (x, xs) = mx_random(g, rows, cols), mx_random(g, batch, cols)
    for a, b in ((0, 250), (250, 0), (0, 240), (2, 252)):
        sw, sx = ws - ws.min() + a, xs - xs.min() + b  # 13 bytes from a and from b on
        sw, sx = sw.clamp(max=254), sx.clamp(max=254)
        y = torch.empty(batch, rows, device="cuda")
        serve.matmul_mxfp4(y, w.cuda(), sw.cuda(), x.cuda(), sx.cuda())
        vx, vw = mx_values(unpack(x), sx.numpy()), mx_values(unpack(w), sw.numpy())
        want, size = vx @ vw.T, np.abs(vx) @ np.abs(vw).T
        assert np.all(np.abs(f64(y) - want) <= (cols // 32 + 2) * (U * size + 2.0 ** -149) + half_step("f32") * np.abs(want))


def test_mx_values_back_to_their_codes(gpu):
    """What every code stands for at the scales 2^-125 to 2^125 comes back as the definition has it."""
    import torch

    from nightrun_amd import serve

    q = torch.arange(16, dtype=torch.uint8).repeat(251, 2)
    packed = (q[:, 0::2] | q[:, 1::2] << 4).contiguous().cuda()
    s = torch.arange(2, 253, dtype=torch.uint8).view(251, 1).cuda()
    y = torch.empty(251, 32, device="cuda")
    serve.dequantize_mxfp4(packed, s, y)
    fine = mx_values(q.numpy().astype(int), s.cpu().numpy()).astype(np.float32)
    assert np.array_equal(y.cpu().numpy(), fine)


# ---- more sequences than a grid has rows, columns past 32-bit offsets, mixed types ----------------------


def test_verify_more_sequences_than_a_grid_has_rows(gpu):
    """70,000 sequences in two launches each; one-hot rows of drafts accepted, refused and counted out."""
    import torch

    from nightrun_amd import serve

    b, n, vocab = 70000, 2, 33
    g = torch.Generator(device="cuda").manual_seed(2)
    best = torch.randint(0, vocab, (b, n + 1), device="cuda", generator=g)
    target = torch.zeros(b, n + 1, vocab, device="cuda").scatter_(2, best[..., None], 1.0)
    drafted = torch.where(torch.rand(b, n, device="cuda", generator=g) < 0.7, best[:, :n],
                          torch.randint(0, vocab, (b, n), device="cuda", generator=g)).to(torch.int32)
    counts = torch.randint(0, n + 1, (b,), device="cuda", generator=g, dtype=torch.int32)
    u = torch.rand(b, n + 1, device="cuda", generator=g)
    tokens, accepted = (torch.full(s, 99, dtype=torch.int32, device="cuda") for s in ((b, n + 1), (b,)))
    serve.verify_drafts(tokens, accepted, target, None, drafted, u, counts=counts)
    j = torch.arange(n, device="cuda")
    took = torch.cumprod(((drafted == best[:, :n]) & (j < counts[:, None])).int(), 1).sum(1)
    # a refused draft is not the row's one token, so that what is left out does not matter
    j = torch.arange(n + 1, device="cuda")
    want = torch.where(j <= took[:, None], best, -1)
    assert torch.equal(accepted.long(), took) and torch.equal(tokens.long(), want)


@pytest.mark.parametrize("batch", [1, 66])
@pytest.mark.parametrize("cols", [2 ** 26, 2 ** 26 + 32])
def test_mx_columns_past_32_bit_offsets(gpu, batch, cols):
    """Rows of 2^25 bytes, of which all but a few values are zeros: whole sums, exact in any order."""
    import torch

    from nightrun_amd import serve

    rows, at = 70, [0, 31, 2 ** 25 - 1, 2 ** 25, 2 ** 26 - 33, 2 ** 26 - 1, cols - 32, cols - 1]
    at = sorted(set(at))
    g = gen(cols % 1000 + batch)
    codes = []

    def sparse(n):
        c = torch.randint(0, 16, (n, len(at)), generator=g)
        q = torch.zeros(n, cols // 2, dtype=torch.uint8, device="cuda")
        for i, a in enumerate(at):
            q[:, a // 2] |= (c[:, i] << 4 * (a % 2)).to(torch.uint8).cuda()
        codes.append(c.numpy())
        return q, torch.full((n, cols // 32), 127, dtype=torch.uint8, device="cuda")

    w, ws = sparse(rows)
    x, xs = sparse(batch)
    y = torch.empty(batch, rows, device="cuda")
    serve.matmul_mxfp4(y, w, ws, x, xs)
    vw, vx = (np.where(c >= 8, -1.0, 1.0) * GRID[c & 7] for c in codes)
    assert np.array_equal(f64(y), vx @ vw.T)


@pytest.mark.parametrize("batch,rows,cols", [(1, 300, 2560), (9, 40, 96), (3, 300, 8192), (40, 70, 640), (100, 300, 1056), (70, 131, 9728)])
@pytest.mark.parametrize("kind,out", [("f32", "bf16"), ("bf16", "f32"), ("f16", "bf16"), ("f32", "f16"), ("f16", "f32"), ("bf16", "f16")])
def test_mx_linear_mixed_types(gpu, kind, out, batch, rows, cols):
    """The activation of one type, the outputs of another."""
    import torch

    from nightrun_amd import serve

    g = gen(rows + batch)
    w, ws = mx_random(g, rows, cols, spread=3)
    x = torch.randn(batch, cols, generator=g).to(dt(kind))
    y = torch.empty(batch, rows, dtype=dt(out), device="cuda")
    serve.linear_mxfp4(y, w.cuda(), ws.cuda(), x.cuda())
    codes, scales = mx_quantize(x.double().numpy())
    check_product(y, codes, scales, unpack(w), ws.numpy(), out)
