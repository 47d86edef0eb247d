"""The operators for trees of drafts (include/nrq_tree.h, nightrun_amd.serve) against their definitions in 64 bits.

Tolerances are bounds on the arithmetic: U = 2^-24 is the most that one f32 rounding changes a value by, relative
to it, half an eps that of a 16-bit output. What is whole (tokens, paths, lengths, values moved) is compared for equality.
"""
import math

import numpy as np
import pytest

from tests.test_gpu_serve import PIECES, U, Cache, dt, f64, freqs, gen, half_step, normal, pool, rope_tolerance, turn

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "bf16"), ("bf16", "f16")]


def trees(seed, seqs, n):
    """Random trees: chains, bushes and anything between, as parents [seqs][n]."""
    rng = np.random.default_rng(seed)
    p = np.full((seqs, n), -1, np.int32)
    for b in range(seqs):
        shape = rng.choice([0.3, 1.0, 3.0])
        for j in range(1, n):
            p[b, j] = min(j - 1, int(j * rng.random() ** shape))
    return p


def way(parents, j):
    """Node j and those above it, the root first."""
    out = []
    while True:
        out.append(j)
        if not 0 <= parents[j] < j:
            return out[::-1]
        j = int(parents[j])


# ---- norms with rotary positions -----------------------------------------------------------------


def norm(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 if w is None else w)


def norm_tolerance(y, m, kind, far, hd):
    """rope_tolerance of the normed rows, and what they are off by themselves: the sum of hd squares by hd + 1 roundings at
    most (half of that in the root), then the division by hd, eps, root and reciprocal (1 each, halves before the
    root) and two products: (hd / 2 + 6) U of the pair's magnitude. Half a step of f16 below its least normal value, 2^-14, is
    2^-25 whatever the value is: its subnormal values are 2^-24 apart."""
    return rope_tolerance(y, m, kind, far) + m * (hd / 2 + 6) * U + (2.0 ** -25 if kind == "f16" else 0.0)


def check_norm(x, pos, w, nf, neox, kind, eps=1e-6, scale=1.0, y=None):
    import torch

    from nightrun_amd import serve

    f = freqs(nf)
    y = torch.full_like(x, 7.0) if y is None else y
    serve.norm_rope(y, x, w, pos, torch.from_numpy(f).cuda(), eps=eps, neox=neox, scale=scale)
    want, m = turn(norm(f64(x), None if w is None else f64(w), eps), pos.cpu().numpy(), f, neox, scale)
    m[..., 2 * nf:] = np.abs(want[..., 2 * nf:])
    far = float(pos.abs().max().item() + 1)
    got = f64(y)
    assert np.all(np.abs(got - want) <= norm_tolerance(want, m, kind, far, x.shape[-1])), float(np.abs(got - want).max())
    return y


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("tokens,heads,hd,nf", [(1, 1, 2, 1), (1, 40, 128, 64), (3, 5, 64, 32), (7, 3, 96, 48),
                                                (130, 8, 128, 32), (5, 2, 66, 33), (9, 3, 80, 11), (2, 1, 1024, 512),
                                                (700, 2, 64, 3), (33, 4, 256, 128), (3, 2, 1024, 1), (2, 3, 1023, 300),
                                                (5, 33, 72, 8), (3000, 3, 32, 16)])
def test_norm_rope(gpu, kind, neox, tokens, heads, hd, nf):
    import torch

    g = gen(tokens * 1000 + hd + nf)
    x = normal(g, tokens, heads, hd, kind=kind, scale=3.0)
    pos = torch.randint(0, 2 ** 20, (tokens,), generator=g, dtype=torch.int32).cuda()
    w = 1 + normal(g, hd, scale=0.3)
    y = check_norm(x, pos, w, nf, neox, kind, scale=1.25)
    z = x.clone()
    assert torch.equal(check_norm_inplace(z, pos, w, nf, neox), y)
    check_norm(x, pos, None, nf, neox, kind, eps=0.5)  # without weights, an eps that counts


def check_norm_inplace(z, pos, w, nf, neox):
    import torch

    from nightrun_amd import serve

    serve.norm_rope(z, z, w, pos, torch.from_numpy(freqs(nf)).cuda(), neox=neox, scale=1.25)
    return z


def test_norm_rope_sizes_of_values(gpu):
    """Rows of zeros, tiny and large ones beside ordinary ones; far and negative positions; an infinity and a NaN, which
    stay in their row; eps 0."""
    import torch

    from nightrun_amd import serve

    g = gen(3)
    x = normal(g, 6, 3, 128)
    x[0, 1] = 0
    x[1] *= 1e-12
    x[2] *= 1e15
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31, -1, 2 ** 30 + 1, 123456789, 0], dtype=torch.int32).cuda()
    w = 1 + normal(g, 128, scale=0.3)
    for neox in (False, True):
        y = check_norm(x, pos, w, 64, neox, "f32")
        assert torch.equal(y[0, 1], torch.zeros_like(y[0, 1]))
        bad = x.clone()
        bad[3, 0, 5], bad[4, 2, 127] = float("inf"), float("nan")
        z = torch.empty_like(bad)
        serve.norm_rope(z, bad, w, pos, torch.from_numpy(freqs(64)).cuda(), neox=neox)
        same = torch.ones(6, 3, dtype=torch.bool)
        same[3, 0] = same[4, 2] = False
        assert torch.equal(z[same.cuda()], y[same.cuda()])
        assert torch.isnan(z[4, 2]).all() and torch.isnan(z[3, 0, 5])
        one = x[1:2] * 1e12
        check_norm(one, pos[1:2].contiguous(), w, 64, neox, "f32", eps=0.0)


def test_norm_rope_strides(gpu):
    """Slices of a wider projection that are not 16-byte aligned, and outputs between others; an input whose rows repeat;
    a row stride that is odd."""
    import torch

    g = gen(5)
    wide = normal(g, 6, 9, 67)
    out = torch.full((6, 4, 70), 3.0, device="cuda")
    pos = torch.arange(6, dtype=torch.int32).cuda()
    w = 1 + normal(g, 64, scale=0.3)
    for neox in (False, True):
        for x in (wide[:, 2:5, 1:65], normal(g, 1, 1, 64).expand(6, 3, 64), normal(g, 6, 3, 72)[..., 8:]):
            out.fill_(3.0)
            check_norm(x, pos, w, 32, neox, "f32", y=out[:, 1:, 3:67])
            got = f64(out)
            assert np.all(got[:, 0] == 3) and np.all(got[..., :3] == 3) and np.all(got[..., 67:] == 3)
        # the output's heads lie between the input's in one tensor
        both = normal(g, 6, 6, 64, kind="bf16")
        check_norm(both[:, :3], pos, w, 32, neox, "bf16", y=both[:, 3:])


@pytest.mark.parametrize("kind,cache", TYPES)
@pytest.mark.parametrize("neox,hd,nf,size,layout,heads,kv", [(True, 128, 64, 16, "heads", 32, 8), (False, 64, 32, 24, "rows", 5, 5),
                                                             (True, 96, 20, 1, "heads", 6, 2), (False, 256, 127, 7, "rows", 4, 1)])
@pytest.mark.parametrize("places", [False, True])
def test_norm_rope_append(gpu, kind, cache, neox, hd, nf, size, layout, heads, kv, places):
    """Slices of one projection; padding rows, places behind the table, entries that are no page: left alone. With `at`
    the rotary positions are others than the places, negative ones among them."""
    import torch

    from nightrun_amd import serve

    seqs, width = 3, 5
    g = gen(hd + size)
    pages = seqs * width + 2
    table = torch.randperm(pages, generator=g)[:seqs * width].to(torch.int32).view(seqs, width)
    table[1, 2], table[2, 0] = -1, pages
    rows = []  # (seq, place)
    for s in range(seqs):
        rows += [(s, p) for p in range(0, width * size, max(1, size // 3))] + [(s, width * size), (s, width * size + 9)]
    rows += [(-1, 3), (seqs, 3), (0, -1), (2 ** 31 - 1, 0), (0, 2 ** 31 - 1)]
    order = torch.randperm(len(rows), generator=g).tolist()
    rows = [rows[i] for i in order]
    n = len(rows)
    seq = torch.tensor([r[0] for r in rows], dtype=torch.int32)
    place = torch.tensor([r[1] for r in rows], dtype=torch.int32)
    pos = torch.randint(-2 ** 20, 2 ** 20, (n,), generator=g, dtype=torch.int32) if places else place
    qkv = normal(g, n, heads + 2 * kv, hd, kind=kind, scale=2.0)
    q, k, v = qkv.split([heads, kv, kv], 1)
    f = freqs(nf)
    wq, wk = (1 + normal(g, hd, scale=0.3) for _ in range(2))
    fd = torch.from_numpy(f).cuda()
    at = dict(at=place.cuda()) if places else {}
    for normed in (True, False):
        if not normed and not places:
            continue  # rope_append as it was
        kp, vp = pool(pages, kv, size, hd, cache, 5.0, layout), pool(pages, kv, size, hd, cache, 6.0, layout)
        y = torch.full((n, heads, hd), 9.0, dtype=dt(kind), device="cuda")

        def call(y, q, kp, vp):
            if normed:
                serve.norm_rope_append(y, q, k, v, wq, wk, pos.cuda(), seq.cuda(), fd, kp, vp, table.cuda(), neox=neox,
                                       scale=0.75, **at)
            else:
                serve.rope_append(y, q, k, v, pos.cuda(), seq.cuda(), fd, kp, vp, table.cuda(), neox=neox, scale=0.75, **at)

        call(y, q, kp, vp)
        far = float(pos.abs().max()) + 1
        xq, xk = f64(q), f64(k)
        if normed:
            xq, xk = norm(xq, f64(wq), 1e-6), norm(xk, f64(wk), 1e-6)
        (rq, mq), (rk, mk) = turn(xq, pos.numpy(), f, neox, 0.75), turn(xk, pos.numpy(), f, neox, 0.75)
        mq[..., 2 * nf:], mk[..., 2 * nf:] = np.abs(rq[..., 2 * nf:]), np.abs(rk[..., 2 * nf:])
        tq, tk = norm_tolerance(rq, mq, kind, far, hd), norm_tolerance(rk, mk, cache, far, hd)
        want_k, tol_k = np.full(kp.shape, 5.0), np.zeros(kp.shape)
        want_v = torch.full(vp.shape, 6.0, dtype=dt(cache))
        gy = f64(y)
        for i, (s, p) in enumerate(rows):
            if not (0 <= s < seqs and p >= 0):
                assert np.all(gy[i] == 9.0), (s, p)
                continue
            assert np.all(np.abs(gy[i] - rq[i]) <= tq[i]), (s, p)
            page = int(table[s, p // size]) if p < width * size else -1
            if 0 <= page < pages:
                want_k[page, :, p % size], tol_k[page, :, p % size] = rk[i], tk[i]
                want_v[page, :, p % size] = v[i].cpu().to(dt(cache))
        assert np.all(np.abs(f64(kp) - want_k) <= tol_k)
        assert torch.equal(vp.cpu(), want_v)
        p2, v2 = pool(pages, kv, size, hd, cache, 5.0, layout), pool(pages, kv, size, hd, cache, 6.0, layout)
        q2 = qkv.clone().split([heads, kv, kv], 1)[0]
        call(q2, q2, p2, v2)  # q in place
        good = (seq >= 0) & (seq < seqs) & (place >= 0)
        assert torch.equal(q2.cpu()[good], y.cpu()[good]) and torch.equal(q2.cpu()[~good], q.cpu()[~good])
        assert torch.equal(p2, kp) and torch.equal(v2, vp)


# ---- attention of a tree's nodes -------------------------------------------------------------------


def tree_attention(q, c, parents, counts, scale, window, gone=()):
    """(out, bound per value, lse, bound) in 64 bits, as attention() of the tests of the serving operators has them:
    scores are off by at most d = (hd + 4) u A + 3 u max |s|, weights by 2 e^(2d) - 2 relative, sums of T weights
    by (T + 8) u; the log-sum by d, what the sum is, and the rounding of the logarithm and of its product with log 2."""
    seqs, new, heads, hd = q.shape
    group = heads // c.kv
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    lse, lse_tol = np.full(q.shape[:3], -np.inf), np.zeros(q.shape[:3])
    for b in range(seqs):
        k, v = c.k[b].double().numpy(), c.v[b].double().numpy()
        n, m = len(k), counts[b]
        base = n - m
        held = np.array([(b, t // c.size) not in gone for t in range(n)], bool)
        for j in range(m):
            nodes = way(parents[b], j)
            sees = np.zeros(n, bool)
            sees[max(0, base + len(nodes) - window) if window else 0:max(0, base)] = True
            for a in nodes[-window:] if window else nodes:
                if base + a >= 0:
                    sees[base + a] = True
            sees &= held
            if not sees.any():
                continue
            kk, vv = k[sees], v[sees]
            for h in range(heads):
                s = kk[:, h // group] @ q[b, j, h] * scale
                size = float((np.abs(kk[:, h // group]) @ np.abs(q[b, j, h])).max()) * abs(scale)
                d = (hd + 4) * U * size + 3 * U * float(np.abs(s).max())
                top = s.max()
                w = np.exp(s - top)
                out[b, j, h] = w @ vv[:, h // group] / w.sum()
                lse[b, j, h] = top + math.log(w.sum())
                weight = w @ np.abs(vv[:, h // group]) / w.sum()
                tol[b, j, h] = weight * (2 * math.expm1(2 * d) + 2 * (len(s) + 8) * U)
                lse_tol[b, j, h] = d + (len(s) + 8) * U + 4 * U * (abs(top) + abs(lse[b, j, h])) + 16 * U
    return out, tol, lse, lse_tol


def check_tree(c, kind, cache, parents, heads, window=0, counts=None, q=None, scale=None, seed=1, gone=(), lse=True):
    import torch

    from nightrun_amd import serve

    seqs, new = parents.shape
    q = normal(gen(seed), seqs, new, heads, c.hd, kind=kind, scale=1.5) if q is None else q
    scale = c.hd ** -0.5 if scale is None else scale
    y = torch.full(q.shape, 11.0, dtype=q.dtype, device="cuda")
    ls = torch.full(q.shape[:3], 12.0, device="cuda") if lse else None
    kp, vp, table, lens = c.dev()
    cnt = torch.tensor(counts, dtype=torch.int32, device="cuda") if counts is not None else None
    serve.tree_attention(y, q, kp, vp, table, lens, torch.from_numpy(parents).cuda(), scale, window=window, counts=cnt,
                         lse=ls)
    use = [min(max(x, 0), new) for x in counts] if counts is not None else [new] * seqs
    want, tol, wl, tl = tree_attention(f64(q), c, parents, use, scale, window, gone)
    got = f64(y)
    for b in range(seqs):
        top = float(c.v[b].abs().max()) if len(c.v[b]) else 0.0
        tol[b] += PIECES[kind, cache] * top
    tol += half_step(kind) * np.abs(want)
    for b in range(seqs):
        assert np.all(got[b, use[b]:] == 11.0)
        bad = np.abs(got[b, :use[b]] - want[b, :use[b]]) > tol[b, :use[b]] + 1e-30
        assert not bad.any() and np.all(np.isfinite(got[b, :use[b]])), \
            (b, np.argwhere(bad)[:3], float(np.abs(got[b, :use[b]] - want[b, :use[b]]).max()))
        if lse:
            gl, w = f64(ls)[b, :use[b]], wl[b, :use[b]]
            none = np.isneginf(w)
            assert np.all(np.isneginf(gl[none]))
            assert np.all(np.abs(gl[~none] - w[~none]) <= tl[b, :use[b]][~none])
            assert np.all(f64(ls)[b, use[b]:] == 12.0)
    return y


@pytest.mark.parametrize("kind,cache", TYPES)
@pytest.mark.parametrize("hd,heads,kv,size,new", [(32, 4, 4, 16, 7), (64, 32, 8, 16, 16), (96, 5, 1, 24, 9),
                                                  (128, 32, 8, 16, 12), (256, 8, 2, 7, 5), (64, 24, 1, 1, 3)])
def test_tree_types_and_heads(gpu, kind, cache, hd, heads, kv, size, new):
    lens = [new, new + 1, 31 + new, 200, 0, 129]
    c = Cache(gen(hd + size), lens, kv, hd, size, cache, layout="rows" if hd == 64 else "heads")
    check_tree(c, kind, cache, trees(new, len(lens), new), heads)


@pytest.mark.parametrize("kind,cache", TYPES)
@pytest.mark.parametrize("hd,heads,kv,new", [(64, 8, 2, 64), (128, 4, 1, 64), (128, 8, 2, 33), (96, 8, 1, 31), (32, 4, 1, 64),
                                             (256, 4, 1, 40), (128, 5, 1, 21)])
def test_tree_many_nodes(gpu, kind, cache, hd, heads, kv, new):
    """More rows than one group of them: many nodes, odd groups of heads, sequences around the size of a tile."""
    lens = [new, 300, 128 + new // 2, 127, 900]
    c = Cache(gen(hd + new), lens, kv, hd, 16, cache)
    check_tree(c, kind, cache, trees(new, len(lens), new), heads)


@pytest.mark.parametrize("new,heads,kv,window,counts", [(5, 32, 8, 0, None), (7, 8, 1, 50, None), (17, 8, 2, 0, None),
                                                        (3, 6, 2, 1, None), (5, 32, 8, 33, [5, 0, 1, 9, -2, 4, 3]),
                                                        (40, 4, 2, 3, [40, 0, 1, 39, 12, 17, 33]), (64, 4, 2, 2, None),
                                                        (64, 8, 2, 200, [64, 3, 64, 0, 63, 64, 50]), (1, 4, 2, 0, None)])
@pytest.mark.parametrize("kind,cache", [("f32", "f16"), ("bf16", "bf16")])
def test_tree_counts_and_windows(gpu, kind, cache, new, heads, kv, window, counts):
    """Trees that begin before the first position, windows shorter than the tree is deep and ones that cut tiles, padding."""
    lens = [300, 5, 1, 128, 64, 0, 257]
    c = Cache(gen(new), lens, kv, 128, 24, cache, width=13)
    check_tree(c, kind, cache, trees(new + window, 7, new), heads, window=window, counts=counts)


@pytest.mark.parametrize("lens,kv,new", [([5000], 1, 16), ([3000, 1, 7000, 0, 130], 2, 20), ([9000], 8, 64),
                                         (list(range(0, 700, 5)), 1, 6), (list(range(0, 1400, 20)), 2, 48)])
def test_tree_long(gpu, lens, kv, new):
    """Sequences that many workgroups share, beside short and empty ones; more than 64 and 128 sequences."""
    import torch

    c = Cache(gen(len(lens)), lens, kv, 64, 16, "f16")
    t = trees(new, len(lens), new)
    y = check_tree(c, "f16", "f16", t, 4 * kv)
    assert torch.equal(y, check_tree(c, "f16", "f16", t, 4 * kv))  # the same bits again


def test_tree_parents_of_any_kind(gpu):
    """Parents that are none: -1 anywhere, the node itself, one behind it, what no tree holds. A chain is paged_attention()."""
    import torch

    from nightrun_amd import serve

    c = Cache(gen(9), [150, 64, 40], 2, 128, 16, "f16")
    t = trees(4, 3, 32)
    t[0, 5], t[0, 9], t[0, 12], t[1, 3], t[1, 31], t[2, 0] = -1, 9, 31, 2 ** 31 - 1, -2 ** 31, 7
    check_tree(c, "f32", "f16", t, 4)
    for new in (6, 40, 64):
        chain = np.tile(np.arange(-1, new - 1, dtype=np.int32), (3, 1))
        for window in (0, 5):
            y = check_tree(c, "bf16", "f16", chain, 4, window=window)
            z = torch.empty_like(y)
            q = normal(gen(1), 3, new, 4, 128, kind="bf16", scale=1.5)
            kp, vp, table, lens = c.dev()
            serve.paged_attention(z, q, kp, vp, table, lens, 128 ** -0.5, window=window)
            # both within the pieces of the exact value and one rounding
            assert np.all(np.abs(f64(y) - f64(z)) <= 2 * half_step("bf16") * np.abs(f64(z)) + 2e-5)


@pytest.mark.parametrize("new", [6, 48])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_tree_masked_garbage(gpu, new, bad):
    """Infinities and NaN behind the length, before the window, on other branches and at unused places of the pages do not reach
    a node; on its own way they do."""
    import torch

    from nightrun_amd import serve

    for window in (0, 30):
        c = Cache(gen(new), [150, 90, new + 3], 2, 128, 16, "f16", garbage=bad)
        t = trees(new, 3, new)
        check_tree(c, "f32", "f16", t, 4, window=window, seed=3)
        q = normal(gen(3), 3, new, 4, 128, kind="f16", scale=1.5)
        want, tol, _, _ = tree_attention(f64(q), c, t, [new] * 3, 128 ** -0.5, window)
        tol += PIECES["f16", "f16"] * max(float(v.abs().max()) for v in c.v) + half_step("f16") * np.abs(want)
        node = new // 2  # holds infinities in its values
        for b, n in enumerate(c.lens):
            p = n - new + node
            c.vp[int(c.table[b, p // 16]), :, p % 16] = bad
            if window:
                for p in range(0, max(0, n - new + 1 - window)):
                    c.vp[int(c.table[b, p // 16]), :, p % 16] = bad
                    c.kp[int(c.table[b, p // 16]), :, p % 16] = float("nan")
        y = torch.empty_like(q)
        kp, vp, table, lens = c.dev()
        serve.tree_attention(y, q, kp, vp, table, lens, torch.from_numpy(t).cuda(), 128 ** -0.5, window=window)
        got = f64(y)
        for b in range(3):
            for j in range(new):
                nodes = way(t[b], j)
                if node in (nodes[-window:] if window else nodes):
                    assert not np.isfinite(got[b, j]).any(), (b, j)
                else:
                    assert np.all(np.abs(got[b, j] - want[b, j]) <= tol[b, j]), (b, j)


def test_tree_bad_pages_and_lengths(gpu):
    """Table entries that are no page, lengths below zero and past the table, nothing to do, tables without columns."""
    import torch

    from nightrun_amd import serve

    c = Cache(gen(9), [100, 80, 64, 1000, -7], 2, 64, 16, "bf16", width=7)
    pages = c.kp.shape[0]
    c.table[0, 2], c.table[1, 0], c.table[1, 4] = -1, pages, 2 ** 31 - 1
    c.table[2, :4] = -5  # nothing left of it
    gone = {(0, 2), (1, 0), (1, 4)} | {(2, i) for i in range(4)}
    for new in (3, 30):
        check_tree(c, "bf16", "bf16", trees(2, 5, new), 8, gone=gone)
        check_tree(c, "f32", "bf16", trees(3, 5, new), 2, window=20, gone=gone)
    kp, vp, table, lens = c.dev()
    par = torch.zeros(5, 0, dtype=torch.int32, device="cuda")
    y = torch.full((5, 0, 4, 64), 1.0, device="cuda")
    serve.tree_attention(y, y, kp, vp, table, lens, par, 1.0)
    serve.tree_attention(y[:0], y[:0], kp, vp, table[:0], lens[:0], par[:0], 1.0)
    for new in (2, 40):
        z = torch.full((2, new, 4, 64), 1.0, device="cuda")
        serve.tree_attention(z, z.clone(), kp[:0], vp[:0], table[:2, :0].contiguous(), lens[:2],
                             torch.zeros(2, new, dtype=torch.int32, device="cuda"), 1.0)
        assert torch.equal(z, torch.zeros_like(z))


@pytest.mark.parametrize("new", [4, 40])
def test_tree_extreme_scores(gpu, new):
    """Rows of very different sizes, f32 queries past f16's range, zeros, a scale of zero; outputs that cancel."""
    import torch

    c = Cache(gen(4), [333, 170], 2, 128, 16, "f16")
    t = trees(6, 2, new)
    q = normal(gen(4), 2, new, 8, 128)
    for i, f in enumerate((1e-30, 1.0, 40.0, 0.0)):
        q[:, i] *= f
    check_tree(c, "f32", "f16", t, 8, q=q)
    check_tree(c, "f32", "f16", t, 8, q=q * 2.0 ** 40, scale=128 ** -0.5 * 2.0 ** -40)
    check_tree(c, "f32", "f16", t, 8, q=q * 2.0 ** -60, scale=128 ** -0.5 * 2.0 ** 60)
    check_tree(c, "f32", "f16", t, 8, scale=0.0)
    check_tree(c, "f32", "f16", t, 8, scale=-0.1)
    assert torch.isfinite(q).all()


@pytest.mark.parametrize("new", [3, 40])
def test_tree_strides_and_far_offsets(gpu, new):
    """q and out as slices of wider tensors, not aligned; pools of more than 2^32 elements, whose last pages are used."""
    import torch

    from nightrun_amd import serve

    hd, kv, size = 128, 2, 16
    pages = 2 ** 32 // (hd * kv * size) + 40
    kp = torch.empty(pages, kv, size, hd, dtype=torch.float16, device="cuda")
    vp = torch.empty(pages, kv, size, hd, dtype=torch.float16, device="cuda")
    g = gen(8)
    lens = [new + 70, new + 33]
    c = Cache(g, lens, kv, hd, size, "f16")
    far = torch.randperm(40, generator=g)[:c.table.numel()].to(torch.int32).view(c.table.shape) + (pages - 40)
    for b in range(2):
        for i in range(c.width):
            kp[far[b, i].long()] = c.kp[c.table[b, i].long()]
            vp[far[b, i].long()] = c.vp[c.table[b, i].long()]
    t = trees(5, 2, new)
    wide = normal(g, 2, new, 7, 133)
    q = wide[:, :, 1:5, 3:131]
    out = torch.full((2, new, 6, 140), 2.0, device="cuda")
    serve.tree_attention(out[:, :, 1:5, 5:133], q, kp, vp, far.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                         torch.from_numpy(t).cuda(), hd ** -0.5)
    want, tol, _, _ = tree_attention(f64(q), c, t, [new, new], hd ** -0.5, 0)
    tol += PIECES["f32", "f16"] * max(float(v.abs().max()) for v in c.v) + U * np.abs(want)
    got = f64(out)
    assert np.all(np.abs(got[:, :, 1:5, 5:133] - want) <= tol)
    got[:, :, 1:5, 5:133] = 2.0
    assert np.all(got == 2.0)


@pytest.mark.parametrize("heads,kv,new,hd,kind,cache", [(64, 1, 64, 64, "bf16", "bf16"), (24, 1, 64, 128, "f32", "f16"), (7, 1, 64, 32, "f16", "f16"),
                                                        (20, 1, 64, 128, "f32", "bf16"), (16, 1, 64, 256, "f16", "f16"), (9, 3, 64, 96, "bf16", "bf16")])
def test_tree_many_rows(gpu, heads, kv, new, hd, kind, cache):
    """Several units for a KV head, the last of them not full, over a sequence that fills the card and short ones."""
    lens = [9000 if hd < 256 else 4000, 64, 200]
    c = Cache(gen(hd), lens, kv, hd, 16, cache)
    check_tree(c, kind, cache, trees(heads, 3, new), heads)


@pytest.mark.parametrize("size", [3, 200, 1000])
@pytest.mark.parametrize("new", [5, 40])
def test_tree_page_sizes(gpu, size, new):
    """Pages longer than a stage, pages that end anywhere in it; a table with room for far more than there is."""
    c = Cache(gen(size), [700, 128 + new, 256, 64 + new], 2, 128, size, "f16", width=4096 // size + 1)
    check_tree(c, "f16", "f16", trees(size, 4, new), 8)
    check_tree(c, "f32", "f16", trees(size, 4, new), 2, window=77)


@pytest.mark.parametrize("new", [4, 40])
def test_tree_one_pool_and_wide_table(gpu, new):
    """Keys and values side by side in one pool; the table is a part of a wider one."""
    import torch

    from nightrun_amd import serve

    c = Cache(gen(new), [300, new, 129], 2, 64, 16, "bf16")
    t = trees(new, 3, new)
    want = check_tree(c, "bf16", "bf16", t, 8)
    kp, vp, table, lens = c.dev()
    for both in (torch.stack((kp, vp), 1), torch.stack((kp.transpose(1, 2), vp.transpose(1, 2)), 2)):
        k, v = (both[:, 0], both[:, 1]) if both.shape[1] == 2 else (both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2))
        wide = torch.full((3, c.width + 5), -1, dtype=torch.int32, device="cuda")
        wide[:, 2:2 + c.width] = table
        q = normal(gen(1), 3, new, 8, 64, kind="bf16", scale=1.5)
        y = torch.empty_like(q)
        serve.tree_attention(y, q, k, v, wide[:, 2:2 + c.width], lens, torch.from_numpy(t).cuda(), 0.125)
        assert torch.equal(y, want)
        # the append and the move into such pools
        x = normal(gen(2), 3, 12, 64, kind="bf16")
        f = torch.from_numpy(freqs(32)).cuda()
        pos = lens - new
        seq = torch.arange(3, dtype=torch.int32, device="cuda")
        out = torch.empty(3, 8, 64, dtype=torch.bfloat16, device="cuda")
        k2, v2 = kp.clone(), vp.clone()
        serve.norm_rope_append(out, x[:, :8], x[:, 8:10], x[:, 10:], None, None, pos, seq, f, k2, v2, table)
        serve.norm_rope_append(out, x[:, :8], x[:, 8:10], x[:, 10:], None, None, pos, seq, f, k, v, wide[:, 2:2 + c.width])
        assert torch.equal(k.nan_to_num(9), k2.nan_to_num(9)) and torch.equal(v.nan_to_num(9), v2.nan_to_num(9))
        path = torch.full((3, new), -1, dtype=torch.int32, device="cuda")
        path[:, 0], path[:, 1] = 1, new - 1
        a, b = torch.empty_like(lens), torch.empty_like(lens)
        serve.keep_path(a, k2, v2, table, lens, path)
        serve.keep_path(b, k, v, wide[:, 2:2 + c.width], lens, path)
        assert torch.equal(a, b) and torch.equal(k.nan_to_num(9), k2.nan_to_num(9)) and torch.equal(v.nan_to_num(9), v2.nan_to_num(9))


@pytest.mark.parametrize("kind,cache,hd", [("f16", "f16", 128), ("f32", "f16", 64), ("f32", "bf16", 128), ("bf16", "bf16", 256)])
def test_tree_bad_queries_stay_alone(gpu, kind, cache, hd):
    """Queries with an infinity or a NaN: their rows alone."""
    import torch

    from nightrun_amd import serve

    c = Cache(gen(hd), [400, 90], 2, hd, 16, cache)
    t = trees(3, 2, 20)
    q = normal(gen(5), 2, 20, 8, hd, kind=kind, scale=1.5)
    want, tol, _, _ = tree_attention(f64(q), c, t, [20, 20], hd ** -0.5, 0)
    tol += PIECES[kind, cache] * max(float(v.abs().max()) for v in c.v) + half_step(kind) * np.abs(want)
    q[0, 3, 1, 7], q[1, 19, 7, hd - 1] = float("nan"), float("inf")
    kp, vp, table, lens = c.dev()
    y = torch.empty_like(q)
    serve.tree_attention(y, q, kp, vp, table, lens, torch.from_numpy(t).cuda(), hd ** -0.5)
    got = f64(y)
    bad = np.zeros(got.shape[:3], bool)
    bad[0, 3, 1] = bad[1, 19, 7] = True
    assert np.all(np.abs(got - want)[~bad] <= tol[~bad]) and not np.isfinite(got[bad]).any()


@pytest.mark.parametrize("kind,cache,hd,heads,kv,new", [("bf16", "bf16", 64, 8, 1, 40), ("f32", "bf16", 128, 4, 1, 50), ("f16", "f16", 256, 4, 1, 30),
                                                        ("f32", "f16", 96, 3, 1, 64), ("f16", "f16", 32, 4, 2, 20), ("bf16", "bf16", 128, 4, 1, 64),
                                                        ("f32", "bf16", 256, 2, 1, 9)])
def test_tree_infinities_in_every_shape(gpu, kind, cache, hd, heads, kv, new):
    """An infinity in one node's values, which its descendants see and no other: with every number of rows and pieces, over
    positions that several workgroups share."""
    import torch

    from nightrun_amd import serve

    lens = [new + 600, new + 3, 130 + new]
    c = Cache(gen(hd + new), lens, kv, hd, 16, cache)
    t = trees(new, 3, new)
    q = normal(gen(3), 3, new, heads, hd, kind=kind, scale=1.5)
    want, tol, _, _ = tree_attention(f64(q), c, t, [new] * 3, hd ** -0.5, 0)
    tol += PIECES[kind, cache] * max(float(v.abs().max()) for v in c.v) + half_step(kind) * np.abs(want)
    node = new // 3
    for b, n in enumerate(lens):
        p = n - new + node
        c.vp[int(c.table[b, p // 16]), :, p % 16, hd - 1] = float("inf")
    kp, vp, table, lens_ = c.dev()
    y = torch.empty_like(q)
    serve.tree_attention(y, q, kp, vp, table, lens_, torch.from_numpy(t).cuda(), hd ** -0.5)
    got = f64(y)
    for b in range(3):
        for j in range(new):
            below = node in way(t[b], j)
            assert np.all(np.abs(got[b, j] - want[b, j])[:, :hd - below] <= tol[b, j][:, :hd - below]), (b, j)
            assert np.all(np.isposinf(got[b, j, :, hd - 1])) == below, (b, j)


def test_tree_broadcast_inputs(gpu):
    """Queries that repeat, sequences of one row of the table, all pages one: strides of 0 are read like any other."""
    import torch

    from nightrun_amd import serve

    g = gen(21)
    for new in (3, 40):
        c = Cache(gen(new), [100 + new], 2, 64, 16, "f16")
        kp, vp, table, _ = c.dev()
        q = normal(g, 1, 1, 4, 64, kind="f16").expand(3, new, 4, 64)
        t = torch.from_numpy(trees(new, 3, new)).cuda()
        lens = torch.tensor([100 + new, 64, 31 + new], dtype=torch.int32, device="cuda")
        y, z = (torch.empty(3, new, 4, 64, dtype=torch.float16, device="cuda") for _ in range(2))
        serve.tree_attention(y, q, kp, vp, table.expand(3, -1), lens, t, 0.125, window=50)
        serve.tree_attention(z, q.contiguous(), kp, vp, table.repeat(3, 1), lens, t, 0.125, window=50)
        assert torch.equal(y, z)
        one = kp[:1].expand(7, -1, -1, -1), vp[:1].expand(7, -1, -1, -1)
        same = torch.zeros_like(table).expand(3, -1)
        serve.tree_attention(y, q, *one, table.clamp(max=6).expand(3, -1), lens, t, 0.125)
        serve.tree_attention(z, q, kp, vp, same, lens, t, 0.125)
        assert torch.equal(y, z)


def test_tree_more_sequences_than_a_grid_has_rows(gpu):
    """70,000 sequences of a few positions, three in four without nodes."""
    import torch

    from nightrun_amd import serve

    n = 70000
    g = gen(22)
    kp, vp = (torch.randn(50, 1, 4, 32, generator=g).half().cuda() for _ in range(2))
    table = torch.randint(0, 50, (n, 2), generator=g, dtype=torch.int32).cuda()
    lens = torch.randint(2, 9, (n,), generator=g, dtype=torch.int32).cuda()
    counts = (2 * (torch.arange(n) % 4 == 0)).to(torch.int32).cuda()
    q = normal(g, n, 2, 1, 32, kind="f16")
    y = torch.full_like(q, 5.0)
    serve.tree_attention(y, q, kp, vp, table, lens, torch.tensor([[-1, 0]], dtype=torch.int32, device="cuda").repeat(n, 1),
                         32 ** -0.5, counts=counts)
    some = torch.arange(0, n, 4, device="cuda")
    k, v = (x[table[some].long()].float().reshape(len(some), 8, 32) for x in (kp, vp))
    hi = lens[some].long()[:, None] - 2 + torch.arange(2, device="cuda")
    s = (q[some, :, 0].float()[:, :, None] * k[:, None]).sum(-1) * 32 ** -0.5
    w = torch.softmax(s.masked_fill(torch.arange(8, device="cuda") > hi[..., None], -math.inf), -1)
    want = (w[..., None] * v[:, None]).sum(2)
    # 36 products and sums of at most |s| times 4 |v| in f32 on either side, and the output's rounding
    assert float((y[some, :, 0].float() - want).abs().max()) <= 2.0 ** -11 * 5 + 1e-4
    y[some] = 5.0
    assert bool((y == 5.0).all())


@pytest.mark.parametrize("kind,cache,hd,heads,new", [("f16", "f16", 64, 1, 1), ("bf16", "bf16", 64, 8, 40), ("f32", "bf16", 128, 4, 20),
                                                     ("f32", "f16", 128, 4, 40), ("bf16", "bf16", 128, 4, 64), ("f16", "f16", 256, 4, 30),
                                                     ("f32", "f16", 32, 2, 5), ("bf16", "f16", 96, 1, 9)])
def test_tree_infinities_of_little_weight(gpu, kind, cache, hd, heads, new):
    """A weight is positive however small: an infinity that a row sees is its output, also where f32 holds no such weight, whether
    the row's largest score is in the same 32 positions, with another wave or with another workgroup, before or behind. Infinities of
    both signs, and a NaN, give NaN. Keys are 0 but the largest's: e^-256 of its weight for all others, so that the output is its value."""
    import torch

    from nightrun_amd import serve

    n, size, pages = 3000, 16, 196
    places = [0, 7, 31, 32, 70, 127, 128, 333, 1000, 1500, 2048, 2900]
    pairs = [(a, b) for a in places for b in places if a != b][::3] + [(7, 31), (31, 7), (7, 32), (32, 7), (7, 70), (70, 7), (333, 1500)]
    seqs = 8
    g = gen(hd + new)
    q = torch.zeros(seqs, new, heads, hd, dtype=dt(kind))
    q[..., 0] = 16.0
    qd, t = q.cuda(), torch.from_numpy(trees(new, seqs, new)).cuda()
    table = torch.arange(seqs * pages, dtype=torch.int32, device="cuda").view(seqs, pages)
    for i in range(0, len(pairs), seqs):
        some = (pairs[i:] + pairs)[:seqs]
        for kinds in ((1,), (-1,), (1, -1), (float("nan"),)):
            k = torch.zeros(seqs, pages * size, hd, dtype=dt(cache))
            v = torch.randn(seqs, pages * size, hd, generator=g).to(dt(cache))
            want = np.zeros((seqs, hd))
            for b, (top, at) in enumerate(some):
                k[b, top, 0] = 16.0
                want[b] = v[b, top].double().numpy()
                for j, sign in enumerate(kinds):  # the second somewhere else
                    v[b, (at + 900 * j) % n if (at + 900 * j) % n != top else top + 1, hd - 3] = sign * float("inf")
            kp, vp = (x.view(-1, 1, size, hd).cuda() for x in (k, v))
            y = torch.empty_like(qd)
            serve.tree_attention(y, qd, kp, vp, table, torch.full((seqs,), n + new, dtype=torch.int32, device="cuda"), t, 1.0)
            got = f64(y)
            hit = got[..., hd - 3]
            if len(kinds) == 2 or kinds[0] != kinds[0]:
                assert np.isnan(hit).all(), (some, kinds, hit[:, 0, 0])
            else:
                assert np.all(hit == kinds[0] * np.inf), (some, kinds, hit[:, 0, 0])
            got[..., hd - 3] = want[:, None, None, hd - 3]
            tol = PIECES[kind, cache] * 8 + half_step(kind) * np.abs(want)
            assert np.all(np.abs(got - want[:, None, None]) <= tol[:, None, None]), (some, kinds)


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("new,width", [(1, 1), (3, 1), (12, 1), (40, 3), (12, 900), (40, 900)])
def test_tree_weights_keep_32_bits(gpu, hd, new, width):
    """bf16 throughout, outputs that cancel. Three positions before the tree weigh 1, a fourth p = exp(-c s), the nodes nothing; in
    dimension h the values are minus the first two bf16 pieces of head h's p, and 1: what is left is the third piece. Values whose third
    piece is 2^-18.5 and more. Wide tables (whose columns are no pages) bring in the units of 128 and 256 rows.

    The numerator is off by: 3 u of the exponent (at most 1 in units of log2) in its unit and product, 2 u in the exponential,
    and 12 products of at most 2 added up, each sum rounded or cut: 24 u for rounding. In all 29 u, below 2^-18.5 / 1.4. The sum of the
    weights, its reciprocal and the product with it: less than 8 u of the output."""
    import torch

    from nightrun_amd import serve

    def bf(x):
        return torch.tensor(x, dtype=torch.float64).bfloat16().double().numpy()

    seqs, heads, s = 16, 8, 0.69
    scale = float(np.float32(s))
    c = np.concatenate([(128 + np.arange(128)) / 256, 1 - np.arange(1, 100) / 256.0])
    c = c[c >= 0.5]
    p = np.exp(-c * scale)
    third = p - bf(p) - bf(p - bf(p))
    c = c[np.abs(third) >= 2.0 ** -18.5]
    assert len(c) >= 5
    cc = c[np.random.default_rng(2).integers(0, len(c), (seqs, heads))]
    p = np.exp(-cc * scale)
    one, two = bf(p), bf(p - bf(p))
    q = np.zeros((seqs, new, heads, hd))
    q[..., 0] = cc[:, None]
    pages = -(-(4 + new) // 16)
    k, v = np.zeros((seqs, pages * 16, hd)), np.zeros((seqs, pages * 16, hd))
    k[:, 3, 0] = -1.0
    k[:, 4:, 0] = -1000.0
    v[:, 0, :heads], v[:, 1, :heads], v[:, 3, :heads] = -one, -two, 1.0
    qd = torch.from_numpy(q).to(torch.bfloat16).cuda()
    kd, vd = (torch.from_numpy(x).to(torch.bfloat16).view(seqs * pages, 1, 16, hd).cuda() for x in (k, v))
    table = torch.full((seqs, width), -1, dtype=torch.int32)
    table[:, :pages] = torch.arange(seqs * pages, dtype=torch.int32).view(seqs, pages)
    y = torch.empty_like(qd)
    serve.tree_attention(y, qd, kd, vd, table.cuda(), torch.full((seqs,), 4 + new, dtype=torch.int32, device="cuda"),
                         torch.from_numpy(trees(new, seqs, new)).cuda(), scale)
    got = f64(y)[:, :, np.arange(heads), np.arange(heads)]
    want = ((p - one - two) / (3 + p))[:, None]
    assert np.all(np.abs(want) >= 2.0 ** -18.5 / 4)
    assert np.all(np.abs(got - want) <= 29 * U / (3 + p[:, None]) + (half_step("bf16") + 8 * U) * np.abs(want))


def test_norm_rope_more_tokens_than_a_grid_has_threads_for(gpu):
    """2^29 tokens and some are two launches: rows around the seam and at the ends."""
    import torch

    from nightrun_amd import serve

    n = 2 ** 29 + 77
    x = torch.tensor([[[3.0, 4.0]]], device="cuda", dtype=torch.bfloat16).expand(n, 1, 2)
    pos = torch.zeros(n, dtype=torch.int32, device="cuda")
    at = [0, 1, 2 ** 29 - 1, 2 ** 29, 2 ** 29 + 1, n - 1]
    for i, p in enumerate(at):
        pos[p] = i + 1
    y = torch.zeros(n, 1, 2, dtype=torch.bfloat16, device="cuda")
    f = torch.ones(1, device="cuda")
    serve.norm_rope(y, x, None, pos, f)
    r = math.sqrt(12.5 + 1e-6)
    for i, p in enumerate(at):
        c, s_ = math.cos(i + 1), math.sin(i + 1)
        w = np.array([3 * c - 4 * s_, 3 * s_ + 4 * c]) / r
        assert np.all(np.abs(f64(y[p, 0]) - w) <= half_step("bf16") * np.abs(w) + 1e-6)
    w = torch.tensor([3 / r, 4 / r], device="cuda").bfloat16()
    bad = (y[:, 0] != w).any(-1)
    assert int(bad.sum()) == len(at)


# ---- acceptance of a path ---------------------------------------------------------------------------


def verify_tree(target, drafted, parents, u, counts):
    """The definition, node by node, in 64 bits."""
    seqs, new, vocab = target.shape
    tokens, path = np.full((seqs, new), -1, np.int32), np.full((seqs, new), -1, np.int32)
    accepted = np.zeros(seqs, np.int32)
    for b in range(seqs):
        if counts[b] == 0:
            continue
        node, gone, left, nodes = 0, set(), 1.0, [0]
        for j in range(1, counts[b]):
            if not 0 <= parents[b, j] < j or parents[b, j] != node:
                continue
            x = int(drafted[b, j])
            p = float(target[b, node, x]) if 0 <= x < vocab and x not in gone else 0.0
            p = p if p > 0 else 0.0
            if p > 0 and float(u[b, j]) * left < p:
                node, gone, left = j, set(), 1.0
                nodes.append(j)
            else:
                gone.add(x)
                left -= p
        row = target[b, node].astype(np.float64)
        row = np.where(row > 0, row, 0.0)
        r = row.copy()
        for x in gone:
            if 0 <= x < vocab:
                r[x] = 0
        if not r.sum() > 0:
            r = row
        c = np.cumsum(r)
        if c[-1] > 0:
            point = max(float(u[b, 0]), 0.0) * c[-1] if u[b, 0] < 1 else np.inf
            over = np.flatnonzero((c > point) & (r > 0))
            draw = int(over[0]) if len(over) else int(np.flatnonzero(r)[-1])
        else:
            draw = -1
        a = len(nodes) - 1
        accepted[b] = a
        path[b, :a + 1] = nodes
        tokens[b, :a] = drafted[b, nodes[1:]]
        tokens[b, a] = draw
    return tokens, path, accepted


def run_verify(target, drafted, parents, u, counts=None, stream=None):
    import torch

    from nightrun_amd import serve

    seqs, new, _ = target.shape
    tokens, path = (torch.full((seqs, new), 77, dtype=torch.int32, device="cuda") for _ in range(2))
    accepted = torch.full((seqs,), 77, dtype=torch.int32, device="cuda")
    serve.verify_tree(tokens, path, accepted, target, drafted, parents, u, counts=counts)
    return tokens, path, accepted


def verify_case(seed, seqs, new, vocab, sharp=6.0):
    import torch

    g = gen(seed)
    logits = torch.randn(seqs, new, vocab, generator=g) * sharp
    target = torch.softmax(logits, -1)
    parents = torch.from_numpy(trees(seed, seqs, new))
    best = (logits + 0.3 * torch.randn(logits.shape, generator=g)).topk(min(8, vocab), -1).indices
    drafted = torch.zeros(seqs, new, dtype=torch.int32)
    for b in range(seqs):
        seen = {}
        for j in range(1, new):
            p = int(parents[b, j])
            k = seen.get(p, 0)
            seen[p] = k + 1
            drafted[b, j] = best[b, p, min(k, best.shape[-1] - 1)]
    return target, drafted, parents, torch.rand(seqs, new, generator=g)


def check_verify(target, drafted, parents, u, counts=None):
    import torch

    use = [min(max(x, 0), target.shape[1]) for x in counts] if counts is not None else [target.shape[1]] * len(target)
    dev = [torch.as_tensor(x).cuda() for x in (target, drafted, parents, u)]
    cnt = torch.tensor(counts, dtype=torch.int32).cuda() if counts is not None else None
    got = run_verify(*dev, counts=cnt)
    want = verify_tree(*(np.asarray(x) for x in (target, drafted, parents, u)), use)
    for g, w, what in zip(got, want, ("tokens", "path", "accepted")):
        assert np.array_equal(g.cpu().numpy(), w), (what, g.cpu().numpy(), w)
    return want


@pytest.mark.parametrize("seqs,new,vocab", [(1, 1, 1), (1, 2, 5), (3, 8, 1000), (2, 64, 4097), (40, 16, 1024), (5, 33, 50257),
                                            (1, 12, 300000), (130, 5, 77)])
def test_verify_tree(gpu, seqs, new, vocab):
    most = 0
    for seed in range(4):
        want = check_verify(*verify_case(seed, seqs, new, vocab, sharp=3.0 + 2 * seed))
        most = max(most, int(want[2].max()))
    assert new < 8 or seqs < 2 or most >= 2  # many trees have paths of some length among them


def test_verify_tree_edges(gpu):
    """Counts, tokens given twice and outside the vocabulary, parents that are none, rows without weight, NaN, uniforms of 0 and
    1 and outside."""
    import torch

    target, drafted, parents, u = verify_case(1, 8, 12, 500)
    check_verify(target, drafted, parents, u, counts=[12, 0, 1, 5, -3, 99, 2, 11])
    d = drafted.clone()
    d[0, 1:] = d[0, 1]  # one token throughout
    d[1, 2], d[1, 3], d[2, 1] = -1, 500, 2 ** 31 - 1
    check_verify(target, d, parents, u)
    p = parents.clone()
    p[0, 3], p[0, 4], p[1, 5], p[2, 6], p[3, 0] = -1, 4, 9, 2 ** 31 - 1, 3
    check_verify(target, drafted, p, u)
    t = target.clone()
    t[0] = 0  # nothing to draw
    t[1, :, ::2] = float("nan")
    t[2] = -t[2]
    t[3, :] = 0
    t[3, :, 7] = 1.0  # certain
    check_verify(t, drafted, parents, u)
    # all weight on the children, all refused by uniforms of 1: drawn from the row as it is
    t = torch.zeros(2, 4, 50)
    t[:, 0, 3], t[:, 0, 9], t[:, 0, 11] = 0.5, 0.25, 0.25
    star = torch.tensor([[-1, 0, 0, 0]] * 2, dtype=torch.int32)
    kids = torch.tensor([[0, 3, 9, 11]] * 2, dtype=torch.int32)
    one = torch.ones(2, 4)
    one[0, 0] = 0.6
    tokens, path, accepted = check_verify(t, kids, star, one)
    assert accepted.tolist() == [0, 0] and tokens[:, 0].tolist() == [9, 11]
    for x in (0.0, 1.0, -0.5, 2.0, float(np.nextafter(np.float32(1), np.float32(0)))):
        check_verify(target, drafted, parents, torch.full_like(u, x))
        v = u.clone()
        v[:, 0] = x
        check_verify(target, drafted, parents, v)


def test_verify_tree_all_children(gpu):
    """A root with 63 children, in every place of the row, the last of them accepted or none."""
    import torch

    vocab = 5000
    g = gen(2)
    target = torch.softmax(torch.randn(6, 64, vocab, generator=g), -1)
    star = torch.full((6, 64), 0, dtype=torch.int32)
    star[:, 0] = -1
    drafted = torch.stack([torch.randperm(vocab, generator=g)[:64] for _ in range(6)]).to(torch.int32)
    drafted[:, 1], drafted[:, 2], drafted[:, 3] = 0, vocab - 1, 1023
    u = torch.ones(6, 64)
    u[3:, 63] = 0
    u[:, 0] = torch.rand(6, generator=g)
    want = check_verify(target, drafted, star, u)
    assert want[2].tolist() == [0, 0, 0, 1, 1, 1]


def test_verify_tree_draws_as_the_target(gpu):
    """What is emitted first, accepted or drawn, comes as often as the target has it: 60,000 sequences of one distribution.
    Counts of n draws lie within 6 standard deviations, sqrt(n p (1 - p)), of n p, but for one time in 5e8 each."""
    import torch

    n, vocab = 60000, 12
    p = torch.tensor([0.3, 0.2, 0.15, 0.1, 0.08, 0.06, 0.04, 0.03, 0.02, 0.01, 0.01, 0.0], dtype=torch.float32)
    target = p.expand(n, 5, vocab).contiguous()
    parents = torch.tensor([[-1, 0, 0, 0, 1]], dtype=torch.int32).repeat(n, 1)
    drafted = torch.tensor([[0, 1, 4, 0, 2]], dtype=torch.int32).repeat(n, 1)
    u = torch.rand(n, 5, generator=gen(7))
    tokens, path, accepted = run_verify(*(x.cuda() for x in (target, drafted, parents, u)))
    first = np.bincount(tokens[:, 0].cpu().numpy(), minlength=vocab)
    for v in range(vocab):
        q = float(p[v] / p.sum())
        assert abs(first[v] - n * q) <= 6 * math.sqrt(n * q * (1 - q)) + 1, (v, first[v], n * q)


def test_verify_tree_more_sequences_than_a_grid_has_rows(gpu):
    import torch

    target, drafted, parents, u = verify_case(3, 500, 4, 40)
    n = 70000
    idx = torch.arange(n) % 500
    got = run_verify(*(x[idx].cuda() for x in (target, drafted, parents, u)))
    want = verify_tree(*(np.asarray(x) for x in (target, drafted, parents, u)), [4] * 500)
    for g, w in zip(got, want):
        assert np.array_equal(g.cpu().numpy(), w[idx.numpy()])


def test_verify_tree_strides(gpu):
    """A target that is a slice, its rows not aligned."""
    import torch

    target, drafted, parents, u = verify_case(5, 3, 9, 1501)
    wide = torch.full((3, 10, 1507), float("nan"), device="cuda")
    wide[:, 1:, 3:1504] = target.cuda()
    got = run_verify(wide[:, 1:, 3:1504], drafted.cuda(), parents.cuda(), u.cuda())
    for g, w in zip(got, verify_tree(*(np.asarray(x) for x in (target, drafted, parents, u)), [9] * 3)):
        assert np.array_equal(g.cpu().numpy(), w)


# ---- the move of an accepted path --------------------------------------------------------------------


def keep(pages, table, lens, path, counts, width, size):
    """The definition, move by move: pages [layers, pages, kv, size, hd] on the host, in place; the new lengths."""
    out = []
    for b, n in enumerate(lens):
        n = min(max(n, 0), width * size)
        base = n - counts[b]
        last, kept = -1, 0
        for i in range(counts[b]):
            j = int(path[b, i])
            if not last < j < counts[b]:
                break
            last = j
            kept += 1
            to, of = base + i, base + j
            if to < 0 or of < 0:
                continue
            d, s = int(table[b, to // size]), int(table[b, of // size])
            if 0 <= d < pages[0].shape[1] and 0 <= s < pages[0].shape[1]:
                for p in pages:
                    p[:, d, :, to % size] = p[:, s, :, of % size].clone()
        out.append(max(base + kept, 0))
    return out


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("layers,kv,hd,size,new,layout", [(1, 8, 128, 16, 8, "heads"), (3, 2, 64, 24, 64, "rows"), (2, 1, 256, 1, 40, "heads"),
                                                          (28, 2, 96, 7, 33, "heads"), (1, 3, 72, 16, 64, "rows"), (2, 1, 40, 5, 20, "heads")])
def test_keep_path(gpu, cache, layers, kv, hd, size, new, layout):
    import torch

    from nightrun_amd import serve

    rng = np.random.default_rng(hd + new)
    g = gen(hd)
    seqs, width = 9, -(-(new + 60) // size)
    count = seqs * width + 2
    shape = (layers, count, size, kv, hd) if layout == "rows" else (layers, count, kv, size, hd)
    host = [torch.randn(shape, generator=g).to(dt(cache)) for _ in range(2)]
    view = [p.transpose(2, 3) if layout == "rows" else p for p in host]
    dev = [p.cuda() for p in host]
    dview = [p.transpose(2, 3) if layout == "rows" else p for p in dev]
    table = torch.randperm(count, generator=g)[:seqs * width].to(torch.int32).view(seqs, width)
    table[3, 1 if width > 1 else 0], table[4, -1] = -1, count
    lens = [new, new + 50, new + 7, new + 40, width * size, 10 ** 6, new // 2, -5, new + 1]
    t = trees(new, seqs, new)
    path = np.full((seqs, new), -1, np.int32)
    for b in range(seqs):
        nodes = way(t[b], int(rng.integers(0, new)))
        path[b, :len(nodes)] = nodes
    path[1] = np.arange(new)                 # nothing moves
    path[2] = np.sort(rng.permutation(new))  # the same
    path[8, :] = -1                          # nothing is kept
    path[5, :3] = [0, new - 1, new - 1]      # ends at what does not grow
    path[6, :2] = [1, new]                   # and at what is no node
    for counts in (None, [new, 3, new, new // 2, new, new, new, 2, 0]):
        a, b = [p.clone() for p in view], [p.clone() for p in dev]
        bv = [p.transpose(2, 3) if layout == "rows" else p for p in b]
        use = [new] * seqs if counts is None else counts
        want = keep(a, table, lens, path, use, width, size)
        new_lens = torch.full((seqs,), -9, dtype=torch.int32, device="cuda")
        args = bv if layers > 1 else [p[0] for p in bv]
        serve.keep_path(new_lens, *args, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                        torch.from_numpy(path).cuda(),
                        counts=None if counts is None else torch.tensor(counts, dtype=torch.int32).cuda())
        assert new_lens.tolist() == want
        for x, y in zip(a, bv):
            assert torch.equal(x.view(torch.int16) if x.is_contiguous() else x, y.cpu().view(torch.int16) if x.is_contiguous() else y.cpu())
    assert dview[0].shape == view[0].shape


def test_keep_path_more_sequences_than_a_grid_has_rows(gpu):
    import torch

    from nightrun_amd import serve

    n, size, new = 70000, 4, 3
    g = gen(1)
    kp, vp = (torch.randn(n, 1, size, 8, generator=g).half().cuda() for _ in range(2))
    table = torch.arange(n, dtype=torch.int32).view(n, 1).cuda()
    lens = torch.full((n,), 4, dtype=torch.int32, device="cuda")
    path = torch.tensor([[0, 2, -1]], dtype=torch.int32).repeat(n, 1).cuda()
    wk, wv = kp.clone(), vp.clone()
    for w in (wk, wv):
        w[:, :, 2] = w[:, :, 3]
    out = torch.empty_like(lens)
    serve.keep_path(out, kp, vp, table, lens, path)
    assert torch.equal(kp, wk) and torch.equal(vp, wv) and bool((out == 3).all())


# ---- refusals from Python, overlaps -------------------------------------------------------------------


def test_tree_refusals(gpu):
    import torch

    from nightrun_amd import NrqError, serve

    x = torch.randn(4, 6, 64, device="cuda")
    pos = torch.arange(4, dtype=torch.int32, device="cuda")
    f = torch.from_numpy(freqs(32)).cuda()
    w = torch.ones(64, device="cuda")
    y = torch.empty_like(x)
    for bad in (dict(w=w[:63]), dict(w=w.half()), dict(w=w.cpu()), dict(pos=pos.long()), dict(pos=pos[:3]), dict(y=y.half())):
        a = dict(y=y, x=x, w=w, pos=pos, f=f)
        a.update(bad)
        with pytest.raises(ValueError):
            serve.norm_rope(*a.values())
    with pytest.raises(NrqError):
        serve.norm_rope(y, x, w, pos, f, eps=-1.0)
    flat = torch.randn(4 * 6 * 64 + 64, device="cuda")
    with pytest.raises(NrqError, match="shares memory"):
        serve.norm_rope(flat[64:].view(4, 6, 64), flat[:-64].view(4, 6, 64), w, pos, f)
    with pytest.raises(NrqError, match="shares memory"):
        serve.norm_rope(flat[:1536].view(4, 6, 64), x, flat[100:164], pos, f)

    c = Cache(gen(1), [40, 30], 2, 64, 16, "f16")
    kp, vp, table, lens = c.dev()
    par = torch.from_numpy(trees(1, 2, 5)).cuda()
    q = torch.randn(2, 5, 4, 64, device="cuda")
    o = torch.empty_like(q)
    for bad in (dict(par=par.long()), dict(par=par[:, :4].contiguous()), dict(par=par.t().contiguous().t()), dict(par=par.cpu()),
                dict(lens=lens[:1])):
        a = dict(o=o, q=q, kp=kp, vp=vp, table=table, lens=lens, par=par)
        a.update(bad)
        with pytest.raises(ValueError):
            serve.tree_attention(*a.values(), 0.1)
    with pytest.raises(NrqError, match="shares memory"):
        serve.tree_attention(q, q, kp, vp, table, lens, par, 0.1)
    long = torch.zeros(2, 65, dtype=torch.int32, device="cuda")
    many = torch.randn(2, 65, 4, 64, device="cuda")
    with pytest.raises(NrqError, match="64"):
        serve.tree_attention(torch.empty_like(many), many, kp, vp, table, lens, long, 0.1)

    target, drafted, parents, u = (x.cuda() for x in verify_case(1, 2, 5, 100))
    t, p, a = torch.empty_like(drafted), torch.empty_like(drafted), torch.empty(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        serve.verify_tree(t, p, a, target, drafted[:, :4], parents, u)
    with pytest.raises(ValueError):
        serve.verify_tree(t, p, a, target.double(), drafted, parents, u)
    for args in ((t, t, a), (drafted, p, a), (t, parents, a), (t, p, t.view(-1)[:2])):
        with pytest.raises(NrqError, match="shares memory"):
            serve.verify_tree(*args, target, drafted, parents, u)
    path = torch.zeros(2, 5, dtype=torch.int32, device="cuda")
    with pytest.raises(NrqError, match="shares memory"):
        serve.keep_path(lens, kp, vp, table, lens, path)
    with pytest.raises(ValueError):
        serve.keep_path(torch.empty_like(lens), kp, vp, table, lens, path[:1])
    with pytest.raises(ValueError):
        serve.keep_path(torch.empty_like(lens), kp[None], vp, table, lens, path)


class Arena:
    """Arguments of a C entry in one block of memory, each at the beginning of a slot of its own. Everything is zeros: whatever a
    call is made of them stays in their memory."""

    SLOT = 8 << 20

    def __init__(self, entry):
        import torch

        from nightrun_amd import _lib

        _lib.init(0)
        self.entry, self.a = entry, getattr(self, entry[len("nrq_dev_"):])()
        self.size = {n: x[0] for n, x in self.a.items() if isinstance(x, tuple)}  # bytes, alignment
        self.align = {n: x[1] for n, x in self.a.items() if isinstance(x, tuple)}
        self.block = torch.zeros(len(self.size) * self.SLOT, dtype=torch.uint8, device="cuda")
        self.at = {n: self.block.data_ptr() + i * self.SLOT for i, n in enumerate(self.size)}

    def call(self, **moved):
        """The status and what went wrong, with arguments moved to other addresses."""
        import ctypes as C

        import torch

        from nightrun_amd import _lib
        from nightrun_amd.serve import PagedKv, PageTable

        self.block.zero_()
        p, args = {**self.at, **moved}, []
        for n, x in self.a.items():
            if n in ("k_pages", "v_pages", "pages"):
                continue
            if n == "kv":
                args.append(C.byref(PagedKv(p["k_pages"], p["v_pages"], *x)))
            elif n == "table":
                args.append(C.byref(PageTable(p["pages"], *x)))
            elif n == "strides":
                args.append((C.c_int64 * len(x))(*x))
            else:
                args.append(p[n] if n in p else x)
        rc = getattr(_lib.lib(), self.entry)(*args, torch._C._cuda_getCurrentRawStream(0))
        torch.cuda.synchronize()
        return rc, _lib.lib().nrq_last_error().decode()

    # ---- arguments in order: (bytes, alignment), or what they are; a cache's three pages of 16 positions of one head of 64

    def pools(self):
        return dict(k_pages=(6144, 16), v_pages=(6144, 16), pages=(16, 4), kv=[1024, 1024, 64, 3, 16, 1, 64, 16], table=[2, 2, 2])

    def norm_rope(self):
        return dict(y=(2048, 4), x=(2048, 4), dtype=0, tokens=4, heads=2, hd=64, strides=[128, 64, 128, 64], weight=(256, 4),
                    eps=1e-6, pos=(16, 4), freqs=(128, 4), nf=32, style=1, scale=1.0)

    def norm_rope_append(self):
        return dict(y=(2048, 4), q=(2048, 4), k=(1024, 4), v=(1024, 4), dtype=0, tokens=4, heads=2,
                    strides=[128, 64, 64, 64, 64, 64, 128, 64], norm=1, q_weight=(256, 4), k_weight=(256, 4), eps=1e-6,
                    pos=(16, 4), seq=(16, 4), at=(16, 4), freqs=(128, 4), nf=32, style=1, scale=1.0, **self.pools())

    def tree_attention(self):
        import ctypes as C

        from nightrun_amd import _lib
        from nightrun_amd.serve import PagedKv

        pools, n = self.pools(), C.c_size_t()
        kv = PagedKv(0, 0, *pools["kv"])
        assert _lib.lib().nrq_tree_attention_workspace(2, 5, 2, C.byref(kv), C.byref(n)) == 0 and n.value < self.SLOT
        return dict(out=(5120, 4), q=(5120, 4), dtype=0, n_new=5, heads=2, strides=[640, 128, 64, 640, 128, 64], **pools,
                    lens=(8, 4), parents=(40, 4), counts=(8, 4), scale=0.1, window=0, lse=(80, 4), ws=(n.value, 16),
                    ws_bytes=n.value)

    def verify_tree(self):
        return dict(tokens=(24, 4), path=(24, 4), accepted=(8, 4), target=(2400, 4), strides=[300, 100], drafted=(24, 4),
                    parents=(24, 4), uniforms=(24, 4), counts=(8, 4), seqs=2, n_new=3, vocab=100, ws=(56, 16), ws_bytes=56)

    def keep_path(self):
        return dict(new_lens=(8, 4), layers=2, layer_stride=4096, **{**self.pools(), "k_pages": (14336, 16), "v_pages": (14336, 16)},
                    lens=(8, 4), path=(24, 4), counts=(8, 4), n_new=3)


OUTPUTS = {"nrq_dev_norm_rope": ["y"], "nrq_dev_norm_rope_append": ["y", "k_pages", "v_pages"],
           "nrq_dev_tree_attention": ["out", "lse", "ws"], "nrq_dev_verify_tree": ["tokens", "path", "accepted", "ws"],
           "nrq_dev_keep_path": ["new_lens", "k_pages", "v_pages"]}


@pytest.mark.parametrize("entry", OUTPUTS)
def test_tree_shared_memory(gpu, entry):
    """Each output over the last bytes of each other argument, and right behind it: refused and taken."""
    a = Arena(entry)
    assert a.call()[0] == 0
    for out in OUTPUTS[entry]:
        for other in a.size:
            if other == out:
                continue
            end, n = a.at[other] + a.size[other], a.align[out]
            rc, text = a.call(**{out: (end - 1) // n * n})
            assert rc == -1 and ("shares memory" in text or "share memory" in text), (out, other, rc, text)
            assert a.call(**{out: -(-end // n) * n})[0] == 0, (out, other)
    if "y" in a.a:
        assert a.call(y=a.at["x" if "x" in a.a else "q"])[0] == 0  # in place


# ---- a step of them together ---------------------------------------------------------------------------


class TreeStep:
    """Norms, rotation and append of a tree's nodes, attention, acceptance of a path, the move of its keys and values
    in every layer."""

    def __init__(self, seed, seqs=3, new=14, layers=2, heads=8, kv=2, hd=64, vocab=2000, kind="f32", cache="f16"):
        import torch

        g = gen(seed)
        self.seqs, self.new, self.layers, self.heads, self.kv, self.hd = seqs, new, layers, heads, kv, hd
        size, width = 16, 9
        self.size = size
        pages = seqs * width
        self.kp0, self.vp0 = (torch.randn(layers, pages, kv, size, hd, generator=g).to(dt(cache)).cuda() for _ in range(2))
        self.kp, self.vp = self.kp0.clone(), self.vp0.clone()
        self.table = torch.randperm(pages, generator=g).to(torch.int32).view(seqs, width).cuda()
        before = torch.randint(3, width * size - new, (seqs,), generator=g, dtype=torch.int32)
        self.before = before
        self.lens = (before + new).cuda()
        target, drafted, parents, u = verify_case(seed, seqs, new, vocab)
        self.target, self.drafted, self.parents, self.u = (x.cuda() for x in (target, drafted, parents, u))
        depth = torch.tensor([[len(way(parents[b].numpy(), j)) - 1 for j in range(new)] for b in range(seqs)], dtype=torch.int32)
        j = torch.arange(new, dtype=torch.int32)
        self.pos, self.at = ((before[:, None] + x).reshape(-1).contiguous().cuda() for x in (depth, j.expand(seqs, new)))
        self.seq = torch.arange(seqs, dtype=torch.int32).repeat_interleave(new).cuda()
        self.qkv = [normal(g, seqs * new, heads + 2 * kv, hd, kind=kind) for _ in range(layers)]
        self.w = [1 + normal(g, hd, scale=0.2) for _ in range(2)]
        self.freqs = torch.from_numpy(freqs(hd // 2)).cuda()
        self.q = torch.empty(layers, seqs * new, heads, hd, dtype=dt(kind), device="cuda")
        self.y = torch.empty(layers, seqs, new, heads, hd, dtype=dt(kind), device="cuda")
        self.tokens, self.path = (torch.empty(seqs, new, dtype=torch.int32, device="cuda") for _ in range(2))
        self.accepted, self.new_lens = (torch.empty(seqs, dtype=torch.int32, device="cuda") for _ in range(2))

    def run(self, stream=None):
        from nightrun_amd import serve

        for i in range(self.layers):
            q, k, v = self.qkv[i].split([self.heads, self.kv, self.kv], 1)
            serve.norm_rope_append(self.q[i], q, k, v, *self.w, self.pos, self.seq, self.freqs, self.kp[i], self.vp[i],
                                   self.table, neox=True, at=self.at, stream=stream)
            serve.tree_attention(self.y[i], self.q[i].view(self.y[i].shape), self.kp[i], self.vp[i], self.table, self.lens,
                                 self.parents, self.hd ** -0.5, stream=stream)
        serve.verify_tree(self.tokens, self.path, self.accepted, self.target, self.drafted, self.parents, self.u, stream=stream)
        serve.keep_path(self.new_lens, self.kp, self.vp, self.table, self.lens, self.path, stream=stream)

    def results(self):
        # what lies in the sequences, not what the tree left behind
        out = [self.q, self.y, self.tokens, self.path, self.accepted, self.new_lens]
        for b, n in enumerate(self.new_lens.tolist()):
            t = np.arange(n)
            pages = self.table[b].cpu().long()[t // self.size].cuda()
            out += [p[:, pages, :, (t % self.size).tolist()] for p in (self.kp, self.vp)]
        return [x.clone() for x in out]

    def reset(self):
        self.kp.copy_(self.kp0)
        self.vp.copy_(self.vp0)
        for x in (self.q, self.y, self.tokens, self.path, self.accepted, self.new_lens):
            x.fill_(3)


def test_tree_step(gpu):
    """Each node's output is what the tokens on its way give one after the other, in a cache that has nothing else; what is kept is
    what a sequence without the tree would hold."""
    import torch

    from nightrun_amd import serve

    s = TreeStep(1)
    s.run()
    got = s.results()
    want = verify_tree(*(x.cpu().numpy() for x in (s.target, s.drafted, s.parents, s.u)), [s.new] * s.seqs)
    for g, w in zip(got[2:5], want):
        assert np.array_equal(g.cpu().numpy(), w)
    assert s.new_lens.tolist() == [int(n) + int(a) + 1 for n, a in zip(s.before, want[2])]
    for b in range(s.seqs):
        nodes = want[1][b][:want[2][b] + 1].tolist()
        n = int(s.before[b]) + len(nodes)
        kp, vp = s.kp0.clone(), s.vp0.clone()
        rows = torch.tensor([b * s.new + j for j in nodes], device="cuda")
        pos = (int(s.before[b]) + torch.arange(len(nodes), dtype=torch.int32)).cuda()
        for i in range(s.layers):
            q, k, v = (x[rows] for x in s.qkv[i].split([s.heads, s.kv, s.kv], 1))
            y = torch.empty_like(q)
            serve.norm_rope_append(y, q, k, v, *s.w, pos, torch.full_like(pos, b), s.freqs, kp[i], vp[i], s.table, neox=True)
            out = torch.empty(1, len(nodes), s.heads, s.hd, device="cuda")
            serve.paged_attention(out, y[None], kp[i], vp[i], s.table[b:b + 1], torch.tensor([n], dtype=torch.int32).cuda(),
                                  s.hd ** -0.5)
            # the same keys, values and queries to the bit; sums in another order, 32 bits both: 200 weights of 2^-24
            # relative, scores within 68 roundings of |q||k| scale <= 64 * 4 * 4 / 8
            assert torch.equal(s.q[i][rows], y)
            assert float((s.y[i][b, nodes] - out[0]).abs().max()) <= 5e-5
        t = np.arange(n)
        pages = s.table[b].cpu().long()[t // s.size].cuda()
        for p, kept in ((kp, s.kp), (vp, s.vp)):
            assert torch.equal(p[:, pages, :, (t % s.size).tolist()], kept[:, pages, :, (t % s.size).tolist()])


def test_tree_step_in_graphs(gpu):
    """Two captured steps, replayed in turn and on two streams at once, with eager work and synchronizations between."""
    import torch

    steps = [TreeStep(2), TreeStep(3, seqs=5, new=40, hd=128, kind="bf16", cache="bf16")]
    want = []
    for s in steps:
        s.run()
        torch.cuda.synchronize()
        want.append(s.results())
    graphs = []
    for s in steps:
        s.reset()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.run()
        graphs.append(g)
    eager = TreeStep(4)
    streams = [torch.cuda.Stream() for _ in steps]
    for turn_ in range(4):
        for s in steps:
            s.reset()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        eager.reset()
        eager.run()
        torch.cuda.synchronize()
        for s, w in zip(steps, want):
            for a, b in zip(s.results(), w):
                assert torch.equal(a, b), turn_


def test_tree_step_on_a_stream(gpu):
    """All calls on a stream that is not the current one, and from two host threads."""
    import threading

    import torch

    steps = [TreeStep(5), TreeStep(6, new=33)]
    want = []
    for s in steps:
        s.run()
        torch.cuda.synchronize()
        want.append(s.results())
        s.reset()
    torch.cuda.synchronize()

    def work(s, st):
        for _ in range(10):
            with torch.cuda.stream(st):
                s.reset()
            s.run(stream=st)
        st.synchronize()

    threads = [threading.Thread(target=work, args=(s, torch.cuda.Stream())) for s in steps]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for s, w in zip(steps, want):
        for a, b in zip(s.results(), w):
            assert torch.equal(a, b)
