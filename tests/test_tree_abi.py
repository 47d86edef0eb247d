"""include/nrq_tree.h without a GPU: its symbols, what it refuses, and what a node of a tree sees
(csrc/nrq_tree_mask.h compiled for the host)."""
import ctypes as C
import os
import random
import re
import subprocess

import pytest

from tests.test_serve_abi import _call, _i64, _kv, _table

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "nrq_tree.h")
ARG, SHAPE, UNSUPPORTED, NOT_INIT = -1, -2, -4, -5
P = 1 << 20  # aligned addresses that nothing reads, 2^32 apart


def at(i):
    return P + (i << 32)


def test_symbols():
    from nightrun_amd import _lib

    names = re.findall(r"^int (nrq_\w+)\(", open(HEADER).read(), flags=re.M)
    assert sorted(names) == sorted(_lib.TREE_SIGNATURES) and len(names) == 7
    L = C.CDLL(_lib.LIB_PATH)
    for n in names:
        assert hasattr(L, n), n


def test_header_is_plain_c(tmp_path):
    src = tmp_path / "t.c"
    src.write_text('#include "nrq_tree.h"\nint main(void) { return sizeof(nrq_paged_kv) == 64 ? 0 : 1; }\n')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.dirname(HEADER), str(src), "-o",
                    str(tmp_path / "t")], check=True)


def _norm():
    return dict(y=at(0), x=at(1), dtype=0, tokens=5, heads=4, hd=128, strides=_i64(512, 128, 512, 128), weight=at(2),
                eps=1e-6, pos=at(3), freqs=at(4), nf=64, style=1, scale=1.0, stream=None)


def _append():
    return dict(y=at(0), q=at(1), k=at(2), v=at(3), dtype=0, tokens=5, heads=32,
                strides=_i64(4096, 128, 1024, 128, 1024, 128, 4096, 128), norm=1, q_weight=at(4), k_weight=at(5),
                eps=1e-6, pos=at(6), seq=at(7), at=at(8), freqs=at(9), nf=64, style=0, scale=1.0,
                kv=_kv(k=at(10), v=at(11)), table=_table(), stream=None)


def _attend():
    return dict(out=at(0), q=at(1), dtype=0, n_new=2, heads=32, strides=_i64(8192, 4096, 128, 8192, 4096, 128),
                kv=_kv(), table=_table(pages=at(2)), lens=at(3), parents=at(4), counts=None, scale=0.1, window=0,
                lse=None, ws=at(5), ws_bytes=1 << 30, stream=None)


def _verify():
    return dict(tokens=at(0), path=at(1), accepted=at(2), target=at(3), strides=_i64(4000, 1000), drafted=at(4),
                parents=at(5), uniforms=at(6), counts=None, seqs=2, n_new=4, vocab=1000, ws=at(7), ws_bytes=1 << 20,
                stream=None)


def _keep():
    return dict(new_lens=at(0), layers=2, layer_stride=10 * 8 * 16 * 128, kv=_kv(), table=_table(pages=at(1)),
                lens=at(2), path=at(3), counts=None, n_new=8, stream=None)


CALLS = {"nrq_dev_norm_rope": _norm, "nrq_dev_norm_rope_append": _append, "nrq_dev_tree_attention": _attend,
         "nrq_dev_verify_tree": _verify, "nrq_dev_keep_path": _keep}

REFUSED = [
    ("nrq_dev_norm_rope", dict(dtype=1), ARG, "unknown type"),
    ("nrq_dev_norm_rope", dict(eps=-1e-6), ARG, "eps"),
    ("nrq_dev_norm_rope", dict(eps=float("nan")), ARG, "eps"),
    ("nrq_dev_norm_rope", dict(eps=float("inf")), ARG, "eps"),
    ("nrq_dev_norm_rope", dict(weight=P + 2), ARG, "aligned"),
    ("nrq_dev_norm_rope", dict(nf=65), SHAPE, "frequencies"),
    ("nrq_dev_norm_rope", dict(tokens=1 << 31), UNSUPPORTED, "tokens"),
    ("nrq_dev_norm_rope", dict(strides=None), ARG, "null"),
    ("nrq_dev_norm_rope", dict(pos=None), ARG, "null"),
    ("nrq_dev_norm_rope", dict(strides=_i64(512, 128, 512, 64)), ARG, "overlap"),
    ("nrq_dev_norm_rope", dict(y=at(1), strides=_i64(1024, 128, 512, 128)), ARG, "in place"),
    ("nrq_dev_norm_rope_append", dict(eps=-1.0), ARG, "eps"),
    ("nrq_dev_norm_rope_append", dict(k_weight=P + 1), ARG, "aligned"),
    ("nrq_dev_norm_rope_append", dict(at=P + 2), ARG, "aligned"),
    ("nrq_dev_norm_rope_append", dict(seq=None), ARG, "null"),
    ("nrq_dev_norm_rope_append", dict(v=None), ARG, "null"),
    ("nrq_dev_norm_rope_append", dict(table=None), ARG, "null"),
    ("nrq_dev_norm_rope_append", dict(heads=0), SHAPE, "no heads"),
    ("nrq_dev_norm_rope_append", dict(kv=_kv(pos_stride=64)), ARG, "overlap"),
    ("nrq_dev_norm_rope_append", dict(kv=_kv(dtype=0)), ARG, "type"),
    ("nrq_dev_tree_attention", dict(n_new=65), UNSUPPORTED, "64"),
    ("nrq_dev_tree_attention", dict(parents=None), ARG, "null"),
    ("nrq_dev_tree_attention", dict(parents=P + 2), ARG, "aligned"),
    ("nrq_dev_tree_attention", dict(heads=31), SHAPE, "31 heads"),
    ("nrq_dev_tree_attention", dict(window=-1), ARG, "window"),
    ("nrq_dev_tree_attention", dict(kv=_kv(head_dim=80)), UNSUPPORTED, "heads of 80"),
    ("nrq_dev_tree_attention", dict(ws_bytes=100), ARG, "workspace of 100"),
    ("nrq_dev_tree_attention", dict(ws=None), ARG, "workspace"),
    ("nrq_dev_tree_attention", dict(strides=_i64(8192, 4096, 128, 8192, 4096, 120)), ARG, "overlap"),
    ("nrq_dev_tree_attention", dict(lens=None), ARG, "null"),
    ("nrq_dev_verify_tree", dict(n_new=65), UNSUPPORTED, "64"),
    ("nrq_dev_verify_tree", dict(n_new=0), SHAPE, "root"),
    ("nrq_dev_verify_tree", dict(vocab=0), SHAPE, "vocabulary"),
    ("nrq_dev_verify_tree", dict(path=None), ARG, "null"),
    ("nrq_dev_verify_tree", dict(parents=None), ARG, "null"),
    ("nrq_dev_verify_tree", dict(uniforms=P + 2), ARG, "aligned"),
    ("nrq_dev_verify_tree", dict(ws_bytes=8), ARG, "workspace"),
    ("nrq_dev_keep_path", dict(n_new=65), UNSUPPORTED, "64"),
    ("nrq_dev_keep_path", dict(layers=4097), UNSUPPORTED, "layers"),
    ("nrq_dev_keep_path", dict(layer_stride=12), ARG, "multiple of 8"),
    ("nrq_dev_keep_path", dict(layer_stride=1024), ARG, "overlap"),
    ("nrq_dev_keep_path", dict(path=None), ARG, "null"),
    ("nrq_dev_keep_path", dict(new_lens=None), ARG, "null"),
    ("nrq_dev_keep_path", dict(lens=P + 1), ARG, "aligned"),
    ("nrq_dev_keep_path", dict(table=_table(width=2 ** 26 + 1, stride=2 ** 27)), UNSUPPORTED, "2^30"),
]


@pytest.mark.parametrize("name,change,code,text", REFUSED, ids=[f"{n[8:]}-{'-'.join(c)}-{i}" for i, (n, c, _, _) in
                                                               enumerate(REFUSED)])
def test_refusals(name, change, code, text):
    rc, msg = _call(name, CALLS[name](), **change)
    assert rc == code and text in msg and msg.startswith(name), (rc, msg)


@pytest.mark.parametrize("name", CALLS)
def test_without_a_device(name):
    """Good arguments: refused for want of nrq_init, never a silent fallback."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("checks the no-GPU failure path")
    assert _call(name, CALLS[name]())[0] == NOT_INIT
    nothing = {"nrq_dev_tree_attention": "n_new", "nrq_dev_verify_tree": "seqs", "nrq_dev_keep_path": "n_new"}
    assert _call(name, CALLS[name](), **{nothing.get(name, "tokens"): 0})[0] == NOT_INIT


def test_workspaces():
    from nightrun_amd import _lib

    L, n = _lib.lib(), C.c_size_t()
    assert L.nrq_verify_tree_workspace(3, 5000, C.byref(n)) == 0 and 0 < n.value <= 3 * 5000 * 16
    assert L.nrq_verify_tree_workspace(3, 5000, None) == ARG
    assert L.nrq_tree_attention_workspace(3, 8, 32, _kv(), C.byref(n)) == 0 and n.value >= 4 * 130 * 4
    assert L.nrq_tree_attention_workspace(3, 65, 32, _kv(), C.byref(n)) == UNSUPPORTED
    assert L.nrq_tree_attention_workspace(3, 8, 33, _kv(), C.byref(n)) == SHAPE
    assert L.nrq_tree_attention_workspace(3, 8, 32, _kv(), None) == ARG


@pytest.mark.parametrize("seqs,width,fits", [(2 ** 20, 2048, True), (2 ** 20, 16128, True), (2 ** 20, 16366, False), (2 ** 20, 16384, False)])
def test_tree_attention_line(seqs, width, fits):
    """One node, one head over one: a sequence is its tiles and what the beginning of a unit counts for; 2^31 of them are
    no int."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("checks the no-GPU failure path")
    rc, msg = _call("nrq_dev_tree_attention", _attend(), n_new=1, heads=1, ws_bytes=1 << 40,
                    strides=_i64(128, 128, 128, 128, 128, 128),
                    kv=_kv(n_kv_heads=1, page_stride=16 * 128), table=_table(pages=at(2), seqs=seqs, width=width, stride=width))
    assert rc == (NOT_INIT if fits else UNSUPPORTED), (rc, msg)
    assert fits or "too much" in msg


@pytest.mark.parametrize("layers,n_kv,hd,fits", [(1024, 2 ** 20, 1, False), (1024, 2 ** 20 - 1, 1, True), (4096, 2 ** 18, 1, False),
                                                 (4096, 2 ** 18 - 1, 1, True), (1024, 2 ** 19, 2, True), (4096, 2 ** 15, 8, True),
                                                 (1024, 1, 2 ** 20, True)])
def test_keep_path_items(layers, n_kv, hd, fits):
    """A thread has eight dimensions of a head's keys or values in a layer: the last are fewer, but a thread. 2^31 of those are no int."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("checks the no-GPU failure path")
    head = -(-hd // 8) * 8
    kv = _kv(k=at(10), v=at(2 ** 15), n_pages=2, page_size=1, n_kv_heads=n_kv, head_dim=hd, head_stride=head,
             pos_stride=n_kv * head, page_stride=n_kv * head)
    rc, msg = _call("nrq_dev_keep_path", _keep(), layers=layers, layer_stride=2 * n_kv * head, kv=kv)
    assert rc == (NOT_INIT if fits else UNSUPPORTED), (rc, msg)
    assert fits or "layers of" in msg


@pytest.mark.parametrize("seqs,fits", [(2 ** 30, True), (2 ** 30 + 1, False), (2 ** 31 - 1, False)])
def test_keep_path_sequences(seqs, fits):
    """Launches go from sequence to sequence in steps of up to 2^15 of them: behind the last, that is an int too."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("checks the no-GPU failure path")
    rc, msg = _call("nrq_dev_keep_path", _keep(), n_new=0, table=_table(pages=at(1), seqs=seqs, width=0, stride=0))
    assert rc == (NOT_INIT if fits else UNSUPPORTED), (rc, msg)
    assert fits or "sequences" in msg


# ---- what a node sees -----------------------------------------------------------------------------


@pytest.fixture(scope="module")
def mask(tmp_path_factory):
    d = tmp_path_factory.mktemp("mask")
    src = d / "mask.cpp"
    src.write_text('''#include "nrq_tree_mask.h"
extern "C" {
int parent(int p, int j) { return nrq::tree_parent(p, j); }
uint32_t sees(uint64_t above, int p0, int base) { return nrq::tree_sees(above, p0, base); }
uint32_t from(int lo, int p0, int base) { return nrq::tree_from(lo, p0, base); }
}
''')
    so = d / "mask.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-Wall", "-Werror", "-fsanitize=undefined",
                    "-fno-sanitize-recover", "-static-libubsan", "-I", os.path.join(ROOT, "nightrun_amd", "csrc"),
                    str(src), "-o", str(so)], check=True)
    L = C.CDLL(str(so))
    L.sees.argtypes, L.sees.restype = [C.c_uint64, C.c_int, C.c_int], C.c_uint32
    getattr(L, "from").restype = C.c_uint32
    return L


def test_parents(mask):
    for j in range(64):
        for p in (-2 ** 31, -1, 0, j - 1, j, j + 1, 63, 64, 2 ** 31 - 1):
            assert mask.parent(p, j) == (p if 0 <= p < j else -1)


def test_bits(mask):
    """Every bit of every 32 positions around the tree, trees before position 0 and at the largest positions among them."""
    rng = random.Random(3)
    low = getattr(mask, "from")
    for base in (-64, -40, -1, 0, 1, 31, 32, 33, 100, 2 ** 30, 2 ** 30 - 64):
        for _ in range(40):
            above = rng.getrandbits(64)
            lo = rng.choice([0, base, base - 1, base - 40, base + 3, base + 70, 2 ** 30, rng.randint(0, 200)])
            lo = max(lo, 0)
            for p0 in {max(0, base + d) for d in (-70, -64, -33, -32, -31, -16, -1, 0, 1, 16, 31, 32, 33, 63, 64, 65, 90)}:
                s, f = mask.sees(above, p0, base), low(lo, p0, base)
                for i in range(32):
                    t = p0 + i
                    r = t - base
                    assert s >> i & 1 == (1 if r < 0 else (above >> r & 1 if r < 64 else 0)), (above, p0, base, i)
                    assert f >> i & 1 == int(t >= lo or r >= 0), (lo, p0, base, i)


# ---- which tensors share memory -----------------------------------------------------------------


@pytest.fixture(scope="module")
def extent(tmp_path_factory):
    d = tmp_path_factory.mktemp("extent")
    src = d / "extent.cpp"
    src.write_text('''#include "nrq_extent.h"
extern "C" int meet(const int64_t* a, const int64_t* b) {
  const int64_t* p[2] = {a, b};
  nrq::Extent e[2];
  for (int i = 0; i < 2; i++)
    e[i] = nrq::Extent{(const void*)p[i][0], (size_t)p[i][1], (int)p[i][2],
                       {{p[i][3], (size_t)p[i][4]}, {p[i][5], (size_t)p[i][6]}, {p[i][7], (size_t)p[i][8]}}};
  return nrq::extents_meet(e[0], nrq::range_of(e[0]), e[1], nrq::range_of(e[1]));
}
''')
    so = d / "extent.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-Wall", "-Werror", "-fsanitize=undefined",
                    "-fno-sanitize-recover", "-static-libubsan", "-I", os.path.join(ROOT, "nightrun_amd", "csrc"),
                    str(src), "-o", str(so)], check=True)
    L = C.CDLL(str(so))
    return lambda a, b: bool(L.meet((C.c_int64 * 9)(*a), (C.c_int64 * 9)(*b)))


def _bytes(first, length, size, *dims):
    out = {0}
    for stride, n in dims:
        out = {o + stride * i for o in out for i in range(n)}
    return {first + (o + k) * size + e for o in out for k in range(length) for e in range(size)}


def test_extents_never_miss(extent):
    """Whatever shares a byte is found; what is apart in ranges is left alone."""
    rng = random.Random(11)
    met = apart = 0
    for _ in range(20000):
        a, b = ([4000 + rng.randint(-200, 200), rng.choice([0, 1, 2, 4, 8]), rng.choice([1, 2, 4])] +
                [x for _ in range(3) for x in (rng.choice([-24, -8, 0, 3, 8, 16, 24, 64, 130]), rng.choice([0, 1, 1, 2, 3]))]
                for _ in range(2))
        x, y = (_bytes(e[0], e[1], e[2], *zip(e[3::2], e[4::2])) for e in (a, b))
        got = extent(a, b)
        assert got == extent(b, a)
        if x & y:
            met += 1
            assert got, (a, b)
        elif not x or not y or max(x) < min(y) or max(y) < min(x):
            apart += 1
            assert not got, (a, b)
    assert met > 500 and apart > 2000


def test_extents_of_layouts(extent):
    """Layouts of one tensor: slices of a projection, keys and values of one pool, heads between heads."""
    base = 1 << 40

    def e(first, length, *dims, size=2):
        dims = list(dims) + [(0, 1)] * (3 - len(dims))
        return [base + first * size, length, size] + [x for d in dims for x in d]

    t, h, kv, hd = 100, 32, 8, 128
    row = (h + 2 * kv) * hd
    q, k, v = e(0, hd, (row, t), (hd, h)), e(h * hd, hd, (row, t), (hd, kv)), e((h + kv) * hd, hd, (row, t), (hd, kv))
    for i, x in enumerate((q, k, v)):
        for j, y in enumerate((q, k, v)):
            assert extent(x, y) == (i == j)
    assert extent(q, e(h * hd - 1, hd, (row, t), (hd, kv)))
    p, size = 50, 16
    one = 2 * kv * size * hd  # [pages][2][heads][positions][hd], [pages][positions][2][heads][hd]
    pools = ([(one, p), (size * hd, kv), (hd, size)], kv * size * hd), ([(one, p), (hd, kv), (2 * kv * hd, size)], kv * hd)
    for dims, off in pools:
        assert not extent(e(0, hd, *dims), e(off, hd, *dims))
        assert extent(e(0, hd, *dims), e(off - 1, hd, *dims))
    extent(e(0, hd, (2 ** 62, 3)), e(hd, hd, (-2 ** 62, 7)))  # past any memory: either answer, no overflow
    assert extent(e(0, hd, (0, 5)), e(1, hd))
    assert not extent(e(0, hd, (row, 0)), e(0, hd))


@pytest.fixture(scope="module")
def copies(tmp_path_factory):
    d = tmp_path_factory.mktemp("copies")
    src = d / "copies.cpp"
    src.write_text('''#include "nrq_extent.h"
extern "C" int meet(const int64_t* a, int64_t other) {
  const nrq::Extent e{(const void*)a[0], (size_t)a[1], (int)a[2], {{a[3], (size_t)a[4]}, {a[5], (size_t)a[6]}, {a[7], (size_t)a[8]}}};
  return nrq::copies_meet(e, (const void*)other);
}
''')
    so = d / "copies.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-Wall", "-Werror", "-fsanitize=undefined",
                    "-fno-sanitize-recover", "-static-libubsan", "-I", os.path.join(ROOT, "nightrun_amd", "csrc"),
                    str(src), "-o", str(so)], check=True)
    L = C.CDLL(str(so))
    return lambda a, other: bool(L.meet((C.c_int64 * 9)(*a), C.c_int64(other)))


def test_copies_meet(copies):
    """Keys and values of any layouts whose rows do not overlap, at any distance: exact."""
    rng = random.Random(5)
    met = between = 0
    for _ in range(30000):
        length, size = rng.choice([0, 1, 2, 4, 8]), rng.choice([1, 2])
        span, dims = length, []
        for _ in range(3):
            stride, n = span + rng.choice([0, 0, 1, 8, span, 2 * span + 3]), rng.choice([0, 1, 1, 2, 3, 4])
            dims.append((stride, n))
            if n > 1:
                span += stride * (n - 1)
        rng.shuffle(dims)
        first = 1 << 20
        other = first + rng.randint(-size * (span + 10), size * (span + 10))
        x = _bytes(first, length, size, *dims)
        y = {i + other - first for i in x}
        got = copies([first, length, size] + [v for d in dims for v in d], other)
        assert got == bool(x & y), (length, size, dims, other - first)
        met += got
        between += not got and bool(x) and max(x) >= min(y) and max(y) >= min(x)
    assert met > 3000 and between > 2000


def test_copies_of_layouts(copies):
    """Keys and values of one pool, some of its pages, some of its heads, at its far end; the same pool twice."""
    base, kv, size, hd, layers, pages = 1 << 40, 8, 16, 128, 28, 1000

    def e(*dims):
        return [base, hd, 2] + [x for d in dims for x in d]

    one = kv * size * hd
    for k, off in ((e((2 * one, pages), (size * hd, kv), (hd, size)), one),  # [pages][2][heads][positions]
                   (e((2 * one, pages), (size * hd, kv // 2), (hd, size)), one // 2),  # and half of the heads
                   (e((2 * one, pages), (hd, kv), (2 * kv * hd, size)), kv * hd),  # [pages][positions][2][heads]
                   (e((2 * one * (pages + 7), layers), (2 * one, pages), (hd, size * kv)), one),  # some pages of each layer
                   (e((one, pages), (size * hd, kv), (hd, size)), one * pages), (e((2 ** 61, 4), (one, 3), (hd, size)), one * 3)):
        gap = one - size * hd if off == one * 3 else 0  # one head's pages at the distance of all heads'
        for sign in (1, -1):
            assert not copies(k, base + 2 * off * sign) and not copies(k, base + 2 * (off - gap) * sign)
            assert copies(k, base + (2 * (off - gap) - 2) * sign) and copies(k, base + 16 * sign)
        assert copies(k, base)


def test_extents_of_four_dimensions(tmp_path):
    """The caches of some layers: layers, pages, heads and positions come down to rows at one distance, whichever of them follow one
    another without gaps. What lies beside a layer's pages in its part of memory is apart from them."""
    src = tmp_path / "four.cpp"
    src.write_text('''#include "nrq_extent.h"
#include <cstdio>
#include <initializer_list>
int main() {
  typedef nrq::Extent E;
  auto meet = [](const E& a, const E& b) { return nrq::extents_meet(a, nrq::range_of(a), b, nrq::range_of(b)); };
  const uintptr_t base = 1l << 40;
  const int64_t hd = 128, size = 16, kv = 8, pages = 50, layers = 5, one = hd * size * kv, gap = 4096;
  const size_t s = size, h = kv, p = pages, l = layers;
  const int64_t layer = pages * one + gap;
  const E dense{(void*)base, (size_t)hd, 2, {{one, p}, {size * hd, h}, {hd, s}, {layer, l}}};
  const E rows{(void*)base, (size_t)hd, 2, {{one, p}, {hd, h}, {kv * hd, s}, {layer, l}}};
  const E two{(void*)base, (size_t)hd, 2, {{2 * one, p}, {size * hd, h}, {hd, s}, {2 * one * pages, l}}};
  int bad = 0;
  for (const E& e : {dense, rows})
    for (int i = 0; i < layers; i++) {
      const uintptr_t end = base + 2 * (layer * i + pages * one);
      bad += meet(E{(void*)end, (size_t)gap, 2, {}}, e) || meet(e, E{(void*)end, (size_t)gap, 2, {}});
      bad += !meet(E{(void*)(end - 4), 1, 4, {}}, e) || !meet(e, E{(void*)(end - 4), 1, 4, {}});
      if (i + 1 < layers) bad += !meet(E{(void*)(end + 4), (size_t)gap, 2, {}}, e);
    }
  for (int i = 0; i < layers * pages; i++) {  // values between the keys
    bad += meet(E{(void*)(base + 2 * (2 * i + 1) * one), (size_t)one, 2, {}}, two);
    bad += !meet(E{(void*)(base + 2 * (2 * i + 1) * one - 4), 1, 4, {}}, two);
  }
  const E copy{(void*)(base + 2 * one), (size_t)hd, 2, {{2 * one, p}, {size * hd, h}, {hd, s}, {2 * one * pages, l}}};
  bad += meet(copy, two) || nrq::copies_meet(two, copy.first) || !nrq::copies_meet(two, (void*)(base + 2 * one - 16));
  bad += !nrq::copies_meet(two, (void*)(base + 4 * one * pages * (layers - 1))) || nrq::copies_meet(two, (void*)(base + 4 * one * pages * layers));
  printf("%d\\n", bad);
  return bad != 0;
}
''')
    subprocess.run(["g++", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-static-libubsan", "-I",
                    os.path.join(ROOT, "nightrun_amd", "csrc"), str(src), "-o", str(tmp_path / "four")], check=True)
    subprocess.run([str(tmp_path / "four")], check=True)


SHARED = [
    ("nrq_dev_norm_rope", "y", "x", 128), ("nrq_dev_norm_rope", "y", "weight", 0), ("nrq_dev_norm_rope", "y", "freqs", 0),
    ("nrq_dev_norm_rope_append", "y", "k", 0), ("nrq_dev_norm_rope_append", "y", "pos", 0),
    ("nrq_dev_tree_attention", "out", "q", 0), ("nrq_dev_tree_attention", "ws", "q", 0), ("nrq_dev_tree_attention", "out", "lens", 0),
    ("nrq_dev_verify_tree", "tokens", "path", 0), ("nrq_dev_verify_tree", "path", "parents", 0),
    ("nrq_dev_verify_tree", "accepted", "uniforms", 4), ("nrq_dev_keep_path", "new_lens", "lens", 0),
]


@pytest.mark.parametrize("name,out,other,by", SHARED)
def test_overlaps_reach_the_check(name, out, other, by):
    """Asked last, behind the device: without one the arguments are otherwise good."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("checks the no-GPU failure path")
    a = CALLS[name]()
    assert _call(name, a, **{out: a[other] + by})[0] == NOT_INIT
