"""include/nrq_serve.h without a GPU: its symbols, what it refuses, and the index
arithmetic of the paged cache (csrc/nrq_page.h compiled for the host)."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "nrq_serve.h")
ARG, SHAPE, UNSUPPORTED, NOT_INIT = -1, -2, -4, -5
P = 1 << 20  # an aligned address that nothing reads


def test_symbols():
    from nightrun_amd import _lib

    names = re.findall(r"^int (nrq_\w+)\(", open(HEADER).read(), flags=re.M)
    assert sorted(names) == sorted(_lib.SERVE_SIGNATURES) and len(names) == 12
    L = C.CDLL(_lib.LIB_PATH)
    for n in names:
        assert hasattr(L, n), n


def test_header_is_plain_c(tmp_path):
    src = tmp_path / "t.c"
    src.write_text('#include "nrq.h"\n#include "nrq_serve.h"\nint main(void) { return sizeof(nrq_paged_kv) == 64 && '
                   'sizeof(nrq_page_table) == 24 ? 0 : 1; }\n')
    exe = tmp_path / "t"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)],
                   check=True)
    assert subprocess.run([str(exe)]).returncode == 0
    from nightrun_amd import serve
    assert C.sizeof(serve.PagedKv) == 64 and C.sizeof(serve.PageTable) == 24


def _call(name, args, **change):
    from nightrun_amd import _lib

    a = dict(args)
    a.update(change)
    L = _lib.lib()
    rc = getattr(L, name)(*a.values())
    return rc, L.nrq_last_error().decode()


def _i64(*v):
    return (C.c_int64 * len(v))(*v)


def _kv(**change):
    from nightrun_amd.serve import PagedKv

    d = dict(k=P, v=P, page_stride=8 * 16 * 128, head_stride=16 * 128, pos_stride=128, n_pages=10, page_size=16,
             n_kv_heads=8, head_dim=128, dtype=16)
    d.update(change)
    return C.byref(PagedKv(*d.values()))


def _table(**change):
    from nightrun_amd.serve import PageTable

    d = dict(pages=P, stride=4, seqs=3, width=4)
    d.update(change)
    return C.byref(PageTable(*d.values()))


def _rope():
    return dict(y=P, x=P + 4096, dtype=0, tokens=5, heads=4, hd=128, strides=_i64(512, 128, 512, 128), pos=P, freqs=P,
                nf=64, style=1, scale=1.0, stream=None)


def _append():
    return dict(y=P, q=P + 4096, k=P, v=P, dtype=0, tokens=5, heads=32,
                strides=_i64(4096, 128, 1024, 128, 1024, 128, 4096, 128), pos=P, seq=P, freqs=P, nf=64, style=0,
                scale=1.0, kv=_kv(), table=_table(), stream=None)


def _attend():
    return dict(out=P, q=P, dtype=0, n_new=2, heads=32, strides=_i64(8192, 4096, 128, 8192, 4096, 128), kv=_kv(),
                table=_table(), lens=P, counts=None, scale=0.1, window=0, lse=None, ws=P, ws_bytes=1 << 30, stream=None)


def _verify():
    return dict(tokens=P, accepted=P, target=P, draft=P, strides=_i64(4000, 1000, 3000, 1000), drafted=P, uniforms=P,
                counts=None, seqs=2, n_new=3, vocab=1000, ws=P, ws_bytes=1 << 20, stream=None)


def _quant():
    return dict(src=P, dtype=0, rows=3, cols=64, stride=64, q=P, s=P, stream=None)


def _dequant():
    return dict(q=P, s=P, rows=3, cols=64, dst=P, dtype=0, stride=64, stream=None)


def _matmul():
    return dict(y=P, dtype=0, ldy=40, w=P, ws=P, x=P, xs=P, rows=40, cols=64, batch=5, wk=None, wk_bytes=0,
                stream=None)


def _linear():
    return dict(y=P, dtype=0, ldy=40, w=P, ws=P, x=P, x_dtype=0, ldx=64, rows=40, cols=64, batch=505, wk=P,
                wk_bytes=1 << 20, stream=None)


CALLS = {"nrq_dev_rope": _rope, "nrq_dev_rope_append": _append, "nrq_dev_paged_attention": _attend,
         "nrq_dev_verify_drafts": _verify, "nrq_dev_quantize_mxfp4": _quant, "nrq_dev_dequantize_mxfp4": _dequant,
         "nrq_dev_matmul_mxfp4": _matmul, "nrq_dev_linear_mxfp4": _linear}

REFUSED = [
    ("nrq_dev_rope", dict(dtype=1), ARG, "unknown type"),
    ("nrq_dev_rope", dict(style=2), ARG, "style"),
    ("nrq_dev_rope", dict(nf=0), SHAPE, "frequencies"),
    ("nrq_dev_rope", dict(nf=65), SHAPE, "frequencies"),
    ("nrq_dev_rope", dict(hd=1026, nf=4), SHAPE, "1026"),
    ("nrq_dev_rope", dict(tokens=1 << 31), UNSUPPORTED, "tokens"),
    ("nrq_dev_rope", dict(heads=1 << 20), UNSUPPORTED, "heads"),
    ("nrq_dev_rope", dict(pos=None), ARG, "null"),
    ("nrq_dev_rope", dict(strides=None), ARG, "null"),
    ("nrq_dev_rope", dict(x=P + 2), ARG, "aligned"),
    ("nrq_dev_rope", dict(strides=_i64(512, 128, 512, 64)), ARG, "overlap"),
    ("nrq_dev_rope", dict(strides=_i64(512, 128, 0, 128)), ARG, "overlap"),
    ("nrq_dev_rope", dict(y=P, x=P, strides=_i64(1024, 128, 512, 128)), ARG, "in place"),
    ("nrq_dev_rope_append", dict(seq=None), ARG, "null"),
    ("nrq_dev_rope_append", dict(k=None), ARG, "null"),
    ("nrq_dev_rope_append", dict(kv=None), ARG, "null"),
    ("nrq_dev_rope_append", dict(table=None), ARG, "null"),
    ("nrq_dev_rope_append", dict(kv=_kv(dtype=0)), ARG, "type"),
    ("nrq_dev_rope_append", dict(kv=_kv(page_size=0)), SHAPE, "positions"),
    ("nrq_dev_rope_append", dict(kv=_kv(pos_stride=129)), ARG, "multiples of 8"),
    ("nrq_dev_rope_append", dict(kv=_kv(k=P + 8)), ARG, "16-byte"),
    ("nrq_dev_rope_append", dict(kv=_kv(v=None)), ARG, "null"),
    ("nrq_dev_rope_append", dict(table=_table(width=-1)), SHAPE, "table"),
    ("nrq_dev_rope_append", dict(table=_table(pages=None)), ARG, "null"),
    ("nrq_dev_paged_attention", dict(dtype=3), ARG, "unknown type"),
    ("nrq_dev_paged_attention", dict(window=-1), ARG, "window"),
    ("nrq_dev_paged_attention", dict(heads=31), SHAPE, "31 heads"),
    ("nrq_dev_paged_attention", dict(kv=_kv(head_dim=80)), UNSUPPORTED, "heads of 80"),
    ("nrq_dev_paged_attention", dict(lens=None), ARG, "null"),
    ("nrq_dev_paged_attention", dict(strides=_i64(8192, 4096, 128, 8192, 4096, 120)), ARG, "overlap"),
    ("nrq_dev_paged_attention", dict(ws_bytes=100), ARG, "workspace of 100"),
    ("nrq_dev_paged_attention", dict(ws=None), ARG, "workspace"),
    ("nrq_dev_paged_attention", dict(ws=P + 8), ARG, "aligned"),
    ("nrq_dev_paged_attention", dict(n_new=70000), UNSUPPORTED, "rows"),
    ("nrq_dev_paged_attention", dict(kv=_kv(n_pages=2 ** 31 - 1)), UNSUPPORTED, "elements"),
    ("nrq_dev_paged_attention", dict(table=_table(width=2 ** 25, stride=2 ** 25, seqs=20)), UNSUPPORTED, "too much"),
    ("nrq_dev_paged_attention", dict(table=_table(width=2 ** 26 + 1, stride=2 ** 27)), UNSUPPORTED, "2^30"),
    ("nrq_dev_rope_append", dict(kv=_kv(page_size=2 ** 31 - 1)), UNSUPPORTED, "elements"),
    ("nrq_dev_verify_drafts", dict(n_new=65), UNSUPPORTED, "64"),
    ("nrq_dev_verify_drafts", dict(vocab=0), SHAPE, "vocabulary"),
    ("nrq_dev_verify_drafts", dict(target=None), ARG, "null"),
    ("nrq_dev_verify_drafts", dict(drafted=None), ARG, "null"),
    ("nrq_dev_verify_drafts", dict(draft=P + 2), ARG, "aligned"),
    ("nrq_dev_verify_drafts", dict(ws_bytes=8), ARG, "workspace"),
    ("nrq_dev_quantize_mxfp4", dict(cols=48), SHAPE, "32"),
    ("nrq_dev_quantize_mxfp4", dict(dtype=9), ARG, "unknown type"),
    ("nrq_dev_quantize_mxfp4", dict(q=P + 4), ARG, "aligned"),
    ("nrq_dev_quantize_mxfp4", dict(s=None), ARG, "null"),
    ("nrq_dev_dequantize_mxfp4", dict(stride=32), ARG, "overlap"),
    ("nrq_dev_dequantize_mxfp4", dict(cols=33), SHAPE, "32"),
    ("nrq_dev_matmul_mxfp4", dict(cols=40), SHAPE, "32"),
    ("nrq_dev_matmul_mxfp4", dict(ldy=39), ARG, "overlap"),
    ("nrq_dev_matmul_mxfp4", dict(x=P + 8), ARG, "aligned"),
    ("nrq_dev_matmul_mxfp4", dict(w=None), ARG, "null"),
    ("nrq_dev_matmul_mxfp4", dict(batch=(1 << 20) + 1), UNSUPPORTED, "batch"),
    ("nrq_dev_matmul_mxfp4", dict(ldy=2560, rows=2560, cols=9728, batch=128), ARG, "workspace"),
    ("nrq_dev_linear_mxfp4", dict(x_dtype=5), ARG, "unknown type"),
    ("nrq_dev_linear_mxfp4", dict(wk_bytes=100), ARG, "workspace"),
    ("nrq_dev_linear_mxfp4", dict(x=None), ARG, "null"),
    # rows that would overlap although each stride alone is wide enough
    ("nrq_dev_rope", dict(strides=_i64(512, 128, 256, 128)), ARG, "overlap"),
    ("nrq_dev_rope", dict(strides=_i64(512, 128, 128, 512)), ARG, "overlap"),
    ("nrq_dev_rope", dict(strides=_i64(512, 128, 512, -128)), ARG, "overlap"),
    ("nrq_dev_paged_attention", dict(strides=_i64(8192, 4096, 128, 4096, 4096, 128)), ARG, "overlap"),
    ("nrq_dev_paged_attention", dict(strides=_i64(8192, 4096, 128, 8192, 4000, 128)), ARG, "overlap"),
    ("nrq_dev_rope_append", dict(kv=_kv(pos_stride=64)), ARG, "overlap"),
    ("nrq_dev_rope_append", dict(kv=_kv(head_stride=0)), ARG, "overlap"),
    ("nrq_dev_rope_append", dict(kv=_kv(page_stride=1024)), ARG, "overlap"),
    ("nrq_dev_rope_append", dict(heads=0), SHAPE, "no heads"),
]


@pytest.mark.parametrize("name,change,code,text", REFUSED, ids=[f"{n[8:]}-{'-'.join(c)}-{i}" for i, (n, c, _, _) in
                                                               enumerate(REFUSED)])
def test_refusals(name, change, code, text):
    rc, msg = _call(name, CALLS[name](), **change)
    assert rc == code and text in msg and msg.startswith(name), (rc, msg)


@pytest.mark.parametrize("name", CALLS)
def test_without_a_device(name):
    """Good arguments: refused for want of nrq_init (also when nothing is to be done), never a silent fallback."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("checks the no-GPU failure path")
    assert _call(name, CALLS[name]())[0] == NOT_INIT
    empty = {"nrq_dev_rope": "tokens", "nrq_dev_rope_append": "tokens", "nrq_dev_paged_attention": "n_new",
             "nrq_dev_verify_drafts": "seqs"}.get(name, "rows")
    assert _call(name, CALLS[name](), **{empty: 0})[0] == NOT_INIT


def test_workspaces():
    from nightrun_amd import _lib

    L, n = _lib.lib(), C.c_size_t()
    assert L.nrq_linear_mxfp4_workspace(40, 64, 505, C.byref(n)) == 0 and n.value == 505 * 32 + 1024
    assert L.nrq_linear_mxfp4_workspace(40, 64, 5, C.byref(n)) == 0 and n.value == 0  # quantized where it is used
    assert L.nrq_linear_mxfp4_workspace(40, 65, 5, C.byref(n)) == SHAPE
    assert L.nrq_matmul_mxfp4_workspace(40, 65, 5, C.byref(n)) == SHAPE
    assert L.nrq_matmul_mxfp4_workspace(40, 64, 5, C.byref(n)) == 0 and n.value == 0
    # planes of sums where few tiles share long rows
    assert L.nrq_matmul_mxfp4_workspace(2556, 9728, 128, C.byref(n)) == 0 and n.value % (128 * 2560 * 4) == 0 < n.value
    planes = n.value
    assert L.nrq_linear_mxfp4_workspace(2556, 9728, 128, C.byref(n)) == 0 and n.value == planes + 128 * 9728 * 17 // 32
    assert L.nrq_verify_workspace(3, 5000, C.byref(n)) == 0 and 0 < n.value <= 3 * 5000 * 16
    assert L.nrq_paged_attention_workspace(3, 1, 32, _kv(), C.byref(n)) == 0 and n.value >= 4 * 130 * 4
    assert L.nrq_paged_attention_workspace(3, 1, 33, _kv(), C.byref(n)) == SHAPE
    assert L.nrq_paged_attention_workspace(3, 1, 32, _kv(), None) == ARG


# ---- the paged cache's index arithmetic ---------------------------------------------------


@pytest.fixture(scope="module")
def page(tmp_path_factory):
    d = tmp_path_factory.mktemp("page")
    src = d / "page.cpp"
    src.write_text('''#include "nrq_page.h"
extern "C" {
uint32_t place(const int* p, int w, int ps, int n, uint32_t a, uint32_t b, int t) { return nrq::page_place(p, w, ps, n, a, b, t); }
void span(int len, int count, int n_new, int64_t held, int window, int tile, int* o) {
  nrq::SeqSpan s = nrq::seq_span(len, count, n_new, held, window, tile);
  o[0] = s.len; o[1] = s.n; o[2] = s.start; o[3] = s.tiles;
}
int start(int w, int t, int n) { return nrq::line_start(w, t, n); }
int owner(int g, int t, int n) { return nrq::line_owner(g, t, n); }
}
''')
    so = d / "page.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-Wall", "-Werror", "-fsanitize=undefined",
                    "-fno-sanitize-recover", "-static-libubsan", "-I", os.path.join(ROOT, "nightrun_amd", "csrc"),
                    str(src), "-o", str(so)], check=True)
    L = C.CDLL(str(so))
    i, q, u = C.c_int, C.c_int64, C.c_uint32
    L.place.argtypes, L.place.restype = [C.c_void_p, i, i, i, u, u, i], u
    L.span.argtypes = [i, i, i, q, i, i, C.c_void_p]
    L.start.argtypes, L.start.restype = [i, i, i], i
    L.owner.argtypes, L.owner.restype = [i, i, i], i
    return L


@pytest.mark.parametrize("size", [1, 2, 16, 24, 1000])
def test_places(page, size):
    """Every position of a table with bad entries: the page's place, or none."""
    table = np.array([3, -1, 7, 8, 0, -2 ** 31, 2 ** 31 - 1, 5], np.int32)
    n_pages, ps, ts, none = 8, 3 * 2 ** 27, 17, 2 ** 32 - 1
    for t in list(range(-3, 8 * size + 3)) + [2 ** 31 - 1, -2 ** 31]:
        want = none
        if 0 <= t < 8 * size and 0 <= table[t // size] < n_pages:
            want = int(table[t // size]) * ps + (t % size) * ts
        assert page.place(table.ctypes.data, 8, size, n_pages, ps, ts, t) == want, t
    assert page.place(table.ctypes.data, 0, size, n_pages, ps, ts, 0) == none


def test_spans(page):
    """What the new tokens see lies in the tiles, which lie within what is held."""
    out = (C.c_int * 4)()
    tile = 128
    for held in (0, 1, 127, 1000, 2 ** 40):
        for length in (-5, 0, 1, 5, 127, 128, 129, 1000, 70000, 2 ** 31 - 1):
            for count, n_new in ((1, 1), (-1, 4), (0, 4), (3, 4), (4, 4), (9, 4)):
                for window in (0, 1, 7, 16, 500, 2 ** 31 - 1):
                    page.span(length, count, n_new, held, window, tile, out)
                    ln, n, start, tiles = out
                    assert n == min(max(count, 0), n_new)
                    assert ln == (0 if n == 0 else min(max(length, 0), held, 2 ** 31 - 1))
                    low = max(0, ln - n + 1 - window) if window else 0
                    assert 0 <= start <= low and low - start < 16 and start % 16 == 0
                    assert tiles >= 1 and start + tiles * tile >= ln
                    assert tiles == 1 or start + (tiles - 1) * tile < ln


@pytest.mark.parametrize("total,wgs", [(1, 1), (7, 3), (7, 7), (1000, 64), (1023, 1024), (999983, 1024),
                                       (2 ** 31 - 1, 1024), (2 ** 31 - 1024, 1023)])
def test_line(page, total, wgs):
    """Every tile has one owner, whose stretch holds it; every workgroup has a stretch."""
    wgs = min(total, wgs)
    starts = [page.start(w, total, wgs) for w in range(wgs + 1)]
    assert starts[0] == 0 and starts[-1] == total and all(a < b for a, b in zip(starts, starts[1:]))
    rng = np.random.default_rng(total % 1000)
    some = range(total) if total < 2000 else [0, total - 1] + [int(x) for x in rng.integers(0, total, 500)] + \
        [s for s in starts[:-1]] + [s - 1 for s in starts[1:]]
    for g in some:
        w = page.owner(g, total, wgs)
        assert 0 <= w < wgs and starts[w] <= g < starts[w + 1], (g, w)


# ---- sizes that no launch takes ---------------------------------------------------------------


@pytest.mark.parametrize("seqs,width,fits", [(2 ** 21, 9, False), (2 ** 21 - 1, 9, True), (2 ** 21, 8, True), (2 ** 23, 8, True)])
def test_attention_units(seqs, width, fits):
    """Eight units a sequence; 2^24 need a grid of 2^32 threads where sequences hold more than a tile of 128."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("checks the no-GPU failure path")
    rc, msg = _call("nrq_dev_paged_attention", _attend(), n_new=1, ws_bytes=1 << 40, strides=_i64(8192, 4096, 128, 4096, 4096, 128),
                    table=_table(seqs=seqs, width=width, stride=width))
    assert rc == (NOT_INIT if fits else UNSUPPORTED), (rc, msg)
    assert fits or "too much" in msg


@pytest.mark.parametrize("name,change,fits", [
    ("nrq_dev_quantize_mxfp4", dict(rows=2 ** 30, cols=64, stride=64), False),
    ("nrq_dev_quantize_mxfp4", dict(rows=2 ** 30 - 64, cols=64, stride=64), True),
    ("nrq_dev_quantize_mxfp4", dict(rows=2 ** 31 - 1023, cols=32, stride=32), False),
    ("nrq_dev_dequantize_mxfp4", dict(rows=2 ** 30, cols=64, stride=64), False),
    ("nrq_dev_dequantize_mxfp4", dict(rows=2 ** 30 - 64, cols=64, stride=64), True),
    ("nrq_dev_matmul_mxfp4", dict(rows=2 ** 31 - 1, batch=1), False),  # rounded up to tiles it would be negative
    ("nrq_dev_matmul_mxfp4", dict(rows=2 ** 31 - 1, cols=0, batch=1), False),
    ("nrq_dev_matmul_mxfp4", dict(rows=2 ** 31 - 1025, batch=1), True),
    ("nrq_dev_matmul_mxfp4", dict(rows=2 ** 30, batch=129, ldy=2 ** 30), False),  # 2^24 tiles
    ("nrq_dev_matmul_mxfp4", dict(rows=2 ** 30 - 1024, batch=129, ldy=2 ** 30), True),
    ("nrq_dev_linear_mxfp4", dict(rows=40, cols=2 ** 16 + 64, batch=2 ** 20, wk_bytes=2 ** 40), False),  # the activation's values
    ("nrq_dev_linear_mxfp4", dict(rows=2 ** 31 - 1, batch=1), False),
    ("nrq_dev_linear_mxfp4", dict(rows=2 ** 30, batch=129, ldy=2 ** 30), False),
    ("nrq_dev_linear_mxfp4", dict(rows=2 ** 30 - 1024, batch=128, ldy=2 ** 30), True)])
def test_mx_sizes(name, change, fits):
    """Sizes that a launch does not hold are refused, those below them are not."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("checks the no-GPU failure path")
    rc, msg = _call(name, CALLS[name](), **change)
    assert rc == (NOT_INIT if fits else UNSUPPORTED), (rc, msg)
