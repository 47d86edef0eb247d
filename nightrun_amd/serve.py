"""Operators of a serving step over torch tensors (the C ABI in include/nrq_serve.h).

    serve.linear_mxfp4(qkv, w, w_scales, x)                     # 4-bit projection
    serve.rope_append(q, q, k, v, pos, seq, freqs, k_pages, v_pages, table)
    serve.paged_attention(y, q, k_pages, v_pages, table, lens, scale=hd ** -0.5)
    serve.verify_drafts(tokens, accepted, target, draft, drafted, uniforms)

Outputs come first and are written in place, as in nightrun_amd.device. Every call is a kernel launch or two
on `stream` (default: torch's current stream) and may be captured into a graph; a
workspace comes from torch's allocator on that stream, so captured graphs and
streams never share one. Tensors live on the library's device, which is the
current one. Wrong types, shapes, layouts or devices raise ValueError before anything
is launched, shapes that the library refuses NrPanic, anything else it refuses NrqError.
"""
from __future__ import annotations

import contextlib
import ctypes as C

import torch

from . import _lib

F32, F16, BF16 = _lib.F32, _lib.F16, _lib.BF16
DTYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


class PagedKv(C.Structure):
    """nrq_paged_kv"""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("page_stride", C.c_int64), ("head_stride", C.c_int64),
                ("pos_stride", C.c_int64), ("n_pages", C.c_int32), ("page_size", C.c_int32),
                ("n_kv_heads", C.c_int32), ("head_dim", C.c_int32), ("dtype", C.c_int32)]


class PageTable(C.Structure):
    """nrq_page_table"""
    _fields_ = [("pages", C.c_void_p), ("stride", C.c_int64), ("seqs", C.c_int32), ("width", C.c_int32)]


_I2, _I4, _I6, _I8 = (C.c_int64 * n for n in (2, 4, 6, 8))


def _start() -> int:
    dev = torch.cuda.current_device()
    _lib.init(dev)
    return dev


def _stream(stream):
    return (stream if stream is not None else torch.cuda.current_stream()).cuda_stream


def _on(t: torch.Tensor, what: str, dev: int) -> int:
    if t.get_device() != dev:
        raise ValueError(f"{what}: expected a tensor on cuda:{dev}, got one on {t.device}")
    return t.data_ptr()


def _ints(t: torch.Tensor, what: str, dev: int, shape) -> int:
    if t.dtype is not torch.int32 or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{what}: expected a contiguous int32 tensor of shape {tuple(shape)}, got {t.dtype} "
                         f"{tuple(t.shape)}")
    return _on(t, what, dev)


def _kind(t: torch.Tensor, what: str) -> int:
    d = DTYPES.get(t.dtype)
    if d is None:
        raise ValueError(f"{what}: expected float32, float16 or bfloat16, got {t.dtype}")
    return d


def _rows(t: torch.Tensor, what: str, dims: int) -> None:
    """`dims` dimensions, the last of them contiguous."""
    if t.dim() != dims or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{what}: expected {dims} dimensions, the last contiguous, got shape {tuple(t.shape)}, "
                         f"strides {t.stride()}")


def _workspace(n: int, dev: int, stream) -> torch.Tensor:
    with torch.cuda.stream(stream) if stream is not None else contextlib.nullcontext():
        return torch.empty(n, dtype=torch.uint8, device=f"cuda:{dev}")


def _paged(k: torch.Tensor, v: torch.Tensor, dev: int) -> PagedKv:
    """Pools [pages, KV heads, positions of a page, head_dim], any strides but the last."""
    _rows(k, "k_pages", 4)
    _rows(v, "v_pages", 4)
    if k.dtype is not v.dtype or k.shape != v.shape or k.stride() != v.stride():
        raise ValueError("k_pages and v_pages differ in type, shape or strides")
    kind = _kind(k, "k_pages")
    if kind == F32:
        raise ValueError("k_pages: expected float16 or bfloat16")
    n, heads, size, hd = k.shape
    sp, sh, st, _ = k.stride()
    return PagedKv(_on(k, "k_pages", dev), _on(v, "v_pages", dev), sp, sh, st, n, size, heads, hd, kind)


def _table(t: torch.Tensor, dev: int) -> PageTable:
    if t.dtype is not torch.int32:
        raise ValueError(f"table: expected int32, got {t.dtype}")
    _rows(t, "table", 2)
    return PageTable(_on(t, "table", dev), t.stride(0), t.shape[0], t.shape[1])


def _same(y: torch.Tensor, x: torch.Tensor, what: str) -> None:
    if y.shape != x.shape or y.dtype is not x.dtype:
        raise ValueError(f"{what}: expected {x.dtype} {tuple(x.shape)}, got {y.dtype} {tuple(y.shape)}")


def _freqs(f: torch.Tensor, dev: int) -> int:
    if f.dtype is not torch.float32 or f.dim() != 1 or not f.is_contiguous():
        raise ValueError("freqs: expected a contiguous float32 vector")
    return _on(f, "freqs", dev)


def rope(y: torch.Tensor, x: torch.Tensor, pos: torch.Tensor, freqs: torch.Tensor, neox: bool = False,
         scale: float = 1.0, stream=None) -> None:
    """Rotary positions of x [tokens, heads, head_dim] at pos int32 [tokens] into y (which may be x). Pair i of the
    first 2 len(freqs) dimensions, (2i, 2i + 1) or with neox (i, i + len(freqs)), turns by pos * freqs[i] (formed in
    64 bits) and is multiplied by scale; the dimensions behind are copied. freqs f32 holds the context scaling."""
    dev = _start()
    _rows(x, "x", 3)
    _rows(y, "y", 3)
    _same(y, x, "y")
    n, heads, hd = x.shape
    s = _I4(x.stride(0), x.stride(1), y.stride(0), y.stride(1))
    _lib.check(_lib.lib().nrq_dev_rope(_on(y, "y", dev), _on(x, "x", dev), _kind(x, "x"), n, heads, hd, s,
                                       _ints(pos, "pos", dev, (n,)), _freqs(freqs, dev), freqs.numel(), int(neox),
                                       scale, _stream(stream)))


def rope_append(y: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor,
                seq: torch.Tensor, freqs: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                table: torch.Tensor, neox: bool = False, scale: float = 1.0, stream=None) -> None:
    """rope() of q [tokens, heads, head_dim] into y (which may be q) and of k [tokens, KV heads, head_dim] into the
    cache, v with it: token t at position pos[t] of sequence seq[t] (both int32). k_pages and v_pages are [pages,
    KV heads, page size, head_dim] in float16 or bfloat16, table int32 [sequences, pages of one]. A token with a
    negative seq or pos is padding and is left alone."""
    dev = _start()
    for t, what in ((q, "q"), (k, "k"), (v, "v"), (y, "y")):
        _rows(t, what, 3)
    _same(y, q, "y")
    _same(v, k, "v")
    n, heads, hd = q.shape
    if k.dtype is not q.dtype or tuple(k.shape) != (n, k_pages.shape[1], hd) or k_pages.shape[3] != hd:
        raise ValueError(f"k: expected {q.dtype} {(n, k_pages.shape[1], hd)}, got {k.dtype} {tuple(k.shape)}; "
                         f"pages {tuple(k_pages.shape)}")
    kv, tab = _paged(k_pages, v_pages, dev), _table(table, dev)
    s = _I8(q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), y.stride(0), y.stride(1))
    _lib.check(_lib.lib().nrq_dev_rope_append(
        _on(y, "y", dev), _on(q, "q", dev), _on(k, "k", dev), _on(v, "v", dev), _kind(q, "q"), n, heads, s,
        _ints(pos, "pos", dev, (n,)), _ints(seq, "seq", dev, (n,)), _freqs(freqs, dev), freqs.numel(), int(neox),
        scale, C.byref(kv), C.byref(tab), _stream(stream)))


def paged_attention(y: torch.Tensor, q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    table: torch.Tensor, lens: torch.Tensor, scale: float, window: int = 0, counts=None, lse=None,
                    stream=None) -> None:
    """Attention of the last tokens q [sequences, new tokens, heads, head_dim] over the cached positions of each
    sequence, theirs among them: lens int32 [sequences]. counts (int32 [sequences]): how many of the rows are new
    tokens, those behind them are left as they were. Row j is position lens - counts + j and attends to itself and
    what is before it, with window > 0 to the last `window` of those. lse (f32 [sequences, new tokens, heads]) gets the
    logarithm of the sum of exponentials."""
    dev = _start()
    _rows(q, "q", 4)
    _rows(y, "y", 4)
    _same(y, q, "y")
    b, n, heads, hd = q.shape
    kv, tab = _paged(k_pages, v_pages, dev), _table(table, dev)
    if tab.seqs != b or kv.head_dim != hd:
        raise ValueError(f"q {tuple(q.shape)} does not go with pages {tuple(k_pages.shape)} and table "
                         f"{tuple(table.shape)}")
    if lse is not None and (lse.dtype is not torch.float32 or tuple(lse.shape) != (b, n, heads) or
                            not lse.is_contiguous()):
        raise ValueError(f"lse: expected a contiguous float32 tensor of shape {(b, n, heads)}")
    L, need = _lib.lib(), C.c_size_t()
    _lib.check(L.nrq_paged_attention_workspace(n, heads, C.byref(kv), C.byref(need)))
    ws = _workspace(need.value, dev, stream)
    s = _I6(q.stride(0), q.stride(1), q.stride(2), y.stride(0), y.stride(1), y.stride(2))
    _lib.check(L.nrq_dev_paged_attention(
        _on(y, "y", dev), _on(q, "q", dev), _kind(q, "q"), n, heads, s, C.byref(kv), C.byref(tab),
        _ints(lens, "lens", dev, (b,)), _ints(counts, "counts", dev, (b,)) if counts is not None else None, scale,
        window, _on(lse, "lse", dev) if lse is not None else None, ws.data_ptr(), need.value, _stream(stream)))


def verify_drafts(tokens: torch.Tensor, accepted: torch.Tensor, target: torch.Tensor, draft, drafted: torch.Tensor,
                  uniforms: torch.Tensor, counts=None, stream=None) -> None:
    """Accepts drafted tokens (int32 [sequences, new tokens]) one after the other while uniform * draft < target of
    the token, draws the one behind them from what the target has more than the draft (or, after the last draft, from
    the target), by the last of the uniforms (f32 [sequences, new tokens + 1]). target f32 [sequences, new tokens + 1,
    vocabulary] and draft (one row less; None: the drafts were certain) hold probabilities. tokens int32 like uniforms gets the accepted
    ones, the drawn one and -1 behind; accepted int32 [sequences] how many there are. counts: drafted tokens of each
    sequence, if fewer."""
    dev = _start()
    _rows(target, "target", 3)
    b, rows, vocab = target.shape
    n = rows - 1
    if target.dtype is not torch.float32 or n < 0:
        raise ValueError("target: expected float32 [sequences, new tokens + 1, vocabulary]")
    if draft is not None:
        _rows(draft, "draft", 3)
        if draft.dtype is not torch.float32 or tuple(draft.shape) != (b, n, vocab):
            raise ValueError(f"draft: expected float32 {(b, n, vocab)}, got {draft.dtype} {tuple(draft.shape)}")
    if uniforms.dtype is not torch.float32 or tuple(uniforms.shape) != (b, rows) or not uniforms.is_contiguous():
        raise ValueError(f"uniforms: expected a contiguous float32 tensor of shape {(b, rows)}")
    L, need = _lib.lib(), C.c_size_t()
    _lib.check(L.nrq_verify_workspace(b, vocab, C.byref(need)))
    ws = _workspace(need.value, dev, stream)
    s = _I4(target.stride(0), target.stride(1), *((draft.stride(0), draft.stride(1)) if draft is not None else (0, 0)))
    _lib.check(L.nrq_dev_verify_drafts(
        _ints(tokens, "tokens", dev, (b, rows)), _ints(accepted, "accepted", dev, (b,)), _on(target, "target", dev),
        _on(draft, "draft", dev) if draft is not None else None, s, _ints(drafted, "drafted", dev, (b, n)),
        _on(uniforms, "uniforms", dev), _ints(counts, "counts", dev, (b,)) if counts is not None else None, b, n,
        vocab, ws.data_ptr(), need.value, _stream(stream)))


def _mx(q: torch.Tensor, s: torch.Tensor, what: str, dev: int):
    """(pointers, rows, columns) of a matrix in MXFP4: q uint8 [rows, cols / 2], scales uint8 [rows, cols / 32]."""
    if q.dtype is not torch.uint8 or s.dtype is not torch.uint8 or q.dim() != 2 or s.dim() != 2 or \
            not q.is_contiguous() or not s.is_contiguous() or q.shape[0] != s.shape[0] or q.shape[1] != 16 * s.shape[1]:
        raise ValueError(f"{what}: expected contiguous uint8 [rows, cols / 2] and [rows, cols / 32], got "
                         f"{tuple(q.shape)} and {tuple(s.shape)}")
    return _on(q, what, dev), _on(s, what, dev), q.shape[0], 2 * q.shape[1]


def quantize_mxfp4(src: torch.Tensor, q: torch.Tensor, scales: torch.Tensor, stream=None) -> None:
    """src [rows, cols] to MXFP4: q uint8 [rows, cols / 2] (the first of two values in the low bits), scales uint8
    [rows, cols / 32], exponents of 2 plus 127."""
    dev = _start()
    _rows(src, "src", 2)
    qp, sp, rows, cols = _mx(q, scales, "q, scales", dev)
    if tuple(src.shape) != (rows, cols):
        raise ValueError(f"src: expected {(rows, cols)}, got {tuple(src.shape)}")
    _lib.check(_lib.lib().nrq_dev_quantize_mxfp4(_on(src, "src", dev), _kind(src, "src"), rows, cols, src.stride(0),
                                                 qp, sp, _stream(stream)))


def dequantize_mxfp4(q: torch.Tensor, scales: torch.Tensor, out: torch.Tensor, stream=None) -> None:
    """The values that q and scales stand for, rounded to out's type."""
    dev = _start()
    _rows(out, "out", 2)
    qp, sp, rows, cols = _mx(q, scales, "q, scales", dev)
    if tuple(out.shape) != (rows, cols):
        raise ValueError(f"out: expected {(rows, cols)}, got {tuple(out.shape)}")
    _lib.check(_lib.lib().nrq_dev_dequantize_mxfp4(qp, sp, rows, cols, _on(out, "out", dev), _kind(out, "out"),
                                                   out.stride(0), _stream(stream)))


def matmul_mxfp4(y: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, x: torch.Tensor, x_scales: torch.Tensor,
                 stream=None) -> None:
    """y [batch, rows] = x w^T, both in MXFP4: w [rows, cols / 2], x [batch, cols / 2] and their scales."""
    dev = _start()
    _rows(y, "y", 2)
    wp, wsp, rows, cols = _mx(w, w_scales, "w, w_scales", dev)
    xp, xsp, batch, xc = _mx(x, x_scales, "x, x_scales", dev)
    if xc != cols or tuple(y.shape) != (batch, rows):
        raise ValueError(f"y {tuple(y.shape)}: x is [{batch}, {xc}], w [{rows}, {cols}]")
    _lib.check(_lib.lib().nrq_dev_matmul_mxfp4(_on(y, "y", dev), _kind(y, "y"), y.stride(0), wp, wsp, xp, xsp, rows,
                                               cols, batch, _stream(stream)))


def linear_mxfp4(y: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, x: torch.Tensor, stream=None) -> None:
    """y [batch, rows] = x w^T with w in MXFP4 and x [batch, cols] quantized to it on the way."""
    dev = _start()
    _rows(y, "y", 2)
    _rows(x, "x", 2)
    wp, wsp, rows, cols = _mx(w, w_scales, "w, w_scales", dev)
    batch = x.shape[0]
    if x.shape[1] != cols or tuple(y.shape) != (batch, rows):
        raise ValueError(f"y {tuple(y.shape)}: x is {tuple(x.shape)}, w [{rows}, {cols}]")
    L, need = _lib.lib(), C.c_size_t()
    _lib.check(L.nrq_linear_mxfp4_workspace(cols, batch, C.byref(need)))
    ws = _workspace(need.value, dev, stream)
    _lib.check(L.nrq_dev_linear_mxfp4(_on(y, "y", dev), _kind(y, "y"), y.stride(0), wp, wsp, _on(x, "x", dev),
                                      _kind(x, "x"), x.stride(0), rows, cols, batch, ws.data_ptr(), need.value,
                                      _stream(stream)))
