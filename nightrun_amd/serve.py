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
is launched, shapes that the library refuses NrPanic, anything else it refuses NrqError: an output of
the MXFP4 functions that shares memory with an input, for one. rope() and rope_append() may run in place (y is x or q, with
the same strides); no other output may overlap an input.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

_lib.lib()  # libnrq.so, which the next one is linked to, and torch before both

from . import _serve  # noqa: E402


class PagedKv(C.Structure):
    """nrq_paged_kv"""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("page_stride", C.c_int64), ("head_stride", C.c_int64),
                ("pos_stride", C.c_int64), ("n_pages", C.c_int32), ("page_size", C.c_int32),
                ("n_kv_heads", C.c_int32), ("head_dim", C.c_int32), ("dtype", C.c_int32)]


class PageTable(C.Structure):
    """nrq_page_table"""
    _fields_ = [("pages", C.c_void_p), ("stride", C.c_int64), ("seqs", C.c_int32), ("width", C.c_int32)]


def _run(fn, stream, *args) -> None:
    if stream is not None:  # the workspace is that stream's too
        with torch.cuda.stream(stream):
            return _run(fn, None, *args)
    dev = torch.cuda.current_device()
    _lib.init(dev)
    rc = fn(*args, dev, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        _lib.check(rc)


def rope(y: torch.Tensor, x: torch.Tensor, pos: torch.Tensor, freqs: torch.Tensor, neox: bool = False,
         scale: float = 1.0, stream=None) -> None:
    """Rotary positions of x [tokens, heads, head_dim] at pos int32 [tokens] into y (which may be x). Pair i of the
    first 2 len(freqs) dimensions, (2i, 2i + 1) or with neox (i, i + len(freqs)), turns by pos * freqs[i] (formed in
    64 bits) and is multiplied by scale; the dimensions behind are copied. freqs f32 holds the context scaling."""
    _run(_serve.rope, stream, y, x, pos, freqs, neox, scale)


def rope_append(y: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor,
                seq: torch.Tensor, freqs: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                table: torch.Tensor, neox: bool = False, scale: float = 1.0, stream=None) -> None:
    """rope() of q [tokens, heads, head_dim] into y (which may be q) and of k [tokens, KV heads, head_dim] into the
    cache, v with it: token t at position pos[t] of sequence seq[t] (both int32). k_pages and v_pages are [pages,
    KV heads, page size, head_dim] in float16 or bfloat16, table int32 [sequences, pages of one]. A token with a
    negative seq or pos is padding and is left alone."""
    _run(_serve.rope_append, stream, y, q, k, v, pos, seq, freqs, k_pages, v_pages, table, neox, scale)


def paged_attention(y: torch.Tensor, q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    table: torch.Tensor, lens: torch.Tensor, scale: float, window: int = 0, counts=None, lse=None,
                    stream=None) -> None:
    """Attention of the last tokens q [sequences, new tokens, heads, head_dim] over the cached positions of each
    sequence, theirs among them: lens int32 [sequences]. counts (int32 [sequences]): how many of the rows are new
    tokens, those behind them are left as they were. Row j is position lens - counts + j and attends to itself and
    what is before it, with window > 0 to the last `window` of those. lse (f32 [sequences, new tokens, heads]) gets the
    logarithm of the sum of exponentials."""
    _run(_serve.paged_attention, stream, y, q, k_pages, v_pages, table, lens, scale, window, counts, lse)


def verify_drafts(tokens: torch.Tensor, accepted: torch.Tensor, target: torch.Tensor, draft, drafted: torch.Tensor,
                  uniforms: torch.Tensor, counts=None, stream=None) -> None:
    """Accepts drafted tokens (int32 [sequences, new tokens]) one after the other while uniform * draft < target of
    the token, draws the one behind them from what the target has more than the draft (or, after the last draft, from
    the target), by the last of the uniforms (f32 [sequences, new tokens + 1]). target f32 [sequences, new tokens + 1,
    vocabulary] and draft (one row less; None: the drafts were certain) hold probabilities. tokens int32 like uniforms gets the accepted
    ones, the drawn one and -1 behind; accepted int32 [sequences] how many there are. counts: drafted tokens of each
    sequence, if fewer."""
    _run(_serve.verify_drafts, stream, tokens, accepted, target, draft, drafted, uniforms, counts)


def quantize_mxfp4(src: torch.Tensor, q: torch.Tensor, scales: torch.Tensor, stream=None) -> None:
    """src [rows, cols] to MXFP4: q uint8 [rows, cols / 2] (the first of two values in the low bits), scales uint8
    [rows, cols / 32], exponents of 2 plus 127."""
    _run(_serve.quantize_mxfp4, stream, src, q, scales)


def dequantize_mxfp4(q: torch.Tensor, scales: torch.Tensor, out: torch.Tensor, stream=None) -> None:
    """The values that q and scales stand for, rounded to out's type."""
    _run(_serve.dequantize_mxfp4, stream, q, scales, out)


def matmul_mxfp4(y: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, x: torch.Tensor, x_scales: torch.Tensor,
                 stream=None) -> None:
    """y [batch, rows] = x w^T, both in MXFP4: w [rows, cols / 2], x [batch, cols / 2] and their scales."""
    _run(_serve.matmul_mxfp4, stream, y, w, w_scales, x, x_scales)


def linear_mxfp4(y: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, x: torch.Tensor, stream=None) -> None:
    """y [batch, rows] = x w^T with w in MXFP4 and x [batch, cols] quantized to it on the way."""
    _run(_serve.linear_mxfp4, stream, y, w, w_scales, x)
