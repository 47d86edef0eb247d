"""Operators of a serving step over torch tensors (the C ABI in include/nrq_serve.h and include/nrq_tree.h).

    serve.linear_mxfp4(qkv, w, w_scales, x)                     # 4-bit projection
    serve.rope_append(q, q, k, v, pos, seq, freqs, k_pages, v_pages, table)
    serve.paged_attention(y, q, k_pages, v_pages, table, lens, scale=hd ** -0.5)
    serve.verify_drafts(tokens, accepted, target, draft, drafted, uniforms)

and where the drafted tokens form a tree, a row of `parents` for each sequence (node 0 is the last token known, the
nodes' keys and values are the last positions of the cache, a node's rotary position counts the nodes above it):

    serve.norm_rope_append(q, q, k, v, q_weight, k_weight, pos, seq, freqs, k_pages, v_pages, table, at=at)
    serve.tree_attention(y, q, k_pages, v_pages, table, lens, parents, scale=hd ** -0.5)
    serve.verify_tree(tokens, path, accepted, target, drafted, parents, uniforms)
    serve.keep_path(new_lens, k_pages, v_pages, table, lens, path)

Outputs come first and are written in place, as in nightrun_amd.device. Every call is a kernel launch or two
on `stream` (default: torch's current stream) and may be captured into a graph; a
workspace comes from torch's allocator on that stream, so captured graphs and
streams never share one. Tensors live on the library's device, which is the
current one. Wrong types, shapes, layouts or devices raise ValueError before anything
is launched, shapes that the library refuses NrPanic, anything else it refuses NrqError: an output of
the MXFP4 functions that shares memory with an input, for one. rope(), rope_append(), norm_rope() and norm_rope_append() may
run in place (y is x or q, with the same strides); no other output may overlap an input.
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
                table: torch.Tensor, neox: bool = False, scale: float = 1.0, stream=None, at=None) -> None:
    """rope() of q [tokens, heads, head_dim] into y (which may be q) and of k [tokens, KV heads, head_dim] into the
    cache, v with it: token t at position pos[t] of sequence seq[t] (both int32). k_pages and v_pages are [pages,
    KV heads, page size, head_dim] in float16 or bfloat16, table int32 [sequences, pages of one]. A token with a
    negative seq or pos is padding and is left alone. at (int32 [tokens]): the cache positions, where they are not the
    rotary ones, as of a tree's nodes; then pos may be negative and at may not."""
    if at is not None:
        return _run(_serve.norm_rope_append, stream, y, q, k, v, False, None, None, pos, seq, freqs, k_pages, v_pages,
                    table, 0.0, neox, scale, at)
    _run(_serve.rope_append, stream, y, q, k, v, pos, seq, freqs, k_pages, v_pages, table, neox, scale)


def norm_rope(y: torch.Tensor, x: torch.Tensor, weight, pos: torch.Tensor, freqs: torch.Tensor, eps: float = 1e-6,
              neox: bool = False, scale: float = 1.0, stream=None) -> None:
    """rope() of x / sqrt(mean of x^2 over the head + eps) * weight, in one pass and rounded once. weight f32
    [head_dim], the same for all heads (None: ones)."""
    _run(_serve.norm_rope, stream, y, x, weight, pos, freqs, eps, neox, scale)


def norm_rope_append(y: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight, k_weight,
                     pos: torch.Tensor, seq: torch.Tensor, freqs: torch.Tensor, k_pages: torch.Tensor,
                     v_pages: torch.Tensor, table: torch.Tensor, eps: float = 1e-6, neox: bool = False,
                     scale: float = 1.0, at=None, stream=None) -> None:
    """rope_append() with q and k normed first, as norm_rope() does it, each with its weight. at (int32 [tokens]): the
    cache positions, where they are not the rotary ones."""
    _run(_serve.norm_rope_append, stream, y, q, k, v, True, q_weight, k_weight, pos, seq, freqs, k_pages, v_pages, table,
         eps, neox, scale, at)


def paged_attention(y: torch.Tensor, q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    table: torch.Tensor, lens: torch.Tensor, scale: float, window: int = 0, counts=None, lse=None,
                    stream=None) -> None:
    """Attention of the last tokens q [sequences, new tokens, heads, head_dim] over the cached positions of each
    sequence, theirs among them: lens int32 [sequences]. counts (int32 [sequences]): how many of the rows are new
    tokens, those behind them are left as they were. Row j is position lens - counts + j and attends to itself and
    what is before it, with window > 0 to the last `window` of those. lse (f32 [sequences, new tokens, heads]) gets the
    logarithm of the sum of exponentials."""
    _run(_serve.paged_attention, stream, y, q, k_pages, v_pages, table, lens, scale, window, counts, lse)


def tree_attention(y: torch.Tensor, q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                   lens: torch.Tensor, parents: torch.Tensor, scale: float, window: int = 0, counts=None, lse=None,
                   stream=None) -> None:
    """paged_attention() where the new tokens, at most 64, are the nodes of a tree: parents int32 [sequences, nodes]
    has the node that each follows, one before it (anything else: none). A node attends to the positions before the tree, to itself
    and to the nodes above it, with window > 0 to the last `window` of those."""
    _run(_serve.tree_attention, stream, y, q, k_pages, v_pages, table, lens, parents, scale, window, counts, lse)


def verify_drafts(tokens: torch.Tensor, accepted: torch.Tensor, target: torch.Tensor, draft, drafted: torch.Tensor,
                  uniforms: torch.Tensor, counts=None, stream=None) -> None:
    """Accepts drafted tokens (int32 [sequences, new tokens]) one after the other while uniform * draft < target of
    the token, draws the one behind them from what the target has more than the draft (or, after the last draft, from
    the target), by the last of the uniforms (f32 [sequences, new tokens + 1]). target f32 [sequences, new tokens + 1,
    vocabulary] and draft (one row less; None: the drafts were certain) hold probabilities. tokens int32 like uniforms gets the accepted
    ones, the drawn one and -1 behind; accepted int32 [sequences] how many there are. counts: drafted tokens of each
    sequence, if fewer."""
    _run(_serve.verify_drafts, stream, tokens, accepted, target, draft, drafted, uniforms, counts)


def verify_tree(tokens: torch.Tensor, path: torch.Tensor, accepted: torch.Tensor, target: torch.Tensor,
                drafted: torch.Tensor, parents: torch.Tensor, uniforms: torch.Tensor, counts=None, stream=None) -> None:
    """Accepts a path through a tree of drafted tokens, from its root (node 0, whose token is known) on: the children
    of the node reached in their order, each while uniform * (what the children refused before it left of 1) < target of its token.
    Then draws a token from that node's row without the refused ones, by the sequence's first uniform. target f32
    [sequences, nodes, vocabulary] holds the probabilities of what follows each node, uniforms f32 and drafted and parents
    int32 are [sequences, nodes], and so are the int32 outputs: tokens gets the accepted ones, the drawn one and -1 behind,
    path the nodes with the root first and -1 behind. accepted int32 [sequences]: how many drafts were. counts: nodes of
    each sequence, if fewer. The drafts count as certain, as the best tokens of a draft are."""
    _run(_serve.verify_tree, stream, tokens, path, accepted, target, drafted, parents, uniforms, counts)


def keep_path(new_lens: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
              lens: torch.Tensor, path: torch.Tensor, counts=None, stream=None) -> None:
    """Moves the keys and values of an accepted path together: of each sequence's last nodes (path.shape[1], or its
    counts) the path's come first, the rest is given up. new_lens int32 [sequences] gets the lengths then. Pages may have layers
    in front ([layers, pages, KV heads, page size, head_dim]), all of which go by the one table. path int32
    [sequences, nodes] as verify_tree() leaves it: nodes that grow, then -1."""
    _run(_serve.keep_path, stream, new_lens, k_pages, v_pages, table, lens, path, counts)


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
