"""Attention over the cached latents of whole sequences: trees of drafted tokens, windows with a few first keys, or every key.

The sparse attention reads the keys that the indexer selected, at most some thousands to a token, each token its own.  These operators read what a
sequence has in the cache through its block table, in the absorbed form (keys of 512 + 64 channels, values their 512), and share what they read
among all heads and all of the sequence's tokens:

* a tree of drafted tokens (``tree_mask``): each sees everything before the tree and, of the tree, what its mask says, its ancestors and itself.
  The nodes' own latents are in the cache already, behind the context, in the order of the nodes;
* a window (``window``, ``sinks``): a token sees the last keys up to its own and the first few of the sequence, which stay visible;
* neither: a token sees all keys up to its own.

Sequences' query tokens lie one behind the other, one or hundreds to a sequence.  ``cache_slots`` makes the beginnings and the masks.  The cache is
that of the sparse attention, in its three arrays or packed.

Calling convention as for the other operators; queries and the output may be strided bare tensors: the last dimension alone has to be contiguous.
"""
from __future__ import annotations

import math

import torch

from . import _native
from .cache_layout_impl import _lengths, _mask, _typed
from .converter import as_rows, as_torch, check_writable, refuse_overlap
from .latent_cache_impl import _cache_tensors
from .prompt_attention_impl import check_window
from .rotary_position_impl import _on_gpu
from .sparse_flash_attention_quant_impl import KV_LORA_RANK, ROPE_DIM


def _attend(op, query_nope, query_rope, parts, names, block_table, cu_seqlens_q, seq_lens, attention_out, softmax_scale, block_size, window, sinks,
            tree_mask, softmax_lse):
    C = _native.load()
    window, sinks = check_window(window, sinks)
    pad = list(parts) + [None] * (3 - len(parts))
    if C.latent_attention_call(query_nope, query_rope, *pad, block_table, cu_seqlens_q, seq_lens, attention_out, softmax_scale, block_size, window or 0, sinks,
                               tree_mask, softmax_lse):
        return None
    qn, qr, out = (as_rows(t, n) for t, n in ((query_nope, "query_nope"), (query_rope, "query_rope"), (attention_out, "attention_out")))
    for t, n, width in ((qn, "query_nope", KV_LORA_RANK), (qr, "query_rope", ROPE_DIM), (out, "attention_out", KV_LORA_RANK)):
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{n}: expected torch.bfloat16, got {t.dtype}")
        if t.dim() != 3 or tuple(t.shape) != (*qn.shape[:2], width) or t.shape[1] < 1:
            raise ValueError(f"{n}: expected shape (total_q, heads, {width}), got {tuple(t.shape)}")
    cache = _cache_tensors(parts, names)
    table = _typed(block_table, "block_table", torch.int32, 2)
    lens = _lengths(seq_lens, "seq_lens", table)
    cu = _typed(cu_seqlens_q, "cu_seqlens_q", torch.int32, 1)
    if cu.shape[0] != lens.shape[0] + 1:
        raise ValueError(f"cu_seqlens_q: expected shape {(lens.shape[0] + 1,)}, got {tuple(cu.shape)}")
    inputs = [(qn, "query_nope"), (qr, "query_rope"), (table, "block_table"), (cu, "cu_seqlens_q"), (lens, "seq_lens")] + list(zip(cache, names))
    mask = lse = None
    if tree_mask is not None:
        if window is not None:
            raise ValueError("tree_mask and window exclude one another")
        mask = _mask(tree_mask, qn.shape[0])
        inputs.append((mask, "tree_mask"))
    check_writable(out, "attention_out")
    if softmax_lse is not None:
        lse = as_torch(softmax_lse, "softmax_lse")
        if lse.dtype != torch.float32:
            raise TypeError(f"softmax_lse: expected torch.float32, got {lse.dtype}")
        if tuple(lse.shape) != tuple(qn.shape[:2]):
            raise ValueError(f"softmax_lse: expected shape {tuple(qn.shape[:2])}, got {tuple(lse.shape)}")
        refuse_overlap(lse, out, "softmax_lse and attention_out")
        for t, n in inputs:
            refuse_overlap(lse, t, f"softmax_lse and {n}")
    for t, n in inputs:
        refuse_overlap(out, t, f"attention_out and {n}")
    if not math.isfinite(float(softmax_scale)):
        raise ValueError("softmax_scale is not finite")
    _on_gpu(op, [t for t, _ in inputs] + [out] + ([lse] if lse is not None else []))
    if not C.latent_attention_call(qn, qr, *(cache + [None] * (3 - len(cache))), table, cu, lens, out, float(softmax_scale), int(block_size), window or 0, sinks,
                                   mask, lse):
        raise RuntimeError(f"{op}: these arguments are not supported")
    return None


def latent_attention(query_nope, query_rope, kv_cache, kr_cache, k_scale_cache, block_table, cu_seqlens_q, seq_lens, attention_out, softmax_scale, block_size,
                     window=None, sinks=0, tree_mask=None, softmax_lse=None):
    """softmax(softmax_scale * (query_nope . latent + query_rope . rope)) . latent over the three-array cache, sequence by sequence.

    query_nope (total_q, heads, 512), query_rope (total_q, heads, 64) bf16, beginning at multiples of 16 bytes, their strides multiples of 8
    elements; kv_cache int8 with rows of 512, kr_cache bf16 of 64, k_scale_cache fp32 of 4; block_table (b, max_blocknum_perbatch), cu_seqlens_q
    (b + 1,), ascending, seq_lens (b,) int32: sequence i's query tokens ``cu_seqlens_q[i] ..`` are the last of its ``seq_lens[i]`` keys;
    attention_out (total_q, heads, 512) bf16, softmax_lse (total_q, heads) fp32 or None: written in place, the latter with the natural logarithm
    of the sum of the exponentials of a row's scores.

    A token sees the keys up to its own; with ``window`` of these the last ``window``, its own among them, and the first ``sinks`` of the sequence;
    with ``tree_mask`` (total_q, words) int64 the keys before the sequence's query tokens and those of query tokens j whose bit j % 64 of word
    j / 64 is set (of fewer keys than query tokens the first tokens have none).  Rows that see no key are zeros (softmax_lse -inf); rows of no
    sequence stay as they were.  What a row does not see may hold anything, infinities and what is no number among it, and has no part in its
    results; the same goes for what lies behind a sequence's last key in its page.  Positions without a page read as zeros, as in
    ``latent_cache_read``.
    """
    return _attend("latent_attention", query_nope, query_rope, (kv_cache, kr_cache, k_scale_cache), ("kv_cache", "kr_cache", "k_scale_cache"), block_table,
                   cu_seqlens_q, seq_lens, attention_out, softmax_scale, block_size, window, sinks, tree_mask, softmax_lse)


def latent_attention_packed(query_nope, query_rope, nope_cache, block_table, cu_seqlens_q, seq_lens, attention_out, softmax_scale, block_size, window=None,
                            sinks=0, tree_mask=None, softmax_lse=None):
    """The same over the packed cache: nope_cache int8 with rows of 656 bytes."""
    return _attend("latent_attention_packed", query_nope, query_rope, (nope_cache,), ("nope_cache",), block_table, cu_seqlens_q, seq_lens, attention_out,
                   softmax_scale, block_size, window, sinks, tree_mask, softmax_lse)
