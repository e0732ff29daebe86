"""A serving step's bookkeeping on the GPU: pages of the cache, and of each new token its position and its cache row.

The operators over the paged cache take block tables, lengths, beginnings of sequences, positions and cache rows.  All of them follow from two
lengths per sequence and from which pages it has; made here, they need no copy to the host and back between two steps, and a captured step
may be replayed with other lengths.  A step's way:

    cache_pages(held, wanted, block_table, free_pages, free_count, free_count, block_size)      # room for the new tokens
    cache_slots(query_lens, seq_lens, block_table, cu_q, cu_k, positions, cache_index, block_size)
    ... rotary tables of `positions`, prologs or cache writes to `cache_index`, attention over `cu_q`, `seq_lens`, `block_table` ...

and after drafted tokens were rejected ``cache_pages`` with the shorter lengths gives their pages back.

Calling convention as for the other operators: outputs are pre-allocated and written in place.
"""
from __future__ import annotations

import torch

from . import _native
from .converter import as_torch, refuse_overlap
from .rotary_position_impl import _on_gpu

MAX_MASK_WORDS = 16


def _typed(x, name, dtype, dim=None):
    t = as_torch(x, name)
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if dim is not None and t.dim() != dim:
        raise ValueError(f"{name}: expected {dim} dimension{'s' if dim > 1 else ''}, got {t.dim()}")
    return t


def _lengths(lens, name, table, b=None):
    t = _typed(lens, name, torch.int32, 1)
    if t.shape[0] < 1 or (b is not None and t.shape[0] != b):
        raise ValueError(f"{name}: expected shape ({'b' if b is None else b},), got {tuple(t.shape)}")
    if table.shape[0] != t.shape[0] or table.shape[1] < 1:
        raise ValueError(f"block_table: expected shape ({t.shape[0]}, max_blocknum_perbatch), got {tuple(table.shape)}")
    return t


def cache_pages(lens_before, lens_after, block_table, free_pages, free_count, free_left, block_size):
    """Pages for sequences that grow, back from sequences that shrink, in one launch.

    lens_before, lens_after (b,) int32: tokens that sequence i's pages hold, and shall hold; block_table (b, max_blocknum_perbatch) int32, written in
    place; free_pages (room,) int32: a stack, its first ``free_count`` (1,) int32 entries are free pages; free_left (1,) int32 receives how many
    there are afterwards, and may be ``free_count`` itself.

    First the pages behind ``lens_after`` go onto the stack, sequence by sequence and block by block (entries below zero are no pages; what the
    stack has no room for is dropped); their entries in the table stay as they were, as nothing reads behind a sequence's length.  Then
    sequences that grow take pages from its top, in the same order.  Where none are left the entries become -1: ``cache_slots`` gives their tokens
    no cache row, and cache writes skip those.  What a table has no column for is not taken.
    """
    C = _native.load()
    if C.cache_pages_call(lens_before, lens_after, block_table, free_pages, free_count, free_left, block_size):
        return None
    table = _typed(block_table, "block_table", torch.int32, 2)
    before = _lengths(lens_before, "lens_before", table)
    after = _lengths(lens_after, "lens_after", table, before.shape[0])
    pages = _typed(free_pages, "free_pages", torch.int32, 1)
    count, left = (_typed(t, n, torch.int32) for t, n in ((free_count, "free_count"), (free_left, "free_left")))
    for t, n in ((count, "free_count"), (left, "free_left")):
        if t.numel() != 1:
            raise ValueError(f"{n}: expected one element, got {tuple(t.shape)}")
    inputs = [(before, "lens_before"), (after, "lens_after")]
    for t, n in inputs + [(pages, "free_pages"), (count, "free_count"), (left, "free_left")]:
        refuse_overlap(table, t, f"block_table and {n}")
    for t, n in inputs + [(count, "free_count"), (left, "free_left")]:
        refuse_overlap(pages, t, f"free_pages and {n}")
    for t, n in inputs:
        refuse_overlap(left, t, f"free_left and {n}")
    _on_gpu("cache_pages", [before, after, table, pages, count, left])
    if not C.cache_pages_call(before, after, table, pages, count, left, int(block_size)):
        raise RuntimeError("cache_pages: these arguments are not supported")
    return None


def cache_slots(query_lens, seq_lens, block_table, cu_seqlens_q, cu_seqlens_k, positions, cache_index, block_size, parents=None, tree_mask=None):
    """Beginnings, positions and cache rows of a step's tokens, from lengths, in one launch.

    query_lens, seq_lens (b,) int32: sequence i's new tokens are the last ``query_lens[i]`` of its ``seq_lens[i]``; block_table (b,
    max_blocknum_perbatch) int32.  Written in place: cu_seqlens_q (b + 1,) int32, cu_seqlens_k (b + 1,) int32 or None, the sums of either
    length; positions, cache_index (t,) int64, token by token: its position and its physical row in the cache, -1 where the table holds no
    page for it.  Tokens of no sequence (t may exceed the sum of ``query_lens``) get position 0 and cache row -1, which writes skip.

    parents (t,) int32 with tree_mask (t, words) int64, 1 to 16 words: a sequence's new tokens are nodes of a tree of drafted tokens; a node's
    parent is given by its number within the sequence, lower than its own, anything else meaning none (a token that goes on from the cached ones).
    ``positions`` then counts depth, ``cache_index`` still numbers, and bit j % 64 of word j / 64 of ``tree_mask`` says whether the node is node j
    or descends from it, for the first 64 * words nodes: what ``latent_attention`` takes.
    """
    C = _native.load()
    if C.cache_slots_call(query_lens, seq_lens, block_table, cu_seqlens_q, cu_seqlens_k, positions, cache_index, block_size, parents, tree_mask):
        return None
    table = _typed(block_table, "block_table", torch.int32, 2)
    ql = _lengths(query_lens, "query_lens", table)
    sl = _lengths(seq_lens, "seq_lens", table, ql.shape[0])
    outs = [(_typed(cu_seqlens_q, "cu_seqlens_q", torch.int32, 1), "cu_seqlens_q"), (_typed(positions, "positions", torch.int64, 1), "positions"),
            (_typed(cache_index, "cache_index", torch.int64, 1), "cache_index")]
    if cu_seqlens_k is not None:
        outs.append((_typed(cu_seqlens_k, "cu_seqlens_k", torch.int32, 1), "cu_seqlens_k"))
    for t, n in outs:
        if n.startswith("cu_") and t.shape[0] != ql.shape[0] + 1:
            raise ValueError(f"{n}: expected shape {(ql.shape[0] + 1,)}, got {tuple(t.shape)}")
    tokens = outs[1][0].shape[0]
    if outs[2][0].shape[0] != tokens:
        raise ValueError(f"cache_index: expected shape {(tokens,)}, got {tuple(outs[2][0].shape)}")
    if (parents is None) != (tree_mask is None):
        raise ValueError("parents and tree_mask come together")
    inputs, up = [(ql, "query_lens"), (sl, "seq_lens"), (table, "block_table")], None
    if parents is not None:
        up = _typed(parents, "parents", torch.int32, 1)
        if up.shape[0] != tokens:
            raise ValueError(f"parents: expected shape {(tokens,)}, got {tuple(up.shape)}")
        inputs.append((up, "parents"))
        outs.append((_mask(tree_mask, tokens), "tree_mask"))
    for i, (t, n) in enumerate(outs):
        for x, m in inputs + outs[:i]:
            refuse_overlap(t, x, f"{n} and {m}")
    _on_gpu("cache_slots", [t for t, _ in inputs + outs])
    by = {n: t for t, n in outs}
    if not C.cache_slots_call(ql, sl, table, by["cu_seqlens_q"], by.get("cu_seqlens_k"), by["positions"], by["cache_index"], int(block_size), up,
                              by.get("tree_mask")):
        raise RuntimeError("cache_slots: these arguments are not supported")
    return None


def _mask(tree_mask, tokens):
    t = _typed(tree_mask, "tree_mask", torch.int64, 2)
    if t.shape[0] != tokens or not 1 <= t.shape[1] <= MAX_MASK_WORDS:
        raise ValueError(f"tree_mask: expected shape ({tokens}, 1 to {MAX_MASK_WORDS}), got {tuple(t.shape)}")
    return t
