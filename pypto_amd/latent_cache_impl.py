"""Writing latents into the quantised cache of the sparse attention, and reading them back.

The cache is what the attention operators take: three arrays (``sparse_flash_attention_quant_d``: 512 int8, 64 bf16 and 4 fp32 a row) or
one packed array of 656-byte rows (``sparse_attention_antiquant_d``).  The MLA prolog writes the three arrays as the last step of its
projections; these operators write either form from latents that are already there (a prompt's, from plain projections), in
fp32: of every 128 channels ``steps = 127 * (1 / max|v|)``, ``code = rint(v * steps)``, ``scale = 1 / steps``, the value stored being
``bf16(code * scale)``.  With ``prolog_steps`` ``steps = 127 / max|v|`` in one rounding, as the prolog divides: rows are then bit for bit
those that it writes for the same latents, which a cache that both write, or whose pages are compared, wants.  (Between the two one scale
in four or five differs in its last bits, and of bf16 latents 4 codes in 10000, in one row of six, by one step.)

Reading gathers positions of sequences through their block tables, de-quantised as the attention does it and packed one sequence behind
the other: the context that a prompt's next chunk makes its keys and values from.

Calling convention as for the other operators; latents, rope keys and the bf16 outputs may be strided bare tensors (slices of a projection's
output): the last dimension alone has to be contiguous.
"""
from __future__ import annotations

import torch

from . import _native
from .converter import as_rows, as_torch, check_writable, refuse_overlap, same_rows
from .rotary_position_impl import DTYPES, _on_gpu
from .sparse_attention_antiquant_impl import PACKED_ROW_BYTES
from .sparse_flash_attention_quant_impl import KV_LORA_RANK, ROPE_DIM

GROUPS = 4


def _cache_tensors(parts, names):
    out = [as_torch(p, n) for p, n in zip(parts, names)]
    widths = (PACKED_ROW_BYTES,) if len(out) == 1 else (KV_LORA_RANK, ROPE_DIM, GROUPS)
    dtypes = (torch.int8, torch.bfloat16, torch.float32)
    for t, n, dt in zip(out, names, dtypes):
        if t.dtype != dt:
            raise TypeError(f"{n}: expected {dt}, got {t.dtype}")
    if out[0].dim() < 2 or out[0].shape[-1] != widths[0]:
        raise ValueError(f"{names[0]}: expected [.., {widths[0]}], got {tuple(out[0].shape)}")
    rows = out[0].numel() // widths[0]
    for t, n, w in zip(out, names, widths):
        if t.numel() != rows * w:
            raise ValueError(f"{n}: expected {rows} rows of {w}, got {tuple(t.shape)}")
    return out


def _rows(t, name, width, dtypes, rows=None):
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: expected {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if t.dim() != 2 or t.shape[1] != width or (rows is not None and t.shape[0] != rows):
        raise ValueError(f"{name}: expected shape ({'rows' if rows is None else rows}, {width}), got {tuple(t.shape)}")
    return t


def _write(op, latent, key_rope, cache_index, parts, names, latent_out, prolog_steps):
    C = _native.load()
    pad = list(parts) + [None] * (3 - len(parts))
    if C.cache_write_call(latent, key_rope, cache_index, *pad, latent_out, prolog_steps):
        return None
    lat = _rows(as_rows(latent, "latent"), "latent", KV_LORA_RANK, DTYPES)
    rope = _rows(as_rows(key_rope, "key_rope"), "key_rope", ROPE_DIM, (lat.dtype,), lat.shape[0])
    idx = as_torch(cache_index, "cache_index")
    if idx.dtype != torch.int64:
        raise TypeError(f"cache_index: expected torch.int64, got {idx.dtype}")
    if idx.numel() != lat.shape[0]:
        raise ValueError(f"cache_index: expected {lat.shape[0]} elements, got {idx.numel()}")
    cache = _cache_tensors(parts, names)
    for c, n in zip(cache, names):
        refuse_overlap(c, lat, f"{n} and latent")
        refuse_overlap(c, rope, f"{n} and key_rope")
        refuse_overlap(c, idx, f"{n} and cache_index")
    for i, j in ((0, 1), (0, 2), (1, 2)) if len(cache) == 3 else ():
        refuse_overlap(cache[i], cache[j], f"{names[i]} and {names[j]}")
    tensors = [lat, rope, idx] + cache
    values = None
    if latent_out is not None:
        values = _rows(as_rows(latent_out, "latent_out"), "latent_out", KV_LORA_RANK, (torch.bfloat16,), lat.shape[0])
        check_writable(values, "latent_out")
        if lat.dtype != values.dtype or not same_rows(values, lat):
            refuse_overlap(values, lat, "latent_out and latent")
        refuse_overlap(values, rope, "latent_out and key_rope")
        refuse_overlap(values, idx, "latent_out and cache_index")
        for c, n in zip(cache, names):
            refuse_overlap(values, c, f"latent_out and {n}")
        tensors.append(values)
    _on_gpu(op, tensors)
    if not C.cache_write_call(lat, rope, idx, *(cache + [None] * (3 - len(cache))), values, bool(prolog_steps)):
        raise RuntimeError(f"{op}: these arguments are not supported")
    return None


def latent_cache_write(latent, key_rope, cache_index, kv_cache, kr_cache, k_scale_cache, latent_out=None, prolog_steps=False):
    """Quantises rows into the three-array cache.

    latent (t, 512), key_rope (t, 64) bf16, fp16 or fp32, both alike; cache_index (t,) int64, the physical row of each token (rows outside the
    cache are skipped; no row may be named twice); kv_cache int8 with rows of 512, kr_cache bf16 of 64, k_scale_cache fp32 of 4, in the
    attention's two or the MLA prolog's four dimensions, written in place.  latent_out (t, 512) bf16 or None receives what the written rows
    stand for (it may be ``latent`` itself).  prolog_steps: codes and scales are those that the MLA prolog writes.
    """
    return _write("latent_cache_write", latent, key_rope, cache_index, (kv_cache, kr_cache, k_scale_cache),
                  ("kv_cache", "kr_cache", "k_scale_cache"), latent_out, prolog_steps)


def latent_cache_write_packed(latent, key_rope, cache_index, nope_cache, latent_out=None, prolog_steps=False):
    """The same into the packed cache: nope_cache int8 with rows of 656 bytes, written in place."""
    return _write("latent_cache_write_packed", latent, key_rope, cache_index, (nope_cache,), ("nope_cache",), latent_out,
                  prolog_steps)


def _read(op, parts, names, block_table, cu_seqlens, latent_out, key_rope_out, block_size, first):
    C = _native.load()
    pad = list(parts) + [None] * (3 - len(parts))
    if C.cache_read_call(*pad, block_table, cu_seqlens, first, latent_out, key_rope_out, block_size):
        return None
    cache = _cache_tensors(parts, names)
    bt, cu = as_torch(block_table, "block_table"), as_torch(cu_seqlens, "cu_seqlens")
    ints = [(bt, "block_table"), (cu, "cu_seqlens")]
    start = None
    if first is not None:
        start = as_torch(first, "first")
        ints.append((start, "first"))
    for t, n in ints:
        if t.dtype != torch.int32:
            raise TypeError(f"{n}: expected torch.int32, got {t.dtype}")
    if bt.dim() != 2 or bt.shape[0] < 1:
        raise ValueError(f"block_table: expected shape (b, max_blocknum_perbatch), got {tuple(bt.shape)}")
    if tuple(cu.shape) != (bt.shape[0] + 1,):
        raise ValueError(f"cu_seqlens: expected shape {(bt.shape[0] + 1,)}, got {tuple(cu.shape)}")
    if start is not None and tuple(start.shape) != (bt.shape[0],):
        raise ValueError(f"first: expected shape {(bt.shape[0],)}, got {tuple(start.shape)}")
    latent = _rows(as_rows(latent_out, "latent_out"), "latent_out", KV_LORA_RANK, (torch.bfloat16,))
    rope = _rows(as_rows(key_rope_out, "key_rope_out"), "key_rope_out", ROPE_DIM, (torch.bfloat16,), latent.shape[0])
    for t, n in ((latent, "latent_out"), (rope, "key_rope_out")):
        check_writable(t, n)
        for c, m in zip(cache, names):
            refuse_overlap(t, c, f"{n} and {m}")
        for i, m in ints:
            refuse_overlap(t, i, f"{n} and {m}")
    refuse_overlap(latent, rope, "latent_out and key_rope_out")
    _on_gpu(op, cache + [t for t, _ in ints] + [latent, rope])
    if not C.cache_read_call(*(cache + [None] * (3 - len(cache))), bt, cu, start, latent, rope, int(block_size)):
        raise RuntimeError(f"{op}: these arguments are not supported")
    return None


def latent_cache_read(kv_cache, kr_cache, k_scale_cache, block_table, cu_seqlens, latent_out, key_rope_out, block_size, first=None):
    """Reads positions of sequences out of the three-array cache, de-quantised.

    block_table (b, max_blocknum_perbatch) int32; cu_seqlens (b + 1,) int32, ascending: rows ``cu_seqlens[i] .. cu_seqlens[i + 1] - 1`` of the
    outputs are positions ``first[i]`` (int32, None: 0) and following of sequence i.  latent_out (rows, 512), key_rope_out (rows, 64) bf16,
    written in place; rows of no sequence stay as they were, positions that the table holds no page for read as zeros.
    """
    return _read("latent_cache_read", (kv_cache, kr_cache, k_scale_cache), ("kv_cache", "kr_cache", "k_scale_cache"), block_table, cu_seqlens,
                 latent_out, key_rope_out, block_size, first)


def latent_cache_read_packed(nope_cache, block_table, cu_seqlens, latent_out, key_rope_out, block_size, first=None):
    """The same out of the packed cache."""
    return _read("latent_cache_read_packed", (nope_cache,), ("nope_cache",), block_table, cu_seqlens, latent_out, key_rope_out, block_size, first)
