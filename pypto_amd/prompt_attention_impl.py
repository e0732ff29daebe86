"""Attention over whole prompts in the multi-head form: causal, grouped heads, packed sequences of different lengths.

A prompt no longer than the indexer's selection sees all of its keys: the sparse attention then computes what plain attention does, over
latents of 512 + 64 channels, 1088 products to a head and key.  In the multi-head form (keys of 128 channels and a rope part of 64 that all
heads share, values of 128) it is 320.  Keys and values come from the latents by a plain matrix product; the rope part stays a tensor of
its own here, so nothing is concatenated or repeated for the heads.

Sequences lie one behind the other; a sequence may have more keys than queries (the earlier chunks' context, read back from the cache;
single tokens).  With grouped heads ``heads / kv_heads`` query heads share a key head.

Calling convention as for the other operators; queries, keys, values and the output may be strided bare tensors (slices of a projection's
output): the last dimension alone has to be contiguous.
"""
from __future__ import annotations

import math

import torch

from . import _native
from .converter import as_rows, as_torch, check_writable, refuse_overlap
from .rotary_position_impl import _on_gpu
from .sparse_flash_attention_quant_impl import ROPE_DIM

HEAD_DIMS = (64, 128)


def prompt_attention(query, key, value, cu_seqlens_q, cu_seqlens_k, attention_out, softmax_scale, query_rope=None, key_rope=None,
                     softmax_lse=None, causal=True):
    """softmax(softmax_scale * (query . key + query_rope . key_rope)) . value, sequence by sequence.

    query (total_q, heads, d), key and value (total_k, kv_heads, d) bf16 or fp16, d 64 or 128, heads a multiple of kv_heads;
    query_rope (total_q, heads, 64) and key_rope (total_k, 64) or (total_k, kv_heads, 64), or None both (with d = 128);
    cu_seqlens_q, cu_seqlens_k (b + 1,) int32, ascending: where each sequence's queries and keys begin, and behind the last one;
    attention_out (total_q, heads, d), softmax_lse (total_q, heads) fp32 or None: written in place, the latter with the natural
    logarithm of the sum of the exponentials of a row's scores.  key, value and key_rope begin at multiples of 16 bytes and their strides are
    multiples of 8 elements.

    causal: the last query of a sequence sees all of its keys, each one before it one key less; otherwise every query sees all keys of
    its sequence.  Rows that see no key are zeros (softmax_lse -inf); rows of no sequence stay as they were.  What lies behind a
    sequence's last key is never looked at; the values of keys of the sequence itself have to be finite, seen or not.
    """
    C = _native.load()
    if C.prompt_attention_call(query, key, value, cu_seqlens_q, cu_seqlens_k, attention_out, softmax_scale, query_rope, key_rope, softmax_lse, causal):
        return None
    q, k, v, out = (as_rows(t, n) for t, n in ((query, "query"), (key, "key"), (value, "value"), (attention_out, "attention_out")))
    cu_q, cu_k = as_torch(cu_seqlens_q, "cu_seqlens_q"), as_torch(cu_seqlens_k, "cu_seqlens_k")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"query: expected torch.bfloat16 or torch.float16, got {q.dtype}")
    for t, n in ((q, "query"), (k, "key"), (v, "value"), (out, "attention_out")):
        if t.dtype != q.dtype:
            raise TypeError(f"{n}: expected {q.dtype}, got {t.dtype}")
        if t.dim() != 3:
            raise ValueError(f"{n}: expected 3 dimensions, got {t.dim()}")
    for t, n in ((cu_q, "cu_seqlens_q"), (cu_k, "cu_seqlens_k")):
        if t.dtype != torch.int32:
            raise TypeError(f"{n}: expected torch.int32, got {t.dtype}")
        if t.dim() != 1 or t.shape[0] < 2 or t.shape != cu_q.shape:
            raise ValueError("cu_seqlens_q, cu_seqlens_k: expected shape (b + 1,) for both, b >= 1")
    total_q, heads, d = q.shape
    total_k, kv_heads = k.shape[:2]
    if d not in HEAD_DIMS:
        raise ValueError(f"query: heads of {d} channels are not supported, only {HEAD_DIMS}")
    if k.shape != v.shape or k.shape[2] != d:
        raise ValueError(f"key, value: expected shape (total_k, kv_heads, {d}) for both, got {tuple(k.shape)} and {tuple(v.shape)}")
    if out.shape != q.shape:
        raise ValueError(f"attention_out: expected shape {tuple(q.shape)}, got {tuple(out.shape)}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"heads must be a multiple of kv_heads, got {heads} and {kv_heads}")
    if (query_rope is None) != (key_rope is None):
        raise ValueError("query_rope and key_rope come together")
    inputs = [(q, "query"), (k, "key"), (v, "value"), (cu_q, "cu_seqlens_q"), (cu_k, "cu_seqlens_k")]
    qr = kr = lse = None
    if query_rope is not None:
        qr, kr = as_rows(query_rope, "query_rope"), as_rows(key_rope, "key_rope")
        for t, n in ((qr, "query_rope"), (kr, "key_rope")):
            if t.dtype != q.dtype:
                raise TypeError(f"{n}: expected {q.dtype}, got {t.dtype}")
        if d != 128:
            raise ValueError("rope parts go with heads of 128 channels")
        if tuple(qr.shape) != (total_q, heads, ROPE_DIM):
            raise ValueError(f"query_rope: expected shape {(total_q, heads, ROPE_DIM)}, got {tuple(qr.shape)}")
        if tuple(kr.shape) not in ((total_k, ROPE_DIM), (total_k, 1, ROPE_DIM), (total_k, kv_heads, ROPE_DIM)):
            raise ValueError(f"key_rope: expected shape {(total_k, ROPE_DIM)} or {(total_k, kv_heads, ROPE_DIM)}, got {tuple(kr.shape)}")
        inputs += [(qr, "query_rope"), (kr, "key_rope")]
    if softmax_lse is not None:
        lse = as_torch(softmax_lse, "softmax_lse")
        if lse.dtype != torch.float32:
            raise TypeError(f"softmax_lse: expected torch.float32, got {lse.dtype}")
        if tuple(lse.shape) != (total_q, heads):
            raise ValueError(f"softmax_lse: expected shape {(total_q, heads)}, got {tuple(lse.shape)}")
        refuse_overlap(lse, out, "softmax_lse and attention_out")
        for t, n in inputs:
            refuse_overlap(lse, t, f"softmax_lse and {n}")
    check_writable(out, "attention_out")
    for t, n in inputs:
        refuse_overlap(out, t, f"attention_out and {n}")
    if not math.isfinite(float(softmax_scale)):
        raise ValueError("softmax_scale is not finite")
    _on_gpu("prompt_attention", [t for t, _ in inputs] + [out] + ([lse] if lse is not None else []))
    if not C.prompt_attention_call(q, k, v, cu_q, cu_k, out, float(softmax_scale), qr, kr, lse, bool(causal)):
        raise RuntimeError("prompt_attention: these arguments are not supported")
    return None
