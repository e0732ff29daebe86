"""Rotary positions: the tables that the prologs take, and the rotation of queries and keys that come from elsewhere.

The prologs (``mla_prolog_quant_d``, ``lightning_indexer_prolog_quant``) take ``cos`` and ``sin`` rows and rotate by themselves;
``rotary_tables`` makes those rows from positions.  A prompt in the multi-head form has its queries and keys from plain
projections: ``rotary_embedding`` rotates them, or a part of every head, in the layouts the path knows:

* ``"half"``           channel i turns with channel i + pairs (the indexer's);
* ``"interleaved"``    channel 2i turns with channel 2i + 1;
* ``"deinterleaved"``  channel 2i turns with channel 2i + 1, and the results go to i and i + pairs (the MLA prolog's).

``rotary_frequencies`` gives the radians per position of every pair, stretched for contexts longer than the trained one if asked
for.  It is made once, on the host; angles are ``position * frequency`` in 64 bits, so far positions keep their bits (angles up to 2^63 are
reduced exactly enough for fp32).

Calling convention as for the other operators: ``from_torch`` wrappers or bare torch tensors, outputs pre-allocated and written in
place, ``None`` returned, asynchronous on the current stream.  Bare tensors may be strided (a slice of a projection's output): the
last dimension alone has to be contiguous.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _native
from .converter import as_rows, as_torch, check_writable, refuse_overlap, same_rows

LAYOUTS = {"half": 0, "interleaved": 1, "deinterleaved": 2}
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
MAX_PAIRS = 128


@dataclass
class RotaryScaling:
    """How frequencies are stretched for contexts ``factor`` times as long as ``original_positions``: pairs that turn more than
    ``beta_fast`` times over the original positions keep their speed, pairs that turn less than ``beta_slow`` times are slowed down
    by ``factor``, those between by a part of it that grows linearly with the pair's number."""
    factor: float = 1.0
    original_positions: int = 4096
    beta_fast: float = 32.0
    beta_slow: float = 1.0


def rotary_frequencies(dim: int, theta: float = 10000.0, scaling: Optional[RotaryScaling] = None, device=None) -> torch.Tensor:
    """Radians per position of the ``dim / 2`` pairs, fp64 ``[dim / 2]``: ``theta ** (-2 i / dim)``, stretched by ``scaling``."""
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary_frequencies: dim must be even and positive, got {dim}")
    if not theta > 1.0:
        raise ValueError(f"rotary_frequencies: theta must exceed 1, got {theta}")
    i = torch.arange(dim // 2, dtype=torch.float64)
    plain = float(theta) ** (-2.0 * i / dim)
    if scaling is not None and scaling.factor != 1.0:
        if scaling.factor <= 0 or scaling.original_positions < 1 or scaling.beta_fast <= 0 or scaling.beta_slow <= 0:
            raise ValueError("rotary_frequencies: factor, original_positions and betas must be positive")

        def pair_of(turns):            # the (fractional) pair that turns so often over the original positions
            return dim * math.log(scaling.original_positions / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))

        lo = max(math.floor(pair_of(scaling.beta_fast)), 0)
        hi = min(math.ceil(pair_of(scaling.beta_slow)), dim - 1)
        slow = ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        plain = plain * (1.0 - slow) + plain / scaling.factor * slow
    return plain.to(device) if device is not None else plain


def rotary_magnitude(factor: float, mscale: float = 1.0) -> float:
    """What stretched models multiply their attention scores' magnitude by: ``0.1 mscale ln(factor) + 1``, 1 up to ``factor`` 1.
    Given to the operators below as ``factor`` it scales cos and sin; its square may go into ``softmax_scale`` instead."""
    return 0.1 * mscale * math.log(factor) + 1.0 if factor > 1.0 else 1.0


def _positions(positions, frequencies, op, multiple):
    pos, freq = as_torch(positions, "positions"), as_torch(frequencies, "frequencies")
    if pos.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"positions: expected torch.int64 or torch.int32, got {pos.dtype}")
    if freq.dtype != torch.float64:
        raise TypeError(f"frequencies: expected torch.float64, got {freq.dtype}")
    if pos.dim() != 1 or freq.dim() != 1:
        raise ValueError("positions and frequencies must be 1-dimensional")
    if freq.shape[0] % multiple or not multiple <= freq.shape[0] <= MAX_PAIRS:
        raise ValueError(f"{op}: the number of pairs must be a multiple of {multiple}, up to {MAX_PAIRS}, got {freq.shape[0]}")
    return pos, freq


def _on_gpu(op, tensors):
    dev = tensors[0].device
    if dev.type != "cuda":
        raise RuntimeError(f"{op}: tensors must live on the GPU (device type 'cuda' on ROCm)")
    if any(t.device != dev for t in tensors):
        raise RuntimeError("not all tensors are on the same device")


def rotary_tables(positions, frequencies, cos_out, sin_out, factor=1.0):
    """``factor * cos`` and ``factor * sin`` of ``positions[t] * frequencies[i]``, in columns i and i + pairs.

    positions (t,) int64 or int32; frequencies (pairs,) fp64, pairs a multiple of 4 up to 128; cos_out, sin_out (t, 2*pairs) bf16, fp16 or
    fp32, written in place: with 32 pairs the ``cos`` / ``sin`` of the prologs.
    """
    C = _native.load()
    if C.rotary_tables_call(positions, frequencies, cos_out, sin_out, factor):
        return None
    pos, freq = _positions(positions, frequencies, "rotary_tables", 4)
    cos, sin = as_torch(cos_out, "cos_out"), as_torch(sin_out, "sin_out")
    for t, name in ((cos, "cos_out"), (sin, "sin_out")):
        if t.dtype not in DTYPES or t.dtype != cos.dtype:
            raise TypeError(f"{name}: expected bf16, fp16 or fp32, both tables alike, got {t.dtype}")
        if tuple(t.shape) != (pos.shape[0], 2 * freq.shape[0]):
            raise ValueError(f"{name}: expected shape {(pos.shape[0], 2 * freq.shape[0])}, got {tuple(t.shape)}")
    refuse_overlap(cos, sin, "cos_out and sin_out")
    for t, name in ((cos, "cos_out"), (sin, "sin_out")):
        refuse_overlap(t, pos, f"{name} and positions")
        refuse_overlap(t, freq, f"{name} and frequencies")
    _on_gpu("rotary_tables", (pos, freq, cos, sin))
    if not C.rotary_tables_call(pos, freq, cos, sin, float(factor)):
        raise RuntimeError("rotary_tables: these arguments are not supported")
    return None


def rotary_embedding(query, key, positions, frequencies, query_out, key_out, layout="half", query_offset=0, key_offset=0, factor=1.0):
    """Rotates ``2 * pairs`` channels of every head of queries and keys, one launch for both.

    query, query_out (t, heads, dim), key, key_out (t, heads, dim) or (t, dim), or None both; bf16, fp16 or fp32, all alike.
    positions (t,) int64 or int32; frequencies (pairs,) fp64, pairs a multiple of 8 up to 128.  Of a head the channels
    ``offset .. offset + 2 * pairs - 1`` turn; the others are copied.  An output may be its input (the other channels then stay as
    they are); otherwise outputs overlap nothing.
    """
    C = _native.load()
    code = LAYOUTS.get(layout) if isinstance(layout, str) else None
    if code is not None and C.rotary_embedding_call(query, key, positions, frequencies, query_out, key_out, code, query_offset, key_offset, factor):
        return None
    if code is None:
        raise ValueError(f"rotary_embedding: layout must be one of {sorted(LAYOUTS)}, got {layout!r}")
    pos, freq = _positions(positions, frequencies, "rotary_embedding", 8)
    if (key is None) != (key_out is None):
        raise ValueError("rotary_embedding: key and key_out come together")
    sides = [("query", as_rows(query, "query"), as_rows(query_out, "query_out"), query_offset)]
    if key is not None:
        sides.append(("key", as_rows(key, "key"), as_rows(key_out, "key_out"), key_offset))
    for name, x, out, offset in sides:
        if x.dtype not in DTYPES or x.dtype != sides[0][1].dtype or out.dtype != x.dtype:
            raise TypeError(f"{name}, {name}_out: expected bf16, fp16 or fp32, all tensors alike, got {x.dtype} and {out.dtype}")
        if x.dim() not in (2, 3) or x.shape[0] != pos.shape[0] or x.shape != out.shape:
            raise ValueError(f"{name}, {name}_out: expected shape ({pos.shape[0]}, heads, dim) for both, got {tuple(x.shape)} and {tuple(out.shape)}")
        if int(offset) < 0 or int(offset) + 2 * freq.shape[0] > x.shape[-1]:
            raise ValueError(f"{name}: {2 * freq.shape[0]} channels from {offset} on do not fit {x.shape[-1]}")
        check_writable(out, f"{name}_out")
        if not same_rows(x, out):
            refuse_overlap(out, x, f"{name} and {name}_out")
        refuse_overlap(out, pos, f"{name}_out and positions")
        refuse_overlap(out, freq, f"{name}_out and frequencies")
    if len(sides) == 2:
        (_, q, qo, _), (_, k, ko, _) = sides
        refuse_overlap(qo, k, "query_out and key")
        refuse_overlap(ko, q, "key_out and query")
        refuse_overlap(qo, ko, "query_out and key_out")
    _on_gpu("rotary_embedding", [pos, freq] + [t for _, x, out, _ in sides for t in (x, out)])
    k = sides[1] if len(sides) == 2 else (None, None, None, 0)
    if not C.rotary_embedding_call(sides[0][1], k[1], pos, freq, sides[0][2], k[2], code, int(query_offset), int(key_offset), float(factor)):
        raise RuntimeError("rotary_embedding: these arguments are not supported")
    return None
