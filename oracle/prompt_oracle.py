"""Plain 64-bit statements of the operators around a prompt: rotary positions, the latent cache's quantisation, attention.

Test infrastructure.  ``attention`` also gives what its results may be off by in a kernel that multiplies 16-bit operands and sums in
fp32 (:func:`attention_bounds`).
"""
from __future__ import annotations

import math

import numpy as np
import torch

F64 = torch.float64


def turn(x, positions, frequencies, layout, offset=0, factor=1.0):
    """x [t, heads, dim] with ``2 * pairs`` channels from ``offset`` on rotated, in 64 bits."""
    pairs = frequencies.numel()
    angle = positions.to(F64)[:, None] * frequencies.to(F64)
    c, s = (factor * angle.cos())[:, None], (factor * angle.sin())[:, None]
    out = x.to(F64).clone()
    part = out[..., offset:offset + 2 * pairs].clone()
    if layout == "half":
        a, b = part[..., :pairs], part[..., pairs:]
    else:
        a, b = part[..., 0::2], part[..., 1::2]
    ra, rb = a * c - b * s, b * c + a * s
    if layout == "interleaved":
        part[..., 0::2], part[..., 1::2] = ra, rb
    else:
        part = torch.cat([ra, rb], dim=-1)
    out[..., offset:offset + 2 * pairs] = part
    return out


def quantise(latent, prolog_steps=False):
    """latent [t, 512] -> codes int8 [t, 512], scales fp32 [t, 4], values fp32 [t, 512] (to be rounded to bf16), in numpy's fp32,
    groups of no number and of next to nothing among them.  prolog_steps: 127 / max rounded once."""
    y = latent.float().cpu().numpy().reshape(-1, 4, 128)
    most = np.abs(y).max(axis=2, keepdims=True)                      # (carries what is no number)
    with np.errstate(all="ignore"):
        steps = ((np.float32(127.0) / most) if prolog_steps else np.float32(127.0) * (np.float32(1) / most).astype(np.float32)).astype(np.float32)
        number, zero = np.isfinite(most), ~np.isfinite(steps)
        codes = np.where(number & ~zero, np.rint((y * steps).astype(np.float32)), 0).astype(np.float32)
        scales = np.where(number, np.where(zero, np.float32(0), (np.float32(1) / steps).astype(np.float32)), np.float32("nan"))
        values = (codes * scales).astype(np.float32)
    t = y.shape[0]
    return (torch.from_numpy(codes.astype(np.int8).reshape(t, 512)), torch.from_numpy(scales.astype(np.float32).reshape(t, 4)),
            torch.from_numpy(values.reshape(t, 512)))


def attention(query, key, value, lens_q, lens_k, scale, query_rope=None, key_rope=None, causal=True):
    """Returns out, lse and, of every row, the mean magnitude of its values (out with |value|), the largest sum of magnitudes of a score's
    products, times |scale|, and how many keys it sees -- all in 64 bits.  Rows of no sequence are NaN."""
    tq, heads, d = query.shape
    kv = key.shape[1]
    g = heads // kv
    new = lambda *s: torch.full(s, math.nan, dtype=F64, device=query.device)  # noqa: E731
    out, mean, lse, reach, seen = new(tq, heads, d), new(tq, heads, d), new(tq, heads), new(tq, heads), new(tq, heads)
    q0 = k0 = 0
    for lq, lk in zip(lens_q, lens_k):
        for h in range(heads):
            q, k, v = query[q0:q0 + lq, h].to(F64), key[k0:k0 + lk, h // g].to(F64), value[k0:k0 + lk, h // g].to(F64)
            if query_rope is not None:
                kr = key_rope if key_rope.dim() == 2 else key_rope[:, h // g if key_rope.shape[1] > 1 else 0]
                q = torch.cat([q, query_rope[q0:q0 + lq, h].to(F64)], dim=1)
                k = torch.cat([k, kr[k0:k0 + lk].to(F64)], dim=1)
            s, size = scale * (q @ k.T), abs(scale) * (q.abs() @ k.abs().T)
            hidden = torch.zeros(lq, lk, dtype=torch.bool, device=query.device)
            if causal:
                i, j = torch.arange(lq, device=query.device)[:, None], torch.arange(lk, device=query.device)
                hidden = j > i + lk - lq
            n = (~hidden).sum(dim=1)
            s = s.masked_fill(hidden, -math.inf)
            top = s.amax(dim=1, keepdim=True) if lk else s.new_full((lq, 1), -math.inf)
            p = torch.exp(s - torch.where(n[:, None] > 0, top, 0.0))
            total = p.sum(dim=1, keepdim=True)
            p = torch.where(n[:, None] > 0, p / total, 0.0)
            out[q0:q0 + lq, h], mean[q0:q0 + lq, h] = p @ v, p @ v.abs()
            lse[q0:q0 + lq, h] = torch.where(n > 0, (top + total.log())[:, 0], -math.inf)
            reach[q0:q0 + lq, h] = size.masked_fill(hidden, 0.0).amax(dim=1) if lk else 0.0
            seen[q0:q0 + lq, h] = n.to(F64)
        q0, k0 = q0 + lq, k0 + lk
    return out, lse, mean, reach, seen


def attention_bounds(dtype, channels, out, lse, mean, reach, seen):
    """What a kernel's out and lse may be off by.  With u half a step of the type and e = 2^-24 half a step of fp32:

    - a score is a sum of `channels` exact products in fp32: off by channels * e * reach; scaling and subtracting the maximum
      rounds values of at most 2 * reach a few times: 4 e * 2 reach.  A probability is then off by that much (relatively), by 2^-22
      from exp2, by u from its rounding, or, in fp16, by 2^-25 of the largest (below its normal numbers);
    - sums over n keys in fp32: n e (relatively to the sum of magnitudes), for the values and for the denominator;
    - the result's own rounding: u.
    """
    u = torch.finfo(dtype).eps / 2
    e = 2.0 ** -24
    p = (channels + 8) * e * reach + 2.0 ** -22
    both = (u + 2 * p + 2 * (seen + 8) * e)[..., None]
    small = 4 * seen[..., None] * 2.0 ** -25 * max(1.0, float(mean.max())) if dtype == torch.float16 and mean.numel() else 0.0
    return u * out.abs() + both * mean + small + 2.0 ** -126, p + (seen + 16) * e + 4 * e * lse.abs().nan_to_num(0, 0, 0)
