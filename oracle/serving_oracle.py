"""Plain statements of a serving step's operators: pages and slots in Python's whole numbers, attention under any mask in 64 bits.

Test infrastructure.  Bounds of the attentions: :func:`oracle.prompt_oracle.attention_bounds`.
"""
from __future__ import annotations

import math

import torch

F64 = torch.float64


def blocks(n, block, columns):
    return min(-(-max(n, 0) // block), columns)


def pages(before, after, table, stack, count, block):
    """table (rows of lists) and stack (a list) are changed; returns how many free pages are left."""
    columns, room = len(table[0]), len(stack)
    top = min(max(count, 0), room)
    for row, x, y in zip(table, before, after):
        for j in range(blocks(y, block, columns), blocks(x, block, columns)):
            if row[j] >= 0 and top < room:
                stack[top] = row[j]
                top += 1
    for row, x, y in zip(table, before, after):
        for j in range(blocks(x, block, columns), blocks(y, block, columns)):
            top -= 1
            row[j] = stack[top] if top >= 0 else -1
    return max(top, 0)


def slots(query_lens, seq_lens, table, tokens, block, parents=None, words=0):
    """cu_q, cu_k, positions, cache rows and (with parents) masks, as lists."""
    cu_q, cu_k, positions, rows, masks = [0], [0], [], [], []
    for b, (n, total) in enumerate(zip(query_lens, seq_lens)):
        n, total = max(n, 0), max(total, 0)
        first, bits, depth = cu_q[-1], [], []
        for r in range(n):
            at = total - n + r
            page = table[b][at // block] if 0 <= at < block * len(table[b]) else -1
            rows.append(page * block + at % block if page >= 0 else -1)
            if parents is None:
                positions.append(at)
                continue
            up = parents[first + r] if first + r < len(parents) else -1
            up = up if 0 <= up < r else -1
            bits.append((1 << r) | (bits[up] if up >= 0 else 0))
            depth.append(depth[up] + 1 if up >= 0 else 0)
            positions.append(total - n + depth[r])
            masks.append([signed((bits[r] >> (64 * w)) & (2 ** 64 - 1)) for w in range(words)])
        cu_q.append(first + n)
        cu_k.append(cu_k[-1] + total)
    spare = tokens - cu_q[-1]
    positions, rows, masks = positions[:tokens] + [0] * spare, rows[:tokens] + [-1] * spare, masks[:tokens] + [[0] * words] * spare
    return cu_q, cu_k, positions, rows, masks


def signed(word):
    return word - 2 ** 64 if word >= 2 ** 63 else word


def seen_keys(n, keys, window=None, sinks=0, mask=None):
    """[n, keys] truth values: what the last n of `keys` positions see.  mask: [n, words] int64, bits of the n."""
    at, j = torch.arange(keys - n, keys)[:, None], torch.arange(keys)
    if mask is not None:
        node = j - (keys - n)                      # (of fewer keys than tokens, the first tokens have none)
        word = (node // 64).clamp(0, mask.shape[1] - 1)
        drafted = ((mask.cpu()[:, word] >> (node % 64)) & 1).bool() & (node < 64 * mask.shape[1])
        return torch.where(node < 0, True, drafted)
    seen = j <= at
    return seen & ((j > at - window) | (j < sinks)) if window is not None else seen


def latents(parts, table_row, keys, block, device=None):
    """Keys [keys, 576] and values [keys, 512] of a sequence, in 64 bits: bf16(code * scale), zeros where there is no page.  parts: the three arrays, or the
    packed one alone."""
    if len(parts) == 1:
        c = parts[0].reshape(-1, 656)
        parts = c[:, :512], c[:, 512:640].view(torch.bfloat16), c[:, 640:].view(torch.float32)
    nope, rope, scales = (p.reshape(-1, w) for p, w in zip(parts, (512, 64, 4)))
    at = torch.arange(keys, device=nope.device)
    page = table_row[at // block].long()
    row = page * block + at % block
    there = (page >= 0) & (row < nope.shape[0])
    row = torch.where(there, row, 0)
    v = (nope[row].float().view(-1, 4, 128) * scales[row][:, :, None]).reshape(-1, 512).to(torch.bfloat16).to(F64)
    v = torch.where(there[:, None], v, 0.0)
    return torch.cat([v, torch.where(there[:, None], rope[row].to(F64), 0.0)], dim=1), v


def attend(q, k, v, scale, seen):
    """q [n, heads, c], k [keys, c], v [keys, d], seen [n, keys]: out, lse, and what :func:`attention_bounds` takes: the mean magnitude of a row's values, the
    largest sum of magnitudes of a score's products (times |scale|), how many keys it sees.  What no row sees may hold anything."""
    q, k, v, seen = q.to(F64), k.to(F64), v.to(F64), seen.to(q.device)
    some = seen.any(dim=0)
    k, v = torch.where(some[:, None], k, 0.0), torch.where(some[:, None], v, 0.0)
    hidden, n = ~seen[:, None, :], seen.sum(dim=1)
    s = (scale * (q @ k.T)).masked_fill(hidden, -math.inf)
    reach = (abs(scale) * (q.abs() @ k.abs().T)).masked_fill(hidden, 0.0)
    empty = (n == 0)[:, None]
    top = torch.where(empty, 0.0, s.amax(dim=2)) if k.shape[0] else s.new_zeros(s.shape[:2])
    p = torch.exp(s - top[..., None])
    total = p.sum(dim=2)
    p = torch.where(empty[..., None], 0.0, p / total[..., None])
    lse = torch.where(empty, -math.inf, top + total.log())
    reach = reach.amax(dim=2) if k.shape[0] else torch.zeros_like(lse)
    return p @ v, lse, p @ v.abs(), reach, n[:, None].to(F64).expand_as(lse)
