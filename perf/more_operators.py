"""The measured operators: a serving step's pages and slots, and attention over parts of what the cache holds.

A step begins with bookkeeping: sequences that grew take pages of the latent cache, sequences that shrank or ended give theirs
back (`cache_pages`), and each new token gets its position and the cache row it is written to (`cache_slots`), for a tree of drafted tokens
its depth and which nodes it sees, too.  Then the new tokens attend over the cache in the absorbed form (`latent_attention`): a tree's nodes over
the context and their ancestors, or single tokens and short chunks over the last keys of a window and a few first ones.  Whole prompts
of such a model attend in the multi-head form (`prompt_window_attention`).  Sizes are those of the repository's tests and benchmark
(128 heads, latents of 512 + 64, pages of 128 positions) or generic ones (64 query heads over 8 key heads, trees of up to 64 nodes).

`run` computes a case in elementary torch operations, or, where `own` is set, through the package's operators.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
PAGE = 128
DN, DR, GROUP = 512, 64, 128           # latent and rope widths of a cache row, channels to a scale
PACKED = DN + 2 * DR + 16              # bytes of a packed row
BF, HALF, F32, F64, I32, I64 = torch.bfloat16, torch.float16, torch.float32, torch.float64, torch.int32, torch.int64
DTYPES = {"bf16": BF, "fp16": HALF}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # a step of 32 sequences that make room for drafted tokens, or give back what was not accepted: one or the other passes a page's end
        dict(name="pages_32", kind="pages", b=32, far=65536, new=40, fresh=0, done=0, block=128, tight=False),
        # a step of a busy server: of 1000 sequences every twentieth ends, every twentieth begins with a prompt, the others take a few
        # tokens or give back what was drafted and not accepted
        dict(name="pages_1000", kind="pages", b=1000, far=16000, new=12, fresh=5, done=5, block=64, tight=False),
        # slots of a decode step, one token to each of 512 sequences
        dict(name="slots_512", kind="slots", b=512, lo=1, hi=1, far=32768, block=128, nodes=0),
        # slots of nine prompts of all lengths, the largest call
        dict(name="slots_prompts", kind="slots", b=9, lo=3000, hi=30000, far=100, block=128, nodes=0),
        # slots, depths and ancestors of 48 drafted trees
        dict(name="slots_trees", kind="slots", b=48, lo=17, hi=63, far=20000, block=64, nodes=64),
        # one sequence's small tree behind 2900 keys, the heads divided over eight GPUs
        dict(name="tree_1", kind="cache", b=1, q_lo=8, q_hi=8, c_lo=2900, c_hi=2900, heads=16, packed=True, nodes=64, window=0, sinks=0, block=128, lse=False),
        # trees of 24 sequences, young and old, all 128 heads: the largest call over the cache
        dict(name="tree_24", kind="cache", b=24, q_lo=25, q_hi=63, c_lo=500, c_hi=9000, heads=128, packed=False, nodes=64, window=0, sinks=0, block=128, lse=False),
        # single tokens of 32 sequences over their last 2048 keys and the first four
        dict(name="window_32", kind="cache", b=32, q_lo=1, q_hi=1, c_lo=300, c_hi=12000, heads=128, packed=True, nodes=0, window=2048, sinks=4, block=128, lse=False),
        # one to four tokens of 90 sequences, a share of the heads, a narrow window, small pages
        dict(name="window_90", kind="cache", b=90, q_lo=1, q_hi=4, c_lo=5, c_hi=30000, heads=16, packed=False, nodes=0, window=1000, sinks=16, block=64, lse=True),
        # a long prompt in the multi-head form: 128 heads, 128 + 64 channels, the last 1024 keys and the first four
        dict(name="prompt_8192", kind="prompt", b=1, q_lo=8192, q_hi=8192, c_lo=0, c_hi=0, heads=128, kv_heads=128, d=128, rope=True, dtype="bf16",
             window=1024, sinks=4, lse=False),
        # nine prompts of different lengths, eight query heads to a key head, a window alone
        dict(name="prompt_packed_9", kind="prompt", b=9, q_lo=70, q_hi=6000, c_lo=0, c_hi=0, heads=64, kv_heads=8, d=128, rope=False, dtype="fp16",
             window=500, sinks=0, lse=True),
        # a chunk of 1024 tokens behind a context of some 15000, the heads divided over eight GPUs
        dict(name="prompt_chunk", kind="prompt", b=1, q_lo=1024, q_hi=1024, c_lo=15001, c_hi=15001, heads=16, kv_heads=16, d=128, rope=True, dtype="bf16",
             window=4096, sinks=64, lse=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _pages_case(rng):
    return dict(kind="pages", b=_log(rng, 1, 1500), far=_log(rng, 100, 32768), new=_log(rng, 1, 200), fresh=rng.choice((0, 3, 10, 100)),
                done=rng.choice((0, 3, 10)), block=rng.choice((128, 128, 64, 16)), tight=rng.random() < 0.2)


def _slots_case(rng):
    tree = rng.random() < 0.4
    b = _log(rng, 1, 300 if tree else 1000)
    lo, hi = sorted(_log(rng, 1, min(200 if tree else 30000, 150000 // b)) for _ in range(2))
    return dict(kind="slots", b=b, lo=lo, hi=hi, far=_log(rng, 10, 100000), block=rng.choice((128, 128, 64, 16)),
                nodes=(hi + 63) // 64 * 64 if tree else 0)


def _cache_case(rng):
    while True:
        tree = rng.random() < 0.5
        b = _log(rng, 1, 100)
        form = "tree" if tree else rng.choice(("tokens", "tokens", "chunk"))
        q = sorted(_log(rng, 1, {"tree": 200, "tokens": 4, "chunk": 600}[form]) for _ in range(2))
        c = sorted(_log(rng, 1, 30000) for _ in range(2))
        case = dict(kind="cache", b=b, q_lo=q[0], q_hi=q[1], c_lo=c[0], c_hi=c[1], heads=rng.choice((128, 128, 64, 40, 16, 5)), packed=rng.random() < 0.5,
                    nodes=(q[1] + 63) // 64 * 64 if tree else 0, window=0 if tree else _log(rng, 16, 6000), sinks=0 if tree else rng.choice((0, 1, 4, 16, 100)),
                    block=rng.choice((128, 128, 64, 16)), lse=rng.random() < 0.5)
        ql, kl = _lengths(case)
        w = work(case)
        # no dearer than the largest listed case, in the scores of the plain form as well
        if w["flops"] <= 1.2e12 and w["bytes"] <= 1.5e9 and sum(x * y for x, y in zip(ql, kl)) * case["heads"] <= 6e8 and sum(kl) <= 400000:
            return case


def _prompt_case(rng):
    while True:
        form = rng.choice(("prompt", "prompt", "chunk", "tokens"))
        d = rng.choice((128, 128, 128, 64))
        kv_heads = rng.choice((1, 2, 4, 8, 16, 32, 128))
        heads = kv_heads * rng.choice((1, 1, 2, 4, 7, 8, 16))
        b = _log(rng, 1, 40 if form == "tokens" else 12)
        q = (1, rng.randint(1, 4)) if form == "tokens" else sorted(_log(rng, 1 if b > 1 else 64, 8192) for _ in range(2))
        c = (0, 0) if form == "prompt" else sorted(_log(rng, 100, 24000) for _ in range(2))
        case = dict(kind="prompt", b=b, q_lo=q[0], q_hi=q[1], c_lo=c[0], c_hi=c[1], heads=heads, kv_heads=kv_heads, d=d, rope=d == 128 and rng.random() < 0.5,
                    dtype=rng.choice(("bf16", "bf16", "fp16")), window=_log(rng, 16, 6000), sinks=rng.choice((0, 0, 1, 4, 64, 200)), lse=rng.random() < 0.5)
        ql, kl = _lengths(case)
        w = work(case)
        if heads <= 128 and w["flops"] <= 6e11 and w["bytes"] <= 4e9 and sum(x * y for x, y in zip(ql, kl)) * heads <= 9e9 and sum(kl) * kv_heads * 2 * d <= 2e9:
            return case


def draw(rng):
    kind = rng.choice(("pages", "slots", "cache", "cache", "cache", "prompt", "prompt"))
    return {"pages": _pages_case, "slots": _slots_case, "cache": _cache_case, "prompt": _prompt_case}[kind](rng)


# ---------------------------------------------------------------- inputs

def _lengths(case):
    """Lengths of a case's sequences, part of its shape, so the same for every seed: (before, after) of pages, else (new tokens, all tokens)."""
    kind = case["kind"]
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if kind == "pages":
        before, after = [], []
        for i in range(case["b"]):
            n, way = r.randint(1, case["far"]), r.randint(0, 99)
            if way < case["fresh"]:
                before.append(0), after.append(n)
            elif way >= 100 - case["done"]:
                before.append(n), after.append(0)
            else:
                before.append(n), after.append(max(n + (r.randint(-case["new"] // 2, case["new"]) if case["new"] > 1 else 1), 0))
        return before, after
    lo, hi, c_lo, c_hi = (case["lo"], case["hi"], 0, case["far"]) if kind == "slots" else (case["q_lo"], case["q_hi"], case["c_lo"], case["c_hi"])
    q = [r.randint(lo, hi) for _ in range(case["b"])]
    return q, [n + r.randint(c_lo, c_hi) for n in q]


class _Maker:
    """Tensors from one seed, made on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEVICE).manual_seed(seed)
        self.r = random.Random(seed)

    def normal(self, shape, dtype=BF):
        return torch.empty(shape, device=DEVICE, dtype=F32).normal_(generator=self.g).to(dtype)

    def uniform(self, shape, lo, hi):
        return torch.empty(shape, device=DEVICE, dtype=F32).uniform_(lo, hi, generator=self.g)

    def whole(self, lo, hi, shape, dtype):
        return torch.randint(lo, hi, shape, device=DEVICE, dtype=dtype, generator=self.g)

    def order(self, n):
        return torch.randperm(n, device=DEVICE, generator=self.g)

    def tree(self, n):
        """A drafted tree: node 0 is the token to go on from, every other hangs on an earlier one, the later ones rather on the last few."""
        return [-1] + [max(self.r.randrange(j), self.r.randrange(j) if self.r.random() < 0.5 else 0) for j in range(1, n)]


def _ints(values):
    return torch.tensor(values, device=DEVICE, dtype=I32)


def _starts(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return _ints(at)


def _pages_of(n, block):
    return -(-n // block)


def _table(m, lengths, block, spare):
    """A block table for sequences of these lengths, pages in random order; how many pages there are; the free ones."""
    per = [_pages_of(n, block) for n in lengths]
    pages = sum(per) + spare
    order = m.order(pages).to(I32)
    wide = max(max(per), 1)
    at = torch.arange(wide, device=DEVICE)[None] < torch.tensor(per, device=DEVICE)[:, None]
    table = torch.full((len(per), wide), -1, device=DEVICE, dtype=I32)
    table[at] = order[:sum(per)]
    return table, pages, order[sum(per):]


def _cache(m, rows, packed):
    """The latent cache, filled: one packed array, or latents, rope and scales."""
    nope, rope, scales = m.whole(-127, 128, [rows, DN], torch.int8), m.normal([rows, DR]), m.uniform([rows, 4], 0.005, 0.02)
    if packed:
        return [torch.cat([nope, rope.view(torch.int8), scales.view(torch.int8)], dim=1).contiguous()]
    return [nope, rope, scales]


def _mask_words(parents, words):
    """Bits of a node and its ancestors, 64 to a word."""
    bits, rows = [], []
    for j, p in enumerate(parents):
        bits.append((1 << j) | (bits[p] if p >= 0 else 0))
        row = [(bits[-1] >> (64 * w)) & (2 ** 64 - 1) for w in range(words)]
        rows.append([x - 2 ** 64 if x >= 2 ** 63 else x for x in row])
    return rows


def prepare(case, seed):
    m, kind = _Maker(seed), case["kind"]
    s = dict(case=case)
    new = lambda *shape, dtype=BF: torch.zeros(shape, device=DEVICE, dtype=dtype)  # noqa: E731
    first, second = _lengths(case)
    if kind == "pages":
        bs = case["block"]
        wide = max(_pages_of(n, bs) for n in first + second)
        takes = sum(max(_pages_of(y, bs) - _pages_of(x, bs), 0) for x, y in zip(first, second))
        table, pages, free = _table(m, first, bs, max(takes // 2, 1) if case["tight"] else takes + 100)
        s.update(before=_ints(first), after=_ints(second), table=torch.cat([table, table.new_full((case["b"], wide - table.shape[1]), -1)], dim=1).contiguous(),
                 free=torch.cat([free, free.new_full((pages - free.numel(),), -1)]), count=_ints([free.numel()]), left=_ints([0]))
    elif kind == "slots":
        tokens = sum(first)
        s.update(query_lens=_ints(first), seq_lens=_ints(second), table=_table(m, second, case["block"], 3)[0],
                 starts_q=new(case["b"] + 1, dtype=I32), starts_k=new(case["b"] + 1, dtype=I32),
                 positions=new(tokens, dtype=I64), slots=new(tokens, dtype=I64), parents=None, mask=None)
        if case["nodes"]:
            s.update(parents=_ints([p for n in first for p in m.tree(n)]), mask=new(tokens, case["nodes"] // 64, dtype=I64))
    elif kind == "cache":
        tq, heads = sum(first), case["heads"]
        table, pages, _ = _table(m, second, case["block"], 3)
        s.update(query=m.normal([tq, heads, DN]), query_rope=m.normal([tq, heads, DR]), cache=_cache(m, pages * case["block"], case["packed"]), table=table,
                 starts_q=_starts(first), seq_lens=_ints(second), scale=192 ** -0.5, out=new(tq, heads, DN), lse=new(tq, heads, dtype=F32) if case["lse"] else None,
                 mask=torch.tensor([row for n in first for row in _mask_words(m.tree(n), case["nodes"] // 64)], device=DEVICE, dtype=I64) if case["nodes"] else None)
    else:
        dt, d, tq, tk = DTYPES[case["dtype"]], case["d"], sum(first), sum(second)
        both = m.normal([tk, case["kv_heads"], 2 * d], dt)          # keys and values as one up-projection leaves them
        s.update(query=m.normal([tq, case["heads"], d], dt), key=both[:, :, :d], value=both[:, :, d:], starts_q=_starts(first), starts_k=_starts(second),
                 query_rope=m.normal([tq, case["heads"], DR], dt) if case["rope"] else None, key_rope=m.normal([tk, DR], dt) if case["rope"] else None,
                 scale=(d + (DR if case["rope"] else 0)) ** -0.5, out=new(tq, case["heads"], d, dtype=dt),
                 lse=new(tq, case["heads"], dtype=F32) if case["lse"] else None)
    return s


# ---------------------------------------------------------------- plain forms

def _flat(counts):
    """Of counts per sequence: for each counted thing its sequence and its number within it."""
    of = torch.repeat_interleave(torch.arange(counts.numel(), device=DEVICE), counts)
    return of, torch.arange(of.numel(), device=DEVICE) - (counts.cumsum(0) - counts)[of]


def _pages(s):
    """Pages of sequences that shrank go on the stack, in order; those that grew take from its top, in order."""
    table, free, bs = s["table"], s["free"], s["case"]["block"]
    had, has = ((s[n].to(I64) + bs - 1).div(bs, rounding_mode="floor").clamp(max=table.shape[1]) for n in ("before", "after"))
    of, at = _flat((had - has).clamp(min=0))
    back = table[of, has[of] + at]
    back = back[back >= 0]
    count = s["count"].to(I64) + back.numel()
    free[s["count"].to(I64) + torch.arange(back.numel(), device=DEVICE)] = back
    of, at = _flat((has - had).clamp(min=0))
    down = count - 1 - torch.arange(of.numel(), device=DEVICE)
    table[of, had[of] + at] = torch.where(down >= 0, free[down.clamp(min=0)], -1)
    return {"table": table, "free": free, "left": (count - of.numel()).clamp(min=0).to(I32)}


def _slots(s):
    ql, sl, bs = s["query_lens"].to(I64), s["seq_lens"].to(I64), s["case"]["block"]
    starts = [torch.cat([x.new_zeros(1), x.cumsum(0)]).to(I32) for x in (ql, sl)]
    of, at = _flat(ql)
    row = (sl - ql)[of] + at
    page = s["table"][of, row // bs].to(I64)
    got = {"starts_q": starts[0], "starts_k": starts[1], "positions": row, "slots": torch.where(page >= 0, page * bs + row % bs, -1)}
    nodes = s["case"]["nodes"]
    if nodes:                          # ancestors by doubling: of a node those within 1, 2, 4 .. steps
        n, first = of.numel(), starts[0].to(I64)[of]
        up = torch.where(s["parents"] >= 0, first + s["parents"], n)
        up = torch.cat([up, up.new_full((1,), n)])
        seen = torch.cat([at[:, None] == torch.arange(nodes, device=DEVICE), torch.zeros(1, nodes, dtype=torch.bool, device=DEVICE)])
        for _ in range(max(nodes - 1, 1).bit_length()):
            seen, up = seen | seen[up], up[up]
        seen = seen[:n]
        got["positions"] = (sl - ql)[of] + seen.sum(dim=1) - 1
        bit = torch.ones((), dtype=I64, device=DEVICE) << torch.arange(64, device=DEVICE)
        got["mask"] = (seen.unflatten(1, (-1, 64)).to(I64) * bit).sum(dim=2)
    return got


def _softmax_product(scores, hidden, values):
    """softmax over the last axis, where nothing is hidden, times values; and the logarithm of the sum of the exponentials."""
    scores.masked_fill_(hidden, -math.inf)
    most = scores.amax(dim=-1, keepdim=True)
    most = torch.where(most > -math.inf, most, 0.0)
    p = scores.sub_(most).exp_()
    total = p.sum(dim=-1, keepdim=True)
    return torch.where(total > 0, (p @ values) / total, 0.0), (most + torch.log(total))[..., 0]


def _hidden(n, keys, window, sinks):
    """[n, keys]: the last of n tokens stands at the last key."""
    at, j = torch.arange(keys - n, keys, device=DEVICE)[:, None], torch.arange(keys, device=DEVICE)
    return (j > at) | ((j <= at - window) & (j >= sinks))


def _parts(cache, packed):
    """Latents, rope and scales of a cache, as views."""
    if not packed:
        return cache
    c = cache[0]
    return c[:, :DN], c[:, DN:DN + 2 * DR].view(BF), c[:, DN + 2 * DR:].view(F32)


def _over_cache(s):
    c = s["case"]
    nope, rope, scales = _parts(s["cache"], c["packed"])
    outs, lses, q0 = [], [], 0
    for i, (n, keys) in enumerate(zip(*_lengths(c))):
        row = torch.arange(keys, device=DEVICE)
        slot = s["table"][i][row // c["block"]].to(I64) * c["block"] + row % c["block"]
        values = (nope[slot].float().unflatten(1, (DN // GROUP, GROUP)) * scales[slot][:, :, None]).flatten(1).to(BF).float()
        q = torch.cat([s["query"][q0:q0 + n], s["query_rope"][q0:q0 + n]], dim=2).float()
        scores = (q.flatten(0, 1) @ torch.cat([values, rope[slot].float()], dim=1).T).mul_(s["scale"]).unflatten(0, (n, -1))
        if c["nodes"]:
            node = torch.arange(n, device=DEVICE)
            drafted = (s["mask"][q0:q0 + n][:, node // 64] >> (node % 64)) & 1 == 0
            hidden = torch.cat([drafted.new_zeros(n, keys - n), drafted], dim=1)
        else:
            hidden = _hidden(n, keys, c["window"], c["sinks"])
        out, lse = _softmax_product(scores, hidden[:, None], values)
        outs.append(out.to(BF)), lses.append(lse)
        q0 += n
    return [torch.cat(outs), torch.cat(lses)] if c["lse"] else [torch.cat(outs)]


def _prompt(s):
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    out = torch.empty(s["query"].shape, device=DEVICE, dtype=dt)
    lse = torch.empty(out.shape[:2], device=DEVICE, dtype=F32)
    g, q0, k0 = c["heads"] // c["kv_heads"], 0, 0
    for n, keys in zip(*_lengths(c)):
        q, k = s["query"][q0:q0 + n].float(), s["key"][k0:k0 + keys].float()
        if c["rope"]:
            q = torch.cat([q, s["query_rope"][q0:q0 + n].float()], dim=2)
            k = torch.cat([k, s["key_rope"][k0:k0 + keys].float()[:, None].expand(-1, c["kv_heads"], -1)], dim=2)
        v, hidden = s["value"][k0:k0 + keys].float(), _hidden(n, keys, c["window"], c["sinks"])
        for h in range(c["kv_heads"]):
            heads = slice(h * g, (h + 1) * g)
            scores = (q[:, heads].flatten(0, 1) @ k[:, h].T.contiguous()).mul_(s["scale"]).unflatten(0, (n, g))
            got, stat = _softmax_product(scores, hidden[:, None], v[:, h].contiguous())
            out[q0:q0 + n, heads], lse[q0:q0 + n, heads] = got.to(dt), stat
        q0, k0 = q0 + n, k0 + keys
    return [out, lse] if c["lse"] else [out]


# ---------------------------------------------------------------- one pass

def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        return {"pages": _pages, "slots": _slots, "cache": _over_cache, "prompt": _prompt}[kind](s)
    import pypto_amd
    if kind == "pages":
        pypto_amd.cache_pages(s["before"], s["after"], s["table"], s["free"], s["count"], s["left"], c["block"])
        return {"table": s["table"], "free": s["free"], "left": s["left"]}
    if kind == "slots":
        pypto_amd.cache_slots(s["query_lens"], s["seq_lens"], s["table"], s["starts_q"], s["starts_k"], s["positions"], s["slots"], c["block"],
                              parents=s["parents"], tree_mask=s["mask"])
        got = {n: s[n] for n in ("starts_q", "starts_k", "positions", "slots")}
        return dict(got, mask=s["mask"]) if c["nodes"] else got
    if kind == "cache":
        op = pypto_amd.latent_attention_packed if c["packed"] else pypto_amd.latent_attention
        op(s["query"], s["query_rope"], *s["cache"], s["table"], s["starts_q"], s["seq_lens"], s["out"], s["scale"], c["block"],
           window=c["window"] or None, sinks=c["sinks"], tree_mask=s["mask"], softmax_lse=s["lse"])
    else:
        pypto_amd.prompt_window_attention(s["query"], s["key"], s["value"], s["starts_q"], s["starts_k"], s["out"], s["scale"], c["window"], sinks=c["sinks"],
                                          query_rope=s["query_rope"], key_rope=s["key_rope"], softmax_lse=s["lse"])
    return [s["out"], s["lse"]] if c["lse"] else [s["out"]]


# ---------------------------------------------------------------- what a pass cannot do without

def _seen(n, keys, window, sinks):
    """Keys that n tokens, the last of which stands at the last key, see together (counted once), and pairs."""
    pairs, low = 0, keys - n + 1
    for sees in range(low, keys + 1):
        pairs += sees if sees <= window + sinks else window + sinks
    first = max(low - window, 0)                       # the first token's window begins here
    return keys - first + min(sinks, first), pairs


def work(case):
    kind = case["kind"]
    first, second = _lengths(case)
    if kind == "pages":
        bs = case["block"]
        moved = sum(abs(_pages_of(y, bs) - _pages_of(x, bs)) for x, y in zip(first, second))
        return dict(bytes=8 * case["b"] + 8 + 8 * moved, flops=moved)
    if kind == "slots":
        t, bs = sum(first), case["block"]
        pages = sum(_pages_of(y, bs) - (y - x) // bs for x, y in zip(first, second))
        return dict(bytes=16 * case["b"] + 8 + 4 * pages + t * (16 + (4 + case["nodes"] // 8 if case["nodes"] else 0)), flops=2 * t)
    heads = case["heads"]
    if kind == "cache":
        if case["nodes"]:              # a drafted token sees the context and, of the tree, some of the nodes before it: counted as none but itself
            seen = [(keys, n * (keys - n + 1)) for n, keys in zip(first, second)]
        else:
            seen = [_seen(n, keys, case["window"], case["sinks"]) for n, keys in zip(first, second)]
        tq = sum(first)
        return dict(bytes=2 * tq * heads * (2 * DN + DR) + sum(k for k, _ in seen) * PACKED + (4 * tq * heads if case["lse"] else 0) + tq * case["nodes"] // 8,
                    flops=2 * heads * sum(p for _, p in seen) * (2 * DN + DR))
    seen = [_seen(n, keys, case["window"], case["sinks"]) for n, keys in zip(first, second)]
    d, r, tq = case["d"], DR if case["rope"] else 0, sum(first)
    return dict(bytes=2 * (tq * heads * (2 * d + r) + sum(k for k, _ in seen) * (case["kv_heads"] * 2 * d + r)) + (4 * tq * heads if case["lse"] else 0),
                flops=2 * heads * sum(p for _, p in seen) * (2 * d + r))


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    if case["kind"] in ("pages", "slots"):
        return None                    # whole numbers
    s = prepare(case, seed)
    ql, kl = _lengths(case)
    heads = case["heads"]
    g = heads // case.get("kv_heads", 1)
    out = torch.zeros(s["query"].shape, device=DEVICE, dtype=F64)
    lse = torch.zeros(out.shape[:2], device=DEVICE, dtype=F64)
    q0 = k0 = 0
    for i, (n, keys) in enumerate(zip(ql, kl)):
        sees = torch.zeros(n, keys, dtype=torch.bool, device=DEVICE)
        if case.get("nodes"):
            words = s["mask"][q0:q0 + n].tolist()
            sees[:, :keys - n] = True
            sees[:, keys - n:] = torch.tensor([[bool(row[j >> 6] >> (j & 63) & 1) for j in range(n)] for row in words], device=DEVICE)
        else:
            sees[:] = True
            sees = sees.tril(keys - n) & (sees.triu(keys - n - case["window"] + 1) | (torch.arange(keys, device=DEVICE) < case["sinks"]))
        if case["kind"] == "cache":
            nope, rope, scales = _parts(s["cache"], case["packed"])
            pages = s["table"][i, :_pages_of(keys, case["block"])].long()
            slots = (pages[:, None] * case["block"] + torch.arange(case["block"], device=DEVICE)).reshape(-1)[:keys]
            v = (nope[slots].float() * scales[slots].repeat_interleave(GROUP, dim=1)).to(BF).double()
            k = torch.cat([v, rope[slots].double()], dim=1)
        for h in range(heads):
            if case["kind"] == "prompt":
                k, v = s["key"][k0:k0 + keys, h // g].double(), s["value"][k0:k0 + keys, h // g].double()
                if case["rope"]:
                    k = torch.cat([k, s["key_rope"][k0:k0 + keys].double()], dim=1)
            q = s["query"][q0:q0 + n, h].double()
            if s["query_rope"] is not None:
                q = torch.cat([q, s["query_rope"][q0:q0 + n, h].double()], dim=1)
            a = torch.where(sees, (q @ k.T) * s["scale"], -math.inf)
            lse[q0:q0 + n, h] = torch.logsumexp(a, dim=1)
            out[q0:q0 + n, h] = torch.softmax(a, dim=1) @ v
        q0, k0 = q0 + n, k0 + keys
    return [out, lse] if case["lse"] else [out]
