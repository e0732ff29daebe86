"""The measured operators: what a prompt needs before and around the sparse path.

A prompt no longer than the selection sees all of its keys, and is cheaper to attend in the model's multi-head form (128 + 64
channels to a query and key, 128 to a value) than over the latent cache: its queries and keys are rotated, its latents
quantised into the cache, earlier chunks' latents read back out of it, and the heads attend over whole sequences.  The cases
are the calls of those operators -- rotary tables, rotation, cache write, cache read, prompt attention -- from one token of a
decode step to whole prompts.  Sizes are those of the repository's tests and benchmark (128 heads, latents of 512 + 64, pages
of 128 positions) or generic ones (64 query heads over 8 key heads).

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
BF, HALF, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
DTYPES = {"bf16": BF, "fp16": HALF, "fp32": F32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # a decode step's cos and sin rows for the prologs: 32 sequences, one position each
        dict(name="tables_32", kind="tables", t=32, far=65536, dtype="bf16"),
        # the rows of several prompts' chunks in one pass, far positions among them
        dict(name="tables_16385", kind="tables", t=16385, far=131072, dtype="fp32"),
        # one decoded token's query and key, whose last 64 channels of 192 turn
        dict(name="rotary_1", kind="rotary", t=1, far=65536, heads=128, dim=192, key_heads=1, layout="deinterleaved", dtype="bf16"),
        # a prompt's queries (the rope part of 192-wide heads) and the one rope key that all heads share
        dict(name="rotary_4096", kind="rotary", t=4096, far=8192, heads=128, dim=192, key_heads=1, layout="interleaved", dtype="bf16"),
        # a decode batch written into the packed cache
        dict(name="write_32", kind="write", t=32, rows=65536, packed=True, values=False, dtype="bf16"),
        # a ragged chunk of prompts written into the three arrays, the values that the cache now stands for wanted too
        dict(name="write_8191", kind="write", t=8191, rows=32768, packed=False, values=True, dtype="bf16"),
        # the context of eleven young and old sequences read back from the packed cache
        dict(name="read_packed_11", kind="read", b=11, lo=190, hi=6000, packed=True),
        # one long sequence's context out of the three arrays
        dict(name="read_65536", kind="read", b=1, lo=65536, hi=65536, packed=False),
        # a whole prompt in the multi-head form: 128 heads, 128 + 64 channels, the rope key shared by all heads
        dict(name="prompt_4096", kind="attention", b=1, q_lo=4096, q_hi=4096, c_lo=0, c_hi=0, heads=128, kv_heads=128, d=128, rope=True,
             dtype="bf16", causal=True, lse=False),
        # nine prompts of different lengths packed one after the other, eight query heads to a key head
        dict(name="prompt_packed_9", kind="attention", b=9, q_lo=1, q_hi=2200, c_lo=0, c_hi=0, heads=64, kv_heads=8, d=128, rope=False,
             dtype="bf16", causal=True, lse=True),
        # a chunk of 1024 tokens behind a context of some 15000, the heads divided over eight GPUs
        dict(name="chunk_1024", kind="attention", b=1, q_lo=1024, q_hi=1024, c_lo=15001, c_hi=15001, heads=16, kv_heads=16, d=128, rope=True,
             dtype="bf16", causal=True, lse=True),
        # single tokens of 32 sequences over their keys, eight query heads to a key head
        dict(name="tokens_32", kind="attention", b=32, q_lo=1, q_hi=1, c_lo=700, c_hi=12000, heads=64, kv_heads=8, d=128, rope=False,
             dtype="fp16", causal=True, lse=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _attention(rng):
    while True:
        form = rng.choice(("prompt", "prompt", "chunk", "tokens"))
        d = rng.choice((128, 128, 128, 64))
        kv_heads = rng.choice((1, 2, 4, 8, 16, 32, 128))
        heads = kv_heads * rng.choice((1, 1, 2, 4, 7, 8, 16))
        b = _log(rng, 1, 40 if form == "tokens" else 12)
        q = (1, rng.randint(1, 4)) if form == "tokens" else sorted(_log(rng, 1 if b > 1 else 64, 4096) for _ in range(2))
        c = (0, 0) if form == "prompt" else sorted(_log(rng, 100, 24000) for _ in range(2))
        case = dict(kind="attention", b=b, q_lo=q[0], q_hi=q[1], c_lo=c[0], c_hi=c[1], heads=heads, kv_heads=kv_heads, d=d,
                    rope=d == 128 and rng.random() < 0.5, dtype=rng.choice(("bf16", "bf16", "fp16")),
                    causal=rng.random() < 0.85, lse=rng.random() < 0.5)
        ql, kl = _lengths(case)
        w = work(case)
        # no dearer than the largest listed case, in the padded scores of the plain form as well
        if heads <= 128 and w["flops"] <= 6.8e11 and w["bytes"] <= 4e9 and b * heads * max(ql) * max(kl) <= 2.1e9 \
                and b * heads * max(kl) * (2 * d) <= 4e9:
            return case


def draw(rng):
    kind = rng.choice(("tables", "rotary", "rotary", "write", "write", "read", "read", "attention", "attention", "attention", "attention"))
    if kind == "tables":
        return dict(kind=kind, t=_log(rng, 1, 40000), far=_log(rng, 4096, 1 << 20), dtype=rng.choice(("bf16", "fp16", "fp32")))
    if kind == "rotary":
        return dict(kind=kind, t=_log(rng, 1, 4096), far=_log(rng, 4096, 1 << 20), heads=rng.choice((128, 64, 40, 16)), dim=rng.choice((192, 128, 64)),
                    key_heads=rng.choice((1, 1, 8)), layout=rng.choice(("half", "interleaved", "deinterleaved")), dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")))
    if kind == "write":
        t = _log(rng, 1, 16000)
        return dict(kind=kind, t=t, rows=PAGE * (t // PAGE + _log(rng, 2, 400)), packed=rng.random() < 0.5, values=rng.random() < 0.6,
                    dtype=rng.choice(("bf16", "bf16", "bf16", "fp16", "fp32")))
    if kind == "read":
        b = _log(rng, 1, 64)
        lo, hi = sorted(_log(rng, 1, 100000 // b) for _ in range(2))
        return dict(kind=kind, b=b, lo=lo, hi=hi, packed=rng.random() < 0.5)
    return _attention(rng)


# ---------------------------------------------------------------- inputs

def _lengths(case):
    """Lengths of a case's sequences, part of its shape, so the same for every seed: of an attention (queries, keys)."""
    if case["kind"] == "read":
        r = random.Random(11 * case["b"] + case["lo"])
        return [r.randint(case["lo"], case["hi"]) for _ in range(case["b"])]
    r = random.Random(7 * case["b"] + case["q_hi"] + case["c_lo"])
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["b"])]
    return q, [n + r.randint(case["c_lo"], case["c_hi"]) for n in q]


class _Maker:
    """Tensors from one seed, made on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(self, shape, dtype=BF):
        return torch.empty(shape, device=DEVICE, dtype=F32).normal_(generator=self.g).to(dtype)

    def uniform(self, shape, lo, hi):
        return torch.empty(shape, device=DEVICE, dtype=F32).uniform_(lo, hi, generator=self.g)

    def whole(self, lo, hi, shape, dtype):
        return torch.randint(lo, hi, shape, device=DEVICE, dtype=dtype, generator=self.g)

    def order(self, n):
        return torch.randperm(n, device=DEVICE, generator=self.g)


def _frequencies():
    """Radians per position of the 32 pairs, stretched 40 times beyond the 4096 positions of training: pairs that turn more
    than 32 times within those keep their speed, pairs that turn less than once are slowed down by all of 40."""
    i = torch.arange(DR // 2, dtype=F64)
    plain = 10000.0 ** (-2 * i / DR)
    pair = lambda turns: DR * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0))  # noqa: E731
    lo, hi = math.floor(pair(32)), math.ceil(pair(1))
    slow = ((i - lo) / (hi - lo)).clamp(0, 1)
    return (plain * (1 - slow) + plain / 40 * slow).to(DEVICE)


def _starts(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, device=DEVICE, dtype=torch.int32)


def _cache(m, rows, packed):
    """The latent cache, filled: one packed array, or latents, rope and scales."""
    nope, rope, scales = m.whole(-127, 128, [rows, DN], torch.int8), m.normal([rows, DR]), m.uniform([rows, 4], 0.005, 0.02)
    if packed:
        return [torch.cat([nope, rope.view(torch.int8), scales.view(torch.int8)], dim=1).contiguous()]
    return [nope, rope, scales]


def prepare(case, seed):
    m, kind = _Maker(seed), case["kind"]
    s = dict(case=case)
    new = lambda *shape, dtype=BF: torch.zeros(shape, device=DEVICE, dtype=dtype)  # noqa: E731
    if kind in ("tables", "rotary"):
        dt, t = DTYPES[case["dtype"]], case["t"]
        s.update(positions=m.whole(0, case["far"], [t], torch.int64), frequencies=_frequencies())
        if kind == "tables":
            s.update(cos=new(t, DR, dtype=dt), sin=new(t, DR, dtype=dt))
        else:                          # the rope part of every head, cut out of the projections' outputs
            s.update(query=m.normal([t, case["heads"], case["dim"]], dt)[:, :, case["dim"] - DR:], key=m.normal([t, case["key_heads"], DR], dt),
                     query_out=new(t, case["heads"], DR, dtype=dt), key_out=new(t, case["key_heads"], DR, dtype=dt))
    elif kind == "write":              # latent and rope key lie side by side, as the down-projection leaves them
        both = m.normal([case["t"], DN + DR], DTYPES[case["dtype"]])
        s.update(latent=both[:, :DN], rope=both[:, DN:], index=m.order(case["rows"])[:case["t"]], cache=_cache(m, case["rows"], case["packed"]),
                 values=new(case["t"], DN) if case["values"] else None)
    elif kind == "read":
        lengths = _lengths(case)
        per = [-(-n // PAGE) for n in lengths]
        pages = sum(per) + 3
        order = m.order(pages).to(torch.int32)
        table = torch.full((len(lengths), max(per)), -1, device=DEVICE, dtype=torch.int32)
        at = 0
        for i, n in enumerate(per):
            table[i, :n] = order[at:at + n]
            at += n
        s.update(cache=_cache(m, pages * PAGE, case["packed"]), table=table, starts=_starts(lengths),
                 latent=new(sum(lengths), DN), rope=new(sum(lengths), DR))
    else:
        ql, kl = _lengths(case)
        dt, d = DTYPES[case["dtype"]], case["d"]
        tq, tk = sum(ql), sum(kl)
        both = m.normal([tk, case["kv_heads"], 2 * d], dt)          # keys and values as one up-projection leaves them
        s.update(query=m.normal([tq, case["heads"], d], dt), key=both[:, :, :d], value=both[:, :, d:], starts_q=_starts(ql), starts_k=_starts(kl),
                 query_rope=m.normal([tq, case["heads"], DR], dt) if case["rope"] else None, key_rope=m.normal([tk, DR], dt) if case["rope"] else None,
                 scale=(d + (DR if case["rope"] else 0)) ** -0.5, most=(max(ql), max(kl)), out=new(tq, case["heads"], d, dtype=dt),
                 lse=new(tq, case["heads"], dtype=F32) if case["lse"] else None)
    return s


# ---------------------------------------------------------------- plain forms

def _turns(s):
    """cos and sin of every token's 32 angles, whose positions take 64 bits."""
    angle = s["positions"].to(F64)[:, None] * s["frequencies"]
    return angle.cos(), angle.sin()


def _tables(s):
    dt = DTYPES[s["case"]["dtype"]]
    return {n: torch.cat([v, v], dim=1).to(dt) for n, v in zip(("cos", "sin"), _turns(s))}


def _turned(x, cos, sin, layout):
    x, c, n = x.float(), cos.float()[:, None, :], x.shape[-1] // 2
    z = sin.float()[:, None, :]
    a, b = (x[..., :n], x[..., n:]) if layout == "half" else (x[..., 0::2], x[..., 1::2])
    a, b = a * c - b * z, b * c + a * z
    return torch.stack([a, b], dim=-1).flatten(-2) if layout == "interleaved" else torch.cat([a, b], dim=-1)


def _rotary(s):
    (cos, sin), layout = _turns(s), s["case"]["layout"]
    return {n: _turned(s[n], cos, sin, layout).to(s[n].dtype) for n in ("query", "key")}


def _parts(cache, packed):
    """Latents, rope and scales of a cache, as views."""
    if not packed:
        return cache
    c = cache[0]
    return c[:, :DN], c[:, DN:DN + 2 * DR].view(BF), c[:, DN + 2 * DR:].view(F32)


def _write(s):
    v = s["latent"].float().unflatten(1, (DN // GROUP, GROUP))
    most = v.abs().amax(dim=2, keepdim=True)
    steps = torch.where(most > 0, 127 / most, 0.0)
    codes = torch.round(v * steps)
    scales = torch.where(most > 0, 1 / steps, 0.0)
    nope, rope, kept = _parts(s["cache"], s["case"]["packed"])
    nope[s["index"]] = codes.flatten(1).to(torch.int8)
    rope[s["index"]] = s["rope"].to(BF)
    kept[s["index"]] = scales[:, :, 0]
    return (codes * scales).flatten(1).to(BF) if s["case"]["values"] else None


def _read(s):
    nope, rope, scales = _parts(s["cache"], s["case"]["packed"])
    starts = s["starts"].to(torch.int64)
    row = torch.arange(s["latent"].shape[0], device=DEVICE)
    of = torch.bucketize(row, starts[1:], right=True)
    at = row - starts[of]
    slot = s["table"][of, at // PAGE].to(torch.int64) * PAGE + at % PAGE
    values = nope[slot].float().unflatten(1, (DN // GROUP, GROUP)) * scales[slot][:, :, None]
    return {"latent": values.flatten(1).to(BF), "rope": rope[slot]}


def _rows(x, starts, most):
    """[sequences, most, heads, channels] of a packed tensor, in 32 bits; rows behind a sequence hold something."""
    at = (starts[:-1, None] + torch.arange(most, device=DEVICE)).clamp(max=x.shape[0] - 1)
    return x[at].float()


def _attend(s):
    c, (mq, mk) = s["case"], s["most"]
    starts_q, starts_k = s["starts_q"].to(torch.int64), s["starts_k"].to(torch.int64)
    ql, kl = starts_q.diff(), starts_k.diff()
    b, kv, g, d = c["b"], c["kv_heads"], c["heads"] // c["kv_heads"], c["d"]
    heads_first = lambda x: x.unflatten(2, (kv, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3).contiguous()  # noqa: E731  [b, kv, g * most, channels]
    q, k, v = (heads_first(_rows(s[n], starts, most)) for n, starts, most in (("query", starts_q, mq), ("key", starts_k, mk), ("value", starts_k, mk)))
    scores = q @ k.transpose(2, 3)
    if c["rope"]:
        scores += heads_first(_rows(s["query_rope"], starts_q, mq)) @ _rows(s["key_rope"], starts_k, mk)[:, None].transpose(2, 3)
    scores *= s["scale"]
    rows, keys = torch.arange(mq, device=DEVICE)[:, None], torch.arange(mk, device=DEVICE)
    sees = kl[:, None] if not c["causal"] else (kl - ql)[:, None] + rows[:, 0] + 1
    hidden = keys >= torch.minimum(sees, kl[:, None])[:, :, None]                       # [b, mq or 1, mk]
    scores.unflatten(2, (g, mq)).masked_fill_(hidden[:, None, None], -math.inf)
    most = scores.amax(dim=3, keepdim=True)
    most = torch.where(most > -math.inf, most, 0.0)
    p = torch.exp(scores.sub_(most))
    total = p.sum(dim=3, keepdim=True)
    out = torch.where(total > 0, (p @ v) / total, 0.0).unflatten(2, (g, mq)).permute(0, 3, 1, 2, 4)   # [b, mq, kv, g, d]
    there = rows[:, 0] < ql[:, None]
    got = [out.flatten(2, 3)[there].to(s["query"].dtype)]
    if c["lse"]:
        got.append((most + torch.log(total)).unflatten(2, (g, mq)).permute(0, 3, 1, 2, 4).flatten(2)[there])
    return got


# ---------------------------------------------------------------- one pass

def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if own:
        import pypto_amd
        if kind == "tables":
            pypto_amd.rotary_tables(s["positions"], s["frequencies"], s["cos"], s["sin"])
        elif kind == "rotary":
            pypto_amd.rotary_embedding(s["query"], s["key"], s["positions"], s["frequencies"], s["query_out"], s["key_out"], layout=c["layout"])
        elif kind == "write":
            op = pypto_amd.latent_cache_write_packed if c["packed"] else pypto_amd.latent_cache_write
            op(s["latent"], s["rope"], s["index"], *s["cache"], s["values"])
        elif kind == "read":
            op = pypto_amd.latent_cache_read_packed if c["packed"] else pypto_amd.latent_cache_read
            op(*s["cache"], s["table"], s["starts"], s["latent"], s["rope"], PAGE)
        else:
            pypto_amd.prompt_attention(s["query"], s["key"], s["value"], s["starts_q"], s["starts_k"], s["out"], s["scale"],
                                       query_rope=s["query_rope"], key_rope=s["key_rope"], softmax_lse=s["lse"], causal=c["causal"])
    if kind == "tables":
        return {"cos": s["cos"], "sin": s["sin"]} if own else _tables(s)
    if kind == "rotary":
        return {"query": s["query_out"], "key": s["key_out"]} if own else _rotary(s)
    if kind == "write":
        values = s["values"] if own else _write(s)
        got = dict(zip(("codes", "rope", "scales"), _parts(s["cache"], c["packed"])))
        return dict(got, values=values) if c["values"] else got
    if kind == "read":
        return {"latent": s["latent"], "rope": s["rope"]} if own else _read(s)
    if not own:
        return _attend(s)
    return [s["out"], s["lse"]] if c["lse"] else [s["out"]]


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind == "tables":
        return dict(bytes=case["t"] * (8 + 2 * DR * SIZE[case["dtype"]]) + 8 * DR // 2, flops=case["t"] * DR)
    if kind == "rotary":
        values = case["t"] * (case["heads"] + case["key_heads"]) * DR
        return dict(bytes=2 * values * SIZE[case["dtype"]] + 8 * case["t"] + 8 * DR // 2, flops=3 * values)
    if kind == "write":
        t = case["t"]
        return dict(bytes=t * ((DN + DR) * SIZE[case["dtype"]] + PACKED + 8 + (2 * DN if case["values"] else 0)), flops=4 * t * DN)
    if kind == "read":
        rows = _lengths(case)
        return dict(bytes=sum(rows) * (PACKED + 2 * (DN + DR)) + 4 * sum(-(-n // PAGE) for n in rows), flops=sum(rows) * DN)
    ql, kl = _lengths(case)
    d, r, n = case["d"], DR if case["rope"] else 0, SIZE[case["dtype"]]
    pairs = sum(q * k - (q * (q - 1) // 2 if case["causal"] else 0) for q, k in zip(ql, kl))
    tq, tk = sum(ql), sum(kl)
    return dict(bytes=n * (tq * case["heads"] * (2 * d + r) + tk * (case["kv_heads"] * 2 * d + r)) + (4 * tq * case["heads"] if case["lse"] else 0),
                flops=2 * case["heads"] * pairs * (2 * d + r))


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("tables", "rotary"):
        turn = torch.polar(torch.ones((), dtype=F64, device=DEVICE), torch.outer(s["positions"].double(), s["frequencies"]))
        if kind == "tables":
            return {"cos": turn.real.repeat(1, 2), "sin": turn.imag.repeat(1, 2)}
        got = {}
        for name in ("query", "key"):
            x = s[name].double()
            pair = x.unflatten(2, (2, -1)).transpose(2, 3) if case["layout"] == "half" else x.unflatten(2, (-1, 2))
            z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn[:, None, :])
            got[name] = (z if case["layout"] == "interleaved" else z.transpose(2, 3)).flatten(2)
        return got
    if kind == "write":
        v = s["latent"].double().reshape(-1, DN // GROUP, GROUP)
        scale = v.abs().max(dim=2).values / 127
        value = ((v / scale[:, :, None]).round() * scale[:, :, None]).reshape(-1, DN)
        _, rope, scales = _parts(s["cache"], case["packed"])
        rope, scales = rope.double(), scales.double()
        rope[s["index"]], scales[s["index"]] = s["rope"].double(), scale
        got = {"codes": None, "rope": rope, "scales": scales}
        return dict(got, values=value) if case["values"] else got
    if kind == "read":
        nope, rope, scales = _parts(s["cache"], case["packed"])
        latent, turned = [], []
        for i, n in enumerate(_lengths(case)):
            pages = s["table"][i, :-(-n // PAGE)].long()
            slots = (pages[:, None] * PAGE + torch.arange(PAGE, device=DEVICE)).reshape(-1)[:n]
            latent.append(nope[slots].double() * scales[slots].double().repeat_interleave(GROUP, dim=1))
            turned.append(rope[slots].double())
        return {"latent": torch.cat(latent), "rope": torch.cat(turned)}
    ql, kl = _lengths(case)
    g = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["query"].shape, device=DEVICE, dtype=F64)
    lse = torch.zeros(out.shape[:2], device=DEVICE, dtype=F64)
    q0 = k0 = 0
    for nq, nk in zip(ql, kl):
        late = torch.arange(nk, device=DEVICE) > torch.arange(nk - nq, nk, device=DEVICE)[:, None]
        kr = s["key_rope"][k0:k0 + nk].double() if case["rope"] else None
        for h in range(case["heads"]):
            a = s["query"][q0:q0 + nq, h].double() @ s["key"][k0:k0 + nk, h // g].double().T
            if kr is not None:
                a += s["query_rope"][q0:q0 + nq, h].double() @ kr.T
            a *= s["scale"]
            if case["causal"]:
                a[late] = -math.inf
            lse[q0:q0 + nq, h] = torch.logsumexp(a, dim=1)
            out[q0:q0 + nq, h] = torch.softmax(a, dim=1) @ s["value"][k0:k0 + nk, h // g].double()
        q0, k0 = q0 + nq, k0 + nk
    return [out, lse] if case["lse"] else [out]
