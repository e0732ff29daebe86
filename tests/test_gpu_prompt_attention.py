"""prompt_attention against attention in 64 bits, with element-wise bounds that count the roundings of 16-bit operands and fp32 sums
(oracle.prompt_oracle.attention_bounds)."""
import math

import pytest
import torch

import pypto_amd
from oracle import prompt_oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HALF = torch.bfloat16, torch.float16


def starts(lengths):
    return torch.tensor([0] + list(torch.tensor(lengths).cumsum(0)), dtype=torch.int32, device=DEV)


class Call:
    def __init__(self, lens_q, lens_k, heads, kv, d, rope=False, dtype=BF, causal=True, seed=0, spare=0, scale=None, shared=True, size=1.0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        new = lambda *s: (size * torch.randn(s, generator=g, device=DEV)).to(dtype)  # noqa: E731
        self.lens_q, self.lens_k, self.causal, self.dtype = lens_q, lens_k, causal, dtype
        tq, tk = sum(lens_q) + spare, sum(lens_k) + spare
        both = new(tk, kv, 2 * d)                                  # keys and values side by side
        self.q, self.k, self.v = new(tq, heads, d), both[:, :, :d], both[:, :, d:]
        self.qr = new(tq, heads, 64) if rope else None
        self.kr = (new(tk, 64) if shared else new(tk, kv, 64)) if rope else None
        self.channels = d + (64 if rope else 0)
        self.scale = self.channels ** -0.5 if scale is None else scale
        self.out = torch.full((tq, heads, d), 7.0, dtype=dtype, device=DEV)
        self.lse = torch.full((tq, heads), 7.0, device=DEV)

    def run(self, lse=True):
        pypto_amd.prompt_attention(self.q, self.k, self.v, starts(self.lens_q), starts(self.lens_k), self.out, self.scale, query_rope=self.qr,
                                   key_rope=self.kr, softmax_lse=self.lse if lse else None, causal=self.causal)
        return self

    def check(self):
        torch.cuda.synchronize()
        n = sum(self.lens_q)
        want = prompt_oracle.attention(self.q, self.k, self.v, self.lens_q, self.lens_k, self.scale, self.qr, self.kr, self.causal)
        out, lse, mean, reach, seen = (x[:n] for x in want)
        may, may_lse = prompt_oracle.attention_bounds(self.dtype, self.channels, out, lse, mean, reach, seen)
        off = (self.out[:n].double() - out).abs()
        assert bool((off <= may).all()), f"{(off / may).max().item():.3g} of what it may be off by, at {tuple((off / may).argmax().unsqueeze(0).tolist())}"
        some = seen > 0
        assert torch.equal(torch.isneginf(self.lse[:n]), ~some)
        assert bool(((self.lse[:n].double() - lse).abs()[some] <= may_lse[some]).all())
        assert bool((self.out[:n][~some] == 0).all())
        assert bool((self.out[n:] == 7).all() and (self.lse[n:] == 7).all()), "rows of no sequence were written"


FORMS = [(64, False), (128, False), (128, True)]


@pytest.mark.parametrize("d,rope", FORMS)
@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv", [(2, 2), (6, 2), (7, 1)])
def test_lengths_around_every_tile(d, rope, dtype, causal, heads, kv):
    lens_q = [1, 2, 31, 32, 33, 0, 63, 64, 65, 100, 255, 256, 257, 300, 1, 5]
    lens_k = [1, 2, 31, 32, 33, 0, 63, 64, 65, 100, 255, 256, 257, 300, 4, 0]
    Call(lens_q, lens_k, heads, kv, d, rope, dtype, causal, seed=1, spare=3).run().check()


@pytest.mark.parametrize("d,rope", FORMS)
@pytest.mark.parametrize("lens_q,lens_k", [
    ([1], [1]), ([1], [64]), ([1], [65]), ([1], [1000]), ([1, 1, 1], [3000, 1, 17]), ([3, 2, 4], [2000, 900, 4]), ([40], [5000]),
    ([257, 1], [1500, 700]), ([5, 0, 3], [2, 9, 3])])
@pytest.mark.parametrize("heads,kv", [(8, 1), (4, 4), (16, 2)])
def test_keys_from_before_the_queries(d, rope, lens_q, lens_k, heads, kv):
    """Chunks and single tokens, with keys divided over workgroups; rows that see nothing where there are fewer keys than queries."""
    Call(lens_q, lens_k, heads, kv, d, rope, seed=2, spare=1).run().check()
    Call(lens_q, lens_k, heads, kv, d, rope, HALF, causal=False, seed=3).run().check()


@pytest.mark.parametrize("d,rope", FORMS)
def test_many_heads_and_sequences(d, rope):
    lens = [int(n) for n in torch.randint(1, 40, (150,), generator=torch.Generator().manual_seed(1))]
    Call(lens, [n + (i * 13) % 50 for i, n in enumerate(lens)], 16, 4, d, rope, seed=4, spare=2).run().check()
    Call([200], [200], 128, 128, d, rope, seed=5).run().check()


@pytest.mark.parametrize("d,rope", FORMS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens_q,lens_k,heads,kv,rows", [
    ([700, 300], [700, 333], 4, 4, 128), ([735, 300], [735, 333], 32, 32, 256), ([65, 1, 0, 80], [400, 1, 7, 80], 15, 1, 128),
    ([600], [700], 64, 32, 256), ([500], [1027], 40, 40, 128), ([513], [1027], 64, 64, 256), ([127], [129], 8, 2, 128)])
def test_workgroups_of_either_size(d, rope, causal, lens_q, lens_k, heads, kv, rows):
    """Around the numbers of rows from which workgroups of 128 channels are twice as large."""
    from pypto_amd import _C
    plan = _C.prompt_attention_plan(len(lens_q), sum(lens_q), sum(lens_k), heads, kv, d, rope, causal)
    assert plan["rows_per_workgroup"] == (rows if d == 128 else 128)
    Call(lens_q, lens_k, heads, kv, d, rope, causal=causal, seed=21, spare=2).run().check()


@pytest.mark.parametrize("d,rope", FORMS)
@pytest.mark.parametrize("lens_q,lens_k", [([600, 0, 500], [6000, 0, 300]), ([1, 700, 400], [1, 200, 7000])])
def test_more_divided_rows_than_waves_among_rows_that_are_not(d, rope, lens_q, lens_k):
    """More rows than the launch that joins the pieces has waves, so a wave has several, of sequences that are divided and of others."""
    from pypto_amd import _C
    plan = _C.prompt_attention_plan(len(lens_q), sum(lens_q), sum(lens_k), 16, 1, d, rope, True)
    assert plan["key_splits"] > 1 and plan["split_keys"] >= 300
    Call(lens_q, lens_k, 16, 1, d, rope, seed=20).run().check()


def test_a_key_head_s_own_rope_part_and_its_one_head_form():
    Call([70, 130], [90, 130], 8, 4, 128, True, seed=6, shared=False).run().check()
    a = Call([70, 130], [90, 130], 8, 4, 128, True, seed=6).run()
    b = Call([70, 130], [90, 130], 8, 4, 128, True, seed=6)
    b.kr = b.kr[:, None]
    b.run().check()
    assert torch.equal(a.out, b.out) and torch.equal(a.lse, b.lse)


@pytest.mark.parametrize("way", ["rising", "falling", "steep", "wide"])
@pytest.mark.parametrize("lens", [([300], [300]), ([2], [2500])])
def test_scores_that_move_the_maximum(way, lens):
    """Scores that rise by many powers of two along the keys, that fall, that one key alone dominates."""
    c = Call(*lens, 4, 2, 64, seed=7, scale=1.0)
    n = lens[1][0]
    ramp = torch.arange(n, device=DEV).float() / n * 60 * (1 if way == "rising" else -1)
    c.q.zero_()
    c.q[..., 0] = 1.0
    if way in ("rising", "falling"):
        c.k[..., 0] = ramp[:, None].to(BF)
    elif way == "steep":
        c.k[..., 0] = 0
        c.k[n // 2, :, 0] = 200.0
    else:
        c.k[..., 0] = (300 * torch.randn(n, 1, device=DEV, generator=torch.Generator(device=DEV).manual_seed(8))).to(BF)
    c.run().check()


@pytest.mark.parametrize("scale", [0.0, -0.11, 3.0])
def test_scales(scale):
    Call([70, 1], [200, 600], 4, 2, 128, True, seed=9, scale=scale).run().check()


def test_what_lies_behind_a_sequence_is_not_looked_at():
    """Infinities and NaN in key and value rows of no sequence, and in other sequences."""
    c = Call([33, 20], [33, 70], 4, 2, 128, True, seed=10, spare=40)
    d = Call([33, 20], [33, 70], 4, 2, 128, True, seed=10, spare=40)
    for t in (d.k, d.v, d.kr):
        t[103:] = math.nan
    d.v[110] = math.inf
    c.run(), d.run()
    assert torch.equal(c.out, d.out) and torch.equal(c.lse, d.lse)
    e = Call([33, 20], [33, 70], 4, 2, 128, True, seed=10, spare=40)
    for t in (e.k, e.v, e.kr):
        t[33:103] = math.nan
    e.run()
    assert torch.equal(c.out[:33], e.out[:33]) and bool(e.out[33:53].isnan().all())


def test_keys_that_are_no_numbers_and_are_not_seen():
    """A key that is no number reaches the rows that see it and no other (its value is a number)."""
    c, d = (Call([100], [100], 4, 4, 64, seed=11) for _ in range(2))
    d.k[60] = math.nan
    c.run(), d.run()
    assert torch.equal(c.out[:60], d.out[:60]) and bool(d.out[60:].isnan().all())


def test_a_score_of_infinity_is_no_number():
    c = Call([3], [90], 2, 2, 64, seed=12)
    c.q[..., 0] = 0
    c.q[1, :, 0] = 3e38
    c.k[5] = 0
    c.k[5, :, 0] = 3e38
    c.run()
    torch.cuda.synchronize()
    assert bool(c.out[1].isnan().all()) and not bool(c.out[0].isnan().any())


@pytest.mark.parametrize("form", ["heads_first", "sliced", "odd_output"])
def test_strides(form):
    a = Call([50, 77], [90, 77], 8, 2, 128, True, seed=13)
    b = Call([50, 77], [90, 77], 8, 2, 128, True, seed=13)
    if form == "heads_first":
        for n in ("q", "k", "v", "qr", "out"):
            setattr(b, n, getattr(b, n).transpose(0, 1).contiguous().transpose(0, 1))
    elif form == "sliced":
        wide = torch.zeros(127, 8, 200, dtype=BF, device=DEV)
        wide[:, :, 3:131], wide[:, :, 131:195] = b.q, b.qr               # (queries promise their element's alignment only)
        b.q, b.qr = wide[:, :, 3:131], wide[:, :, 131:195]
    else:
        b.out = torch.full((127, 8, 131), 7.0, dtype=BF, device=DEV)[:, :, 1:129]
    a.run(), b.run()
    b.check()
    assert torch.equal(a.out, b.out) and torch.equal(a.lse, b.lse)


@pytest.mark.parametrize("lens_q,lens_k", [([1], [70000]), ([300], [70000])])
def test_offsets_past_32_bits(lens_q, lens_k):
    """Key rows 64 KiB apart: the last ones lie more than 4 GiB behind the first."""
    n = lens_k[0]
    c = Call(lens_q, lens_k, 2, 1, 64, seed=14)
    for name in ("k", "v"):
        big = torch.empty(n, 1, 32768, dtype=BF, device=DEV)[:, :, 64:128]
        big.copy_(getattr(c, name))
        setattr(c, name, big)
    c.run().check()


def test_the_same_call_gives_the_same_bits_and_lse_is_optional():
    a, b = (Call([1, 400, 30], [3000, 700, 30], 8, 2, 128, True, seed=15) for _ in range(2))
    a.run(), b.run(lse=False)
    torch.cuda.synchronize()
    assert torch.equal(a.out, b.out) and bool((b.lse == 7).all())
    first = a.out.clone()
    a.out.fill_(3.0)
    a.run()
    assert torch.equal(a.out, first)


def test_tables_of_beginnings_that_leave_the_tensors_stay_inside():
    """Beginnings past the tensors' ends are moved to them: what is there is computed, nothing outside is touched."""
    c = Call([40], [60], 4, 2, 64, seed=16)
    pypto_amd.prompt_attention(c.q, c.k, c.v, torch.tensor([0, 1 << 30], dtype=torch.int32, device=DEV),
                               torch.tensor([0, 1 << 30], dtype=torch.int32, device=DEV), c.out, c.scale, softmax_lse=c.lse)
    c.check()


def test_empty_calls():
    for lens_q, lens_k in (([0], [0]), ([0, 0], [5, 0]), ([4], [0])):
        Call(lens_q, lens_k, 4, 2, 64, seed=17).run().check()


@pytest.mark.parametrize("lens_q,lens_k", [([0], [0]), ([0, 0], [5, 0]), ([4], [0]), ([0], [9])])
def test_empty_calls_with_rope_parts(lens_q, lens_k):
    """(Empty tensors have no address.)"""
    Call(lens_q, lens_k, 4, 2, 128, True, seed=17).run().check()


def test_statistics_in_the_memory_of_an_input_are_refused():
    c = Call([20], [20], 4, 4, 128, True, seed=22, shared=False)
    for name in ("q", "qr", "out"):
        t = getattr(c, name).contiguous()
        setattr(c, name, t)
        c.lse = t.view(-1).view(torch.float32)[:80].view(20, 4)
        with pytest.raises(ValueError, match="overlap"):
            c.run()


@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("form", ["sliced", "odd_output", "sign", "many_keys"])
def test_the_larger_workgroups_in_every_form(form, rope):
    """Queries and outputs that promise their element's alignment only, a negative scale, keys divided over workgroups."""
    from pypto_amd import _C
    lens = [513, 600] if form == "many_keys" else [600]
    keys, heads = ([5000, 4900], 16) if form == "many_keys" else ([700], 48)
    plan = _C.prompt_attention_plan(len(lens), sum(lens), sum(keys), heads, heads, 128, rope, True)
    assert plan["rows_per_workgroup"] == 256 and (plan["key_splits"] > 1) == (form == "many_keys")
    c = Call(lens, keys, heads, heads, 128, rope, HALF, seed=23, scale=-0.09 if form == "sign" else None)
    if form == "sliced":
        wide = torch.zeros(600, heads, 200, dtype=HALF, device=DEV)
        wide[:, :, 3:131] = c.q
        c.q = wide[:, :, 3:131]
        if rope:
            wide[:, :, 131:195] = c.qr
            c.qr = wide[:, :, 131:195]
    elif form == "odd_output":
        c.out = torch.full((600, heads, 131), 7.0, dtype=HALF, device=DEV)[:, :, 1:129]
    c.run().check()


def test_pieces_of_keys_joined_by_their_statistics():
    """Two calls over parts of the keys, joined by softmax_lse, are the call over all of them."""
    c = Call([50], [300], 4, 2, 128, causal=False, seed=18).run()
    parts = []
    for lo, hi in ((0, 130), (130, 300)):
        p = Call([50], [hi - lo], 4, 2, 128, causal=False, seed=18)
        p.q, p.k, p.v = c.q, c.k[lo:hi], c.v[lo:hi]
        parts.append(p.run())
    torch.cuda.synchronize()
    w = torch.softmax(torch.stack([p.lse for p in parts]), dim=0)
    joined = sum(x[..., None] * p.out.float() for x, p in zip(w, parts))
    # each part is off by its rounding and its probabilities', 2 * 2^-8 of values of magnitude below 5; so is the whole
    assert float((joined - c.out.float()).abs().max()) <= 4 * 2.0 ** -8 * 1.5


def test_another_stream_and_replays_of_a_captured_call():
    c, e = (Call([1, 200, 3], [4000, 200, 900], 8, 2, 128, True, seed=19) for _ in range(2))
    cu_q, cu_k = starts(c.lens_q), starts(c.lens_k)

    def call(x):
        pypto_amd.prompt_attention(x.q, x.k, x.v, cu_q, cu_k, x.out, x.scale, query_rope=x.qr, key_rope=x.kr, softmax_lse=x.lse)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(c)
    torch.cuda.current_stream().wait_stream(side)
    call(e)
    torch.cuda.synchronize()
    assert torch.equal(c.out, e.out)
    graphs = []
    for _ in range(2):                                             # two graphs, each with a workspace of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(c)
        graphs.append(graph)
    g = torch.Generator(device=DEV).manual_seed(20)
    for _ in range(4):
        c.q.normal_(generator=g)
        e.q.copy_(c.q)
        for graph in graphs:
            c.out.fill_(5.0)
            graph.replay()
            call(e)
            torch.cuda.synchronize()
            assert torch.equal(c.out, e.out) and torch.equal(c.lse, e.lse)


def test_replays_with_other_lengths_and_on_two_streams_at_once():
    """A captured launch follows the tables of beginnings as they are when it is replayed; two graphs run side by side."""
    calls = [Call([1, 200, 3], [4000, 200, 900], 8, 2, 128, True, seed=24 + i) for i in range(2)]
    cu = [[starts(c.lens_q), starts(c.lens_k)] for c in calls]
    graphs, streams = [], [torch.cuda.Stream() for _ in calls]
    for c, (cu_q, cu_k) in zip(calls, cu):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pypto_amd.prompt_attention(c.q, c.k, c.v, cu_q, cu_k, c.out, c.scale, query_rope=c.qr, key_rope=c.kr, softmax_lse=c.lse)
        graphs.append(graph)
    for lens_q, lens_k in (([1, 200, 3], [4000, 200, 900]), ([150, 4, 50], [100, 3900, 1100]), ([0, 0, 204], [5000, 99, 1])):
        for c, (cu_q, cu_k) in zip(calls, cu):
            c.lens_q, c.lens_k = lens_q, lens_k
            cu_q.copy_(starts(lens_q))
            cu_k.copy_(starts(lens_k))
            c.out.fill_(7.0)
            c.lse.fill_(7.0)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for c in calls:
            c.check()


def plan_and_items(c, heads, kv, d, rope):
    """The call's plan, and how many (key head, row tile, piece of its keys) there are for its workgroups."""
    from pypto_amd import _C
    plan = _C.prompt_attention_plan(len(c.lens_q), sum(c.lens_q), sum(c.lens_k), heads, kv, d, rope, c.causal)
    pieces = [min(max(-(-k // plan["split_keys"]), 1), plan["key_splits"]) for k in c.lens_k]
    return plan, kv * sum(-(-q * (heads // kv) // plan["rows_per_workgroup"]) * n for q, n in zip(c.lens_q, pieces))


@pytest.mark.parametrize("d,rope,rows,heads,kv,causal,lens_q,lens_k", [
    (64, False, 128, 32, 16, True, [1236, 460, 345, 641], [9255, 1733, 564, 5608]),
    (128, False, 128, 64, 32, False, [52, 578, 26, 102], [1365, 11556, 126, 1256]),
    (128, True, 128, 32, 32, True, [2, 2, 2, 2, 1, 2, 2, 2, 2, 2, 2, 1, 1, 2, 1, 1, 1, 2, 1],
     [2876, 2377, 2364, 2929, 1586, 2645, 2547, 646, 163, 2416, 2907, 646, 1798, 214, 1816, 2506, 569, 215, 1391]),
    (128, False, 256, 128, 16, False, [91, 34, 532], [2089, 1245, 5243]),
    (128, True, 256, 128, 16, True, [100, 612], [912, 4692])])
def test_workgroups_that_take_a_second_item(d, rope, rows, heads, kv, causal, lens_q, lens_k):
    """More items of a divided launch than workgroups: one that has written its results begins anew, over the LDS that they came through."""
    c = Call(lens_q, lens_k, heads, kv, d, rope, causal=causal, seed=30)
    plan, items = plan_and_items(c, heads, kv, d, rope)
    assert plan["key_splits"] > 1 and plan["rows_per_workgroup"] == rows and items > 1.05 * plan["workgroups"]
    c.run().check()
    first = c.out.clone(), c.lse.clone()
    c.out.fill_(3.0)
    c.run()
    assert torch.equal(c.out, first[0]) and torch.equal(c.lse, first[1])


@pytest.mark.parametrize("d,rope,tiles", [(128, False, 33), (128, True, 30), (64, False, 50)])
def test_second_items_beyond_the_first_64_sequences(d, rope, tiles):
    """Sequences are looked through 64 at a time, from the first on for every item."""
    lens_k = [64 * tiles + 5] * 65
    for i in range(4):
        lens_k[7 * i + 3] = 60
    c = Call([1] * 65, lens_k, 11, 11, d, rope, seed=31)
    plan, items = plan_and_items(c, 11, 11, d, rope)
    assert plan["key_splits"] > 1 and items > plan["workgroups"]
    c.run().check()


@pytest.mark.parametrize("d,rope", FORMS)
@pytest.mark.parametrize("causal", [True, False])
def test_divided_keys_of_more_than_64_sequences(d, rope, causal):
    lens_k = [(i * i * 37) % 5000 + 2000 * (i % 3) for i in range(150)]
    lens_q = [(i * 5) % 4 for i in range(150)]
    c = Call(lens_q, lens_k, 8, 4, d, rope, causal=causal, seed=32, spare=2)
    plan, _ = plan_and_items(c, 8, 4, d, rope)
    assert plan["key_splits"] > 1 and min(lens_k) < plan["split_keys"] < max(lens_k)
    c.run().check()
