"""latent_attention against attention in 64 bits, with element-wise bounds that count the roundings of bf16 operands and fp32 sums
(oracle.prompt_oracle.attention_bounds)."""
import math
import random

import pytest
import torch

import pypto_amd
from oracle import prompt_oracle, serving_oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF = torch.bfloat16


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def starts(lengths):
    return ints([0] + list(torch.tensor(lengths).cumsum(0)))


class Call:
    """Random latents in a cache whose other rows -- of no sequence, or behind a sequence's last -- are no numbers."""

    def __init__(self, lens_q, lens_k, heads, block=128, packed=False, window=None, sinks=0, words=0, seed=0, spare=0, scale=192 ** -0.5, columns=0, size=1.0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        r = random.Random(seed)
        new = lambda *s: (size * torch.randn(s, generator=g, device=DEV)).to(BF)  # noqa: E731
        self.lens_q, self.lens_k, self.heads, self.block, self.window, self.sinks, self.scale = lens_q, lens_k, heads, block, window, sinks, scale
        per = [-(-n // block) for n in lens_k]
        pages = sum(per) + 2
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table = torch.full((len(lens_k), max(max(per), 1) + columns), -1, dtype=torch.int32)
        rows, at = [], 0
        for i, n in enumerate(lens_k):
            self.table[i, :per[i]] = torch.tensor(order[at:at + per[i]], dtype=torch.int32)
            rows += [order[at + j // block] * block + j % block for j in range(n)]
            at += per[i]
        self.table = self.table.to(DEV)
        rows = torch.tensor(rows, dtype=torch.int64, device=DEV)
        nope = torch.full((pages * block, 512), 100, dtype=torch.int8, device=DEV)
        rope = torch.full((pages * block, 64), math.nan, dtype=BF, device=DEV)
        scales = torch.full((pages * block, 4), math.nan, device=DEV)
        nope[rows] = torch.randint(-127, 128, (len(rows), 512), generator=g, device=DEV, dtype=torch.int8)
        rope[rows], scales[rows] = new(len(rows), 64), 0.005 + 0.015 * torch.rand(len(rows), 4, generator=g, device=DEV)
        self.cache = [torch.cat([nope, rope.view(torch.int8), scales.view(torch.int8)], dim=1).contiguous()] if packed else [nope, rope, scales]
        tq = sum(lens_q) + spare
        self.qn, self.qr = new(tq, heads, 512), new(tq, heads, 64)
        self.mask = None
        if words:
            masks = []
            for n in lens_q:
                bits = []
                for j in range(n):
                    up = r.randrange(-1, j) if j else -1
                    bits.append((1 << j) | (bits[up] if up >= 0 else 0))
                    masks.append([serving_oracle.signed((bits[j] >> (64 * w)) & (2 ** 64 - 1)) for w in range(words)])
            self.mask = ints(masks + [[-1] * words] * spare, torch.int64).view(tq, words)
        self.out = torch.full((tq, heads, 512), 7.0, dtype=BF, device=DEV)
        self.lse = torch.full((tq, heads), 7.0, device=DEV)
        self.cu, self.lens = starts(lens_q), ints(lens_k)

    def parts(self):
        if len(self.cache) == 3:
            return self.cache
        c = self.cache[0]
        return [c[:, :512], c[:, 512:640].view(BF), c[:, 640:].view(torch.float32)]

    def row_of(self, i, key):
        return int(self.table[i, key // self.block]) * self.block + key % self.block

    def run(self, lse=True):
        op = pypto_amd.latent_attention if len(self.cache) == 3 else pypto_amd.latent_attention_packed
        op(self.qn, self.qr, *self.cache, self.table, self.cu, self.lens, self.out, self.scale, self.block, window=self.window, sinks=self.sinks,
           tree_mask=self.mask, softmax_lse=self.lse if lse else None)
        return self

    def want(self, i, begin, n):
        keys = self.lens_k[i]
        k, v = serving_oracle.latents(self.cache, self.table[i], keys, self.block)
        seen = serving_oracle.seen_keys(n, keys, self.window, self.sinks, self.mask[begin:begin + n] if self.mask is not None else None)
        q = torch.cat([self.qn[begin:begin + n], self.qr[begin:begin + n]], dim=2)
        return serving_oracle.attend(q, k, v, self.scale, seen)

    def check(self):
        torch.cuda.synchronize()
        begin = 0
        for i, n in enumerate(self.lens_q):
            if n:
                out, lse, mean, reach, seen = self.want(i, begin, n)
                may, may_lse = prompt_oracle.attention_bounds(BF, 576, out, lse, mean, reach, seen)
                got, got_lse = self.out[begin:begin + n], self.lse[begin:begin + n]
                off = (got.double() - out).abs()
                assert bool((off <= may).all()), f"sequence {i}: {(off / may).max().item():.3g} of what it may be off by"
                some = seen > 0
                assert torch.equal(torch.isneginf(got_lse), ~some)
                assert bool(((got_lse.double() - lse).abs()[some] <= may_lse[some]).all())
                assert bool((got[~some] == 0).all())
            begin += n
        assert bool((self.out[begin:] == 7).all() and (self.lse[begin:] == 7).all()), "rows of no sequence were written"


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("heads", [128, 16, 1, 40])
def test_lengths_around_every_tile(heads, packed):
    keys = [1, 31, 32, 33, 64, 65, 100, 127, 128, 129]
    Call([1] * 10, keys, heads, packed=packed, seed=heads).run().check()
    Call([1, 5, 3, 2, 64, 7, 1, 4, 0, 2], keys, heads, packed=packed, seed=heads + 1, spare=3).run().check()


@pytest.mark.parametrize("block", [1, 2, 5, 16, 48, 64, 128, 1024])
def test_pages_of_all_sizes(block):
    Call([3, 1, 9], [200, 77, 1030], 16, block=block, packed=block % 2 == 0, seed=block).run().check()


@pytest.mark.parametrize("lens_q,lens_k,heads", [([1], [30000], 16), ([2], [9000], 128), ([1], [5000], 1), ([40, 1, 30], [40, 8000, 3000], 128), ([300], [300], 128), ([1] * 70, [900] * 70, 16),
                                                 ([1] * 200, [40] * 200, 8), ([130] * 3, [130, 400, 2000], 64)])
def test_keys_divided_and_joined(lens_q, lens_k, heads):
    Call(lens_q, lens_k, heads, seed=len(lens_q)).run().check()


@pytest.mark.parametrize("lens_q,lens_k", [([1], [1]), ([8], [3000]), ([63, 1, 17, 64], [63, 500, 1017, 95]), ([64, 64], [64, 100]), ([31] * 5, [40, 63, 64, 65, 2000])])
@pytest.mark.parametrize("heads", [128, 16])
def test_trees(lens_q, lens_k, heads):
    Call(lens_q, lens_k, heads, words=1, seed=heads, packed=heads == 16, spare=2).run().check()


@pytest.mark.parametrize("words,lens_q,lens_k", [(2, [128, 65], [1128, 70]), (4, [200, 256, 3], [300, 256, 90]), (16, [700], [801])])
def test_trees_of_more_words(words, lens_q, lens_k):
    Call(lens_q, lens_k, 16, words=words, seed=words).run().check()


def test_masks_that_leave_rows_empty_and_nodes_beyond_the_mask():
    c = Call([40, 70, 5], [40, 75, 5], 16, words=1, seed=3)
    c.mask[::3] = 0
    c.run().check()                                                # (some rows see nothing at all, the second sequence's the context)
    c.mask[:] = -1
    c.run().check()                                                # nodes 64 .. 69 are beyond the mask and seen by none


def test_any_mask_whether_a_tree_or_not():
    c = Call([64, 33], [300, 33], 40, words=1, seed=4)
    c.mask.copy_(torch.randint(-2 ** 63, 2 ** 63 - 1, c.mask.shape, dtype=torch.int64))
    c.run().check()


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 4), (32, 0), (33, 33), (64, 100), (500, 4), (1000, 0), (5000, 16), (100, 5000)])
@pytest.mark.parametrize("heads", [128, 8])
def test_windows(window, sinks, heads):
    Call([1, 4, 70, 1], [2000, 999, 300, 20], heads, window=window, sinks=sinks, seed=window, packed=heads == 8).run().check()


@pytest.mark.parametrize("window,sinks", [(700, 4), (64, 0), (3000, 128)])
def test_windows_of_whole_prompts_and_of_many_sequences(window, sinks):
    Call([600], [1600], 16, window=window, sinks=sinks, seed=1).run().check()
    Call([1, 2, 1] * 30, [50, 4000, 1500] * 30, 16, window=window, sinks=sinks, seed=2, packed=True).run().check()


def test_more_than_64_sequences_some_of_them_empty():
    r = random.Random(5)
    lens_q = [r.choice((0, 0, 1, 2, 30)) for _ in range(300)]
    Call(lens_q, [n + r.choice((0, 1, 200, 700)) for n in lens_q], 16, seed=5).run().check()
    Call(lens_q, [n + r.choice((0, 1, 200, 700)) for n in lens_q], 16, window=50, sinks=2, seed=6).run().check()


def test_more_tokens_than_keys_and_no_keys():
    Call([5, 3, 2], [3, 0, 1], 16, seed=7).run().check()
    Call([5, 3, 2], [3, 0, 1], 16, window=2, sinks=1, seed=7).run().check()
    c = Call([5, 3, 2], [5, 0, 2], 16, words=1, seed=7)
    c.run().check()


@pytest.mark.parametrize("scale", [0.0, -192 ** -0.5, 1e-30, 0.5])
def test_scales(scale):
    Call([1, 9], [300, 1000], 16, scale=scale, seed=8).run().check()


@pytest.mark.parametrize("way", ["rising", "falling", "one"])
def test_scores_that_move_the_maximum(way):
    """Scores whose maximum grows from tile to tile, falls, or jumps once."""
    c = Call([2], [2000], 16, seed=9)
    nope, rope, scales = c.cache
    at = torch.arange(2000, device=DEV)
    rows = c.table[0].long()[at // c.block] * c.block + at % c.block
    size = {"rising": at / 100.0, "falling": 20 - at / 100.0, "one": torch.where(at == 1500, 30.0, 0.1)}[way]
    rope[rows] = (size[:, None] * torch.ones(64, device=DEV)).to(BF)
    c.qr.fill_(1.0)
    c.run().check()


@pytest.mark.parametrize("form", ["window", "tree", "causal"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, 1e38])
def test_what_a_row_does_not_see_may_hold_anything(form, bad):
    """A key that some rows do not see, with a scale that is no number or too large: the others are what they would be without it."""
    lens_q, lens_k = [6, 3], [150, 400]
    kw = dict(window=dict(window=20, sinks=3), tree=dict(words=1), causal={})[form]
    c, d = (Call(lens_q, lens_k, 16, seed=10, **kw) for _ in range(2))
    key = {"window": 120, "tree": 146, "causal": 147}[form]
    row = c.row_of(0, key)
    c.cache[2][row, 2] = bad
    c.cache[1][row, 5] = bad
    c.run(), d.run().check()
    torch.cuda.synchronize()
    seen = serving_oracle.seen_keys(6, 150, c.window, c.sinks, c.mask[:6] if c.mask is not None else None)[:, key].to(DEV)
    assert bool((~seen).any()) and (form == "window" or bool(seen.any()))
    assert torch.equal(c.out[:6][~seen], d.out[:6][~seen]) and torch.equal(c.out[6:], d.out[6:]) and torch.equal(c.lse[:6][~seen], d.lse[:6][~seen])
    assert not bool(torch.isfinite(c.out[:6][seen]).any())


def test_positions_without_a_page_read_as_zeros():
    c = Call([2, 3], [400, 700], 16, block=64, seed=11)
    c.table[0, 2] = -1
    c.table[1, 0] = 10 ** 6
    c.table[1, 5] = 2 ** 31 - 1
    c.run().check()


def test_lengths_beyond_the_table_are_the_table_s():
    c, d = (Call([2, 3], [384, 700], 16, seed=12, columns=n) for n in (0, 0))
    c.table, d.table = c.table[:, :3].contiguous(), d.table[:, :3].contiguous()
    c.lens.copy_(ints([384, 2 ** 31 - 1]))
    d.lens.copy_(ints([384, 384]))
    c.run(), d.run()
    torch.cuda.synchronize()
    assert torch.equal(c.out, d.out)


def test_tables_of_beginnings_that_leave_the_tensors_stay_inside():
    c = Call([3, 4, 2], [50, 60, 70], 16, seed=13)
    for table in ([-5, 3, 100, 7], [9, 3, 2, 1], [0, 2 ** 31 - 1, -2 ** 31, 9]):
        c.cu.copy_(ints(table))
        c.run()
        torch.cuda.synchronize()


@pytest.mark.parametrize("form", ["heads first", "slices", "out"])
def test_strides(form):
    c = Call([3, 1, 40], [100, 1500, 90], 16, seed=14)
    if form == "heads first":                                      # as a batched product over heads leaves them
        c.qn = c.qn.transpose(0, 1).contiguous().transpose(0, 1)
        c.qr = c.qr.transpose(0, 1).contiguous().transpose(0, 1)
    elif form == "slices":
        both = torch.cat([c.qn, c.qr, c.qr], dim=2)
        c.qn, c.qr = both[:, :, :512], both[:, :, 512:576]
    else:
        wide = torch.full((44, 16, 515), 7.0, dtype=BF, device=DEV)
        c.out = wide[:, :, 1:513]
    c.run().check()
    if form == "out":
        assert bool((wide[:, :, 0] == 7).all() and (wide[:, :, 513:] == 7).all())


def test_the_same_call_gives_the_same_bits_and_lse_is_optional():
    c, d = (Call([40, 1], [900, 7000], 128, words=1, seed=15) for _ in range(2))
    c.run()
    d.run(lse=False)
    torch.cuda.synchronize()
    assert torch.equal(c.out, d.out) and bool((d.lse == 7).all())


def test_empty_calls():
    Call([0, 0], [10, 0], 16, seed=16).run().check()
    Call([0], [100], 128, words=1, seed=16).run().check()


def test_cache_rows_past_32_bits():
    """A cache of more than 4 GiB: rows at its far end."""
    block, pages = 128, 70000                                      # 8.96 M rows: 4.6 GB of latents
    c = Call([2, 3], [300, 500], 16, block=block, seed=17)
    big = [torch.zeros(pages * block, w, dtype=t.dtype, device=DEV) for t, w in zip(c.cache, (512, 64, 4))]
    used = c.cache[0].shape[0]
    for b, t in zip(big, c.cache):
        b[-used:] = t
    c.cache = big
    c.table = torch.where(c.table >= 0, c.table + pages - used // block, c.table)
    c.run().check()


def test_another_stream_and_replays_with_other_lengths_and_two_graphs():
    calls = [Call([20, 1, 40], [3000, 500, 900], 16, words=1, seed=18 + i, packed=i == 1, columns=10) for i in range(2)]
    graphs, streams = [], [torch.cuda.Stream() for _ in calls]
    for c in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.run()
        graphs.append(graph)
    for lens_q, lens_k in (([20, 1, 40], [3000, 500, 900]), ([1, 50, 0], [2000, 500, 0]), ([0, 0, 61], [10, 10, 900]), ([20, 1, 40], [2999, 499, 870])):
        for c in calls:
            c.lens_q, c.lens_k = lens_q, lens_k
            c.cu.copy_(starts(lens_q))
            c.lens.copy_(ints(lens_k))
            c.out.fill_(7.0)
            c.lse.fill_(7.0)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for c in calls:
            c.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls[0].run()
    side.synchronize()
    calls[0].check()
