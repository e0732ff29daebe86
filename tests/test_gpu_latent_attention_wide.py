"""latent_attention where sequences fill 128 rows and the table has room for many keys: the form with 128 rows to a workgroup, at the sizes and masks where it can go
wrong.  Statements and bounds are those of the other form's tests."""
import ctypes
import math
import random

import pytest
import torch

from oracle import serving_oracle
from test_gpu_latent_attention import BF, DEV, Call, ints, starts
from tests.test_serving_refusals import LIB, Latent

pytestmark = pytest.mark.gpu


class Wide(Call):
    """Room in the table for as many keys as the form asks for."""

    def __init__(self, lens_q, lens_k, heads, block=128, window=None, **kw):
        rows = (sum(lens_q) + kw.get("spare", 0)) * heads
        super().__init__(lens_q, lens_k, heads, block=block, window=window,
                         columns=-(-32 * 41 * 256 * 64 // (rows * block)) if window is None else -(-(window + kw.get("sinks", 0)) // block) + 1, **kw)
        a = Latent(*([4096] * 8), None, 4096, None, 4096, 1 << 40, len(lens_q), self.qn.shape[0], heads, 1000, block, self.table.shape[1], *([512] * 6), window or 0,
                   self.sinks, 0, 0.1, 0)
        n = ctypes.c_size_t()
        assert ctypes.CDLL(LIB).pto_latent_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == 0
        cus = torch.cuda.get_device_properties(0).multi_processor_count
        assert n.value >= 2 * cus * 128 * 514 * 4, "not the form with 128 rows"


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("heads", [128, 16, 40])
def test_lengths_around_every_tile(heads, packed):
    keys = [1, 31, 32, 33, 64, 65, 100, 127, 128, 129]
    n = 96 * 10 // heads // 10 + 1
    Wide([n] * 10, [max(k, n) for k in keys], heads, packed=packed, seed=heads).run().check()
    Wide([1, 5, 3, 2, 64, 7, 1, 4, 0, 2], [1, 31, 32, 33, 64, 65, 100, 127, 128, 129], heads, packed=packed, seed=heads + 1, spare=3).run().check()


@pytest.mark.parametrize("block", [1, 2, 5, 12, 16, 48, 64, 100, 1024])
def test_pages_of_all_sizes(block):
    Wide([30, 11, 9], [200, 77, 1030], 16, block=block, packed=block % 2 == 0, seed=block).run().check()


@pytest.mark.parametrize("lens_q,lens_k,heads", [([8], [30000], 16), ([2], [9000], 128), ([40, 1, 30], [40, 8000, 3000], 128), ([300], [300], 128),
                                                 ([8] * 70, [900] * 70, 16), ([130] * 3, [130, 400, 2000], 64), ([400], [9000], 1)])
def test_keys_divided_and_joined(lens_q, lens_k, heads):
    Wide(lens_q, lens_k, heads, seed=len(lens_q)).run().check()


@pytest.mark.parametrize("lens_q,lens_k", [([8], [3000]), ([63, 1, 17, 64], [63, 500, 1017, 95]), ([64, 64], [64, 100]), ([31] * 5, [40, 63, 64, 65, 2000])])
@pytest.mark.parametrize("heads", [128, 16])
def test_trees(lens_q, lens_k, heads):
    Wide(lens_q, lens_k, heads, words=1, seed=heads, packed=heads == 16, spare=2).run().check()


@pytest.mark.parametrize("words,lens_q,lens_k", [(2, [128, 65], [1128, 70]), (4, [200, 256, 3], [300, 256, 90]), (16, [700], [801])])
def test_trees_of_more_words(words, lens_q, lens_k):
    Wide(lens_q, lens_k, 16, words=words, seed=words).run().check()


def test_any_mask_empty_rows_and_nodes_beyond_the_mask():
    c = Wide([40, 70, 5], [40, 75, 5], 16, words=1, seed=3)
    c.mask.copy_(torch.randint(-2 ** 63, 2 ** 63 - 1, c.mask.shape, dtype=torch.int64))
    c.mask[::3] = 0
    c.run().check()
    c.mask[:] = -1
    c.run().check()


@pytest.mark.parametrize("window,sinks", [(1, 0), (31, 4), (33, 33), (64, 100), (500, 4), (1000, 0), (100, 5000)])
def test_windows(window, sinks):
    """Enough rows, as the keys that a row tile can see are few."""
    tiles = -(-sinks // 32) + -(-(window + 1) // 32) + 1           # (of 64 rows, 64 heads: one token)
    n = 41 * 256 // tiles + 64
    Wide([n // 2, n - n // 2], [n // 2 + 700, n - n // 2], 64, window=window, sinks=sinks, seed=window, packed=window % 2 == 0).run().check()


def test_more_than_256_sequences_some_of_them_empty():
    r = random.Random(5)
    lens_q = [r.choice((0, 0, 1, 2, 30)) for _ in range(600)]
    assert sum(lens_q) * 16 >= 96 * 600
    Wide(lens_q, [n + r.choice((0, 1, 200, 700)) for n in lens_q], 16, seed=5).run().check()


def test_more_tokens_than_keys_and_no_keys():
    Wide([50, 30, 20], [3, 0, 19], 16, seed=7).run().check()
    Wide([0, 0, 40], [5, 0, 0], 16, words=1, seed=7).run().check()


@pytest.mark.parametrize("scale", [0.0, -192 ** -0.5, 1e-30, 0.5])
def test_scales(scale):
    Wide([10, 9], [300, 1000], 16, scale=scale, seed=8).run().check()


@pytest.mark.parametrize("way", ["rising", "falling", "one"])
def test_scores_that_move_the_maximum(way):
    c = Wide([8], [2000], 16, seed=9)
    at = torch.arange(2000, device=DEV)
    rows = c.table[0].long()[at // c.block] * c.block + at % c.block
    size = {"rising": at / 100.0, "falling": 20 - at / 100.0, "one": torch.where(at == 1500, 30.0, 0.1)}[way]
    c.cache[1][rows] = (size[:, None] * torch.ones(64, device=DEV)).to(BF)
    c.qr.fill_(1.0)
    c.run().check()


@pytest.mark.parametrize("form", ["tree", "causal"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, 1e38])
def test_what_a_row_does_not_see_may_hold_anything(form, bad):
    kw = dict(tree=dict(words=1), causal={})[form]
    c, d = (Wide([6, 30], [150, 400], 16, seed=10, **kw) for _ in range(2))
    key = {"tree": 146, "causal": 147}[form]
    row = c.row_of(0, key)
    c.cache[2][row, 2] = bad
    c.cache[1][row, 5] = bad
    c.run(), d.run().check()
    torch.cuda.synchronize()
    seen = serving_oracle.seen_keys(6, 150, c.window, c.sinks, c.mask[:6] if c.mask is not None else None)[:, key].to(DEV)
    assert bool((~seen).any()) and bool(seen.any())
    assert torch.equal(c.out[:6][~seen], d.out[:6][~seen]) and torch.equal(c.out[6:], d.out[6:]) and torch.equal(c.lse[:6][~seen], d.lse[:6][~seen])
    assert not bool(torch.isfinite(c.out[:6][seen]).any())


def test_positions_without_a_page_read_as_zeros():
    c = Wide([20, 30], [400, 700], 16, block=64, seed=11)
    c.table[0, 2] = -1
    c.table[1, 0] = 10 ** 6
    c.table[1, 5] = 2 ** 31 - 1
    c.run().check()


def test_tables_of_beginnings_that_leave_the_tensors_stay_inside():
    c = Wide([30, 40, 20], [50, 60, 70], 16, seed=13)
    for table in ([-5, 3, 100, 7], [9, 3, 2, 1], [0, 2 ** 31 - 1, -2 ** 31, 90]):
        c.cu.copy_(ints(table))
        c.run()
        torch.cuda.synchronize()


@pytest.mark.parametrize("form", ["heads first", "slices", "out"])
def test_strides(form):
    c = Wide([3, 1, 40], [100, 1500, 90], 16, seed=14)
    if form == "heads first":
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


def test_both_forms_give_what_the_other_does():
    """A table with more columns, the same sequences: either is within its bounds of the statement, and lse is optional to both."""
    c, d = Wide([40, 9], [900, 7000], 128, words=1, seed=15), Call([40, 9], [900, 7000], 128, words=1, seed=15)
    e = Wide([40, 9], [900, 7000], 128, words=1, seed=15)
    c.run().check(), d.run().check()
    e.run(lse=False)
    torch.cuda.synchronize()
    assert torch.equal(c.out, e.out) and bool((e.lse == 7).all())


def test_replays_with_other_lengths_and_two_graphs():
    calls = [Wide([20, 1, 40], [3000, 500, 900], 16, words=1, seed=18 + i, packed=i == 1) for i in range(2)]
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
