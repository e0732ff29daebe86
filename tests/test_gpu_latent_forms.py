"""Which of latent_attention's two forms takes a call, of 64 or of 128 rows to a workgroup: lengths decide, on the device, or row counts that the host knows, and never the width of the
block table.  And the cases of the form with 128 rows again, where rows are many."""
import ctypes
import inspect
import itertools

import pytest
import torch

import test_gpu_latent_attention_wide as wide_cases
from test_gpu_latent_attention import DEV, Call, ints, starts
from tests.test_serving_refusals import LIB, Latent

pytestmark = pytest.mark.gpu
cus = torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 256


def form(c):
    """Rows to a workgroup of this call: what the host chose, or what the device wrote behind the workspace's other parts."""
    lib = ctypes.CDLL(LIB)
    parts = [t.data_ptr() for t in c.cache] + [None] * (3 - len(c.cache))
    out, lse = torch.zeros_like(c.out), torch.zeros_like(c.lse)
    tq, heads = c.qn.shape[:2]
    a = Latent(c.qn.data_ptr(), c.qr.data_ptr(), *parts, c.table.data_ptr(), c.cu.data_ptr(), c.lens.data_ptr(), c.mask.data_ptr() if c.mask is not None else None,
               out.data_ptr(), lse.data_ptr(), None, 0, len(c.lens), tq, heads, c.cache[0].shape[0], c.block, c.table.shape[1], c.qn.stride(0), c.qn.stride(1), c.qr.stride(0),
               c.qr.stride(1), out.stride(0), out.stride(1), c.window or 0, c.sinks, c.mask.shape[1] if c.mask is not None else 0, c.scale, len(c.cache) == 1)
    n = ctypes.c_size_t()
    assert lib.pto_latent_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == 0
    work = torch.full((n.value,), 85, dtype=torch.uint8, device=DEV)
    a.workspace, a.workspace_bytes = work.data_ptr(), n.value
    assert lib.pto_latent_attention_launch(ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    torch.cuda.synchronize()
    rows, keys = tq * heads, c.table.shape[1] * c.block
    if c.window:
        keys = min(keys, 32 * (-(-c.sinks // 32) + -(-(c.window + 62 // heads + 1) // 32) + 1))
    many, unpadded = rows >= 3 * cus // 2 * 64, heads % 128 == 0 or rows >= 1024 * len(c.lens)
    if rows < 96 * len(c.lens) or not (many or rows * -(-keys // 32) >= 40 * cus * 64):
        return 64
    if many and unpadded:
        return 128
    word = work[-16:-12].view(torch.int32).item()
    assert word in (0, 1)
    return 128 if word else 64


@pytest.mark.parametrize("lens_q,lens_k,heads", [([1], [500], 128), ([1], [30000], 128), ([2], [9000], 128), ([1] * 8, [2000] * 8, 128), ([8], [3000], 16), ([9] * 20, [700] * 20, 16),
                                                 ([40, 3], [900, 40], 64), ([1] * 128, [60] * 128, 128)])
def test_the_table_s_width_decides_nothing(lens_q, lens_k, heads):
    want = None
    for wider in (1, 2, 4, 16, 256):
        c = Call(lens_q, lens_k, heads, seed=1, columns=(wider - 1) * -(-max(lens_k) // 128))
        assert form(c) == 64, wider
        c.run()
        torch.cuda.synchronize()
        want = want or (c.out.clone(), c.lse.clone())
        assert torch.equal(c.out, want[0]) and torch.equal(c.lse, want[1]), wider
    c.check()


@pytest.mark.parametrize("n,heads,long", [(1, 128, 330000), (8, 16, 180001), (3, 96, 200000)])
def test_lengths_decide_in_a_captured_call(n, heads, long):
    """One graph, short and long sequences in turn: either form, and back."""
    c = Call([n], [long], heads, seed=2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run()
    took = []
    for keys in (300, long, 40, 20000, long - 77, n):
        c.lens_k = [keys]
        c.lens.copy_(ints([keys]))
        c.out.fill_(7.0), c.lse.fill_(7.0)
        graph.replay()
        c.check()
        took.append(form(c))
    assert took == [64, 128 if heads != 96 else 64, 64, 64, 128 if heads != 96 else 64, 64], took       # (3 * 96 rows fill five tiles of 64, three of 128)


def test_rows_that_128_would_leave_empty_stay_with_64():
    assert form(Call([9] * 300, [40] * 300, 16, seed=3)) == 64     # 144 rows: three of 64, two of 128
    assert form(Call([8] * 400, [40] * 400, 16, seed=3)) == 128
    assert form(Call([1] * 200, [40] * 200, 128, seed=3)) == 128
    assert form(Call([1] * 100, [40] * 100, 128, seed=3)) == 64


def test_two_graphs_of_calls_that_both_forms_might_take():
    calls = [Call([8], [170000], 16, seed=4 + i, packed=i == 1) for i in range(2)]
    graphs, streams = [], [torch.cuda.Stream() for _ in calls]
    for c in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.run()
        graphs.append(graph)
    for lens in ((170000, 90), (3000, 169999), (170000, 170000)):
        for c, n in zip(calls, lens):
            c.lens_k = [n]
            c.lens.copy_(ints([n]))
            c.out.fill_(7.0), c.lse.fill_(7.0)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for c in calls:
            c.check()


class Filled(Call):
    """With one more sequence, of rows enough for the form with 128."""

    def __init__(self, lens_q, lens_k, heads, **kw):
        fill = 3 * cus // 2 * 64 // heads + 1
        super().__init__(list(lens_q) + [fill], list(lens_k) + [fill + 40], heads, **kw)

    def check(self):
        assert form(self) == 128
        super().check()


def cases():
    left_out = ("tables_of_beginnings", "strides", "replays")      # (of a fixed number of tokens: below)
    for name, f in vars(wide_cases).items():
        if name.startswith("test_") and not any(x in name for x in left_out):
            names, values = [], []
            for mark in getattr(f, "pytestmark", ()):
                names.append([x.strip() for x in mark.args[0].split(",")])
                values.append([v if len(names[-1]) > 1 else (v,) for v in mark.args[1]])
            for chosen in itertools.product(*values):
                yield pytest.param(f, {n: v for ns, vs in zip(names, chosen) for n, v in zip(ns, vs)}, id=name[5:] + "-" + "-".join(str(v) for vs in chosen for v in vs)[:60])


@pytest.mark.parametrize("case,args", cases())
def test_many_rows(case, args, monkeypatch):
    if args.get("heads") == 1:
        args = dict(args, heads=8)                             # (24577 tokens of one head would be 600 million scores)
    monkeypatch.setattr(wide_cases, "Wide", Filled)
    assert "Wide" in inspect.getsource(case)
    case(**args)


@pytest.mark.parametrize("form_of", ["heads first", "slices", "out"])
def test_strides_of_many_rows(form_of):
    c = Filled([3, 1, 40], [100, 1500, 90], 16, seed=14)
    n = c.qn.shape[0]
    if form_of == "heads first":
        c.qn, c.qr = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (c.qn, c.qr))
    elif form_of == "slices":
        both = torch.cat([c.qn, c.qr, c.qr], dim=2)
        c.qn, c.qr = both[:, :, :512], both[:, :, 512:576]
    else:
        around = torch.full((n, 16, 515), 7.0, dtype=c.out.dtype, device=DEV)
        c.out = around[:, :, 1:513]
    c.run().check()
    if form_of == "out":
        assert bool((around[:, :, 0] == 7).all() and (around[:, :, 513:] == 7).all())


def test_replays_of_many_rows():
    c = Filled([20, 1, 40], [3000, 500, 900], 16, words=1, seed=18, spare=50, columns=9)
    fill = c.lens_q[-1]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run()
    for lens_q, lens_k in (([20, 1, 40], [3000, 500, 900]), ([1, 50, 0], [2000, 500, 0]), ([0, 0, 61], [10, 10, 900]), ([20, 1, 40], [2999, 499, 870])):
        c.lens_q, c.lens_k = lens_q + [fill], lens_k + [fill + 3]
        c.cu.copy_(starts(c.lens_q))
        c.lens.copy_(ints(c.lens_k))
        c.out.fill_(7.0), c.lse.fill_(7.0)
        graph.replay()
        c.check()
