"""prompt_window_attention against attention in 64 bits, with element-wise bounds that count the roundings of 16-bit operands and fp32 sums
(oracle.prompt_oracle.attention_bounds)."""
import pytest
import torch

import pypto_amd
from oracle import prompt_oracle, serving_oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HALF = torch.bfloat16, torch.float16
FORMS = [(64, False), (128, False), (128, True)]


def starts(lengths):
    return torch.tensor([0] + list(torch.tensor(lengths).cumsum(0)), dtype=torch.int32, device=DEV)


class Call:
    def __init__(self, lens_q, lens_k, heads, kv, d, rope, window, sinks, dtype=BF, seed=0, spare=0, scale=None):
        g = torch.Generator(device=DEV).manual_seed(seed)
        new = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)  # noqa: E731
        self.lens_q, self.lens_k, self.window, self.sinks, self.dtype = lens_q, lens_k, window, sinks, dtype
        tq, tk = sum(lens_q) + spare, sum(lens_k) + spare
        both = new(tk, kv, 2 * d)                                  # keys and values side by side
        self.q, self.k, self.v = new(tq, heads, d), both[:, :, :d], both[:, :, d:]
        self.qr, self.kr = (new(tq, heads, 64), new(tk, 64)) if rope else (None, None)
        self.channels = d + (64 if rope else 0)
        self.scale = self.channels ** -0.5 if scale is None else scale
        self.out = torch.full((tq, heads, d), 7.0, dtype=dtype, device=DEV)
        self.lse = torch.full((tq, heads), 7.0, device=DEV)
        self.cu_q, self.cu_k = starts(lens_q), starts(lens_k)

    def run(self, lse=True):
        pypto_amd.prompt_window_attention(self.q, self.k, self.v, self.cu_q, self.cu_k, self.out, self.scale, self.window, sinks=self.sinks, query_rope=self.qr,
                                          key_rope=self.kr, softmax_lse=self.lse if lse else None)
        return self

    def check(self):
        torch.cuda.synchronize()
        g, q0, k0 = self.q.shape[1] // self.k.shape[1], 0, 0
        for i, (n, keys) in enumerate(zip(self.lens_q, self.lens_k)):
            seen = serving_oracle.seen_keys(n, keys, self.window, self.sinks)
            for h in range(self.k.shape[1]) if n else ():
                heads = slice(h * g, (h + 1) * g)
                q, k = self.q[q0:q0 + n, heads], self.k[k0:k0 + keys, h]
                if self.qr is not None:
                    q, k = torch.cat([q, self.qr[q0:q0 + n, heads]], dim=2), torch.cat([k, self.kr[k0:k0 + keys]], dim=1)
                out, lse, mean, reach, count = serving_oracle.attend(q, k, self.v[k0:k0 + keys, h], self.scale, seen)
                may, may_lse = prompt_oracle.attention_bounds(self.dtype, self.channels, out, lse, mean, reach, count)
                got, got_lse = self.out[q0:q0 + n, heads], self.lse[q0:q0 + n, heads]
                off = (got.double() - out).abs()
                assert bool((off <= may).all()), f"sequence {i}, key head {h}: {(off / may).max().item():.3g} of what it may be off by"
                some = count > 0
                assert torch.equal(torch.isneginf(got_lse), ~some)
                assert bool(((got_lse.double() - lse).abs()[some] <= may_lse[some]).all())
                assert bool((got[~some] == 0).all())
            q0, k0 = q0 + n, k0 + keys
        assert bool((self.out[q0:] == 7).all() and (self.lse[q0:] == 7).all()), "rows of no sequence were written"


@pytest.mark.parametrize("d,rope", FORMS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (63, 0), (64, 64), (65, 4), (200, 1), (300, 129), (2000, 5)])
def test_windows_around_every_tile(d, rope, window, sinks):
    lens = [1, 63, 64, 65, 130, 400]
    Call(lens, lens, 4, 2, d, rope, window, sinks, dtype=HALF if window % 2 else BF, seed=window, spare=2).run().check()


@pytest.mark.parametrize("d,rope", FORMS)
@pytest.mark.parametrize("lens_q,lens_k,heads,kv", [([900, 1300], [900, 1300], 16, 16), ([300], [5000], 8, 1), ([1] * 9, [3000] * 9, 16, 2), ([2, 600, 1], [2000, 4000, 30], 28, 4),
                                                    ([3, 5], [0, 2], 4, 4), ([1], [9000], 2, 1)])
@pytest.mark.parametrize("window,sinks", [(256, 4), (1000, 70)])
def test_keys_from_before_the_queries(d, rope, lens_q, lens_k, heads, kv, window, sinks):
    Call(lens_q, lens_k, heads, kv, d, rope, window, sinks, seed=heads).run().check()


@pytest.mark.parametrize("d,rope", [(128, False), (128, True)])
def test_the_larger_workgroups(d, rope):
    Call([1500, 700], [1500, 2700], 64, 64, d, rope, 300, 10, seed=3).run().check()


def test_many_sequences():
    lens = [(7 * i) % 90 for i in range(150)]
    Call(lens, [n + (13 * i) % 400 for i, n in enumerate(lens)], 4, 1, 128, True, 100, 3, seed=4).run().check()


def test_a_window_longer_than_everything_is_no_window():
    c = Call([300, 40], [700, 40], 8, 2, 128, True, 1 << 30, 0, seed=5).run()
    out = torch.zeros_like(c.out)
    pypto_amd.prompt_attention(c.q, c.k, c.v, c.cu_q, c.cu_k, out, c.scale, query_rope=c.qr, key_rope=c.kr)
    c.check()
    # either is off by half a step of its probabilities and one of its result, 2 * 2^-8 of sums of values that stay below 5
    assert float((out.float() - c.out.float()).abs().max()) <= 2 * 2 * 2.0 ** -8 * 5


@pytest.mark.parametrize("sinks", [0, 4, 128])
def test_keys_that_no_query_sees_may_be_left_out(sinks):
    """The first keys and those that the windows reach, without what lies between: the same results."""
    n, keys, window = 100, 4000, 500
    c = Call([n], [keys], 8, 8, 128, True, window, sinks, seed=6).run()
    kept = torch.cat([torch.arange(sinks), torch.arange(keys - (n - 1 + window), keys)]).to(DEV)
    d = Call([n], [len(kept)], 8, 8, 128, True, window, sinks, seed=6)
    d.q, d.qr, d.k, d.v, d.kr = c.q, c.qr, c.k[kept].contiguous(), c.v[kept].contiguous(), c.kr[kept].contiguous()
    d.run().check()
    c.check()


def test_the_same_call_gives_the_same_bits_and_replays_follow_the_lengths():
    c, e = (Call([1, 200, 3], [4000, 200, 900], 8, 2, 128, True, 400, 5, seed=7) for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run()
    for lens_q, lens_k in (([1, 200, 3], [4000, 200, 900]), ([150, 4, 50], [100, 3900, 1100]), ([0, 0, 204], [5000, 99, 1])):
        for x in (c, e):
            x.lens_q, x.lens_k = lens_q, lens_k
            x.cu_q.copy_(starts(lens_q)), x.cu_k.copy_(starts(lens_k))
            x.out.fill_(7.0), x.lse.fill_(7.0)
        graph.replay()
        e.run()
        c.check()
        assert torch.equal(c.out, e.out) and torch.equal(c.lse, e.lse)


def test_empty_calls():
    Call([0, 0], [10, 0], 4, 2, 128, False, 5, 1, seed=8).run().check()
    Call([0], [0], 4, 2, 128, True, 5, 1, seed=8).run().check()
