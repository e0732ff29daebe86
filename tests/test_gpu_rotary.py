"""rotary_tables and rotary_embedding against rotations in 64 bits.

Bounds: cos and sin are series in fp32 of an angle of at most pi/4 known to 2^-24 of its size; with the series' own roundings they are off by
at most 2^-22.  A rotated channel a c - b s is off by that times |a| + |b|, twice a rounding of fp32 more (2^-21 in all), and by
half a step of its type."""
import math

import pytest
import torch

import pypto_amd
from oracle import prompt_oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HALF, F32 = torch.bfloat16, torch.float16, torch.float32
LAYOUTS = ("half", "interleaved", "deinterleaved")


def normal(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def positions_of(t, far, seed=0, dtype=torch.int64):
    p = torch.randint(-far, far + 1, (t,), generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV, dtype=dtype)
    if t > 2:
        p[0], p[-1] = 0, far
    return p


def near(got, x, pos, freq, layout, offset, factor, in_place=False):
    want = prompt_oracle.turn(x, pos, freq, layout, offset, factor)
    size = prompt_oracle.turn(x.abs(), torch.zeros_like(pos), freq, "half" if layout == "half" else layout, offset, 1.0)
    n = freq.numel()
    part = size[..., offset:offset + 2 * n]
    both = (part[..., :n] + part[..., n:] if layout != "interleaved" else part[..., 0::2] + part[..., 1::2])
    both = torch.cat([both, both], -1) if layout != "interleaved" else both.repeat_interleave(2, -1)
    may = torch.zeros_like(want)
    u = torch.finfo(got.dtype).eps / 2
    may[..., offset:offset + 2 * n] = u * want[..., offset:offset + 2 * n].abs() + 2.0 ** -21 * abs(factor) * both + (2.0 ** -25 if got.dtype == HALF else 0)
    off = (got.double() - want).abs()
    assert bool((off <= may).all()), (off - may).max()


@pytest.mark.parametrize("dtype", [BF, HALF, F32])
@pytest.mark.parametrize("t,pairs,far", [(1, 32, 65536), (2, 4, 5), (33, 32, 131071), (1000, 20, 1 << 20), (17, 128, 1 << 40)])
def test_tables(dtype, t, pairs, far):
    pos = positions_of(t, far)
    freq = pypto_amd.rotary_frequencies(2 * pairs, device=DEV)
    cos, sin = (torch.full((t, 2 * pairs), 7.0, dtype=dtype, device=DEV) for _ in range(2))
    pypto_amd.rotary_tables(pos, freq, cos, sin, 1.25)
    angle = pos.double()[:, None] * freq
    u = torch.finfo(dtype).eps / 2
    for got, want in ((cos, 1.25 * angle.cos()), (sin, 1.25 * angle.sin())):
        # (angles of 2^40 are themselves known to 2^40 * 2^-53)
        may = u * want.abs() + 1.25 * (2.0 ** -22 + 2.0 * angle.abs() * 2.0 ** -53) + (2.0 ** -25 if dtype == HALF else 0)
        assert bool(((got.double() - want.repeat(1, 2)).abs() <= may.repeat(1, 2)).all())


def test_tables_of_narrow_positions_and_of_no_token():
    freq = pypto_amd.rotary_frequencies(64, device=DEV)
    pos = positions_of(100, 70000)
    a, b = (torch.zeros(2, 100, 64, dtype=BF, device=DEV) for _ in range(2))
    pypto_amd.rotary_tables(pos, freq, a[0], a[1])
    pypto_amd.rotary_tables(pos.to(torch.int32), freq, b[0], b[1])
    assert torch.equal(a, b)
    none = torch.zeros(0, 64, dtype=BF, device=DEV)
    pypto_amd.rotary_tables(pos[:0], freq, none, none.clone())


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", [BF, HALF, F32])
@pytest.mark.parametrize("t,heads,kh,dim,offset,pairs", [
    (1, 128, 1, 192, 128, 32), (1, 1, 1, 16, 0, 8), (5, 3, 2, 128, 0, 32), (9, 5, 5, 100, 4, 40), (700, 16, 1, 64, 0, 32), (3000, 3, 1, 72, 1, 32),
    (2, 7, 7, 256, 0, 128), (40, 130, 2, 97, 1, 48), (4500, 2, 1, 128, 64, 16)])
def test_rotation_out_of_place(layout, dtype, t, heads, kh, dim, offset, pairs):
    freq = pypto_amd.rotary_frequencies(2 * pairs, scaling=pypto_amd.RotaryScaling(40.0), device=DEV)
    pos = positions_of(t, 131071, seed=t)
    q, k = normal((t, heads, dim), dtype, 1), normal((t, kh, dim), dtype, 2)
    qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    pypto_amd.rotary_embedding(q, k, pos, freq, qo, ko, layout=layout, query_offset=offset, key_offset=offset, factor=0.9)
    near(qo, q, pos, freq, layout, offset, 0.9)
    near(ko, k, pos, freq, layout, offset, 0.9)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", [BF, HALF, F32])
@pytest.mark.parametrize("t,heads,dim,offset,pairs", [(3, 130, 192, 128, 32), (1500, 6, 80, 0, 40), (50, 9, 256, 0, 128), (8, 4, 24, 8, 8)])
def test_rotation_in_place_is_the_rotation_out_of_place(layout, dtype, t, heads, dim, offset, pairs):
    freq = pypto_amd.rotary_frequencies(2 * pairs, device=DEV)
    pos = positions_of(t, 131071, seed=t, dtype=torch.int32)
    both = normal((t, heads + 1, dim), dtype, 3)                   # queries and one key head, in place in one tensor
    q, k = both[:, :heads], both[:, heads:]
    want_q, want_k = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty_like(k, memory_format=torch.contiguous_format)
    pypto_amd.rotary_embedding(q, k, pos, freq, want_q, want_k, layout=layout, query_offset=offset, key_offset=offset)
    pypto_amd.rotary_embedding(q, k, pos, freq, q, k, layout=layout, query_offset=offset, key_offset=offset)
    assert torch.equal(q, want_q) and torch.equal(k, want_k)


def test_the_rope_part_of_strided_heads_alone_and_a_key_of_two_dimensions():
    freq = pypto_amd.rotary_frequencies(64, device=DEV)
    pos = positions_of(77, 9000)
    q, kv = normal((77, 16, 192), BF, 4), normal((77, 576), BF, 5)
    qo, ko = torch.zeros(77, 16, 64, dtype=BF, device=DEV), torch.zeros(77, 64, dtype=BF, device=DEV)
    pypto_amd.rotary_embedding(q[:, :, 128:], kv[:, 512:], pos, freq, qo, ko, layout="deinterleaved")
    near(qo, q[:, :, 128:], pos, freq, "deinterleaved", 0, 1.0)
    near(ko[:, None], kv[:, None, 512:], pos, freq, "deinterleaved", 0, 1.0)
    alone = torch.zeros_like(qo)
    pypto_amd.rotary_embedding(q[:, :, 128:], None, pos, freq, alone, None, layout="deinterleaved")
    assert torch.equal(alone, qo)
    pypto_amd.rotary_embedding(q[:0], None, pos[:0], freq, alone[:0].repeat(1, 1, 3), None)


def test_tables_and_rotation_are_what_the_prologs_compute():
    """Keys turned by the operator are the MLA prolog's rope keys turned with the operator's tables, to the rounding of the tables to bf16."""
    from oracle import mlap_oracle
    freq = pypto_amd.rotary_frequencies(64, device=DEV)
    pos = positions_of(50, 65536)
    cos, sin = (torch.zeros(50, 64, dtype=BF, device=DEV) for _ in range(2))
    pypto_amd.rotary_tables(pos, freq, cos, sin)
    k = normal((50, 1, 64), BF, 6)
    ko = torch.zeros_like(k)
    pypto_amd.rotary_embedding(k, None, pos, freq, ko, None, layout="deinterleaved")
    want = torch.from_numpy(mlap_oracle.rope_deinterleaved(k[:, 0].float().cpu().numpy(), cos.float().cpu().numpy(), sin.float().cpu().numpy()))
    x = k[:, 0].float().cpu().abs()
    both = (x[:, 0::2] + x[:, 1::2]).repeat(1, 2)
    # the tables' entries are off by half a step (2^-8 of at most 1), both results by half a step of theirs
    assert bool(((ko[:, 0].float().cpu() - want).abs() <= 2.0 ** -8 * both + 2.0 ** -7 * want.abs() + 2.0 ** -20).all())


def test_another_stream_and_replays():
    freq = pypto_amd.rotary_frequencies(64, device=DEV)
    pos = positions_of(64, 4096)
    q, k = normal((64, 8, 64), BF, 7), normal((64, 1, 64), BF, 8)
    got, want = (torch.zeros(64, 9, 64, dtype=BF, device=DEV) for _ in range(2))
    cos, sin, wc, ws = (torch.zeros(64, 64, dtype=BF, device=DEV) for _ in range(4))

    def call(o, c, s):
        pypto_amd.rotary_tables(pos, freq, c, s)
        pypto_amd.rotary_embedding(q, k, pos, freq, o[:, :8], o[:, 8:])

    call(want, wc, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(got, cos, sin)
    for i in range(3):
        pos.add_(i * 17)
        q.normal_()
        graph.replay()
        call(want, wc, ws)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(cos, wc) and torch.equal(sin, ws)


@pytest.mark.parametrize("which", ["tables", "rotation"])
def test_the_series_leave_out_nothing_that_fp32_shows(which):
    """Errors of fp32 cosines and sines next to pi/4, where the series' next terms are largest.  The roundings: of the angle left (2^-25,
    through the other function's at most 0.88), of its square (2^-25, through at most 1/2), of the sums inside (2^-26 times 0.62, 2^-26 / 6,
    2^-27 times 0.49 twice), of the result (2^-25), and 2e-9 for what the series leave out: below 7.7e-8 in all.  Roundings fall to both sides, a term
    left out to one: over n angles the mean error is below six times 7.7e-8 / sqrt(n) and 1e-9 for the coefficients' own roundings (2^-24 of
    z^2 / 24), while the cosine without its tenth power is 1.4e-8 off on average (x^10 / 10! from 0.7 to pi/4)."""
    t = 40000
    freq = pypto_amd.rotary_frequencies(64, device=DEV)
    pos = positions_of(t, 1 << 20, seed=11)
    if which == "tables":
        cos, sin = (torch.zeros(t, 64, device=DEV) for _ in range(2))
        pypto_amd.rotary_tables(pos, freq, cos, sin)
        cos, sin = cos[:, :32], sin[:, :32]
    else:                                                          # (1, 0) turned is (cos, sin), and no rounding more
        one = torch.zeros(t, 1, 64, device=DEV)
        one[..., :32] = 1
        pypto_amd.rotary_embedding(one, None, pos, freq, one, None)
        cos, sin = one[:, 0, :32], one[:, 0, 32:]
    angle = pos.double()[:, None] * freq
    quarter = torch.round(angle * (2 / math.pi))
    left, odd = angle - quarter * (math.pi / 2), quarter.long() % 2 == 1
    even_cos = torch.where(odd, sin, cos).double().abs() - left.cos()                  # |cos| or |sin| of the angle is the cosine of what is left
    even_sin = torch.where(odd, cos, sin).double().abs() - left.sin().abs()
    near_border = left.abs() > 0.7
    n = int(near_border.sum())
    assert n > 50000
    for off in (even_cos, even_sin):
        assert float(off.abs().max()) <= 7.7e-8 + 2.0 ** 21 * 2.0 ** -53
        assert abs(float(off[near_border].mean())) <= 6 * 7.7e-8 * n ** -0.5 + 1e-9


@pytest.mark.parametrize("which", ["tables", "rotation"])
def test_positions_at_the_ends_of_64_bits(which):
    """Angles are positions times frequencies in 64 bits, and their cosines and sines are those of that number, however far it is."""
    freq = pypto_amd.rotary_frequencies(64, device=DEV)
    pos = torch.tensor([2 ** 63 - 1, -2 ** 63, 2 ** 62 + 12345678901, -(10 ** 18), 10 ** 17 + 1, 2 ** 53 + 1, -(10 ** 15), 2 ** 50, 10 ** 14, 0], device=DEV)
    pos = torch.cat([pos, torch.randint(-2 ** 62, 2 ** 62, (500,), generator=torch.Generator().manual_seed(1)).to(DEV)])
    t = len(pos)
    if which == "tables":
        cos, sin = (torch.zeros(t, 64, device=DEV) for _ in range(2))
        pypto_amd.rotary_tables(pos, freq, cos, sin)
        cos, sin = cos[:, :32], sin[:, :32]
    else:
        one = torch.zeros(t, 1, 64, device=DEV)
        one[..., :32] = 1
        pypto_amd.rotary_embedding(one, None, pos, freq, one, None)
        cos, sin = one[:, 0, :32], one[:, 0, 32:]
    angle = pos.cpu().double()[:, None] * freq.cpu()
    # the series' 2^-23; the reduction subtracts multiples of pi/2 (known to 2^-107) below 2^63, in steps below 2^12 times 2^-53
    assert float((cos.cpu().double() - angle.cos()).abs().max()) <= 2.0 ** -22
    assert float((sin.cpu().double() - angle.sin()).abs().max()) <= 2.0 ** -22


@pytest.mark.parametrize("in_place", [True, False])
def test_offsets_past_32_bits(in_place):
    """Tokens 128 KiB apart: the last ones lie more than 8 GiB behind the first."""
    t = 70000
    freq = pypto_amd.rotary_frequencies(64, device=DEV)
    pos = positions_of(t, 131071, seed=12)
    x = torch.empty(t, 1, 65536, dtype=BF, device=DEV)[:, :, 100:164]
    x.copy_(normal((t, 1, 64), BF, 13))
    was = x.contiguous()
    out = x if in_place else torch.zeros_like(was)
    pypto_amd.rotary_embedding(x, None, pos, freq, out, None, layout="interleaved")
    near(out.contiguous(), was, pos, freq, "interleaved", 0, 1.0)
    if not in_place:
        pypto_amd.rotary_embedding(was, None, pos, freq, x, None, layout="interleaved")      # (written that far away, too)
        assert torch.equal(x, out)
