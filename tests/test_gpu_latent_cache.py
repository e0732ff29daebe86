"""latent_cache_write and latent_cache_read: every step is one IEEE operation, so codes, scales and values are equal bit for bit to numpy's,
and what is read is what the attention's oracle de-quantises."""
import math

import pytest
import torch

import pypto_amd
from oracle import mlap_oracle, prompt_oracle, sfa_oracle
from pypto_amd.synthetic import gen_block_table, pack_nope_cache

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HALF, F32 = torch.bfloat16, torch.float16, torch.float32


def cache_of(rows, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randint(-127, 128, (rows, 512), generator=g, device=DEV, dtype=torch.int8),
            torch.randn(rows, 64, generator=g, device=DEV).to(BF), 0.005 + 0.015 * torch.rand(rows, 4, generator=g, device=DEV)]


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def latents(t, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(t, 576, generator=g, device=DEV) * torch.logspace(-3, 3, t, device=DEV)[:, None]
    return x.clamp(-6e4, 6e4).to(dtype)


def expected(cache, latent, rope, index):
    codes, scales, values = prompt_oracle.quantise(latent)
    want = [c.clone().cpu() for c in cache]
    for t, row in enumerate(index.tolist()):
        if 0 <= row < want[0].shape[0]:
            want[0][row], want[1][row], want[2][row] = codes[t], rope[t].to(BF).cpu(), scales[t]
    return want, values.to(BF)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", [BF, HALF, F32])
@pytest.mark.parametrize("t", [1, 3, 32, 257])
def test_rows_written(packed, dtype, t):
    cache = cache_of(384)
    both = latents(t, dtype, t)
    both[t // 2, 128:256] = 0                                      # a group of zeros
    both[t - 1, 7] = -0.0
    index = torch.randperm(384, device=DEV)[:t]
    if t > 2:
        index[1], index[2] = -1, 384                               # rows outside the cache are skipped
    want, values = expected(cache, both[:, :512], both[:, 512:], index)
    got_values = torch.full((t, 512), 7.0, dtype=BF, device=DEV)
    if packed:
        one = pack_nope_cache(*cache)
        pypto_amd.latent_cache_write_packed(both[:, :512], both[:, 512:], index, one, got_values)
        assert same(one.cpu(), pack_nope_cache(*want))
    else:
        pypto_amd.latent_cache_write(both[:, :512], both[:, 512:], index, *cache, got_values)
        assert all(same(c.cpu(), w) for c, w in zip(cache, want))
    assert torch.equal(got_values.cpu(), values)


def test_codes_and_scales_are_the_prolog_s_but_for_a_rounding():
    """The prolog's steps are rounded once where these are rounded twice: 2 steps of fp32 apart at most, so are the scales (which round
    once more), and a code of at most 127 moves by 127 * 2^-22, that is to its neighbour, and only next to a border."""
    x = latents(200, BF, 5)[:, :512]
    codes, scales = (torch.from_numpy(v) for v in mlap_oracle.quant_rows_f32(x.float().cpu().numpy().reshape(200, 4, 128)))
    cache = cache_of(200)
    pypto_amd.latent_cache_write(x, torch.zeros(200, 64, dtype=BF, device=DEV), torch.arange(200, device=DEV), *cache)
    assert bool(((cache[2].cpu() - scales).abs() <= 2.0 ** -21 * scales).all())
    moved = (cache[0].cpu().int() - codes.reshape(200, 512).int()).abs()
    assert int(moved.max()) <= 1
    part = x.float().cpu().double().reshape(200, 4, 128) / scales.double()[..., None]
    assert bool(((part - part.floor() - 0.5).abs()[moved.reshape(200, 4, 128) > 0] <= 127 * 2.0 ** -20).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_groups_that_hold_no_number_read_as_such(bad):
    x = latents(4, BF, 6)
    x[1, 130] = bad
    cache, plain = cache_of(4), cache_of(4)
    pypto_amd.latent_cache_write(x[:, :512], x[:, 512:], torch.arange(4, device=DEV), *cache)
    y = x.clone()
    y[1, 130] = 1.0
    pypto_amd.latent_cache_write(y[:, :512], y[:, 512:], torch.arange(4, device=DEV), *plain)
    latent, rope = torch.zeros(4, 512, dtype=BF, device=DEV), torch.zeros(4, 64, dtype=BF, device=DEV)
    pypto_amd.latent_cache_read(*cache, torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([0, 4], dtype=torch.int32, device=DEV), latent, rope, 4)
    assert bool(latent[1, 128:256].isnan().all()) and int(latent.isnan().sum()) == 128
    for c, p in zip(cache, plain):                                 # the other groups do not notice
        c[1, 128:256] = 0 if c.shape[1] == 512 else c[1, 128:256]
        p[1, 128:256] = 0 if p.shape[1] == 512 else p[1, 128:256]
    assert torch.equal(cache[0], plain[0]) and torch.equal(cache[2].nan_to_num(0)[:, [0, 2, 3]], plain[2][:, [0, 2, 3]])


def test_magnitudes_at_the_ends_of_fp32():
    x = torch.zeros(6, 512, device=DEV)
    for i, top in enumerate((3.3e38, 1e-36, 5e-37, 3e-37, 1e-38, 1e-44)):
        x[i] = top * torch.linspace(-1, 1, 512, device=DEV)
    cache = cache_of(6)
    want, values = expected(cache, x, torch.zeros(6, 64, device=DEV), torch.arange(6))
    got = torch.zeros(6, 512, dtype=BF, device=DEV)
    pypto_amd.latent_cache_write(x, torch.zeros(6, 64, device=DEV), torch.arange(6, device=DEV), *cache, got)
    assert all(same(c.cpu(), w) for c, w in zip(cache, want))
    assert torch.equal(got.cpu(), values)


def test_values_in_the_place_of_the_latents_and_the_prolog_s_four_dimensions():
    x = latents(50, BF, 7)
    cache = [c.view(3, 128, 1, -1) for c in cache_of(384)]
    index = torch.arange(100, 150, device=DEV)
    _, values = expected([c.reshape(384, -1) for c in cache], x[:, :512].clone(), x[:, 512:], index)
    pypto_amd.latent_cache_write(x[:, :512], x[:, 512:], index, *cache, x[:, :512])
    assert torch.equal(x[:, :512].cpu(), values)
    pypto_amd.latent_cache_write(x[:0, :512], x[:0, 512:], index[:0], *cache)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("block_size", [128, 16, 5])
@pytest.mark.parametrize("lengths", [[1], [130, 0, 7, 1, 64, 300], [33] * 90, [0, 0, 5]])
def test_rows_read(packed, block_size, lengths):
    g = torch.Generator().manual_seed(3)
    firsts = [(i * 37) % 90 for i in range(len(lengths))]
    blocks, table = gen_block_table([a + n for a, n in zip(firsts, lengths)], block_size, g)
    blocks = max(blocks, 1)
    cache = cache_of(blocks * block_size + 3, seed=4)
    cu = torch.tensor([0] + list(torch.tensor(lengths).cumsum(0)), dtype=torch.int32)
    spare, n = 2, sum(lengths)
    latent, rope = torch.full((n + spare, 512), 7.0, dtype=BF, device=DEV), torch.full((n + spare, 64), 7.0, dtype=BF, device=DEV)
    args = (table.to(DEV), cu.to(DEV), latent, rope, block_size)
    first = torch.tensor(firsts, dtype=torch.int32, device=DEV)
    if packed:
        pypto_amd.latent_cache_read_packed(pack_nope_cache(*cache), *args, first=first)
    else:
        pypto_amd.latent_cache_read(*cache, *args, first=first)
    slots = [int(table[i, (a + j) // block_size]) * block_size + (a + j) % block_size for i, (a, m) in enumerate(zip(firsts, lengths)) for j in range(m)]
    want = sfa_oracle.dequant_kn(cache[0].cpu()[slots], cache[2].cpu()[slots])
    assert torch.equal(latent[:n].cpu(), want) and torch.equal(rope[:n].cpu(), cache[1].cpu()[slots])
    assert bool((latent[n:] == 7).all() and (rope[n:] == 7).all())


def test_pages_that_are_not_there_read_as_zeros():
    cache = cache_of(256)
    table = torch.tensor([[1, -1, 2, 0], [0, 1, 2 ** 31 - 1, -5]], dtype=torch.int32, device=DEV)
    cu = torch.tensor([1, 601, 1100], dtype=torch.int32, device=DEV)
    latent, rope = torch.full((1100, 512), 7.0, dtype=BF, device=DEV), torch.full((1100, 64), 7.0, dtype=BF, device=DEV)
    pypto_amd.latent_cache_read(*cache, table, cu, latent, rope, 128, first=torch.tensor([0, -3], dtype=torch.int32, device=DEV))
    flat = sfa_oracle.dequant_kn(cache[0].cpu(), cache[2].cpu())
    zero = torch.zeros(600, 512, dtype=BF)
    want = [torch.full((1, 512), 7.0, dtype=BF), flat[128:], zero[:256], flat[:128], zero[:88], zero[:3], flat[:256], zero[:240]]
    assert torch.equal(latent.cpu(), torch.cat(want))


def test_a_table_without_first_positions_and_strided_outputs():
    cache = cache_of(512, seed=8)
    table = torch.tensor([[3, 1], [0, 2]], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 200, 330], dtype=torch.int32, device=DEV)
    both = torch.zeros(330, 576, dtype=BF, device=DEV)
    pypto_amd.latent_cache_read(*cache, table, cu, both[:, :512], both[:, 512:], 128)
    order = torch.cat([torch.arange(384, 512), torch.arange(128, 200), torch.arange(0, 128), torch.arange(256, 258)])
    assert torch.equal(both[:, :512].cpu(), sfa_oracle.dequant_kn(cache[0].cpu()[order], cache[2].cpu()[order]))
    assert torch.equal(both[:, 512:], cache[1][order.to(DEV)])


def test_rows_past_32_bits():
    """Packed rows that lie more than 4 GiB into the cache."""
    rows = (5 << 30) // 656 // 128 * 128
    one = torch.empty(rows, 656, dtype=torch.int8, device=DEV)
    x = latents(100, BF, 9)
    index = torch.arange(rows - 100, rows, device=DEV)
    values = torch.zeros(100, 512, dtype=BF, device=DEV)
    pypto_amd.latent_cache_write_packed(x[:, :512], x[:, 512:], index, one, values)
    back, rope = torch.zeros_like(values), torch.zeros(100, 64, dtype=BF, device=DEV)
    table = torch.tensor([[rows // 128 - 1]], dtype=torch.int32, device=DEV)
    pypto_amd.latent_cache_read_packed(one, table, torch.tensor([0, 100], dtype=torch.int32, device=DEV), back, rope, 128,
                                       first=torch.tensor([28], dtype=torch.int32, device=DEV))
    assert torch.equal(back, values) and torch.equal(rope, x[:, 512:]) and torch.equal(values.cpu(), prompt_oracle.quantise(x[:, :512])[2].to(BF))


def test_replays():
    cache, other = cache_of(256, 1), cache_of(256, 1)
    x = latents(60, BF, 10)
    index = torch.randperm(256, device=DEV)[:60]
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 256], dtype=torch.int32, device=DEV)
    outs = [[torch.zeros(256, 512, dtype=BF, device=DEV), torch.zeros(256, 64, dtype=BF, device=DEV)] for _ in range(2)]

    def call(c, o):
        pypto_amd.latent_cache_write(x[:, :512], x[:, 512:], index, *c)
        pypto_amd.latent_cache_read(*c, table, cu, *o, 128)

    call(other, outs[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(cache, outs[0])
    for _ in range(3):
        x.normal_()
        graph.replay()
        call(other, outs[1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(cache + outs[0], other + outs[1]))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", [BF, HALF, F32])
def test_rows_with_the_prolog_s_steps_are_the_prolog_s(packed, dtype):
    """Codes and scales bit for bit those of the MLA prolog's oracle, which the prolog itself is held to; 3000 rows of normally distributed
    latents, of which the two-rounding steps would miss hundreds of codes in 16 bits and a fifth of the scales in any type."""
    t = 3000
    x = torch.randn(t, 576, generator=torch.Generator(device=DEV).manual_seed(12), device=DEV).to(dtype)
    x[5, :128] = 0
    codes, scales = (torch.from_numpy(v) for v in mlap_oracle.quant_rows_f32(x[:, :512].float().cpu().numpy().reshape(t, 4, 128)))
    cache, index, got = cache_of(t + 7), torch.randperm(t + 7, device=DEV)[:t], torch.zeros(t, 512, dtype=BF, device=DEV)
    want = [c.clone().cpu() for c in cache]
    want[0][index.cpu()], want[1][index.cpu()], want[2][index.cpu()] = codes.reshape(t, 512), x[:, 512:].to(BF).cpu(), scales
    assert int((prompt_oracle.quantise(x[:, :512])[1] != scales).sum()) > t // 4                # (the default's are others)
    if packed:
        one = pack_nope_cache(*cache)
        pypto_amd.latent_cache_write_packed(x[:, :512], x[:, 512:], index, one, got, prolog_steps=True)
        assert same(one.cpu(), pack_nope_cache(*want))
    else:
        pypto_amd.latent_cache_write(x[:, :512], x[:, 512:], index, *cache, got, prolog_steps=True)
        assert all(same(c.cpu(), w) for c, w in zip(cache, want))
    assert torch.equal(got.cpu(), (codes.float() * scales[..., None]).reshape(t, 512).to(BF))


def test_the_ends_of_fp32_and_what_is_no_number_with_the_prolog_s_steps():
    x = torch.zeros(9, 512, device=DEV)
    for i, top in enumerate((3.3e38, 1e38, 1e-36, 5e-37, 3.8e-37, 3e-37, 1e-44)):
        x[i] = top * torch.linspace(-1, 1, 512, device=DEV)
    x[7, 130], x[8, 300] = math.nan, -math.inf
    codes, scales, values = prompt_oracle.quantise(x, prolog_steps=True)
    cache, got = cache_of(9), torch.zeros(9, 512, dtype=BF, device=DEV)
    pypto_amd.latent_cache_write(x, torch.zeros(9, 64, device=DEV), torch.arange(9, device=DEV), *cache, got, prolog_steps=True)
    assert torch.equal(cache[0].cpu(), codes) and torch.equal(cache[2].cpu().nan_to_num(7.0), scales.nan_to_num(7.0))
    assert torch.equal(got.cpu().isnan(), values.isnan()) and torch.equal(got.cpu().nan_to_num(0), values.to(BF).nan_to_num(0))
