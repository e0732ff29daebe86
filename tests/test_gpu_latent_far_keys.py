"""latent_attention over sequences whose keys are numbered up to the largest number that a block table may hold, 2^31 - 16: tiles at the end, and those asked for ahead of their
use, have numbers past 31 bits.  Windows keep the keys that are seen few."""
import pytest
import torch

import pypto_amd
from oracle import prompt_oracle, serving_oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF = torch.bfloat16
MOST = 2 ** 31 - 16


def check(keys, block, columns, n, heads, window, sinks, packed=False, seed=0):
    """Pages are there for the table's first columns and its last ones, as far as they are no longer than the cache; other positions read as zeros."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    new = lambda *s: torch.randn(s, generator=g, device=DEV).to(BF)  # noqa: E731
    ends = -(-(n + window) // block) + 1
    pages = 2 * ends + 2 if block < 10 ** 6 else 1
    rows = max(pages * block if block < 10 ** 6 else 4096, 4096)
    nope, rope = torch.randint(-127, 128, (rows, 512), generator=g, device=DEV, dtype=torch.int8), new(rows, 64)
    scales = 0.005 + 0.015 * torch.rand(rows, 4, generator=g, device=DEV)
    cache = [torch.cat([nope, rope.view(torch.int8), scales.view(torch.int8)], dim=1).contiguous()] if packed else [nope, rope, scales]
    table = torch.full((1, columns), -1, dtype=torch.int32, device=DEV)
    table[0, 0] = 0
    if pages > 1:
        table[0, -ends:] = torch.arange(1, ends + 1, dtype=torch.int32, device=DEV)
    qn, qr = new(n, heads, 512), new(n, heads, 64)
    out, lse = torch.full((n, heads, 512), 7.0, dtype=BF, device=DEV), torch.full((n, heads), 7.0, device=DEV)
    cu, lens = torch.tensor([0, n], dtype=torch.int32, device=DEV), torch.tensor([keys], dtype=torch.int32, device=DEV)
    op = pypto_amd.latent_attention_packed if packed else pypto_amd.latent_attention
    op(qn, qr, *cache, table, cu, lens, out, 192 ** -0.5, block, window=window, sinks=sinks, softmax_lse=lse)
    torch.cuda.synchronize()
    # the keys that any token sees: the first ones and the last
    seen_keys = torch.cat([torch.arange(sinks, device=DEV), torch.arange(keys - (n - 1 + window), keys, device=DEV)])
    page = table[0, seen_keys // block].long()
    row = page * block + seen_keys % block
    there = ((page >= 0) & (row < rows))[:, None]
    row = torch.where(there[:, 0], row, 0)
    values = (nope[row].float().view(-1, 4, 128) * scales[row][:, :, None]).reshape(-1, 512).to(BF).double()
    k = torch.where(there, torch.cat([values, rope[row].double()], dim=1), 0.0)
    want = serving_oracle.attend(torch.cat([qn, qr], dim=2), k, k[:, :512], 192 ** -0.5, serving_oracle.seen_keys(n, k.shape[0], window, sinks))
    may, may_lse = prompt_oracle.attention_bounds(BF, 576, *want)
    assert bool(((out.double() - want[0]).abs() <= may).all()) and bool(((lse.double() - want[1]).abs() <= may_lse).all())


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("before_the_last", [0, 1, 16, 31, 32, 63, 100, 130, 1000])
def test_the_last_keys_of_the_longest_table(before_the_last, packed):
    check(MOST - before_the_last, 16, MOST // 16, 3, 16, 100, 40, packed=packed, seed=before_the_last)


@pytest.mark.parametrize("before_the_last", [0, 17, 140])
def test_many_rows(before_the_last):
    check(MOST - before_the_last, 16, MOST // 16, 700, 128, 90, 4, seed=before_the_last)


@pytest.mark.parametrize("block", [2 ** 30 - 8, 2 ** 30 - 9])
@pytest.mark.parametrize("n,heads", [(2, 16), (700, 128)])
def test_two_pages_of_the_largest_size(block, n, heads):
    for keys in (2 * block, 2 * block - 50, block + 3):
        check(keys, block, 2, n, heads, 70, 33, seed=n)
