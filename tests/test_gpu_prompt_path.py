"""The operators around a prompt as they are used together: a prompt in two chunks -- rotation, cache write, context read back, the
up-projection's product, attention -- and then the sparse attention's decode over the cache that the prompt left."""
import pytest
import torch

import pypto_amd
from oracle import prompt_oracle
from pypto_amd.synthetic import gen_block_table

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF = torch.bfloat16
HEADS, PAGE = 16, 128


def relative(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("packed", [True, False])
def test_a_prompt_in_two_chunks_and_the_sparse_attention_over_its_cache(packed):
    g = torch.Generator(device=DEV).manual_seed(1)
    new = lambda *s, std=1.0: (std * torch.randn(s, generator=g, device=DEV)).to(BF)  # noqa: E731
    lengths, cut = [300, 77, 130], [256, 40, 1]                    # sequences, and where their second chunks begin
    total = sum(lengths)
    blocks, table = gen_block_table(lengths, PAGE, torch.Generator().manual_seed(2))
    table = table.to(DEV)
    freq = pypto_amd.rotary_frequencies(64, scaling=pypto_amd.RotaryScaling(40.0), device=DEV)
    scale = 192 ** -0.5
    w_uk, w_uv = new(HEADS, 128, 512, std=512 ** -0.5), new(HEADS, 128, 512, std=512 ** -0.5)
    hidden_q = [new(n, HEADS, 192) for n in lengths]               # the projections' outputs
    hidden_kv = [new(n, 576) for n in lengths]
    cache = [torch.zeros(blocks * PAGE, 656, dtype=torch.int8, device=DEV)] if packed else [
        torch.zeros(blocks * PAGE, w, dtype=dt, device=DEV) for w, dt in ((512, torch.int8), (64, BF), (4, torch.float32))]
    write = pypto_amd.latent_cache_write_packed if packed else pypto_amd.latent_cache_write
    read = pypto_amd.latent_cache_read_packed if packed else pypto_amd.latent_cache_read
    outs = [torch.zeros(n, HEADS, 128, dtype=BF, device=DEV) for n in lengths]
    turned = [torch.zeros(n, HEADS, 64, dtype=BF, device=DEV) for n in lengths]
    starts = lambda ns: torch.tensor([0] + list(torch.tensor(ns).cumsum(0)), dtype=torch.int32, device=DEV)  # noqa: E731

    for begin, end in (([0, 0, 0], cut), (cut, lengths)):
        ns = [b - a for a, b in zip(begin, end)]
        q = torch.cat([x[a:b] for x, a, b in zip(hidden_q, begin, end)])
        kv = torch.cat([x[a:b] for x, a, b in zip(hidden_kv, begin, end)])
        pos = torch.cat([torch.arange(a, b, device=DEV) for a, b in zip(begin, end)])
        slot = torch.cat([table[i].long()[torch.arange(a, b, device=DEV) // PAGE] * PAGE + torch.arange(a, b, device=DEV) % PAGE
                          for i, (a, b) in enumerate(zip(begin, end))])
        q_rope, k_rope = torch.zeros(len(pos), HEADS, 64, dtype=BF, device=DEV), torch.zeros(len(pos), 64, dtype=BF, device=DEV)
        pypto_amd.rotary_embedding(q[:, :, 128:], kv[:, 512:], pos, freq, q_rope, k_rope, layout="deinterleaved")
        values = torch.zeros(len(pos), 512, dtype=BF, device=DEV)
        write(kv[:, :512], k_rope, slot, *cache, values)
        latent, rope = torch.zeros(sum(end), 512, dtype=BF, device=DEV), torch.zeros(sum(end), 64, dtype=BF, device=DEV)
        cu_k = starts(end)
        read(*cache, table, cu_k, latent, rope, PAGE)
        at = torch.cat([torch.arange(int(c) + a, int(c) + b, device=DEV) for c, a, b in zip(cu_k, begin, end)])
        assert torch.equal(latent[at], values) and torch.equal(rope[at], k_rope)    # the chunk reads as what was written
        up = torch.matmul(latent.float(), torch.cat([w_uk, w_uv], 1).reshape(-1, 512).T.float()).to(BF).view(-1, HEADS, 256)
        out = torch.zeros(len(pos), HEADS, 128, dtype=BF, device=DEV)
        lse = torch.zeros(len(pos), HEADS, device=DEV)
        pypto_amd.prompt_attention(q[:, :, :128], up[:, :, :128], up[:, :, 128:], starts(ns), cu_k, out, scale, query_rope=q_rope,
                                   key_rope=rope, softmax_lse=lse)
        torch.cuda.synchronize()
        want = prompt_oracle.attention(q[:, :, :128], up[:, :, :128], up[:, :, 128:], ns, end, scale, q_rope, rope)
        may, may_lse = prompt_oracle.attention_bounds(BF, 192, *want)
        assert bool(((out.double() - want[0]).abs() <= may).all()) and bool(((lse.double() - want[1]).abs() <= may_lse).all())
        for o, t, qt, x, a, b in zip(outs, turned, q_rope.split(ns), out.split(ns), begin, end):
            o[a:b], t[a:b] = x, qt

    # The last token of every sequence as a decode step of the sparse attention that selects all keys: queries absorbed, results through
    # w_uv.  Both ways round keys or queries, probabilities, values and results to bf16 (2^-8 each); of the scores, sums of 192 products
    # of magnitude 1 scaled to 1, the rounding of one operand is 2^-8 in the mean square.  Eight roundings: 3 % covers their sum.
    topk = max(lengths)
    last = torch.stack([x[-1] for x in hidden_q])
    absorbed = torch.einsum("thc,hcl->thl", last[:, :, :128].float(), w_uk.float()).to(BF)
    select = torch.arange(topk, device=DEV, dtype=torch.int32).repeat(3, 1)
    sparse = torch.zeros(3, 1, HEADS, 512, dtype=BF, device=DEV)
    act = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    op = pypto_amd.sparse_attention_antiquant_d if packed else pypto_amd.sparse_flash_attention_quant_d
    op(absorbed.reshape(-1, 512).contiguous(), torch.stack([t[-1] for t in turned]).reshape(-1, 64), *cache, select, table, act, sparse, HEADS, 1, scale,
       topk, PAGE, table.shape[1], None)
    torch.cuda.synchronize()
    through = torch.einsum("thl,hcl->thc", sparse[:, 0].float(), w_uv.float())
    assert total == sum(o.shape[0] for o in outs)
    assert relative(through, torch.stack([o[-1] for o in outs])) <= 0.03


def test_outputs_in_the_memory_of_positions_tables_and_indices_are_refused():
    """Nothing is launched, whichever output and index meet."""
    z = lambda *s, dtype=BF: torch.zeros(s, dtype=dtype, device=DEV)  # noqa: E731
    within = lambda t, dtype, *s: t.reshape(-1).view(dtype)[:torch.Size(s).numel()].view(s)  # noqa: E731
    I32, I64, F64, I8 = torch.int32, torch.int64, torch.float64, torch.int8

    def refused(op, args, at, value, **kw):
        with pytest.raises(ValueError, match="overlap"):
            op(*(value if i == at else x for i, x in enumerate(args)), **kw)

    freq = pypto_amd.rotary_frequencies(64, device=DEV)
    tables = [z(5, dtype=I64), freq, z(5, 64), z(5, 64)]
    turn = [z(5, 4, 80), z(5, 1, 64), z(5, dtype=I64), freq, z(5, 4, 80), z(5, 1, 64)]
    write = [z(3, 512), z(3, 64), z(3, dtype=I64), z(256, 512, dtype=I8), z(256, 64), z(256, 4, dtype=torch.float32), z(3, 512)]
    read = write[3:6] + [z(2, 3, dtype=I32), z(3, dtype=I32), z(9, 512), z(9, 64), 128]
    attend = [z(6, 4, 128), z(9, 2, 128), z(9, 2, 128), torch.tensor([0, 6], dtype=I32, device=DEV), torch.tensor([0, 9], dtype=I32, device=DEV), z(6, 4, 128), 0.1]
    for out in (2, 3):
        refused(pypto_amd.rotary_tables, tables, 0, within(tables[out], I64, 5))
        refused(pypto_amd.rotary_tables, tables, 1, within(tables[out], F64, 32))
    for out in (4, 5):
        refused(pypto_amd.rotary_embedding, turn, 2, within(turn[out], I64, 5))
        refused(pypto_amd.rotary_embedding, turn, 3, within(turn[out], F64, 32))
    for out in (3, 4, 5, 6):
        refused(pypto_amd.latent_cache_write, write, 2, within(write[out], I64, 3))
    refused(pypto_amd.latent_cache_write, write, 4, within(write[3], BF, 256, 64))
    refused(pypto_amd.latent_cache_write, write, 5, within(write[3], torch.float32, 256, 4))
    refused(pypto_amd.latent_cache_write, write, 5, within(write[4], torch.float32, 256, 4))
    for out in (5, 6):
        refused(pypto_amd.latent_cache_read, read, 3, within(read[out], I32, 2, 3))
        refused(pypto_amd.latent_cache_read, read, 4, within(read[out], I32, 3))
        refused(pypto_amd.latent_cache_read, read, 9, None, first=within(read[out], I32, 2))
    lse = z(6, 4, dtype=torch.float32)
    for at in (3, 4):
        refused(pypto_amd.prompt_attention, attend, at, within(attend[5], I32, 2))
        refused(pypto_amd.prompt_attention, attend, at, within(lse, I32, 2), softmax_lse=lse)
    for t in tables[2:] + turn[4:] + write[3:] + read[5:7] + [attend[5], lse]:
        assert not bool(t.any())
