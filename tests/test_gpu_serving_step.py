"""A serving step's operators as they are used together: captured steps in which sequences draft trees, keep a path of them, end and begin; and a prompt with a
window, its first chunks through the cache, against single tokens over the same cache."""
import random

import pytest
import torch

import pypto_amd
from oracle import prompt_oracle, serving_oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, I32, I64 = torch.bfloat16, torch.int32, torch.int64
HEADS = 16


def ints(x, dtype=I32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def new_cache(rows, packed):
    # (what no token was written to is no number)
    nan = float("nan")
    parts = [torch.full((rows, 512), 100, dtype=torch.int8, device=DEV), torch.full((rows, 64), nan, dtype=BF, device=DEV), torch.full((rows, 4), nan, device=DEV)]
    return [torch.cat([parts[0], parts[1].view(torch.int8), parts[2].view(torch.int8)], dim=1).contiguous()] if packed else parts


@pytest.mark.parametrize("packed", [False, True])
def test_steps_that_draft_trees_and_keep_a_path(packed):
    b, block, columns, pages, tokens, nodes = 5, 16, 40, 60, 120, 24
    r, g = random.Random(3), torch.Generator(device=DEV).manual_seed(4)
    freq = pypto_amd.rotary_frequencies(64, device=DEV)
    scale = 192 ** -0.5
    cache = new_cache(pages * block, packed)
    write = pypto_amd.latent_cache_write_packed if packed else pypto_amd.latent_cache_write
    attend = pypto_amd.latent_attention_packed if packed else pypto_amd.latent_attention
    table = torch.full((b, columns), -1, dtype=I32, device=DEV)
    free, count = ints(r.sample(range(pages), pages)), ints([pages])
    held, lens, new_lens, parents = (torch.zeros(n, dtype=I32, device=DEV) for n in (b, b, b, tokens))
    z = lambda *s, dtype=BF: torch.zeros(s, dtype=dtype, device=DEV)  # noqa: E731
    q, q_rope, kv = z(tokens, HEADS, 512), z(tokens, HEADS, 64), z(tokens, 576)
    turned, k_rope, values, mask = z(tokens, HEADS, 64), z(tokens, 64), z(tokens, 512), z(tokens, 1, dtype=I64)
    cu_q, cu_k, positions, rows = z(b + 1, dtype=I32), z(b + 1, dtype=I32), z(tokens, dtype=I64), z(tokens, dtype=I64)
    out, lse = z(tokens, HEADS, 512), z(tokens, HEADS, dtype=torch.float32)

    def step():
        pypto_amd.cache_pages(held, lens, table, free, count, count, block)
        pypto_amd.cache_slots(new_lens, lens, table, cu_q, cu_k, positions, rows, block, parents, mask)
        pypto_amd.rotary_embedding(q_rope, kv[:, None, 512:], positions, freq, turned, k_rope[:, None], layout="deinterleaved")
        write(kv[:, :512], k_rope, rows, *cache, values)
        attend(q, turned, *cache, table, cu_q, lens, out, scale, block, tree_mask=mask, softmax_lse=lse)

    step()                                                         # (nothing: all lengths are zero)
    assert count.item() == pages
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()

    kept = [torch.zeros(0, 576, dtype=BF, device=DEV) for _ in range(b)]         # per sequence: its accepted tokens' latents and ropes
    for turn in range(8):
        counts = [r.choice((0, 1, r.randint(2, nodes))) for _ in range(b)]
        if turn == 0:
            counts = [nodes] * b
        old = [k.shape[0] for k in kept]
        held.copy_(ints(old)), lens.copy_(ints([o + n for o, n in zip(old, counts)])), new_lens.copy_(ints(counts))
        up = [[r.randint(max(-1, j - 3), j - 1) if j else -1 for j in range(n)] for n in counts]
        flat = [x for u in up for x in u]
        parents.fill_(-1)
        parents[:len(flat)] = ints(flat)
        for t in (q, q_rope, kv):
            t.copy_(torch.randn(t.shape, generator=g, device=DEV))
        out.fill_(7.0), lse.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()

        at = 0
        for i, (o, n) in enumerate(zip(old, counts)):
            if n:
                mine = slice(at, at + n)
                depth = []
                for j, x in enumerate(up[i]):
                    depth.append(depth[x] + 1 if x >= 0 else 0)
                assert positions[mine].tolist() == [o + d for d in depth]
                keys = torch.cat([kept[i], torch.cat([values[mine], k_rope[mine]], dim=1)])
                want = serving_oracle.attend(torch.cat([q[mine], turned[mine]], dim=2), keys, keys[:, :512], scale, seen(o, up[i]))
                may, may_lse = prompt_oracle.attention_bounds(BF, 576, *want)
                assert bool(((out[mine].double() - want[0]).abs() <= may).all()) and bool(((lse[mine].double() - want[1]).abs() <= may_lse).all())
            at += n
        assert bool((out[at:] == 7).all() and (lse[at:] == 7).all()) and rows[at:].tolist() == [-1] * (tokens - at)

        # a path of each tree stays: its latents move to the positions behind the kept ones, the rest's pages go back; some sequences end
        moved, accepted, at = [], [], 0
        for i, n in enumerate(counts):
            path, j = [], r.randrange(n) if n else -1
            while j >= 0:
                path.append(j)
                j = up[i][j]
            path = [at + j for j in reversed(path)]
            accepted.append(len(path)), moved.extend(path)
            kept[i] = torch.cat([kept[i], torch.cat([values[path], k_rope[path]], dim=1)])
            at += n
        with_drafts, shorter = lens.clone(), ints([k.shape[0] for k in kept])
        index = z(len(moved), dtype=I64)
        pypto_amd.cache_slots(ints(accepted), shorter, table, z(b + 1, dtype=I32), None, z(len(moved), dtype=I64), index, block)
        pypto_amd.latent_cache_write_packed(kv[moved, :512], k_rope[moved], index, *cache) if packed else \
            pypto_amd.latent_cache_write(kv[moved, :512], k_rope[moved], index, *cache)
        for i in range(b):
            if r.random() < 0.2:
                kept[i] = kept[i][:0]
        after = [k.shape[0] for k in kept]
        pypto_amd.cache_pages(with_drafts, ints(after), table, free, count, count, block)
        torch.cuda.synchronize()
        in_use = [table[i, j].item() for i, n in enumerate(after) for j in range(-(-n // block))]
        assert sorted(in_use + free[:count.item()].tolist()) == list(range(pages)), "every page is in use once, or free"


def seen(context, up):
    """[nodes, context + nodes]: what each node sees."""
    bits = torch.zeros(len(up), context + len(up), dtype=torch.bool)
    for j, x in enumerate(up):
        if x >= 0:
            bits[j] = bits[x]
        bits[j, :context] = True
        bits[j, context + j] = True
    return bits


@pytest.mark.parametrize("window,sinks", [(100, 4), (37, 0), (400, 70)])
def test_a_prompt_with_a_window_and_single_tokens_over_the_cache_it_left(window, sinks):
    g = torch.Generator(device=DEV).manual_seed(1)
    new = lambda *s, std=1.0: (std * torch.randn(s, generator=g, device=DEV)).to(BF)  # noqa: E731
    lengths, cut, block = [300, 77, 130], [256, 40, 0], 64
    freq, scale = pypto_amd.rotary_frequencies(64, device=DEV), 192 ** -0.5
    w_uk, w_uv = new(HEADS, 128, 512, std=512 ** -0.5), new(HEADS, 128, 512, std=512 ** -0.5)
    hidden_q, hidden_kv = [new(n, HEADS, 192) for n in lengths], [new(n, 576) for n in lengths]
    table = torch.full((3, 8), -1, dtype=I32, device=DEV)
    free, count, cache = ints(list(range(16))), ints([16]), new_cache(16 * block, False)
    z = lambda *s, dtype=BF: torch.zeros(s, dtype=dtype, device=DEV)  # noqa: E731

    for begin, end in (([0, 0, 0], cut), (cut, lengths)):
        ns, total = [b - a for a, b in zip(begin, end)], sum(end) - sum(begin)
        q = torch.cat([x[a:b] for x, a, b in zip(hidden_q, begin, end)])
        kv = torch.cat([x[a:b] for x, a, b in zip(hidden_kv, begin, end)])
        cu_q, cu_k, positions, rows = z(4, dtype=I32), z(4, dtype=I32), z(total, dtype=I64), z(total, dtype=I64)
        pypto_amd.cache_pages(ints(begin), ints(end), table, free, count, count, block)
        pypto_amd.cache_slots(ints(ns), ints(end), table, cu_q, cu_k, positions, rows, block)
        q_rope, k_rope = z(total, HEADS, 64), z(total, 64)
        pypto_amd.rotary_embedding(q[:, :, 128:], kv[:, None, 512:], positions, freq, q_rope, k_rope[:, None], layout="deinterleaved")
        pypto_amd.latent_cache_write(kv[:, :512], k_rope, rows, *cache)
        latent, rope = z(sum(end), 512), z(sum(end), 64)
        pypto_amd.latent_cache_read(*cache, table, cu_k, latent, rope, block)
        up = torch.matmul(latent.float(), torch.cat([w_uk, w_uv], 1).reshape(-1, 512).T.float()).to(BF).view(-1, HEADS, 256)
        out, lse = z(total, HEADS, 128), z(total, HEADS, dtype=torch.float32)
        pypto_amd.prompt_window_attention(q[:, :, :128], up[:, :, :128], up[:, :, 128:], cu_q, cu_k, out, scale, window, sinks=sinks, query_rope=q_rope, key_rope=rope,
                                          softmax_lse=lse)
        torch.cuda.synchronize()
        q0 = k0 = 0
        for n, keys in zip(ns, end):
            sees = serving_oracle.seen_keys(n, keys, window, sinks)
            for h in range(HEADS) if n else ():
                one = torch.cat([q[q0:q0 + n, h:h + 1, :128], q_rope[q0:q0 + n, h:h + 1]], dim=2)
                want = serving_oracle.attend(one, torch.cat([up[k0:k0 + keys, h, :128], rope[k0:k0 + keys]], dim=1), up[k0:k0 + keys, h, 128:], scale, sees)
                may, may_lse = prompt_oracle.attention_bounds(BF, 192, *want)
                assert bool(((out[q0:q0 + n, h:h + 1].double() - want[0]).abs() <= may).all())
                assert bool(((lse[q0:q0 + n, h:h + 1].double() - want[1]).abs() <= may_lse).all())
            q0, k0 = q0 + n, k0 + keys

    # The same queries absorbed, over the cache: keys or queries, probabilities, values and results are rounded to bf16 (2^-8 each) either way; of the
    # scores, sums of 192 products scaled to magnitude 1, the rounding of one operand is 2^-8 in the mean square.  Eight roundings: 3 % covers their sum.
    absorbed = torch.stack([q[:, h, :128].float() @ w_uk[h].float() for h in range(HEADS)], dim=1).to(BF)
    latent_out, latent_lse = z(total, HEADS, 512), z(total, HEADS, dtype=torch.float32)
    pypto_amd.latent_attention(absorbed, q_rope, *cache, table, cu_q, ints(lengths), latent_out, scale, block, window=window, sinks=sinks, softmax_lse=latent_lse)
    torch.cuda.synchronize()
    through = torch.stack([latent_out[:, h].float() @ w_uv[h].float().T for h in range(HEADS)], dim=1)
    assert float((through - out.float()).norm() / out.float().norm()) <= 0.03
    assert float((latent_lse - lse).abs().max()) <= 0.03 * float(lse.abs().max())


def test_what_is_refused_on_the_device():
    """Outputs in the memory of inputs, addresses and strides that the kernels do not take: nothing is launched."""
    z = lambda *s, dtype=BF: torch.zeros(s, dtype=dtype, device=DEV)  # noqa: E731
    within = lambda t, dtype, *s: t.reshape(-1).view(dtype)[:torch.Size(s).numel()].view(s)  # noqa: E731

    def refused(text, op, args, at=None, value=None, kind=ValueError, **kw):
        with pytest.raises(kind, match=text):
            op(*(value if i == at else x for i, x in enumerate(args)), **kw)

    pages = [z(3, dtype=I32), z(3, dtype=I32), z(3, 5, dtype=I32), z(20, dtype=I32), z(1, dtype=I32), z(1, dtype=I32), 128]
    refused("overlap", pypto_amd.cache_pages, pages, 0, within(pages[2], I32, 3))
    refused("overlap", pypto_amd.cache_pages, pages, 3, pages[2].view(-1)[3:])
    refused("overlap", pypto_amd.cache_pages, pages, 5, pages[3][:1])
    refused("block_size", pypto_amd.cache_pages, pages, 6, 0, kind=(ValueError, RuntimeError))
    slots = [z(3, dtype=I32), z(3, dtype=I32), z(3, 5, dtype=I32), z(4, dtype=I32), z(4, dtype=I32), z(9, dtype=I64), z(9, dtype=I64), 128]
    refused("overlap", pypto_amd.cache_slots, slots, 6, slots[5])
    refused("overlap", pypto_amd.cache_slots, slots, 0, within(slots[5], I32, 3))
    refused("overlap", pypto_amd.cache_slots, slots, parents=within(slots[6], I32, 9), tree_mask=z(9, 1, dtype=I64))
    refused("mask", pypto_amd.cache_slots, slots, parents=z(9, dtype=I32), tree_mask=z(9, 17, dtype=I64))
    latent = [z(6, 4, 512), z(6, 4, 64), z(256, 512, dtype=torch.int8), z(256, 64), z(256, 4, dtype=torch.float32), z(2, 3, dtype=I32), z(3, dtype=I32), z(2, dtype=I32),
              z(6, 4, 512), 0.1, 128]
    op = pypto_amd.latent_attention
    for at, shape, dtype in ((0, (6, 4, 512), BF), (5, (2, 3), I32), (6, (3,), I32), (7, (2,), I32)):
        refused("overlap", op, latent, at, within(latent[8], dtype, *shape))
    refused("overlap", op, latent, softmax_lse=within(latent[0], torch.float32, 6, 4))
    refused("overlap", op, latent, tree_mask=within(latent[8], I64, 6, 1))
    refused("exclude", op, latent, tree_mask=z(6, 1, dtype=I64), window=3)
    refused("window", op, latent, window=0)
    refused("tree_mask", op, latent, tree_mask=z(5, 1, dtype=I64))
    refused("16-byte", op, latent, 0, z(6 * 4 * 512 + 4)[4:].view(6, 4, 512), kind=(ValueError, RuntimeError))
    refused("multiples of 8", op, latent, 1, z(6, 4, 68)[:, :, :64], kind=(ValueError, RuntimeError))
    refused("GPU|device", op, latent, 7, torch.zeros(2, dtype=I32), kind=(ValueError, RuntimeError))
    prompt = [z(6, 4, 128), z(9, 2, 128), z(9, 2, 128), ints([0, 6]), ints([0, 9]), z(6, 4, 128), 0.1, 5]
    refused("overlap", pypto_amd.prompt_window_attention, prompt, 5, prompt[0])
    refused("overlap", pypto_amd.prompt_window_attention, prompt, 3, within(prompt[5], I32, 2))
    refused("window", pypto_amd.prompt_window_attention, prompt, 7, 0)


def test_calls_on_two_streams_at_once():
    """Each with its own workspace: the results of either are those it has alone."""
    from test_gpu_latent_attention import Call
    calls = [Call([30, 1, 40], [3000, 9000, 900], HEADS, words=1, seed=i, packed=i == 1) for i in range(4)]
    alone = []
    for c in calls:
        c.run()
        alone.append((c.out.clone(), c.lse.clone()))
        c.out.fill_(7.0), c.lse.fill_(7.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        for c, s in zip(calls, streams):
            with torch.cuda.stream(s):
                c.run()
    torch.cuda.synchronize()
    for c, (out, lse) in zip(calls, alone):
        c.check()
        assert torch.equal(c.out, out) and torch.equal(c.lse, lse)
