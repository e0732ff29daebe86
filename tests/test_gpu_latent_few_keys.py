"""latent_attention with a tree mask over sequences that have fewer keys than query tokens: the tokens are the last of the keys, so the first ones have none, and key k is that of
token k + tokens - keys, as without a mask and as cache_slots numbers rows."""
import pytest
import torch

import pypto_amd
from oracle import prompt_oracle, serving_oracle
from test_gpu_latent_attention import BF, DEV, Call, ints
from test_gpu_latent_attention_wide import Wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", [Call, Wide])
@pytest.mark.parametrize("lens_q,lens_k,words", [([5, 40, 70], [3, 21, 69], 1), ([130, 9], [97, 30], 3), ([64, 100], [1, 36], 2)])
def test_each_key_is_its_token_s(form, lens_q, lens_k, words):
    c = form(lens_q, lens_k, 16, words=words, seed=sum(lens_k))
    c.mask.copy_(torch.randint(-2 ** 63, 2 ** 63 - 1, c.mask.shape, dtype=torch.int64, generator=torch.Generator().manual_seed(1)))
    c.run()
    torch.cuda.synchronize()
    begin = 0
    for i, (n, keys) in enumerate(zip(lens_q, lens_k)):
        k, v = serving_oracle.latents(c.cache, c.table[i], keys, c.block)
        words_of = c.mask[begin:begin + n].tolist()
        seen = torch.zeros(n, keys, dtype=torch.bool)
        for t in range(n):
            for j in range(n):
                key = keys - n + j
                if key >= 0:
                    seen[t, key] = j < 64 * words and bool(words_of[t][j // 64] >> (j % 64) & 1)
                    # (keys in front of the query tokens are seen by all)
            seen[t, :max(keys - n, 0)] = True
        assert torch.equal(seen, serving_oracle.seen_keys(n, keys, mask=c.mask[begin:begin + n]))
        q = torch.cat([c.qn[begin:begin + n], c.qr[begin:begin + n]], dim=2)
        want = serving_oracle.attend(q, k, v, c.scale, seen)
        may, may_lse = prompt_oracle.attention_bounds(BF, 576, *want)
        some = want[4] > 0
        assert bool(((c.out[begin:begin + n].double() - want[0]).abs() <= may).all())
        assert bool(((c.lse[begin:begin + n].double() - want[1]).abs()[some] <= may_lse[some]).all()) and torch.equal(torch.isneginf(c.lse[begin:begin + n]), ~some)
        begin += n


@pytest.mark.parametrize("form", [Call, Wide])
def test_a_causal_mask_is_no_mask(form):
    """Masks that say what is seen without them: the same bits, whether the first tokens have keys or not."""
    lens_q, lens_k = [60, 33, 50], [41, 33, 200]
    with_mask, without = (form(lens_q, lens_k, 16, words=w, seed=5) for w in (1, 0))
    rows = [(1 << (t + 1)) - 1 for n in lens_q for t in range(n)]
    with_mask.mask.copy_(ints([[serving_oracle.signed(x)] for x in rows], torch.int64))
    with_mask.run(), without.run()
    torch.cuda.synchronize()
    assert torch.equal(with_mask.lse, without.lse) and torch.equal(with_mask.out, without.out)
