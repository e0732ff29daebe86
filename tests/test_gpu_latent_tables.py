"""latent_attention with tables of beginnings that do not ascend: sequences that overlap ask for more rows than there are.  Nothing outside the outputs is touched, and the
next call is what it is without them."""
import pytest
import torch

from test_gpu_latent_attention import Call, DEV, ints
from test_gpu_latent_attention_wide import Wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", [Call, Wide])
@pytest.mark.parametrize("b", [3, 40, 700])
def test_sequences_that_overlap(form, b):
    n = 4 * b if b > 3 else 90
    c = form([n // b] * b, [n // b + 40] * b, 64, seed=b)
    total = c.qn.shape[0]
    good = c.cu.clone()
    around = torch.full((total + 64, 64, 512), 7.0, dtype=c.out.dtype, device=DEV)
    c.out = around[32:32 + total]
    c.out.fill_(7.0)
    for table in ([0, total] * b, [total, 0] * b, [0, total, 5] * b, [-2 ** 31, 2 ** 31 - 1] * b):
        c.cu.copy_(ints(table[:b + 1]))
        c.run()
        torch.cuda.synchronize()
        assert bool((around[:32] == 7).all() and (around[32 + total:] == 7).all())
    c.cu.copy_(good)
    c.out.fill_(7.0)
    c.lse.fill_(7.0)
    c.run().check()
