"""latent_attention with tables of beginnings that leave the tensors, do not ascend or overlap: nothing around the outputs is touched, neither results nor statistics, and the next call is what it
is without them."""
import pytest
import torch

from test_gpu_latent_attention import DEV, Call, ints
from test_gpu_latent_attention_wide import Wide
from test_gpu_latent_forms import Filled

pytestmark = pytest.mark.gpu
BORDER = 200


def guarded(c):
    """The call's outputs inside larger tensors, and a check of what is around them."""
    n, heads = c.lse.shape
    out = torch.full((n + 2 * BORDER, heads, 512), 7.0, dtype=c.out.dtype, device=DEV)
    lse = torch.full((n + 2 * BORDER, heads), 7.0, device=DEV)
    c.out, c.lse = out[BORDER:BORDER + n], lse[BORDER:BORDER + n]

    def check():
        torch.cuda.synchronize()
        for t in (out, lse):
            assert bool((t[:BORDER] == 7).all() and (t[BORDER + n:] == 7).all())
    return check


@pytest.mark.parametrize("form", [Call, Wide, Filled])
@pytest.mark.parametrize("kw", [{}, dict(words=1), dict(window=30, sinks=5)])
def test_nothing_around_the_outputs_is_touched(form, kw):
    lens_q, lens_k = [30, 40, 20], [50, 600, 70]
    if form is Wide and "window" in kw:
        lens_q, lens_k = [3000, 4000, 2000], [3050, 4600, 2070]    # (rows enough for that form)
    c = form(lens_q, lens_k, 16, seed=13, **kw)
    around = guarded(c)
    good, n = c.cu.clone(), c.qn.shape[0]
    most, least = 2 ** 31 - 1, -2 ** 31
    for table in ([-5, 3, 100, 7], [9, 3, 2, 1], [0, most, least, n], [n, n, n, n], [n + 1, n + 5, most, most], [least, -1, 0, n + 3], [0, 0, n + 100, n + 100], [n - 1, most, 0, n]):
        c.cu.copy_(ints((table + [table[-1]])[:len(c.cu)]))
        c.run()
        around()
    c.cu.copy_(good)
    c.out.fill_(7.0), c.lse.fill_(7.0)
    c.run().check()
    around()


@pytest.mark.parametrize("form", [Call, Filled])
def test_lengths_that_are_no_lengths(form):
    """Lengths of keys below zero or beyond the table, and none at all: inside the outputs rows of such sequences see what there is."""
    c = form([30, 40, 20], [50, 600, 70], 16, seed=14)
    around = guarded(c)
    good = c.lens.clone()
    for lens in ([-1, -2 ** 31, 2 ** 31 - 1], [0, 0, 0], [2 ** 31 - 1] * 3, [1, 10 ** 9, -7]):
        c.lens[:3].copy_(ints(lens))
        c.run()
        around()
    c.lens.copy_(good)
    c.out.fill_(7.0), c.lse.fill_(7.0)
    c.run().check()
    around()
