"""cache_slots over deep trees and masks of many words: a node's ancestors are walked up once, whatever the number of words, and words that the walk steps over are empty."""
import pytest
import torch

import pypto_amd
from test_gpu_cache_layout import check_slots, ints

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("words", [1, 2, 3, 16])
@pytest.mark.parametrize("form", ["chain", "star", "steps", "tree"])
def test_words_that_a_walk_steps_over(form, words, monkeypatch):
    def parents(r, n):
        return {"chain": lambda j: j - 1, "star": lambda j: 0 if j else -1, "steps": lambda j: j - 150 if j >= 150 else -1,
                "tree": lambda j: r.randrange(-1, j)}[form]

    monkeypatch.setattr("test_gpu_cache_layout.tree", lambda r, n: [parents(r, n)(j) for j in range(n)])
    lens = [1, 1500, 0, 64, 65, 1024, 2]
    check_slots(lens, [n + 90 for n in lens], 64, 30, words=words, seed=words, spare=2)


def test_words_do_not_multiply_the_walk():
    """A chain of 1000 nodes: with 16 words a tenth more is stored than with one, and the walk, nearly all of the time, is the same."""
    n, times = 1000, {}
    chain, lens, table = ints([j - 1 for j in range(n)]), [ints([n]), ints([n + 50])], ints([list(range(20))])
    z = lambda *s, dtype=torch.int64: torch.zeros(s, dtype=dtype, device=DEV)  # noqa: E731
    for words in (1, 16):
        args = [*lens, table, z(2, dtype=torch.int32), None, z(n), z(n), 64, chain, z(n, words)]
        taken = []
        for _ in range(25):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            pypto_amd.cache_slots(*args)
            end.record()
            torch.cuda.synchronize()
            taken.append(begin.elapsed_time(end))
        times[words] = sorted(taken)[len(taken) // 2]
    assert times[16] < 4 * times[1], times
