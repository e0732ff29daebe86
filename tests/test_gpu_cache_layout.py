"""cache_pages and cache_slots against their statements in Python's whole numbers, number for number."""
import random

import pytest
import torch

import pypto_amd
from oracle import serving_oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def pages_case(b, block, columns, far, seed, free, room, holes=False):
    r = random.Random(seed)
    before = [r.choice((0, r.randint(0, far), r.randint(-2, 3))) for _ in range(b)]
    after = [r.choice((0, n, n + 1, n + r.randint(0, 3 * block), r.randint(0, far), -1)) for n in before]
    numbers = list(range(b * columns + free + 5))
    r.shuffle(numbers)
    table = [[numbers.pop() if j < serving_oracle.blocks(n, block, columns) and not (holes and r.random() < 0.3) else -1 for j in range(columns)] for n in before]
    stack = [numbers.pop() for _ in range(min(free, room))] + [-7] * max(room - free, 0)
    return before, after, table, stack, min(free, room)


def check_pages(before, after, table, stack, count, block, same=True):
    args = [ints(before), ints(after), ints(table), ints(stack), ints([count])]
    left = args[4] if same else ints([-5])
    pypto_amd.cache_pages(*args, left, block)
    torch.cuda.synchronize()
    want = serving_oracle.pages(before, after, table, stack, count, block)
    assert left.item() == want
    assert args[2].tolist() == table and args[3].tolist() == stack
    assert args[0].tolist() == before and args[1].tolist() == after and (same or args[4].item() == count)


@pytest.mark.parametrize("b,block,columns,far", [(1, 128, 1, 128), (3, 1, 9, 9), (33, 128, 12, 1500), (64, 16, 70, 1100), (1023, 64, 7, 400), (1024, 64, 5, 320),
                                                 (1025, 128, 4, 512), (2500, 7, 3, 20), (5, 64, 3000, 150000)])
def test_pages(b, block, columns, far):
    check_pages(*pages_case(b, block, columns, far, b, b * columns, 3 * b * columns), block, same=b % 2 == 0)


@pytest.mark.parametrize("free,room", [(0, 500), (3, 500), (40, 45), (0, 0), (7, 7)])
def test_stacks_that_run_out_of_pages_or_of_room(free, room):
    check_pages(*pages_case(40, 32, 10, 320, free, free, room), 32)


def test_entries_without_a_page_are_not_given_back():
    check_pages(*pages_case(1500, 32, 10, 320, 5, 100, 20000, holes=True), 32)


@pytest.mark.parametrize("count", [-3, 1000])
def test_counts_outside_the_stack(count):
    before, after, table, stack, _ = pages_case(20, 32, 10, 320, 6, 30, 60)
    check_pages(before, after, table, [abs(x) for x in stack], count, 32)


def test_lengths_far_beyond_the_table():
    before, after = [2 ** 31 - 1, 5, 0, -2 ** 31], [3, 2 ** 31 - 1, 2 ** 31 - 1, 4]
    check_pages(before, after, [[9, 8, 7], [6, -1, -1], [-1] * 3, [-1] * 3], list(range(10, 30)) + [-1] * 10, 20, 2)


def tree(r, n):
    return [r.choice((-1, r.randrange(-1, j) if j else -1, j - 1)) for j in range(n)]


def check_slots(query_lens, seq_lens, block, columns, spare=0, words=0, seed=0, short=0, odd_parents=False, cu_k=True):
    r = random.Random(seed)
    b = len(query_lens)
    table = [[r.randrange(1 << 20) if r.random() < 0.95 else -1 for _ in range(columns)] for _ in range(b)]
    tokens = sum(max(n, 0) for n in query_lens) + spare - short
    parents = None
    if words:
        parents = [p for n in query_lens for p in tree(r, n)] + [3] * spare
        if odd_parents:
            parents = [r.choice((p, -5, 10 ** 6, 2 ** 31 - 1)) for p in parents]
        parents = parents[:tokens]
    new = lambda *s, dtype=torch.int64: torch.full(s, 77, dtype=dtype, device=DEV)  # noqa: E731
    cq, ck = new(b + 1, dtype=torch.int32), new(b + 1, dtype=torch.int32) if cu_k else None
    pos, row, mask = new(tokens), new(tokens), new(tokens, words) if words else None
    pypto_amd.cache_slots(ints(query_lens), ints(seq_lens), ints(table), cq, ck, pos, row, block, parents=ints(parents) if words else None, tree_mask=mask)
    torch.cuda.synchronize()
    want = serving_oracle.slots(query_lens, seq_lens, table, tokens, block, parents, words)
    assert cq.tolist() == want[0] and (not cu_k or ck.tolist() == want[1])
    assert pos.tolist() == want[2]
    assert row.tolist() == want[3]
    assert not words or mask.tolist() == want[4]


@pytest.mark.parametrize("b,lo,hi,block,columns", [(1, 1, 1, 128, 4), (32, 1, 1, 128, 40), (512, 1, 1, 16, 30), (1025, 0, 3, 64, 3), (4, 0, 9000, 128, 80), (3000, 0, 2, 7, 5),
                                                   (2, 100000, 150000, 128, 2000), (70, 0, 600, 1, 900)])
def test_slots(b, lo, hi, block, columns):
    r = random.Random(b)
    ql = [r.randint(lo, hi) for _ in range(b)]
    check_slots(ql, [n + r.randint(0, max(block * columns - n, 0)) for n in ql], block, columns, seed=b, cu_k=b % 2 == 0)


@pytest.mark.parametrize("spare", [0, 1, 300, 5000])
def test_tokens_of_no_sequence(spare):
    check_slots([5, 0, 200, 1], [50, 3, 200, 900], 64, 20, spare=spare)
    check_slots([5, 0, 20, 1], [50, 3, 200, 900], 64, 20, spare=spare, words=1)
    check_slots([0, 0], [0, 0], 64, 20, spare=spare)


def test_fewer_positions_than_tokens():
    check_slots([5, 300, 200], [50, 700, 200], 64, 20, short=230)


@pytest.mark.parametrize("lens,words", [([1], 1), ([64], 1), ([65, 3, 0, 64], 2), ([63] * 48, 1), ([200, 1, 130, 256], 4), ([1000, 1024, 30], 16), ([100, 90], 1), ([3000], 2),
                                        ([2] * 2100, 1)])
def test_trees(lens, words):
    r = random.Random(len(lens))
    check_slots(lens, [n + r.randint(0, 500) for n in lens], 64, 60, words=words, seed=words)
    check_slots(lens, [n + r.randint(0, 500) for n in lens], 64, 60, words=words, seed=words, odd_parents=True, spare=3)


def test_lengths_below_zero_beyond_the_table_and_shorter_than_the_new_tokens():
    check_slots([3, -2, 4, 2, 5], [10, 20, -5, 10 ** 6, 3], 16, 4)
    check_slots([3, -2, 4, 2, 5], [2 ** 31 - 1, 20, -5, 10 ** 6, 3], 16, 4, cu_k=False)


def test_sums_that_pass_31_bits_stay_below():
    cq, ck = (torch.zeros(4, dtype=torch.int32, device=DEV) for _ in range(2))
    pos, row = (torch.zeros(3, dtype=torch.int64, device=DEV) for _ in range(2))
    pypto_amd.cache_slots(ints([1, 1, 1]), ints([2 ** 31 - 1] * 3), torch.zeros(3, 2, dtype=torch.int32, device=DEV), cq, ck, pos, row, 16)
    torch.cuda.synchronize()
    assert cq.tolist() == [0, 1, 2, 3] and ck.tolist() == [0] + [2 ** 31 - 1] * 3 and pos.tolist() == [2 ** 31 - 2] * 3 and row.tolist() == [-1] * 3


def test_steps_replayed_with_other_lengths_and_on_another_stream():
    """A captured step -- pages, slots -- follows its lengths, and takes its pages from where the last replay left the stack."""
    r = random.Random(9)
    b, block, columns, room = 24, 16, 40, 700
    held = ints([0] * b)
    wanted, ql = ints([0] * b), ints([0] * b)
    table, stack, count = ints([[-1] * columns] * b), ints(list(range(room))), ints([room])
    cq, ck = (torch.zeros(b + 1, dtype=torch.int32, device=DEV) for _ in range(2))
    pos, row = (torch.zeros(400, dtype=torch.int64, device=DEV) for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pypto_amd.cache_pages(held, wanted, table, stack, count, count, block)
        pypto_amd.cache_slots(ql, wanted, table, cq, ck, pos, row, block)
        held.copy_(wanted)
    state = dict(held=[0] * b, table=[[-1] * columns for _ in range(b)], stack=list(range(room)), count=room)
    for step in range(6):
        new = [r.choice((0, 1, 1, r.randint(1, 30))) for _ in range(b)]
        to = [0 if r.random() < 0.1 else min(h + n, 600) for h, n in zip(state["held"], new)]
        new = [min(n, t) for n, t in zip(new, to)]
        ql.copy_(ints(new))
        wanted.copy_(ints(to))
        stream = torch.cuda.Stream() if step % 2 else torch.cuda.current_stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        state["count"] = serving_oracle.pages(state["held"], to, state["table"], state["stack"], state["count"], block)
        state["held"] = to
        want = serving_oracle.slots(new, to, state["table"], 400, block)
        assert count.item() == state["count"] and table.tolist() == state["table"] and stack.tolist() == state["stack"], step
        assert (cq.tolist(), ck.tolist(), pos.tolist(), row.tolist()) == want[:4], step
