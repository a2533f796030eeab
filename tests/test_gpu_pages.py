"""The page tables of a cache in pages against a walk over the rows: every number is equal."""
import random

import pytest
import torch

from oracle import page_oracle as PO

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import slotpage_hip as P

ints = lambda x: torch.tensor(x, dtype=torch.int32)


class State:
    """The GPU's state and the walk's, the table a strided view between columns that nobody may touch."""

    def __init__(self, R, M, pages, page, seed=0, free=None):
        g = torch.Generator().manual_seed(seed)
        order = torch.randperm(pages, generator=g).to(torch.int32)
        self.page, self.R, self.M = page, R, M
        self.wide = torch.full((R, M + 3), 77, dtype=torch.int32, device="cuda")
        self.table = self.wide[:, 1: M + 1]
        self.table.fill_(-1)
        self.lens = torch.zeros(R, dtype=torch.int32, device="cuda")
        self.free = torch.cat((ints([pages if free is None else free]), order)).cuda()
        self.pull()

    def pull(self):
        self.h = [self.lens.tolist(), self.table.cpu().tolist(), self.free.tolist()]

    def same(self):
        torch.cuda.synchronize()
        lens, table, free = self.h
        assert self.lens.tolist() == lens and self.table.cpu().tolist() == table and self.free.tolist() == free
        edge = self.wide.cpu()
        assert bool((edge[:, 0] == 77).all()) and bool((edge[:, self.M + 1:] == 77).all())

    def extend(self, new, N):
        step = P.page_extend(ints(new).cuda(), self.lens, self.table, self.free, self.page, N)
        starts, ends, slots, pos = PO.extend(new, *self.h, self.page, N)
        self.same()
        assert step.starts.tolist() == starts and step.ends.tolist() == ends and step.slots.tolist() == slots and step.pos.tolist() == pos
        assert step.slots.dtype == torch.int64 and step.pos.dtype == step.starts.dtype == step.ends.dtype == torch.int32
        return step

    def trim(self, keep):
        P.page_trim(ints(keep).cuda(), self.lens, self.table, self.free, self.page)
        PO.trim(keep, *self.h, self.page)
        self.same()


@pytest.mark.parametrize("R,M,page,pages,top", [
    (1, 1, 16, 1, 16), (3, 4, 16, 9, 30), (64, 20, 16, 300, 90), (65, 3, 4096, 100, 5000), (200, 40, 32, 900, 300), (1000, 6, 16, 2000, 40),
    (1025, 4, 64, 700, 100), (3000, 3, 16, 2500, 20)])
def test_many_steps(R, M, page, pages, top):
    """Sequences that grow, are cut and freed, with pages that run out and rows that fill up; the batch is at times too small."""
    print("pages", R, M, page, pages, flush=True)
    rng = random.Random(R * 31 + page)
    s = State(R, M, pages, page)
    for step in range(12 if R < 500 else 5):
        kind = rng.choice(["one", "some", "many"])
        new = [rng.choice([0, -5, 1, 1, 1] if kind == "one" else [0, 1, rng.randrange(1, top)] if kind == "some" else [rng.randrange(top)])
               for _ in range(R)]
        total = sum(max(x, 0) for x in new)
        s.extend(new, rng.choice([total, total + 7, max(0, total - 3), total // 2]))
        if step % 3 == 2:
            s.trim([rng.choice([0, x, x // 2, x + 5, -1, max(0, x - 1)]) for x in s.h[0]])


def test_one_row_takes_thousands_of_pages_and_gives_them_back():
    s = State(2, 5000, 9000, 16, seed=3)
    s.extend([70000, 3], 70003)                          # more tokens than the rows' workgroup writes itself
    s.extend([1, 9990], 9991)
    s.trim([17, 9993])
    s.extend([9000, 0], 9000)
    s.trim([0, 0])
    assert s.h[2][0] == 9000


def test_trimming_to_the_lengths_before_undoes_an_extension():
    s = State(40, 10, 300, 16, seed=5)
    rng = random.Random(1)
    s.extend([rng.randrange(100) for _ in range(40)], 4000)
    before = [list(x) for x in (s.h[0], s.h[2])] + [[list(r) for r in s.h[1]]]
    s.extend([rng.randrange(9) for _ in range(40)], 400)
    assert s.h[2] != before[1]
    s.trim(before[0])
    assert [s.h[0], s.h[2], s.h[1]] == before


def test_a_row_that_waits_is_not_overtaken_but_by_rows_that_need_no_page():
    s = State(4, 8, 5, 16, seed=7)
    s.extend([10, 16, 0, 0], 26)
    step = s.extend([4, 60, 1, 16], 81)                  # the second asks for 4 pages of 3, the third and fourth behind it for 1 each
    assert step.ends.tolist() == [14, 0, 0, 0] and s.h[2][0] == 3
    assert step.starts.tolist() == [0, 4, 64, 65, 81] and set(step.slots.tolist()[4:]) == {-1}


def test_no_tokens_no_pages():
    s = State(5, 2, 0, 16)
    s.extend([3, 0, 0, 0, 1], 4)                         # no page at all
    s.extend([0] * 5, 0)
    s.trim([0] * 5)
    lens, table, free = P.page_state(3, 4, 7)
    assert free.tolist() == [7, 6, 5, 4, 3, 2, 1, 0] and table.shape == (3, 4) and not bool(lens.any())


def test_states_that_hold_nonsense_stay_in_bounds():
    """Counts past the pool, lengths past the table, pages that are not there: as the walk has it, and nothing around is touched."""
    for count in (-4, 99, 2 ** 31 - 1):
        s = State(6, 3, 4, 16, seed=2, free=count)
        s.lens.copy_(ints([-3, 40, 48, 2 ** 31 - 1, 5, 0]))
        s.table.copy_(ints([[9, -7, 2 ** 31 - 1]] * 6))
        s.pull()
        s.extend([1, 5, 1, 2 ** 31 - 1, 20, 2], 64)
        s.trim([0, 3, 2 ** 31 - 1, 7, -2 ** 31, 1])
        s.extend([30, 1, 1, 1, 1, 1], 40)


def test_captured_steps_follow_the_lengths():
    s = State(7, 6, 40, 16, seed=9)
    new = ints([1, 0, 16, 3, 1, 40, 2]).cuda()
    graph = torch.cuda.CUDAGraph()
    s.extend(new.tolist(), 70)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        step = P.page_extend(new, s.lens, s.table, s.free, 16, 70)
    torch.cuda.current_stream().wait_stream(side)
    s.same()                                             # a capture runs nothing
    for i, x in enumerate(([1, 1, 1, 1, 1, 1, 1], [0, 20, 0, 2, 17, 9, 1], [5, 0, 0, 0, 0, 0, 0])):
        new.copy_(ints(x))
        graph.replay()
        want = PO.extend(x, *s.h, 16, 70)
        s.same()
        assert [y.tolist() for y in step] == [list(y) for y in want]
        if i == 1:
            s.trim([3] * 7)


def test_more_rows_than_fit_on_chip_and_no_batch():
    """Room for no token: no row gets any, and there are no tokens to place."""
    s = State(5000, 2, 7, 16)
    s.extend([1] * 5000, 0)
    s.extend([0] * 5000, 0)
    s.extend([1] * 5000, 5000)
