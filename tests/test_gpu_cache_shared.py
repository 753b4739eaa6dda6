"""GPU: acceptance of drafted rows in pages that sequences share, exactly, with
the reference counts and without them."""
import random

import pytest
import torch

import ops_b200
from oracle import cache_oracle as C
from test_gpu_cache import SHAPES, Both, ints

pytestmark = pytest.mark.gpu

COUNTS = pytest.mark.parametrize("counts", [True, False], ids=["counts", "table"])


class Shared(Both):
    counts = True

    def accept(self, acc, drafted):
        got = ops_b200.paged_cache_accept(self.g_pools, self.g_table, self.g_lens, ints(acc).view(len(drafted), -1),
                                          ints(drafted), refcounts=self.g_refs if self.counts else None)
        keep = C.accept(self.pools, self.table, self.lens, acc, drafted, self.refs if self.counts else None)
        assert got.tolist() == keep
        return keep


def cache(counts, *args):
    c = Shared(*args)
    c.counts = counts
    return c


@COUNTS
@pytest.mark.parametrize("both", [True, False])
def test_a_fork_of_drafted_rows(counts, both):
    # five rows, then 30 drafted ones over pages of 16; a fork shares the two whole pages of them
    c = cache(counts, 3, 4, 12, SHAPES[0], 1)
    c.reserve([5, 0, 7])
    c.reserve([30, 0, 30])
    c.fork([0], [1])
    c.same()
    path = [0, 3, 9, 29]
    keep = c.accept([path, path if both else [-1] * 4, path], [30, 30 if both else 0, 30])
    assert keep == [-1, -1 if both else 35, 11]          # sequence 2 shares nothing
    c.same()
    c.trim(keep)
    c.same()
    # once one of the two is gone, the other one's pages are its own
    c.trim([-1, 0, -1])
    assert c.accept([path, [-1] * 4, [-1] * 4], [30, 0, 0]) == [9, 0, 11]
    c.same()


@COUNTS
def test_only_pages_that_are_written_matter(counts):
    # the prefix's pages are shared, the drafted rows' are not; rows that stay where they are write nothing
    c = cache(counts, 3, 6, 20, SHAPES[0], 2)
    c.reserve([32, 0, 0])
    c.fork([0], [1])
    c.reserve([20, 20, 0])
    assert c.accept([[1, 2, 19], [0, 2, -1], [-1] * 3], [20, 20, 0]) == [35, 34, 0]
    c.same()
    c.trim([48, 0, 0])
    c.fork([0], [1])                                      # all of it whole pages
    c.same()
    assert c.accept([[0, 1, 2], [0, 1, -1], [-1] * 3], [16, 16, 0]) == [35, 34, 0]
    c.same()
    assert c.accept([[0, 1, 3], [0, 1, 2], [-1] * 3], [16, 16, 0]) == [-1, 35, 0]
    c.same()


@COUNTS
def test_a_shared_page_late_in_a_long_path(counts):
    # 150 rows, several lists of the kernel's; only the page of the last moved row is shared, and only there does a
    # row move: nothing of the sequence may
    c = cache(counts, 2, 12, 30, [((16, 8), torch.int16)] * 3, 3)
    c.reserve([160, 0])
    c.g_table[1, 0] = c.table[1][0] = c.table[0][8]       # rows 128 .. 143
    c.refs[c.table[0][8]] += 1
    c.g_refs[c.table[0][8]] += 1
    c.lens[1] = 16
    c.g_lens[1] = 16
    stay = list(range(140))
    assert c.accept([stay + [150], [-1] * 141], [160, 0]) == [-1, 16]
    c.same()
    assert c.accept([[1] + list(range(2, 120)) + [-1] * 22, [-1] * 141], [160, 0]) == [119, 16]   # does not reach it
    c.same()
    # one sequence that holds a page twice
    c.trim([0, 0])
    c.reserve([160, 0])
    c.g_table[0, 9] = c.table[0][9] = c.table[0][0]
    c.refs[c.table[0][0]] += 1
    c.g_refs[c.table[0][0]] += 1
    assert c.accept([[2, 5] + [-1] * 139, [-1] * 141], [160, 0]) == [-1, 0]
    c.same()


@COUNTS
@pytest.mark.parametrize("shapes", SHAPES, ids=["vectors", "bytes", "large"])
@pytest.mark.parametrize("n,width,pages,seed", [(9, 6, 40, 1), (40, 4, 200, 2), (3, 12, 18, 3)])
def test_random_histories_with_forks_before_acceptance(counts, shapes, n, width, pages, seed):
    r, c = random.Random(seed), cache(counts, n, width, pages, shapes, seed)
    for step in range(30):
        op = r.choice(["reserve", "trim", "fork", "accept", "accept"])
        if op == "reserve":
            c.reserve([r.choice([0, 1, r.randint(0, 3 * c.page)]) for _ in range(n)])
        elif op == "trim":
            c.trim([r.choice([0, 0, r.randint(0, width * c.page)]) if r.random() < 0.3 else -1 for _ in range(n)])
        elif op == "fork":
            f = r.randint(0, n)
            c.fork([r.randint(0, n - 1) for _ in range(f)], [r.randint(0, n - 1) for _ in range(f)])
        else:
            drafted = [r.randint(0, length) for length in c.lens]
            acc = [sorted(r.sample(range(d), r.randint(0, min(d, 70)))) for d in drafted]
            wide = max(map(len, acc))
            c.trim(c.accept([a + [-1] * (wide - len(a)) for a in acc], drafted))
        c.same(f"step {step}: {op}")


@COUNTS
@pytest.mark.parametrize("shapes", SHAPES, ids=["vectors", "bytes", "large"])
@pytest.mark.parametrize("n,width,pages,seed", [(9, 6, 60, 1), (40, 5, 250, 2), (4, 12, 50, 3)])
def test_drafts_forked_and_accepted(counts, shapes, n, width, pages, seed):
    # every step: room for drafts in a third of the rows, those forked into the empty ones, acceptance on all
    r, c = random.Random(seed), cache(counts, n, width, pages, shapes, seed)
    refused = moved = 0
    for step in range(8):
        c.trim([0 if r.random() < 0.5 else -1 for _ in range(n)])
        c.reserve([r.randint(0, 2 * c.page) if s % 3 == 0 else 0 for s in range(n)])
        empty, full = ([s for s in range(n) if (c.lens[s] == 0) == e] for e in (True, False))
        c.fork([r.choice(full) for _ in empty if full], empty if full else [])
        drafted = [r.randint(0, length) for length in c.lens]
        acc = [sorted(r.sample(range(d), r.randint(0, min(d, 70)))) for d in drafted]
        wide = max(map(len, acc))
        keep = c.accept([a + [-1] * (wide - len(a)) for a in acc], drafted)
        refused += sum(k < 0 for k in keep)
        moved += sum(k >= 0 and a != list(range(len(a))) for k, a in zip(keep, acc))
        c.same(f"step {step}")
        c.trim(keep)
        c.same(f"step {step}: trim")
    assert moved and (refused or n < 9)        # the history has both answers (few rows: not always)


def test_counts_in_a_graph():
    c = cache(False, 3, 4, 12, SHAPES[0], 1)
    c.reserve([35, 0, 37])
    c.fork([0], [1])
    path, drafted = ints([[0, 3, 9, 29]] * 3), ints([30, 30, 30])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep = ops_b200.paged_cache_accept(c.g_pools, c.g_table, c.g_lens, path, drafted)
    for expect in ([-1, -1, 11], [9, -1, 11]):
        if expect[0] > 0:
            c.trim([-1, 0, -1])
        graph.replay()
        assert C.accept(c.pools, c.table, c.lens, [[0, 3, 9, 29]] * 3, [30, 30, 30]) == expect
        assert keep.tolist() == expect
        c.same()
