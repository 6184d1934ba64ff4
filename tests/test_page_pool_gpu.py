"""GPU tests of the pages dealt to sequences (page_pool.py over csrc/page_pool.hip) against lists on the CPU: whole numbers,
so everything is equal."""

import copy
import random

import pytest
import torch

import _hip
from page_pool import PagePool, row_positions

pytestmark = pytest.mark.gpu
DEV = "cuda"


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


class Lists:
    """The pool's definition."""

    def __init__(self, pages, seqs, width, page):
        self.stack, self.table, self.width, self.page = list(range(pages - 1, -1, -1)), [[] for _ in range(seqs)], width, page
        self.lengths, self.missing = [0] * seqs, [0] * seqs

    def resize(self, lengths):
        self.lengths = [min(max(n, 0), 1 << 30) for n in lengths]
        want = [min(-(-n // self.page), self.width) for n in self.lengths]
        for mine, w in reversed(list(zip(self.table, want))):
            while len(mine) > w:
                self.stack.append(mine.pop())
        for mine, w in zip(self.table, want):
            while len(mine) < w and self.stack:
                mine.append(self.stack.pop())
        self.missing = [w - len(mine) for mine, w in zip(self.table, want)]

    def extend(self, new, tokens):
        new = [max(n, 0) for n in new]
        held = self.lengths
        self.resize([h + n for h, n in zip(held, new)])
        offsets = [0]
        for n in new:
            offsets.append(min(offsets[-1] + n, tokens))
        positions, slots = [0] * tokens, [-1] * tokens
        for b, h in enumerate(held):
            for r in range(offsets[b], offsets[b + 1]):
                positions[r] = h + r - offsets[b]
                at = positions[r] // self.page
                if at < len(self.table[b]):
                    slots[r] = self.table[b][at] * self.page + positions[r] % self.page
        return offsets, held, positions, slots


def same(pool, lists):
    assert pool.lengths.tolist() == lists.lengths
    assert pool.owned.tolist() == [len(m) for m in lists.table]
    assert pool.table.tolist() == [m + [-1] * (lists.width - len(m)) for m in lists.table]
    assert pool.missing.tolist() == lists.missing
    assert pool.left.tolist() == [len(lists.stack)] and pool.free[:len(lists.stack)].tolist() == lists.stack


CASES = [(1, 1, 1, 32), (7, 3, 4, 32), (100, 5, 40, 64), (40, 17, 6, 1), (500, 64, 30, 96), (3000, 1025, 9, 64),
         (9000, 2500, 5, 32), (20, 2100, 2, 64), (0, 4, 3, 32), (5, 2, 0, 32), (6, 0, 3, 32)]


@pytest.mark.parametrize("pages,seqs,width,page", CASES)
def test_steps(pages, seqs, width, page):
    """Growth, drafts taken back, sequences that end and others that take their place, pages that run out."""
    print(f"pool of {pages} pages of {page}, {seqs} x {width}", flush=True)
    rng = random.Random(pages + seqs)
    pool, lists = PagePool(pages, seqs, width, page_size=page), Lists(pages, seqs, width, page)
    same(pool, lists)
    for step in range(12):
        most = rng.choice([1, 1, 3, page, 2 * page + 5])
        if seqs > 1000:
            most = min(most, 3)
        new = [rng.choice([0, 1, rng.randint(-3, most)]) for _ in range(seqs)]
        tokens = sum(max(n, 0) for n in new) + rng.choice([0, 0, 9])
        got, want = pool.extend(int32(new), tokens=tokens), lists.extend(new, tokens)
        for g, w in zip(got, want):
            assert g.tolist() == w
        same(pool, lists)
        lengths = [max(h - rng.randint(0, most), 0) if rng.random() < 0.6 else rng.choice([h, 0, h + most, -4])
                   for h in lists.lengths]
        if step % 4 == 3:
            lengths = [0 if rng.random() < 0.5 else rng.randint(0, width * page + 3) for _ in lengths]
        pool.resize(int32(lengths))
        lists.resize(lengths)
        same(pool, lists)


def test_prompts_of_many_rows():
    """More rows than one workgroup takes; pages that come back are taken in the same call; all of it again."""
    pages, seqs, width, page = 700, 30, 40, 32
    pool, lists = PagePool(pages, seqs, width, page_size=page), Lists(pages, seqs, width, page)
    rng = random.Random(1)
    for step in range(4):
        stay = [0 if rng.random() < 0.5 else h for h in lists.lengths]
        pool.resize(int32(stay))
        lists.resize(stay)
        new = [rng.randint(0, 600) for _ in range(seqs)]
        got, want = pool.extend(int32(new), tokens=sum(new) + 3), lists.extend(new, sum(new) + 3)
        for g, w in zip(got, want):
            assert g.tolist() == w
        same(pool, lists)
    swap = [h if b % 2 else 0 for b, h in enumerate(lists.lengths)]
    swap[0] = 1200
    pool.resize(int32(swap))
    lists.resize(swap)
    same(pool, lists)


def test_a_step_taken_back_and_made_again():
    pool = PagePool(50, 6, 8, page_size=32)
    pool.extend(int32([40, 0, 31, 64, 100, 1]), tokens=236)
    held, table = pool.lengths.clone(), pool.table.clone()
    pool.extend(int32([8] * 6), tokens=48)
    after = pool.table.clone()
    pool.resize(held)
    assert torch.equal(pool.table, table)
    pool.extend(int32([8] * 6), tokens=48)
    assert torch.equal(pool.table, after)


def test_lengths_that_are_the_pools_own_and_far_too_long():
    pool = PagePool(9, 3, 4, page_size=32)
    pool.resize(int32([200, 2 ** 31 - 1, 5]))
    assert pool.lengths.tolist() == [200, 1 << 30, 5] and pool.owned.tolist() == [4, 4, 1] and pool.missing.tolist() == [0, 0, 0]
    pool.resize(pool.lengths)
    assert pool.owned.tolist() == [4, 4, 1] and pool.left.tolist() == [0]
    rows = pool.extend(int32([2 ** 31 - 1, 2 ** 31 - 1, 1]), tokens=5)
    assert rows.offsets.tolist() == [0, 5, 5, 5] and pool.lengths.tolist() == [1 << 30, 1 << 30, 6]
    assert rows.positions.tolist() == [200, 201, 202, 203, 204] and rows.slots.tolist() == [-1] * 5


def test_captured():
    pool, lists = PagePool(60, 4, 10, page_size=32), Lists(60, 4, 10, 32)
    new, stay = int32([0] * 4), int32([0] * 4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.resize(stay)
        rows = pool.extend(new, tokens=90)
    rng = random.Random(3)
    for _ in range(5):
        n, s = [rng.randint(0, 20) for _ in range(4)], [max(0, h - rng.randint(0, 30)) for h in lists.lengths]
        new.copy_(int32(n)), stay.copy_(int32(s))
        graph.replay()
        torch.cuda.synchronize()
        lists.resize(s)
        want = lists.extend(n, 90)
        for g, w in zip(rows, want):
            assert g.tolist() == w
        same(pool, lists)


def test_row_positions():
    for held, counts, tokens in (([5], [3], 3), ([0, 7, 100, 2], [2, 0, 5, 1], 10), ([4] * 300, [i % 4 for i in range(300)], 460),
                                 ([], [], 2), ([1, 2], [0, 0], 3)):
        offsets = [0]
        for c in counts:
            offsets.append(offsets[-1] + c)
        want = [h + i for h, c in zip(held, counts) for i in range(c)]
        assert row_positions(int32(held), int32(offsets), tokens).tolist() == want + [0] * (tokens - len(want))
    # rows before the first sequence's
    assert row_positions(int32([9]), int32([2, 4]), 5).tolist() == [0, 0, 9, 10, 0]


def test_refusals():
    for kw in (dict(pages=-1, seqs=1, width=1), dict(pages=1, seqs=-1, width=1), dict(pages=1, seqs=1 << 20, width=1 << 11),
               dict(pages=1, seqs=1, width=1, page_size=0)):
        with pytest.raises(ValueError):
            PagePool(**kw)
    with pytest.raises(_hip.GPTQ2DError):
        PagePool(1, 1, 1, device="cpu")
    pool = PagePool(4, 3, 2)
    for bad in (torch.zeros(3, dtype=torch.int64, device=DEV), int32([0, 0]), torch.zeros(3, dtype=torch.int32), int32([0] * 6)[::2]):
        with pytest.raises(ValueError):
            pool.resize(bad)
        with pytest.raises(ValueError):
            pool.extend(bad, tokens=0)
    with pytest.raises(ValueError):
        pool.extend(int32([0, 0, 0]), tokens=-1)
    for held, offsets in ((int32([1, 2]), int32([0, 1])), (int32([1]).long(), int32([0, 1])), (int32([1]), int32([0, 1]).long())):
        with pytest.raises(ValueError):
            row_positions(held, offsets, 1)


def test_copies_have_pages_of_their_own():
    """A deep copy goes on from the same state without touching its original, also once that is gone."""
    pool, other = PagePool(9, 3, 4, page_size=32), Lists(9, 3, 4, 32)
    for p in (pool, other):
        p.extend(int32([40, 0, 65]) if p is pool else [40, 0, 65], tokens=105)
    twin = copy.deepcopy(pool)
    was = [t.clone() for t in (pool.table, pool.lengths, pool.owned, pool.free, pool.left)]
    for lengths in ([10, 90, 0], [128, 0, 128]):
        twin.resize(int32(lengths))
        other.resize(lengths)
        assert [[p for p in row if p >= 0] for row in twin.table.tolist()] == other.table
        assert twin.lengths.tolist() == other.lengths and twin.missing.tolist() == other.missing
        assert all(torch.equal(a, b) for a, b in zip(was, (pool.table, pool.lengths, pool.owned, pool.free, pool.left)))
