"""GPU tests of the page pool at the most tokens that a sequence may hold, 2^30."""

import pytest
import torch

from page_pool import PagePool

pytestmark = pytest.mark.gpu
DEV, MOST = "cuda", 1 << 30


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def pool_of(lengths):
    """Sequences of these lengths, in pages of 2^20 tokens with room for more than 2^30."""
    pool = PagePool(3000, len(lengths), 1030, page_size=1 << 20)
    pool.resize(int32(lengths))
    return pool


@pytest.mark.parametrize("tokens", [17, 5000])  # one launch, and two
def test_rows_across_the_bound(tokens):
    pool = pool_of([MOST - 5, 3])
    rows = pool.extend(int32([10, 7]), tokens=tokens)
    at = list(range(MOST - 5, MOST)) + [MOST] * 5 + list(range(3, 10))
    assert rows.positions.tolist() == at + [0] * (tokens - 17)
    table = pool.table.tolist()
    places = [-1 if p == MOST else table[i >= 10][p >> 20] * (1 << 20) + p % (1 << 20) for i, p in enumerate(at)]
    assert rows.slots.tolist() == places + [-1] * (tokens - 17) and min(places[:5] + places[10:]) >= 0
    assert pool.lengths.tolist() == [MOST, 10] and pool.owned.tolist() == [1024, 1]


def test_more_rows_than_positions():
    """2^30 held and more than 2^30 new: their sum is no number of 32 bits."""
    new = MOST + 3000
    pool = pool_of([MOST, 3])
    rows = pool.extend(int32([new, 7]), tokens=new + 9)
    assert rows.offsets.tolist() == [0, new, new + 7] and rows.held.tolist() == [MOST, 3]
    assert rows.positions[:new].aminmax() == (MOST, MOST) and rows.slots[:new].aminmax() == (-1, -1)
    assert rows.positions[new:].tolist() == [*range(3, 10), 0, 0]
    first = int(pool.table[1, 0]) * (1 << 20)
    assert rows.slots[new:].tolist() == [first + i for i in range(3, 10)] + [-1, -1]
    assert pool.lengths.tolist() == [MOST, 10]
