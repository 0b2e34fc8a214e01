"""Where CachedDecodeStep puts the next tokens (infer_amd/chain.py,
next_slots), on the CPU: every length, in the table or not."""
import pytest
import torch

from infer_amd.chain import next_slots


def slots(lens, table, page, pages=2 ** 31):
    """next_slots, -1 where it says that there is none."""
    at, there = next_slots(lens, table, page, pages)
    assert at.dtype == torch.int64 and there.dtype == torch.bool
    assert torch.all(there | (at < 0) | (at >= pages * page))
    return torch.where(there, at, -1).tolist()


def plain(lens, table, page, pages=2 ** 31):
    got = []
    for b, n in enumerate(lens):
        full = n < 0 or n >= len(table[b]) * page
        got.append(-1 if full or not 0 <= table[b][n // page] < pages else table[b][n // page] * page + n % page)
    return got


@pytest.mark.parametrize("page", [1, 7, 16])
def test_slots(page):
    table = [[3, 0, 2 ** 20], [5, -1, 1], [-1, 4, 2 ** 31 - 1]]
    for n in (0, 1, page - 1, page, 2 * page - 1, 2 * page, 3 * page - 1, 3 * page, 3 * page + 1, 2 ** 31 - 1,
              -1, -2, -page, -page - 1, -2 ** 31):
        lens = [n, 0, n]
        got = slots(torch.tensor(lens, dtype=torch.int32), torch.tensor(table, dtype=torch.int32), page)
        assert got == plain(lens, table, page), n


def test_slots_in_a_part_of_a_table():
    wide = torch.arange(24, dtype=torch.int32).view(3, 8)
    lens = torch.tensor([0, 9, 31], dtype=torch.int32)
    assert slots(lens, wide[:, 2:5], 10) == [20, 109, -1]


def test_pages_outside_the_pool():
    table = [[3, 8, 9], [9, 0, 2 ** 31 - 1]]
    for n in range(12):
        got = slots(torch.tensor([n, n]), torch.tensor(table, dtype=torch.int32), 4, 9)
        assert got == plain([n, n], table, 4, 9), n
