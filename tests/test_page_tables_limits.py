"""Page bookkeeping at the ends of its ranges: counts whose sum passes 31 bits."""
import pytest
import torch

from bitstack_b200 import _lib, glue

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
MOST = 2 ** 31 - 1


def _i(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("listed", [40, 2000])          # written by the first launch, and by the second
@pytest.mark.parametrize("lens,new", [([0, 0, 3], [5, MOST, 4]), ([7, 2, 0], [0, MOST - 2, MOST]), ([100, 0, 9], [30, MOST, -4])])
def test_positions_of_a_list_longer_than_31_bits(lens, new, listed):
    ps, width = 1 << 30, 2                              # (no cache stands behind these pages: bookkeeping alone)
    table = torch.full((3, width), -1, dtype=torch.int32, device=DEV)
    free = _i(*range(40, 50))
    count = _i(10)
    for b, n in enumerate(lens):
        table[b, :-(-n // ps)] = 60 + b
    want_slots, want_positions = [], []
    held_first, top = [60 + b if n else None for b, n in enumerate(lens)], 49
    for b, (n, add) in enumerate(zip(lens, new)):
        pages = [held_first[b]] if n else []
        while len(pages) < -(-(n + max(add, 0)) // ps):
            pages.append(top)
            top -= 1
        for p in range(n, n + min(max(add, 0), listed - len(want_positions))):
            want_positions.append(p)
            want_slots.append(pages[p // ps] * ps + p % ps)
    total = sum(max(a, 0) for a in new)
    want_positions += [-1] * (listed - len(want_positions))
    want_slots += [-1] * (listed - len(want_slots))
    slots, positions, offsets, last = glue.page_tables(_i(*lens), _i(*new), table, free, count, ps, listed)
    assert positions.tolist() == want_positions and slots.tolist() == want_slots
    assert last.tolist() == [n + a - 1 if a > 0 else -1 for n, a in zip(lens, new)]
    assert offsets.tolist() == [min(sum(max(a, 0) for a in new[:b]), MOST) for b in range(4)]
    assert total > listed
    with pytest.raises(_lib.BitStackDeviceIndexError):  # the list was cut
        _lib.check_device_status()


@pytest.mark.parametrize("listed", [2 ** 31, 2 ** 62, -1])
def test_lists_beyond_31_bits_are_refused_before_they_are_allocated(listed):
    free = torch.cuda.memory_reserved()
    lens = _i(1, 2)
    with pytest.raises(ValueError, match="max_tokens"):
        glue.page_tables(lens, _i(1, 1), torch.zeros(2, 3, dtype=torch.int32, device=DEV), _i(1), _i(1), 4, listed)
    assert torch.cuda.memory_reserved() - free < 1 << 22 and lens.tolist() == [1, 2]
