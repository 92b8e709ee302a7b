"""PagedKVCache.next_slots and decode_step want one position for each sequence of the table (CPU)."""
import pytest
import torch

from tests.test_paged_cache import cache


@pytest.mark.parametrize("n", [0, 1, 3])
@pytest.mark.parametrize("length", [0, 20])
def test_other_numbers_of_positions(n, length):
    c = cache()
    t = c.block_tables([c.allocate(length), c.allocate(length)])
    for call in (c.next_slots, c.decode_step):
        with pytest.raises(ValueError, match="one position"):
            call(t, torch.zeros(n, dtype=torch.int32))
        with pytest.raises(ValueError, match="one position"):
            call(t, torch.zeros(2, 1, dtype=torch.int32))
