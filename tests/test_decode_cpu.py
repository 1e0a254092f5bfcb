"""Host side of the example decoder: pages are handed out once, returned and refused."""
import numpy as np
import pytest

from gpreempt_b200.decode import Pages


def test_pages_grow_with_the_sequences_and_are_returned():
    p = Pages(6, 16, 3, 64)
    assert p.grow([17, 0, 1]).tolist() == [0, 17, 17, 18]
    assert p.context.tolist() == [17, 0, 1]
    used = [int(x) for x in p.table[p.table >= 0]]
    assert len(used) == 3 and len(set(used)) == 3
    p.grow([15, 16, 15])  # up to the ends of their pages: one more page
    assert len(p.free) == 2 and np.array_equal(p.context, [32, 16, 16])
    p.grow([1, 1, 0])
    assert not p.free
    with pytest.raises(MemoryError):
        p.grow([0, 0, 1])
    p.release(0)
    assert len(p.free) == 3 and p.context[0] == 0
    p.grow([0, 0, 1])
    assert len({int(x) for s in range(3) for x in p.table[s, :-(-int(p.context[s]) // 16)]}) == 4


def test_a_sequence_longer_than_its_table_row_is_refused():
    p = Pages(100, 16, 1, 64)
    with pytest.raises(MemoryError):
        p.grow([65])
