"""The example layer's bounds (CPU): a step past the rotation's tables or the
sequences' pages is refused, and leaves the cache as it was."""
import numpy as np
import pytest

import attention


def cache_of(seqs, pages, page, used):
    c = attention.Cache.__new__(attention.Cache)
    c.page, c.seqs, c.used = page, seqs, list(used)
    c.table = np.arange(seqs * pages, dtype=np.int32).reshape(seqs, pages)
    return c


@pytest.mark.parametrize("counts", [[0, 2], [9, 0], [3, 3]])
def test_pages_are_full(counts):
    c = cache_of(2, 2, 4, [0, 7])
    with pytest.raises(ValueError):
        c.room(counts)
    assert c.used == [0, 7]
    slot, pos, seq = c.room([8, 1])
    assert list(slot) == list(range(8)) + [15] and list(pos) == list(range(8)) + [7] and c.used == [8, 8]


@pytest.mark.parametrize("counts", [[0, 4], [11, 0]])
def test_positions_past_the_tables(counts):
    layer = attention.Layer.__new__(attention.Layer)
    layer.cos = np.zeros((10, 4), np.int64)
    c = cache_of(2, 8, 4, [0, 7])
    with pytest.raises(ValueError):
        layer.batch(c, counts)
    assert c.used == [0, 7]
