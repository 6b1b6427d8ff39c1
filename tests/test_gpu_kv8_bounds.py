"""Attention over an 8-bit cache where tables lead outside it."""
import numpy as np
import pytest

from test_gpu_kv8 import Attend, cache  # noqa: F401 (a fixture)
from test_gpu_kv8_uneven import check

pytestmark = pytest.mark.gpu

# Blocks of the table that lead outside the cache, for a stream each.
LOST = [[], [0], [1, 2, 3], [0, 1, 2, 3, 4, 5, 6, 7], [17], list(range(18))]


@pytest.mark.parametrize("most", [320, 8192])
@pytest.mark.parametrize("group,dim", [(1, 64), (3, 64), (1, 128)])
@pytest.mark.parametrize("counts", [None, [300] * 6, [20, 33, 300, 299, 16, 300]])
def test_a_block_outside_the_cache_weighs_nothing(cache, counts, group, dim, most):
    """Rows take their keys from the blocks that are there, whatever block 0, which
    stands at the place of the others for the kernel, holds: a stream's, or
    numbers that are not finite."""
    c = cache(6, 2, dim, positions=300)
    c.table[c.table == 0] = max(set(range(c.blocks)) - set(c.table.reshape(-1)))
    c.tables.upload(c.table)
    c.fill([300] * 6)
    table = c.table.copy()
    for s, blocks in enumerate(LOST):
        table[s, blocks] = [c.blocks + s, -1 - s][s % 2]
    c.tables.upload(table)
    n = counts or [1] * 6
    scales = c.scales.download(c.scales0.shape)
    for block0 in (1.0, 3.0e7, np.nan):
        changed = scales.copy()
        changed[1, 0] = block0
        c.scales.upload(changed)
        a = Attend(c, [300 - x for x in n], counts, group, most=most)
        check(c, a, a.run(), LOST, 2)
