"""Attention over an 8-bit cache at the ends of what it takes: tables that lead outside
it, numbers that are not finite, a full batch's workspace for a smaller one."""
import ctypes

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


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("counts", [None, [20, 33]])
@pytest.mark.parametrize("group,dim", [(1, 64), (4, 128)])
def test_a_query_that_is_not_finite(cache, counts, group, dim, bad):
    """Its row does not come out finite, whatever the newest block's keys make of it
    in fp32, and is said; the other rows and heads come out as without it."""
    c = cache(2, 2, dim, positions=200)
    k, v = c.random_rows(400)
    k[:, :, 3] = np.abs(k[:, :, 3]) + 0.5  # infinite scores are of one sign
    c.write([0, 0], [193, 199], k[:392], v[:392])
    n = counts or [1, 1]
    for most in (200, 8192):
        a = Attend(c, [193 - n[0], 199 - n[1]], counts, group, most=most)
        want = a.run()
        assert c.st() == 0
        row = n[0] - 1  # the newest block has its key alone
        q = a.q.copy()
        q[row, 0, 3] = bad
        a.dq.upload(q.reshape(a.total, -1))
        got = a.run()
        assert c.st() == 1
        assert not np.isfinite(got[row, 0]).any()
        got[row, 0] = want[row, 0]
        assert np.array_equal(got[:, ::group], want[:, ::group])


@pytest.mark.parametrize("most", [64, 8192])
@pytest.mark.parametrize("bad", [np.inf, -np.inf])
def test_a_query_that_is_not_finite_over_a_first_block(cache, bad, most):
    c = cache(2, 2, 64, positions=30)
    k, v = c.random_rows(14)
    k[:, :, 3] = np.abs(k[:, :, 3]) + 0.5
    c.write([0, 0], [3, 11], k, v)
    a = Attend(c, [2, 10], None, 1, most=most)
    want = a.run()
    assert c.st() == 0
    q = a.q.copy()
    q[0, 1, 3] = bad
    a.dq.upload(q.reshape(a.total, -1))
    got = a.run()
    assert c.st() == 1
    assert not np.isfinite(got[0, 1]).any()
    got[0, 1] = want[0, 1]
    assert np.array_equal(got, want)


@pytest.mark.parametrize("most", [64, 300, 8192])
@pytest.mark.parametrize("counts", [None, [20, 33]])
def test_scores_that_are_all_minus_infinity(cache, counts, most):
    """Products of large finite keys and queries that pass fp32: no weights are left,
    and that is said."""
    c = cache(2, 2, 64, positions=60)
    k, v = c.random_rows(120)
    k = -np.abs(k) * np.float32(1e20)
    c.write([0, 0], [55, 60], k[:115], v[:115])
    n = counts or [1, 1]
    a = Attend(c, [55 - n[0], 60 - n[1]], counts, 1, most=most)
    a.q = np.abs(a.q) * np.float32(1e20)
    a.dq.upload(a.q.reshape(a.total, -1))
    got = a.run()
    assert c.st() == 1 and not np.isfinite(got).any()


@pytest.mark.parametrize("streams,counts,most", [(23, None, 3136), (7, None, 3136), (1, None, 8192),
                                                 (2, [30, 5], 3136), (1, [1], 8192)])
def test_a_full_batch_s_workspace_holds_a_smaller_one(cache, streams, counts, most):
    """Fewer streams may be dealt to more work-groups than 24, or runs of 64 rows."""
    c = cache(24, 8, 64, positions=130)
    c.fill([130] * 24)
    full = c.call_rows([0] * 24, counts and [64] * 24)
    size = c.lib.pgpu_kv8_attention_bytes(ctypes.byref(c.kv), ctypes.byref(full), 1, most)
    c.n = streams
    n = counts or [1] * streams
    a = Attend(c, [130 - x for x in n], counts, 1, most=most)
    a.bytes, a.work = size, c.up(np.full(max(16, size), 0xFF, np.uint8))
    check(c, a, a.run())
