"""The 4-bit paged KV cache on the GPU where calls meet: streams that share blocks, calls on
several queues at once, graphs of writes and evictions, workspaces taken for larger batches,
contexts of tens of thousands of rows, caches past 4 GiB."""
import ctypes

import numpy as np
import pytest

import kv4_model as model
from test_gpu_kv4 import (BLOCK, Attend, Evict, both_layers, cache, check_evicted,  # noqa: F401
                          tied_sums)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,dim,length,keep", [(1, 64, 8192, 8000), (2, 64, 8193, 300),
                                                   (1, 128, 19999, 9001)])
def test_evictions_of_very_long_streams(cache, heads, dim, length, keep):
    """More rows than the threads of a work-group hold; ties that pass them."""
    c = cache(2, heads, dim, positions=length)
    c.fill([length, keep + 1])
    both_layers(c)
    sums = tied_sums(c, length + 5)
    sums[0, 0, 0] = np.where(np.arange(length + 5) % 3 == 0, 2, 1)  # a third, then the first
    e = Evict(c, keep, 4, 100, sums)
    assert e.enqueue(), c.pkg.last_error(c.lib)
    assert c.st() == 0
    check_evicted(c, e, c.table)


def test_evictions_of_values_that_only_differ_in_their_last_bits(cache):
    c = cache(2, 2, 64, positions=1500)
    c.fill([1500, 1200])
    both_layers(c)
    sums = np.full((2, 2, 2, 1500), 1.0, np.float32)
    sums += c.rng.integers(0, 40, sums.shape).astype(np.float32) * np.float32(2 ** -23)
    sums[1, 0, 0] = 0
    sums[1, 0, 1] = -0.0
    sums[1, 1, 0] *= np.float32(2.0 ** -140)  # subnormal
    sums[1, 1, 1, ::2] = np.inf
    e = Evict(c, 700, 0, 33, sums)
    assert e.enqueue()
    assert c.st() == 0
    check_evicted(c, e, c.table)


@pytest.mark.parametrize("group,dim", [(1, 64), (4, 128)])
def test_a_context_of_many_thousand_rows(cache, group, dim):
    """One row and runs behind 69 999 keys, their parts joined, with sums."""
    c = cache(2, 1, dim, positions=70000)
    c.fill([60000, 130])
    c.write([60000, 130], [9930, 0], *c.random_rows(9930))
    c.write([69930, 130], [70, 70], *c.random_rows(140))
    for first, counts, most in (([69999, 199], None, None), ([69999, 199], None, 1 << 20),
                                ([69930, 130], [70, 70], None), ([69997, 140], [3, 60], 100000)):
        a = Attend(c, first, counts, group, most=most)
        got = a.run()
        assert c.st() == 0
        a.check(got)
        b = Attend(c, first, counts, group, most=most, sums=40)
        got = b.run()
        assert c.st() == 0
        b.check(got, added=b.added())


@pytest.mark.parametrize("sums", [None, 20])
@pytest.mark.parametrize("group,dim", [(1, 64), (3, 128)])
def test_keys_and_values_too_large_for_the_fast_way(cache, group, dim, sums):
    """Scales up to the largest, some blocks of them, beside ordinary rows: runs and one row."""
    c = cache(3, 2, dim, positions=500)
    k, v = c.random_rows(1150)
    for x, rows in ((k, slice(100, 164)), (v, slice(150, 170)), (k, slice(600, 601)), (v, slice(700, 900))):
        x[rows] *= 55000 / np.abs(x[rows]).max()
    c.write([0] * 3, [480, 170, 500], k, v)
    assert c.st() == 0
    for first, counts in (([479, 169, 499], None), ([400, 0, 263], [80, 170, 237])):
        a = Attend(c, first, counts, group, sums=sums, spread=1e-4)
        got = a.run()
        assert c.st() == 0
        a.check(got, added=a.added() if sums else None)


@pytest.mark.parametrize("counts", [None, [40, 40, 40, 40]])
@pytest.mark.parametrize("group,dim", [(1, 64), (4, 128)])
def test_streams_that_share_a_prefix(cache, counts, group, dim):
    """The blocks of a prefix stand in several tables, and one stream twice in the batch."""
    c = cache(4, 2, dim, positions=700)
    k, v = c.random_rows(640)
    n = counts or [1] * 4
    c.write([0] * 4, [640] * 4, *(np.concatenate([x] * 4) for x in (k, v)))
    a = Attend(c, [640 - m for m in n], counts, group, sums=33)
    a.q[:] = np.concatenate([a.q[:n[0]]] * 4)
    a.dq.upload(a.q.reshape(len(a.q), -1))
    a.before0[:] = a.before0[:1]
    a.before.upload(a.before0)
    want, added = a.run(), a.added()
    a.check(want, added=added)
    shared = c.table.copy()
    shared[1:3, :30] = shared[0, :30]
    shared[3] = shared[0]
    c.tables.upload(shared)
    assert np.array_equal(a.run(), want) and np.array_equal(a.added(), added)
    assert c.st() == 0


def test_a_workspace_for_the_largest_batch_serves_smaller_ones(cache):
    """Filled with what is not a number, taken by calls of fewer streams, rows, positions."""
    for heads, dim, group in ((8, 64, 1), (2, 128, 4), (8, 64, 2)):
        c = cache(6, heads, dim, positions=5000)
        c.fill([5000, 1, 17, 900, 64, 300])
        first = [n - 1 for n in c.lengths()]
        big = Attend(c, first, None, group, sums=1)
        for streams, most, sums in ((6, None, 1), (1, 5000, None), (1, 5000, 1), (2, 5000, 1), (6, 5000, None)):
            c.n, n = streams, c.n
            a = Attend(c, first[:streams], None, group, most=most, sums=sums)
            assert a.bytes <= big.bytes
            a.bytes, a.work = big.bytes, big.work
            big.work.upload(np.full(max(16, big.bytes), 0xFF, np.uint8))
            got = a.run()
            a.check(got, added=a.added() if sums else None)
            c.n = n
        counts = [200, 1, 17, 65, 64, 300]
        first = [m - x for m, x in zip(c.lengths(), counts)]
        big = Attend(c, first, counts, group, sums=1000)
        for part, most, sums in (([200, 1, 17, 65, 64, 300], 5000, 1000), ([200, 1, 17, 65, 64, 300], 5000, None),
                                 ([20, 0, 0, 0, 0, 0], 5000, 1), ([1, 1, 1, 1, 1, 1], 5000, None)):
            a = Attend(c, [m - x for m, x in zip(c.lengths(), part)], part, group, most=most, sums=sums)
            assert a.bytes <= big.bytes
            a.bytes, a.work = big.bytes, big.work
            big.work.upload(np.full(max(16, big.bytes), 0xFF, np.uint8))
            got = a.run()
            a.check(got, added=a.added() if sums else None)
        assert c.st() == 0


def test_calls_on_several_queues_at_once(cache):
    """Caches, workspaces and results of their own: what each gives alone."""
    made, streams = [], []
    try:
        for i, (heads, dim, group, counts) in enumerate([(8, 64, 1, None), (2, 128, 4, None), (8, 64, 1, [90, 33, 200]),
                                                         (2, 128, 2, [20, 300, 7])]):
            c = cache(3, heads, dim, positions=900, seed=i)
            n = counts or [1] * 3
            c.fill([500 + n[0], 17 + n[1], 600 + n[2]])
            both_layers(c)
            a = Attend(c, [500, 17, 600], counts, group, sums=40)
            want, added = a.run(), a.added()
            e = Evict(c, 200, 4, 50, tied_sums(c, 900))
            a.dout.upload(a.mark)
            a.after.upload(a.after0)
            s = ctypes.c_void_p()
            assert c.lib.pgpu_stream_create(ctypes.byref(s))
            streams.append((c.lib, s))
            made.append((c, a, e, s, want, added))
        for turn in range(3):
            for c, a, e, s, want, added in made:
                assert a.enqueue(s)
        for c, a, e, s, want, added in made:
            assert e.enqueue(s)
        for c, a, e, s, want, added in made:
            assert c.lib.pgpu_stream_sync(s)
            assert np.array_equal(a.result(), want) and np.array_equal(a.added(), added)
            check_evicted(c, e, c.table)
            assert c.st() == 0
    finally:
        for lib, s in streams:
            lib.pgpu_stream_destroy(s)


def test_writes_and_evictions_replay_from_a_graph(cache):
    """A frame's write, then an eviction of both layers, captured once in global mode and
    replayed over caches that are set back in between: the same bits each time."""
    c = cache(3, 2, 64, positions=400)
    lib = c.lib
    c.fill([300, 20, 390])
    both_layers(c)
    start = c.raw()
    e = Evict(c, 100, 3, 20, tied_sums(c, 400))
    k, v = c.random_rows(3)
    dk, dv = c.up(k.reshape(3, -1)), c.up(v.reshape(3, -1))
    rows = c.call_rows(c.lengths())
    lengths = c.up(np.array([301, 21, 391], np.int32))
    e.lengths = lengths

    def enqueue(stream):
        return all(lib.pgpu_kv4_write(stream, ctypes.byref(c.kv), layer, ctypes.byref(rows), dk.ptr,
                                      dv.ptr, 128, c.status.ptr) for layer in range(2)) and e.enqueue(stream)

    c.note(c.lengths(), [1, 1, 1], k, v)
    stream, exec_ = ctypes.c_void_p(), ctypes.c_void_p()
    assert lib.pgpu_stream_create(ctypes.byref(stream))
    try:
        assert lib.pgpu_graph_begin_global(stream)
        enqueued = enqueue(stream)
        ended = lib.pgpu_graph_end(stream, ctypes.byref(exec_))
        assert enqueued and ended, c.pkg.last_error(lib)
        for replay in range(4):
            c.values.upload(start[0])
            c.scales.upload(start[1])
            e.sums.upload(e.sums0)
            e.kept.upload(e.kept0)
            if replay == 2:
                assert enqueue(None)  # the program's own, between replays
                check_evicted(c, e, c.table)
                continue
            assert lib.pgpu_graph_launch(exec_, stream) and lib.pgpu_stream_sync(stream)
            check_evicted(c, e, c.table)
            assert c.st() == 0
    finally:
        lib.pgpu_graph_destroy(exec_)
        lib.pgpu_stream_destroy(stream)


@pytest.mark.parametrize("counts", [None, [40, 1, 130]])
def test_a_cache_past_4_gib(cache, counts):
    """Blocks whose bytes lie past 2^32, in a second layer: the bits of a small cache."""
    c = cache(3, 8, 128, positions=600)
    n = counts or [1] * 3
    rows = c.random_rows(500 + 17 + 333 + sum(n))
    a = Attend(c, [500, 17, 333], counts, 1, sums=40)
    sums = tied_sums(c, 600)

    def go():
        c.rows = [[np.zeros((0, 8, 128), np.float32)] * 2 for _ in range(3)]
        c.write([0] * 3, [500 + n[0], 17 + n[1], 333 + n[2]], *rows)
        got = [c.raw_read(), a.run(), a.added()]
        e = Evict(c, 100, 4, 20, sums)
        assert c.lib.pgpu_kv4_evict(None, ctypes.byref(c.kv), 1, 1, c.tables.ptr, None, c.stride, e.lengths.ptr, 3,
                                    100, 4, 20, e.sums.ptr, e.sums.ptr, 600, e.kept.ptr, c.status.ptr)
        c.rows = [[x[:100] for x in r] for r in c.rows]
        got += [c.raw_read(), e.kept.download(e.kept0.shape, np.int32)[:1]]
        assert c.st() == 0
        return got

    c.raw_read = lambda: np.stack(c.read([0] * 3, c.lengths()))
    small = go()
    blocks = 300000
    values, scales = (c.pkg.DeviceBuffer(c.lib, b) for b in (2 * blocks * 16384, 2 * blocks * 1024))
    c.keep += [values, scales]
    assert blocks * 16384 > 1 << 32
    c.kv = c.pkg.PgpuKv4(values.ptr, scales.ptr, 2, 8, 128, blocks)
    c.tables.upload(np.where(c.table % 3 == 0, c.table, blocks - 1 - c.table).astype(np.int32))
    for x, y in zip(small, go()):
        assert np.array_equal(x, y)


@pytest.mark.parametrize("first", [32, 47])
def test_evictions_of_streams_that_share_their_first_blocks(cache, first):
    """Blocks whose rows are all among the first stay where they are, in every table."""
    c = cache(3, 2, 64, positions=600)
    k, v = c.random_rows(1500)
    c.write([0] * 3, [600, 300, 600], k, v)
    for s, n in ((1, 300), (2, 600)):  # streams 1 and 2 begin as stream 0 does
        c.table[s, :2] = c.table[0, :2]
        c.rows[s] = [np.concatenate([a[:32], b[32:]]) for a, b in zip(c.rows[0], c.rows[s])]
    c.tables.upload(c.table)
    both_layers(c)
    e = Evict(c, 300, first, 20, tied_sums(c, 600))
    shared = [x[:, c.table[0, :2]] for x in c.raw()]
    assert e.enqueue()
    assert c.st() == 0
    check_evicted(c, e, c.table)
    for x, y in zip(shared, c.raw()):
        assert np.array_equal(x, y[:, c.table[0, :2]])


@pytest.mark.parametrize("dim", [64, 128])
def test_streams_left_with_rows_of_a_block_take_more(cache, dim):
    """After an eviction that ends inside a block, new rows go behind the kept ones."""
    c = cache(2, 2, dim, positions=500)
    c.fill([400, 90])
    both_layers(c)
    e = Evict(c, 75, 3, 9, tied_sums(c, 500))
    assert e.enqueue()
    kept = check_evicted(c, e, c.table)
    k, v = c.random_rows(30)
    c.rows = [[np.stack([x[kept[1, s, h, :75], h] for h in range(2)], 1) for x in r]
              for s, r in enumerate(c.rows)]
    c.write([75, 75], [20, 10], k, v)
    got = c.read([0, 0], c.lengths())
    for x, r in zip(got, range(2)):
        assert np.array_equal(x.astype(np.float64), np.concatenate([model.seen(c.rows[s][r]) for s in range(2)]))
    a = Attend(c, [75, 75], [20, 10], 2, sums=4)
    a.check(a.run(), added=a.added())
    assert c.st() == 0
