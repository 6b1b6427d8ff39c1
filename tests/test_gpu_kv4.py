"""The 4-bit paged KV cache on the GPU against a plain model in 64 bits: rows written in any
number of calls and read back, attention one row a stream and in runs with the sums of its
weights, evictions; odd and empty lengths, strides, grouped heads, both head widths, bounds
that are broken, what is not finite, graphs."""
import ctypes

import numpy as np
import pytest

import kv4_model as model

pytestmark = pytest.mark.gpu
BLOCK = 16


class Cache:
    """A cache of 2 layers with its tables, and the rows that layer 1 holds (layer 0 stays
    as it was made)."""

    def __init__(self, lib, pkg, streams, heads=8, dim=64, positions=200, seed=1):
        self.lib, self.pkg, self.n, self.heads, self.dim = lib, pkg, streams, heads, dim
        self.rng = rng = np.random.default_rng(seed)
        self.stride = -(-positions // BLOCK)
        self.blocks = streams * self.stride + 2
        self.keep = []
        self.values0 = rng.integers(0, 256, (2, self.blocks, heads, 2, dim // 64, 512), np.uint8)
        self.scales0 = rng.integers(0, 65536, (2, self.blocks, heads, dim // 64, BLOCK, 2),
                                    np.uint16)  # any bits: NaN and infinities among them
        self.values, self.scales = self.up(self.values0), self.up(self.scales0)
        self.table = rng.permutation(self.blocks)[:streams * self.stride].astype(np.int32)
        self.table = self.table.reshape(streams, self.stride)
        self.tables = self.up(self.table)
        self.status = self.up(np.zeros(1, np.int32))
        self.kv = pkg.PgpuKv4(self.values.ptr, self.scales.ptr, 2, heads, dim, self.blocks)
        self.rows = [[np.zeros((0, heads, dim), np.float32)] * 2 for _ in range(streams)]

    def up(self, a):
        a = np.ascontiguousarray(a)
        b = self.pkg.DeviceBuffer(self.lib, max(16, a.nbytes))
        if a.nbytes:
            b.upload(a)
        self.keep.append(b)
        return b

    def call_rows(self, first, counts=None):
        first = np.asarray(first, np.int32)
        if counts is None:
            return self.pkg.PgpuKv4Rows(self.tables.ptr, self.stride, self.up(first).ptr, None,
                                        self.n, self.n, 1)
        offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        return self.pkg.PgpuKv4Rows(self.tables.ptr, self.stride, self.up(first).ptr,
                                    self.up(offsets).ptr, self.n, int(offsets[-1]),
                                    int(max(counts)))

    def st(self):
        """The status word, and clears it."""
        s = int(self.status.download((1,), np.int32)[0])
        self.status.upload(np.zeros(1, np.int32))
        return s

    def write(self, first, counts, k, v, pad=0, one=False, stream=None):
        width = self.heads * self.dim
        rows = self.call_rows(first, None if one else counts)
        wide = np.full((2, max(1, len(k)), width + pad), np.nan, np.float32)
        wide[0, :len(k), :width], wide[1, :len(k), :width] = (k.reshape(len(k), -1),
                                                               v.reshape(len(v), -1))
        dk, dv = self.up(wide[0]), self.up(wide[1])
        assert self.lib.pgpu_kv4_write(stream, ctypes.byref(self.kv), 1, ctypes.byref(rows),
                                       dk.ptr, dv.ptr, width + pad, self.status.ptr), \
            self.pkg.last_error(self.lib)
        self.note(first, counts, k, v)

    def note(self, first, counts, k, v):
        at = 0
        for s, (f, n) in enumerate(zip(first, counts)):
            if f >= 0:
                self.rows[s] = [np.concatenate([old[:f], new[at:at + n], old[f + n:]])
                                for old, new in zip(self.rows[s], (k, v))]
            at += n

    def lengths(self):
        return [len(r[0]) for r in self.rows]

    def random_rows(self, count):
        gain = np.exp(self.rng.standard_normal((1, self.heads, self.dim)) * 0.5)
        return [(self.rng.standard_normal((count, self.heads, self.dim)) * gain).astype(np.float32)
                for _ in range(2)]

    def fill(self, lengths):
        self.write([0] * self.n, lengths, *self.random_rows(sum(lengths)))

    def read(self, first, counts, pad=0, lengths=None, tables=None):
        width = self.heads * self.dim
        rows = self.call_rows(first, counts)
        if tables is not None:
            rows.tables = tables.ptr
        total = sum(counts)
        mark = np.full((total + 3, width + pad), 7.5, np.float32)
        dk, dv = self.up(mark), self.up(mark)
        dl = self.up(np.asarray(self.lengths() if lengths is None else lengths, np.int32))
        assert self.lib.pgpu_kv4_read(None, ctypes.byref(self.kv), 1, ctypes.byref(rows), dl.ptr,
                                      dk.ptr, dv.ptr, width + pad, self.status.ptr)
        k, v = dk.download(mark.shape), dv.download(mark.shape)
        for x in (k, v):  # rows behind the last and columns past the width: left as they were
            assert (x[total:] == 7.5).all() and (x[:, width:] == 7.5).all()
        return [x[:total, :width].reshape(total, self.heads, self.dim) for x in (k, v)]

    def raw(self):
        return (self.values.download(self.values0.shape, np.uint8),
                self.scales.download(self.scales0.shape, np.uint16))

    def want(self):
        """What the buffers hold, from the rows written to layer 1."""
        values, scales = self.values0.copy(), self.scales0.copy()
        for s, (k, v) in enumerate(self.rows):
            (qk, sk), (qv, sv) = model.quantise(k), model.quantise(v)
            for b in range(-(-len(k) // BLOCK)):
                lo, hi = b * BLOCK, min(len(k), b * BLOCK + BLOCK)
                for h in range(self.heads):
                    # Rows of the block that nothing was written to keep their bits.
                    mask = model.tile(*(np.repeat((np.arange(BLOCK) < hi - lo)[:, None] * -1,
                                                  self.dim, 1) for _ in range(2)))
                    pad = ((0, BLOCK - hi + lo), (0, 0))
                    new = model.tile(np.pad(qk[lo:hi, h], pad), np.pad(qv[lo:hi, h], pad))
                    t = values[1, self.table[s, b], h]
                    values[1, self.table[s, b], h] = (t & ~mask) | (new & mask)
                pair = np.stack([sk[lo:hi], sv[lo:hi]], -1).astype(np.float16).view(np.uint16)
                scales[1, self.table[s, b], :, :, :hi - lo] = pair.transpose(1, 2, 0, 3)
        return values, scales

    def close(self):
        for b in self.keep:
            b.free()


@pytest.fixture
def cache(lib, pkg):
    made = []

    def make(*args, **kw):
        made.append(Cache(lib, pkg, *args, **kw))
        return made[-1]
    yield make
    for c in made:
        c.close()


def check_contents(c):
    for got, want in zip(c.raw(), c.want()):
        assert np.array_equal(got, want)


@pytest.mark.parametrize("heads,dim", [(8, 64), (3, 128), (1, 64)])
@pytest.mark.parametrize("pad", [0, 20])
def test_rows_written_in_runs_are_the_model_s_bits(cache, heads, dim, pad):
    """Runs that start and end inside blocks, at their borders, of one row and of none, with
    an empty place in the batch; rows written again; whatever the cache held before."""
    c = cache(6, heads, dim)
    plan = [([1, 15, 16, 17, 0, 33], [0] * 6),
            ([15, 1, 1, 30, 5, 0], [0] * 6),
            ([3, 16, 31, 2, 11, 100], [0] * 6),
            ([45, 0, 16, 15, 48, 1], [0, 0, 0, 0, 0, -1])]
    for counts, empty in plan:
        first = [-1 if e else n for e, n in zip(empty, c.lengths())]
        c.write(first, counts, *c.random_rows(sum(counts)), pad)
        assert c.st() == 0
        check_contents(c)
    c.write([3, 0, 20, 17, 63, 0], [2, 16, 9, 1, 1, 40], *c.random_rows(69), pad)  # again
    assert c.st() == 0
    check_contents(c)
    n = c.lengths()
    for first, counts in (([0] * 6, n),
                          ([5, 16, n[2] - 1, 0, n[4] // 16 * 16, 31], [n[0] - 9, 1, 1, 0, n[4] % 16, 2])):
        k, v = c.read(first, counts, pad)
        at = 0
        for s in range(6):
            for got, rows in zip((k, v), c.rows[s]):
                want = model.seen(rows[first[s]:first[s] + counts[s]])
                assert np.array_equal(got[at:at + counts[s]].astype(np.float64), want)
            at += counts[s]
    assert c.st() == 0


def test_rows_of_one_call_or_of_many_are_the_same_bits(cache):
    a, b = cache(2, 2, 64, seed=3), cache(2, 2, 64, seed=3)
    k, v = a.random_rows(90)
    a.write([0, 0], [53, 37], k, v)
    for i in range(53):
        n = [1, 1 if i < 37 else 0]
        pick = [i, 53 + i][:sum(n)]
        b.write([i, i], n, k[pick], v[pick])
    assert all(np.array_equal(x, y) for x, y in zip(a.raw(), b.raw()))
    # One row a stream, without offsets.
    b.write([53, -1], [1, 1], k[:2], v[:2], one=True)
    check_contents(b)
    assert b.st() == 0


def test_magnitudes_and_ties(cache):
    """Rows from nothing to the largest that fits, values on and beside the ties of their
    scale, rows of one sign."""
    c = cache(1, 2, 64, positions=600)
    rng = c.rng
    rows = []
    for spread in (0.0, 1e-9, 2.0 ** -18, 1e-4, 1.0, 1e3, 1.4e4):
        x = rng.standard_normal((16, 2, 64)).astype(np.float32) * np.float32(spread)
        rows += [np.clip(x, -57000, 57000), np.abs(x).clip(0, 57000), -np.abs(x).clip(0, 57000)]
    x = rng.standard_normal((64, 2, 64)).astype(np.float32)
    s = model.scale_of(x)
    n = rng.integers(-8, 7, x.shape) + 0.5
    top = np.abs(x) == np.abs(x).max(-1, keepdims=True)
    for step in (0, np.inf, -np.inf):
        y = (n * s[..., None]).astype(np.float32)
        y = np.nextafter(y, np.float32(step)) if step else y
        y = np.where(top, x, np.clip(y, x.min(-1, keepdims=True), x.max(-1, keepdims=True)))
        rows.append(y.astype(np.float32))
    k = np.concatenate(rows)
    c.write([0], [len(k)], k, k[::-1].copy())
    assert c.st() == 0
    check_contents(c)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 57200.0, -65400.0])
@pytest.mark.parametrize("which", [0, 1])
def test_a_row_that_does_not_fit_is_nan_and_said(cache, dim, bad, which):
    c = cache(2, 2, dim, positions=100)
    rows = c.random_rows(100)
    clean = [x.copy() for x in rows]
    at = [(0, 1, 3), (17, 0, dim - 1), (70, 1, dim // 2)]
    for r, h, d in at:
        rows[which][r, h, d] = bad
    c.write([0, 0], [40, 60], *rows)
    assert c.st() == 1
    k, v = c.read([0, 0], [40, 60])
    lost = np.zeros((100, 2), bool)
    for r, h, _ in at:
        lost[r, h] = True
    for got, x in zip((k, v), clean):
        assert np.isnan(got[lost]).all()
        assert np.array_equal(got[~lost].astype(np.float64), model.seen(x)[~lost])


class Attend:
    """An attention call over a cache's layer 1, its last counts[s] rows a stream."""

    def __init__(self, c, first, counts, group, pad=0, most=None, sums=None, spread=1.0):
        self.c, self.first, self.counts, self.group, self.pad = c, list(first), counts, group, pad
        self.n = counts or [1] * c.n
        self.total = sum(self.n)
        self.most = c.stride * BLOCK if most is None else most
        self.scale = c.dim ** -0.5
        self.width = c.heads * c.dim * group
        self.q = (c.rng.standard_normal((self.total, c.heads * group, c.dim)) * spread).astype(
            np.float32)
        wide = np.full((self.total, self.width + pad), np.nan, np.float32)
        wide[:, :self.width] = self.q.reshape(self.total, -1)
        self.dq = c.up(wide)
        self.mark = np.full((self.total + 2, self.width + pad), 5.5, np.float32)
        self.dout = c.up(self.mark)
        self.rows = c.call_rows(first, counts)
        self.sums, self.counted = None, sums
        if sums:
            shape = (c.n, c.heads, self.most + 3)
            self.before0 = np.exp(c.rng.standard_normal(shape)).astype(np.float32)
            for s, f in enumerate(first):  # what stands there for new rows is not read
                self.before0[s, :, max(0, f):] = np.nan
            self.before = c.up(self.before0)
            self.after0 = np.full(shape, 9.5, np.float32)
            self.after = c.up(self.after0)
            self.sums = c.pkg.PgpuKv4Sums(self.before.ptr, self.after.ptr, shape[-1], sums)
        self.bytes = c.lib.pgpu_kv4_attention_bytes(ctypes.byref(c.kv), ctypes.byref(self.rows),
                                                    group, self.most, 1 if sums else 0)
        self.work = c.up(np.full(max(16, self.bytes), 0xFF, np.uint8))

    def enqueue(self, stream=None):
        c = self.c
        return c.lib.pgpu_kv4_attention(
            stream, ctypes.byref(c.kv), 1, ctypes.byref(self.rows), self.dq.ptr,
            self.width + self.pad, self.group, self.scale, self.most, self.dout.ptr,
            self.width + self.pad, ctypes.byref(self.sums) if self.sums else None, self.work.ptr,
            self.bytes, c.status.ptr)

    def result(self):
        got = self.dout.download(self.mark.shape)
        assert (got[self.total:] == 5.5).all() and (got[:, self.width:] == 5.5).all()
        return got[:self.total, :self.width].reshape(self.q.shape)

    def added(self):
        return self.after.download(self.after0.shape)

    def run(self):
        self.dout.upload(self.mark)
        assert self.enqueue(), self.c.pkg.last_error(self.c.lib)
        return self.result()

    def check(self, got, lost=None, added=None):
        """Against the model, over what the cache holds; lost[s]: blocks of stream s that
        weigh nothing."""
        at = 0
        for s, (f, n) in enumerate(zip(self.first, self.n)):
            rows = slice(at, at + n)
            at += n
            if f < 0:
                assert (got[rows] == 0).all()
                if self.sums:
                    assert (added[s] == 9.5).all()
                continue
            k, v = (model.seen(x[:f + n]) for x in self.c.rows[s])
            there = np.ones(f + n, bool)
            for b in lost[s] if lost else []:
                there[b * BLOCK:(b + 1) * BLOCK] = False
            want, bound, weights, off = model.attention(self.q[rows], k, v, f, self.scale, there)
            worst = np.abs(got[rows] - want) - bound
            assert (worst <= 0).all(), (s, worst.max())
            if self.sums and n:
                w, b = model.sums(self.before0[s], weights, off, f, self.counted, self.c.heads)
                miss = np.abs(added[s, :, :f + n] - w) - b
                assert (miss <= 0).all(), (s, miss.max())
                assert (added[s, :, f + n:] == 9.5).all()


SHAPES = [(8, 64, 1), (2, 64, 3), (3, 128, 4), (1, 128, 1), (2, 64, 16), (5, 64, 2)]


@pytest.mark.parametrize("heads,dim,group", SHAPES)
@pytest.mark.parametrize("most", [None, 2048, 16384])
def test_one_row_a_stream(cache, heads, dim, group, most):
    """Contexts from one key on, at and beside the borders of blocks, 64 and 256 keys; an
    empty place; strides; with sums and without: the same bits."""
    c = cache(9, heads, dim, positions=1100)
    c.fill([1, 16, 17, 63, 64, 66, 257, 700, 1090])
    first = [n - 1 for n in c.lengths()]
    first[3] = -1
    a = Attend(c, first, None, group, pad=8, most=most)
    got = a.run()
    assert c.st() == 0
    a.check(got)
    b = Attend(c, first, None, group, most=most, sums=1)
    b.check(b.run(), added=b.added())
    assert c.st() == 0


@pytest.mark.parametrize("heads,dim,group", SHAPES)
@pytest.mark.parametrize("counted", [0, 1000, 30, 1])
def test_runs_of_rows(cache, heads, dim, group, counted):
    """Runs of one row to some hundreds, behind nothing, inside blocks and behind more than
    they are; one of none and an empty place; all rows counted, some, one."""
    c = cache(8, heads, dim, positions=400)
    plan = [(0, 1), (0, 16), (0, 33), (5, 130), (250, 17), (100, 0), (383, 1), (64, 64)]
    c.fill([f + n for f, n in plan])
    first, counts = [f for f, _ in plan], [n for _, n in plan]
    a = Attend(c, first, counts, group, pad=4, sums=counted)
    got = a.run()
    assert c.st() == 0
    a.check(got, added=a.added() if counted else None)
    first[3] = -1
    a = Attend(c, first, counts, group, sums=counted)
    a.check(a.run(), added=a.added() if counted else None)


@pytest.mark.parametrize("group,dim", [(1, 64), (2, 128)])
def test_a_long_run(cache, group, dim):
    c = cache(2, 1, dim, positions=1500)
    c.fill([1400, 901])
    a = Attend(c, [0, 600], [1400, 301], group, sums=5000)
    a.check(a.run(), added=a.added())
    assert c.st() == 0


@pytest.mark.parametrize("counts", [None, [20, 33, 150]])
@pytest.mark.parametrize("group,dim", [(1, 64), (3, 64), (4, 128)])
def test_uneven_rows_and_queries(cache, counts, group, dim):
    """Keys and values whose sizes differ by 2^24 from row to row and dim to dim, queries
    that are peaked: scores up to some hundreds."""
    c = cache(3, 2, dim, positions=300)
    k, v = c.random_rows(800)
    v *= np.exp2(c.rng.integers(-12, 13, (800, 2, 1))).astype(np.float32)
    v *= np.exp2(c.rng.integers(-3, 4, (1, 2, dim))).astype(np.float32)
    k *= np.exp2(c.rng.integers(-6, 4, (800, 2, 1))).astype(np.float32)
    c.write([0] * 3, [300, 201, 299], np.clip(k, -5e4, 5e4), np.clip(v, -5e4, 5e4))
    n = counts or [1] * 3
    first = [x - y for x, y in zip(c.lengths(), n)]
    a = Attend(c, first, counts, group, sums=40, spread=4.0)
    a.q *= np.exp2(c.rng.integers(-10, 3, a.q.shape)).astype(np.float32)
    a.dq.upload(a.q.reshape(a.total, -1))
    got = a.run()
    assert c.st() == 0
    a.check(got, added=a.added())


LOST = [[], [0], [1, 2, 3], [0, 1, 2, 3, 4, 5, 6, 7], [17], list(range(19))]


@pytest.mark.parametrize("most", [None, 8192])
@pytest.mark.parametrize("group,dim", [(1, 64), (3, 64), (1, 128)])
@pytest.mark.parametrize("counts", [None, [300] * 6, [20, 33, 300, 299, 16, 300]])
def test_a_block_outside_the_cache_weighs_nothing(cache, counts, group, dim, most):
    """Rows take their keys from the blocks that are there, whatever block 0 holds."""
    c = cache(6, 2, dim, positions=300)
    c.table[c.table == 0] = max(set(range(c.blocks)) - set(c.table.reshape(-1)))
    c.tables.upload(c.table)
    c.fill([300] * 6)
    table = c.table.copy()
    for s, blocks in enumerate(LOST):
        table[s, blocks] = [c.blocks + s, -1 - s][s % 2]
    c.tables.upload(table)
    n = counts or [1] * 6
    scales = c.scales.download(c.scales0.shape, np.uint16)
    for block0 in (0x3C00, 0x7E00, 0x7BFF):  # 1, NaN, the largest
        scales[1, 0] = block0
        c.scales.upload(scales)
        a = Attend(c, [300 - x for x in n], counts, group, most=most, sums=50)
        got = a.run()
        assert c.st() == 2
        a.check(got, LOST, a.added())


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("counts", [None, [20, 33]])
@pytest.mark.parametrize("group,dim", [(1, 64), (4, 128)])
def test_a_query_that_is_not_finite(cache, counts, group, dim, bad):
    """Its row does not come out finite, is said, and adds nothing; the other rows and heads
    come out as without it."""
    c = cache(2, 2, dim, positions=200)
    c.fill([193, 199])
    n = counts or [1, 1]
    for most in (None, 8192):
        a = Attend(c, [193 - n[0], 199 - n[1]], counts, group, most=most, sums=100)
        want = a.run()
        assert c.st() == 0
        row = n[0] - 1
        q = a.q.copy()
        q[row, 0, 3] = bad
        a.dq.upload(q.reshape(a.total, -1))
        got = a.run()
        assert c.st() == 1
        assert not np.isfinite(got[row, 0]).any()
        got[row, 0] = want[row, 0]
        assert np.array_equal(got, want)
        added = a.added()
        assert np.isfinite(added).all()
        # Without that row: the first head's sums as if its query were not there.
        _, _, w, off = model.attention(a.q[:n[0]], *(model.seen(x) for x in c.rows[0]),
                                       193 - n[0], a.scale)
        w[row, 0] = off[row, 0] = 0
        total, bound = model.sums(a.before0[0], w, off, 193 - n[0], 100, 2)
        assert (np.abs(added[0, :, :193] - total) <= bound).all()


@pytest.mark.parametrize("most", [None, 300, 8192])
@pytest.mark.parametrize("counts", [None, [20, 33]])
def test_scores_that_are_all_minus_infinity(cache, counts, most):
    """Products of large finite keys and queries that pass fp32: no weights are left, and
    that is said."""
    c = cache(2, 2, 64, positions=60)
    k, v = c.random_rows(115)
    c.write([0, 0], [55, 60], -np.abs(k) * np.float32(1e3), v)
    n = counts or [1, 1]
    a = Attend(c, [55 - n[0], 60 - n[1]], counts, 1, most=most, sums=9)
    a.q = np.abs(a.q) * np.float32(1e37)
    a.dq.upload(a.q.reshape(a.total, -1))
    got = a.run()
    assert c.st() == 1 and not np.isfinite(got).any()
    assert np.isfinite(a.added()[:, :, :50]).all()


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("group,dim", [(1, 64), (3, 128)])
@pytest.mark.parametrize("counts", [None, [90, 60, 33]])
def test_a_stored_row_that_is_not_finite_reaches_the_rows_that_see_it(cache, counts, group, dim, which):
    c = cache(3, 2, dim, positions=700)
    rows = c.random_rows(1000)
    c.write([0] * 3, [600, 300, 100], *rows)
    n = counts or [1] * 3
    first = [x - y for x, y in zip((600, 300, 100), n)]
    a = Attend(c, first, counts, group, sums=1000)
    want, added = a.run(), a.added()
    a.check(want, added=added)
    at = [555, 900]  # of stream 0, inside the run; of stream 1, past its end
    rows[which][at[0], 1, 7] = np.nan
    c.write([0] * 3, [600, 300, 100], *rows)
    assert c.st() == 1
    got = a.run()
    assert c.st() == 1
    sees = max(0, min(n[0], 555 - first[0]))  # rows before it
    hit = np.zeros(got.shape[:2], bool)
    hit[sees:n[0], group:] = True
    assert not np.isfinite(got[hit]).any()
    assert np.array_equal(got[~hit], want[~hit])
    assert np.isfinite(a.added()[:, :, :100]).all()


def test_calls_flag_what_they_cannot_cover(cache):
    """Streams outside their table or offsets, and block ids outside the cache: flagged and
    left out, the others written."""
    c = cache(4, 2, 64, positions=32)
    k, v = c.random_rows(40)
    before = c.raw()

    def go(first, counts, change=None):
        rows = c.call_rows(first, counts)
        if change:
            change(rows)
        dk, dv = c.up(k), c.up(v)
        assert c.lib.pgpu_kv4_write(None, ctypes.byref(c.kv), 1, ctypes.byref(rows), dk.ptr, dv.ptr,
                                    128, c.status.ptr)
        return c.st()
    assert go([30, -1, -1, -1], [3, 0, 0, 0]) == 2          # past the table
    assert go([0, -1, -1, -1], [20, 0, 0, 0], lambda r: setattr(r, "max_rows", 19)) == 2
    bad = c.up(np.array([0, 5, 3, 2 ** 31 - 1, -4], np.int32))
    assert go([0] * 4, [5, 5, 5, 5], lambda r: setattr(r, "offsets", bad.ptr) or
              setattr(r, "first", c.up(np.array([-1, 0, 0, 0], np.int32)).ptr)) == 2
    assert go([2 ** 31 - 1, -1, -1, -1], [2, 0, 0, 0]) == 2
    assert all(np.array_equal(x, y) for x, y in zip(before, c.raw()))
    table = c.table.copy()
    table[0, 0] = c.blocks
    c.tables.upload(table)
    assert go([0, 0, -1, -1], [17, 16, 0, 0]) == 2           # block 0 of stream 0 lost
    c.tables.upload(c.table)
    c.note([-1, 0, -1, -1], [17, 16, 0, 0], k, v)
    got = c.read([0, 0, 0, 0], [0, 16, 0, 0])
    assert np.array_equal(got[0].astype(np.float64), model.seen(k[17:33]))
    # Reads past what a stream holds; attention past max_positions.
    rows = c.call_rows([0, 0, 0, 0], [0, 17, 0, 0])
    out = c.up(np.full((17, 128), 3.5, np.float32))
    dl = c.up(np.array([0, 16, 0, 0], np.int32))
    assert c.lib.pgpu_kv4_read(None, ctypes.byref(c.kv), 1, ctypes.byref(rows), dl.ptr, out.ptr,
                               out.ptr, 128, c.status.ptr)
    assert c.st() == 2 and (out.download((17, 128)) == 3.5).all()
    for counts in (None, [1, 4, 1, 1]):
        n = counts or [1] * 4
        a = Attend(c, [-1, 16 - n[1], -1, -1], counts, 1, most=15, sums=3)
        got = a.run()
        assert c.st() == 2
        assert (got[n[0]:n[0] + n[1]] == 5.5).all() and (a.added() == 9.5).all()


@pytest.mark.parametrize("counts", [None, [20, 3, 40]])
def test_attention_replays_from_a_graph(cache, counts):
    """Captured once in global mode (nothing is allocated), replayed with the program's own
    work between; streams of one row grow between replays, as the captured indexes do."""
    c = cache(3, 2, 64, positions=400)
    lib, n = c.lib, counts or [1] * 3
    c.fill([150 + n[0], 1 + n[1], 300 + n[2]])
    a = Attend(c, [150, 1, 300], counts, 2, most=400, sums=30)
    a.before0 = np.abs(np.nan_to_num(a.before0, nan=1.0))
    a.before.upload(a.before0)
    stream, exec_ = ctypes.c_void_p(), ctypes.c_void_p()
    assert lib.pgpu_stream_create(ctypes.byref(stream))
    try:
        a.check(a.run(), added=a.added())
        assert lib.pgpu_graph_begin_global(stream)
        enqueued = a.enqueue(stream)
        ended = lib.pgpu_graph_end(stream, ctypes.byref(exec_))
        assert enqueued and ended, c.pkg.last_error(lib)
        for replay in range(4):
            a.dout.upload(a.mark)
            a.after.upload(a.after0)
            assert lib.pgpu_graph_launch(exec_, stream) and lib.pgpu_stream_sync(stream)
            got, added = a.result(), a.added()
            a.check(got, added=added)
            assert np.array_equal(got, a.run()) and np.array_equal(added, a.added()), replay
            if counts is None:
                c.write(c.lengths(), [1] * 3, *c.random_rows(3), one=True)
                a.first = [f + 1 for f in a.first]
                at = np.asarray(a.first, np.int32)
                assert lib.pgpu_copy_h2d(None, a.rows.first, at.ctypes.data, at.nbytes)
    finally:
        lib.pgpu_graph_destroy(exec_)
        lib.pgpu_stream_destroy(stream)


@pytest.mark.parametrize("counts", [None, [1, 33, 130]])
def test_attention_gives_the_same_bits_every_time(cache, counts):
    c = cache(3, 8, 64, positions=1500)
    n = counts or [1] * 3
    c.fill([700 + n[0], 17 + n[1], 1300 + n[2]])
    a = Attend(c, [700, 17, 1300], counts, 1, sums=77)
    want, added = a.run(), a.added()
    for _ in range(5):
        assert np.array_equal(a.run(), want) and np.array_equal(a.added(), added)


def test_sums_in_place_and_from_nothing(cache):
    """before = after, and before NULL, over three frames."""
    c = cache(2, 2, 64, positions=100)
    c.fill([70, 33])
    total = np.zeros((2, 2, 112))
    bound = np.zeros_like(total)
    held = c.up(np.full((2, 2, 112), np.nan, np.float32))
    for frame in range(3):
        a = Attend(c, [n - 1 for n in c.lengths()], None, 2, sums=1)
        a.sums = c.pkg.PgpuKv4Sums(held.ptr if frame else None, held.ptr, 112, 1)
        got = a.run()
        for s, n in enumerate(c.lengths()):
            k, v = (model.seen(x) for x in c.rows[s])
            _, _, w, off = model.attention(a.q[s:s + 1], k, v, n - 1, a.scale)
            total[s, :, :n], b = model.sums(total[s] if frame else None, w, off, n - 1, 1, 2)
            bound[s, :, :n] += b
            assert np.isfinite(got).all()
            have = held.download(total.shape)
            assert (np.abs(have[s, :, :n] - total[s, :, :n]) <= bound[s, :, :n]).all()
        c.write(c.lengths(), [1, 1], *c.random_rows(2))


class Evict:
    """An eviction over both layers of a cache."""

    def __init__(self, c, keep, first, newest, sums, elsewhere=None):
        self.c, self.k, self.first, self.newest, self.sums0 = c, keep, first, newest, sums
        self.sums = c.up(sums)
        self.kept0 = np.full((2, c.n, c.heads, keep), -7, np.int32)
        self.kept = c.up(self.kept0)
        self.lengths = c.up(np.asarray(c.lengths(), np.int32))
        self.to_sums = self.sums
        self.to = None
        if elsewhere is not None:
            self.to = c.up(elsewhere)
            self.to_sums = c.up(np.full(sums.shape, 4.5, np.float32))

    def enqueue(self, stream=None):
        c = self.c
        return c.lib.pgpu_kv4_evict(stream, ctypes.byref(c.kv), 0, 2, c.tables.ptr,
                                    self.to.ptr if self.to else None, c.stride, self.lengths.ptr,
                                    c.n, self.k, self.first, self.newest, self.sums.ptr,
                                    self.to_sums.ptr, self.sums0.shape[-1], self.kept.ptr,
                                    c.status.ptr)


def both_layers(c):
    """Layer 0 holds what layer 1 does."""
    for b, a0, t in ((c.values, c.values0, np.uint8), (c.scales, c.scales0, np.uint16)):
        a = b.download(a0.shape, t)
        a[0] = a[1]
        b.upload(a)


def tied_sums(c, stride):
    x = np.exp(2 * c.rng.standard_normal((2, c.n, c.heads, stride))).astype(np.float32)
    x = np.where(x < 0.5, np.round(x * 8) / 8, x).astype(np.float32)
    x[:, :, 0, ::5] = 0
    x[:, :, -1] = 1.5  # all equal
    return x


def check_evicted(c, e, table):
    """Layer by layer and head by head: what is kept, its sums, the rows' bits."""
    kept = e.kept.download(e.kept0.shape, np.int32)
    after = e.to_sums.download(e.sums0.shape)
    old = [[model.quantise(x) for x in r] for r in c.rows]
    values, scales = c.raw()
    for layer in range(2):
        for s, n in enumerate(c.lengths()):
            m = min(n, e.k)
            for h in range(c.heads):
                want = model.keep(e.sums0[layer, s, h], n, e.k, e.first, e.newest)
                assert np.array_equal(kept[layer, s, h, :m], want), (layer, s, h)
                assert (kept[layer, s, h, m:] == -1).all()
                w = e.sums0[layer, s, h][want]
                assert np.array_equal(after[layer, s, h, :m], np.where(np.isnan(w), 0, w))
                for b in range(-(-m // BLOCK)):
                    lo, hi = b * BLOCK, min(m, b * BLOCK + BLOCK)
                    rows = want[lo:hi]
                    pad = ((0, BLOCK - hi + lo), (0, 0))
                    (qk, sk), (qv, sv) = old[s]
                    new = model.tile(np.pad(qk[rows, h], pad), np.pad(qv[rows, h], pad))
                    mask = model.tile(*(np.repeat((np.arange(BLOCK) < hi - lo)[:, None] * -1,
                                                  c.dim, 1) for _ in range(2)))
                    got = values[layer, table[s][b], h]
                    assert np.array_equal(got & mask, new & mask), (layer, s, h, b)
                    pair = np.stack([sk[rows, h], sv[rows, h]], -1).astype(np.float16)
                    assert np.array_equal(scales[layer, table[s][b], h, :, :hi - lo],
                                          pair.view(np.uint16).transpose(1, 0, 2))
    return kept


@pytest.mark.parametrize("heads,dim", [(8, 64), (3, 128)])
@pytest.mark.parametrize("keep,first,newest", [(100, 4, 30), (1, 0, 0), (64, 64, 0), (64, 0, 64),
                                               (257, 1, 1), (48, 17, 31), (2500, 0, 7)])
@pytest.mark.parametrize("elsewhere", [False, True])
def test_evictions_keep_what_weighs_most(cache, heads, dim, keep, first, newest, elsewhere):
    """Streams of none, one, less than keep, one more, and many; ties, all equal, NaN."""
    c = cache(7, heads, dim, positions=1400)
    c.fill([0, 1, 47, keep % 1300, min(keep + 1, 1390), 1100, 1391])
    both_layers(c)
    sums = tied_sums(c, 1400)
    sums[0, 5, 0, 3:400:7] = np.nan
    sums[1, 6, 0] = -sums[1, 6, 0]
    table = c.table
    if elsewhere:  # stream 5's kept rows into blocks that no row is in; the others in place
        free = [b for b in range(c.blocks) if b not in c.table] + list(c.table[0]) + list(c.table[1, 1:])
        table = c.table.copy()
        need = -(-min(keep, 1100) // BLOCK)
        table[5, :need] = free[:need]
    e = Evict(c, keep, first, newest, sums, table if elsewhere else None)
    source = c.raw()
    assert e.enqueue(), c.pkg.last_error(c.lib)
    assert c.st() == 0
    check_evicted(c, e, table)
    if elsewhere and keep < 1100:  # the source blocks of stream 5 are as they were
        values, scales = c.raw()
        assert np.array_equal(values[:, c.table[5]], source[0][:, c.table[5]])
        assert np.array_equal(scales[:, c.table[5]], source[1][:, c.table[5]])


def test_evictions_in_place_touch_nothing_else(cache):
    c = cache(3, 2, 64, positions=600)
    c.fill([500, 20, 333])
    both_layers(c)
    before = c.raw()
    e = Evict(c, 100, 3, 20, tied_sums(c, 600))
    assert e.enqueue()
    assert c.st() == 0
    check_evicted(c, e, c.table)
    after = c.raw()
    mine = set(c.table[0, :7]) | set(c.table[2, :7])
    rest = [b for b in range(c.blocks) if b not in mine]
    for x, y in zip(before, after):
        assert np.array_equal(x[:, rest], y[:, rest])


def test_evictions_leave_out_what_they_cannot_cover(cache):
    """Lengths past the table or the sums, block ids outside the cache, empty places: left as
    they are; the others shrunk."""
    c = cache(6, 2, 64, positions=300)
    c.fill([300, 200, 250, 300, 299, 120])
    both_layers(c)
    before = c.raw()
    e = Evict(c, 64, 2, 10, tied_sums(c, 304))
    lengths = np.array([c.stride * 16 + 1, -1, 305, 300, 299, 120], np.int32)
    e.lengths.upload(lengths)
    table = c.table.copy()
    table[3, 11] = c.blocks
    table[4, 0] = -5
    c.tables.upload(table)
    assert e.enqueue()
    assert c.st() == 2
    kept = e.kept.download(e.kept0.shape, np.int32)
    assert (kept[:, :5] == -1).all()
    c.tables.upload(c.table)
    after = c.raw()
    for x, y in zip(before, after):
        for s in range(5):
            assert np.array_equal(x[:, c.table[s]], y[:, c.table[s]])
    sums = e.sums.download(e.sums0.shape)
    assert np.array_equal(sums[:, :5], e.sums0[:, :5])
    for h in range(2):
        assert np.array_equal(kept[1, 5, h], model.keep(e.sums0[1, 5, h], 120, 64, 2, 10))


def test_a_server_s_life_with_a_budget(cache, lib):
    """The operators as a server uses them: prompts written and attended with their weights
    summed, frames one at a time, evictions whenever a stream has passed its budget, and on,
    every result against a model that holds the same rows."""
    heads, group, dim, budget, room = 2, 2, 64, 96, 32
    c = cache(3, heads, dim, positions=budget + room + 80)
    held = c.up(np.zeros((3, heads, c.stride * BLOCK), np.float32))
    kept = c.up(np.zeros((3, heads, budget), np.int32))
    # What each stream and head holds: rows as they were read back.
    hold = [[[np.zeros((0, dim))] * 2 for _ in range(heads)] for _ in range(3)]
    sums = [[np.zeros(0) for _ in range(heads)] for _ in range(3)]
    length = [0, 0, 0]

    def step(counts, one):
        k, v = c.random_rows(sum(counts))
        first = list(length)
        c.write(first, counts, k, v, one=one)
        a = Attend(c, first, None if one else counts, group, sums=8)
        a.sums = c.pkg.PgpuKv4Sums(held.ptr, held.ptr, c.stride * BLOCK, 8)
        got = a.run()
        assert c.st() == 0
        have = held.download((3, heads, c.stride * BLOCK))
        at = 0
        for s, n in enumerate(counts):
            f = first[s]
            for h in range(heads):
                hold[s][h] = [np.concatenate([old, model.seen(new[at:at + n, h])])
                              for old, new in zip(hold[s][h], (k, v))]
                q = a.q[at:at + n, h * group:(h + 1) * group]
                kk, vv = (x[:, None] for x in hold[s][h])
                want, bound, w, off = model.attention(q, kk, vv, f, a.scale)
                assert (np.abs(got[at:at + n, h * group:(h + 1) * group] - want) <= bound).all()
                total, b = model.sums(np.concatenate([sums[s][h], np.zeros(n)])[None], w, off, f, 8, 1)
                assert (np.abs(have[s, h, :f + n] - total[0]) <= b[0]).all()
                sums[s][h] = have[s, h, :f + n].astype(np.float64)
            length[s] += n
            at += n

    def evict():
        dl = c.up(np.asarray(length, np.int32))
        one = c.pkg.PgpuKv4(c.kv.values, c.kv.scales, 2, heads, dim, c.blocks)
        assert lib.pgpu_kv4_evict(None, ctypes.byref(one), 1, 1, c.tables.ptr, None, c.stride,
                                  dl.ptr, 3, budget, 4, 24, held.ptr, held.ptr, c.stride * BLOCK,
                                  kept.ptr, c.status.ptr)
        assert c.st() == 0
        have = kept.download((3, heads, budget), np.int32)
        for s in range(3):
            m = min(length[s], budget)
            for h in range(heads):
                want = model.keep(sums[s][h].astype(np.float32), length[s], budget, 4, 24)
                assert np.array_equal(have[s, h, :m], want)
                hold[s][h] = [x[want] for x in hold[s][h]]
                sums[s][h] = sums[s][h][want]
            length[s] = m

    step([150, 17, 77], False)
    evict()
    for frame in range(70):
        step([1, 1, 1], True)
        if max(length) > budget + room:
            evict()
    step([9, 40, 1], False)
    evict()
    step([1, 1, 1], True)
    assert max(length) <= budget + 1 and min(length) > 60
