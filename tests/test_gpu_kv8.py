"""The 8-bit paged KV cache on the GPU against a plain model in 64 bits: rows
written in any number of calls, rotated and normalised on their way, read back,
and attended to; one row a stream and runs of rows, odd and empty lengths,
strides, grouped heads, both head widths, bounds that are broken, graphs."""
import ctypes

import numpy as np
import pytest

import kv8_model as model

pytestmark = pytest.mark.gpu
BLOCK = 16


class Cache:
    """A cache of 2 layers with its tables, and the rows that were written to
    layer 1 of it (layer 0 stays as it was made)."""

    def __init__(self, lib, pkg, streams, heads=8, dim=64, positions=200, seed=1):
        self.lib, self.pkg, self.n, self.heads, self.dim = lib, pkg, streams, heads, dim
        self.rng = np.random.default_rng(seed)
        self.stride = -(-positions // BLOCK)
        self.blocks, self.slots = streams * self.stride + 2, streams + 1
        self.keep = []
        rng = self.rng
        self.values0 = rng.integers(-128, 128, (2, self.blocks, heads, 2, BLOCK * dim), np.int8)
        self.scales0 = rng.standard_normal((2, self.blocks, heads, 2)).astype(np.float32)
        self.open0 = rng.standard_normal((2, self.slots, heads, 2, BLOCK, dim)).astype(np.float32)
        self.values, self.scales, self.open = (self.up(a) for a in
                                               (self.values0, self.scales0, self.open0))
        self.table = rng.permutation(self.blocks)[:streams * self.stride].astype(np.int32)
        self.table = self.table.reshape(streams, self.stride)
        self.slot = rng.permutation(self.slots)[:streams].astype(np.int32)
        self.tables, self.slotd = self.up(self.table), self.up(self.slot)
        self.status = self.up(np.zeros(1, np.int32))
        self.kv = pkg.PgpuKv8(self.values.ptr, self.scales.ptr, self.open.ptr, 2, heads, dim,
                              self.blocks, self.slots)
        self.rows = [[np.zeros((0, heads, dim), np.float32)] * 2 for _ in range(streams)]

    def up(self, a):
        a = np.ascontiguousarray(a)
        b = self.pkg.DeviceBuffer(self.lib, max(16, a.nbytes))
        if a.nbytes:
            b.upload(a)
        self.keep.append(b)
        return b

    def call_rows(self, first, counts=None):
        """pgpu_kv8_rows of counts[s] rows a stream from first[s] on (None: one)."""
        first = np.asarray(first, np.int32)
        if counts is None:
            return self.pkg.PgpuKv8Rows(self.tables.ptr, self.stride, self.slotd.ptr,
                                        self.up(first).ptr, None, self.n, self.n, 1)
        offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        return self.pkg.PgpuKv8Rows(self.tables.ptr, self.stride, self.slotd.ptr,
                                    self.up(first).ptr, self.up(offsets).ptr, self.n,
                                    int(offsets[-1]), int(max(counts)))

    def st(self):
        """The status word, and clears it."""
        s = int(self.status.download((1,), np.int32)[0])
        self.status.upload(np.zeros(1, np.int32))
        return s

    def write(self, first, counts, k, v, pad=0, one=False):
        """k, v: [rows][heads][dim] fp32."""
        width = self.heads * self.dim
        rows = self.call_rows(first, None if one else counts)
        wide = np.full((2, max(1, len(k)), width + pad), np.nan, np.float32)
        wide[0, :len(k), :width], wide[1, :len(k), :width] = (k.reshape(len(k), -1),
                                                               v.reshape(len(v), -1))
        dk, dv = self.up(wide[0]), self.up(wide[1])
        assert self.lib.pgpu_kv8_write(None, ctypes.byref(self.kv), 1, ctypes.byref(rows), dk.ptr,
                                       dv.ptr, width + pad, self.status.ptr), \
            self.pkg.last_error(self.lib)
        self.note(first, counts, k, v)

    def note(self, first, counts, k, v):
        at = 0
        for s, (f, n) in enumerate(zip(first, counts)):
            if f >= 0:
                assert len(self.rows[s][0]) == f
                self.rows[s] = [np.concatenate([self.rows[s][0], k[at:at + n]]),
                                np.concatenate([self.rows[s][1], v[at:at + n]])]
            at += n

    def lengths(self):
        return [len(r[0]) for r in self.rows]

    def random_rows(self, count):
        gain = np.exp(self.rng.standard_normal((1, self.heads, self.dim)) * 0.5)
        return [(self.rng.standard_normal((count, self.heads, self.dim)) * gain).astype(np.float32)
                for _ in range(2)]

    def fill(self, lengths):
        k, v = self.random_rows(sum(lengths))
        self.write([0] * self.n, lengths, k, v)

    def read(self, first, counts, pad=0, lengths=None):
        width = self.heads * self.dim
        rows = self.call_rows(first, counts)
        total = sum(counts)
        mark = np.full((total + 3, width + pad), 7.5, np.float32)
        dk, dv = self.up(mark), self.up(mark)
        dl = self.up(np.asarray(self.lengths() if lengths is None else lengths, np.int32))
        assert self.lib.pgpu_kv8_read(None, ctypes.byref(self.kv), 1, ctypes.byref(rows), dl.ptr,
                                      dk.ptr, dv.ptr, width + pad, self.status.ptr)
        k, v = dk.download(mark.shape), dv.download(mark.shape)
        for x in (k, v):  # rows behind the last and columns past the width: left as they were
            assert (x[total:] == 7.5).all() and (x[:, width:] == 7.5).all()
        return [x[:total, :width].reshape(total, self.heads, self.dim) for x in (k, v)]

    def raw(self):
        return (self.values.download(self.values0.shape, np.int8),
                self.scales.download(self.scales0.shape), self.open.download(self.open0.shape))

    def want(self):
        """What the buffers hold, from the rows written to layer 1."""
        values, scales, opened = self.values0.copy(), self.scales0.copy(), self.open0.copy()
        for s, pair in enumerate(self.rows):
            for b in range(len(pair[0]) // BLOCK):
                q = [model.quantise(x[b * BLOCK:(b + 1) * BLOCK].transpose(1, 0, 2)) for x in pair]
                for h in range(self.heads):
                    values[1, self.table[s, b], h] = model.tile(q[0][0][h], q[1][0][h])
                scales[1, self.table[s, b]] = np.stack([q[0][1], q[1][1]], -1)
            for i in range(2):  # row j of the slot: the newest row written at a position % 16 = j
                for p, row in enumerate(pair[i]):
                    opened[1, self.slot[s], :, i, p % BLOCK] = row
        return values, scales, opened

    def check_slots(self, opened):
        """The newest block's rows of every slot."""
        for s, pair in enumerate(self.rows):
            n = len(pair[0])
            lo = max(0, n - 1) // BLOCK * BLOCK
            for i in range(2):
                got = opened[1, self.slot[s], :, i, :n - lo]
                assert np.array_equal(got, pair[i][lo:].transpose(1, 0, 2)), (s, i)

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
    values, scales, opened = c.raw()
    want = c.want()
    assert np.array_equal(values, want[0])
    assert np.array_equal(scales.view(np.uint32), want[1].view(np.uint32))
    c.check_slots(opened)
    # Layer 0, and the slots of no stream, are left as they were.
    assert np.array_equal(opened[0], c.open0[0])
    free = [i for i in range(c.slots) if i not in c.slot]
    assert np.array_equal(opened[1, free], c.open0[1, free])


@pytest.mark.parametrize("heads,dim", [(8, 64), (3, 128), (1, 64)])
@pytest.mark.parametrize("pad", [0, 20])
def test_rows_written_in_runs_are_the_model_s_bits(cache, heads, dim, pad):
    """Runs that start and end inside blocks, at their borders, of one row and
    of none, with an empty place in the batch."""
    c = cache(6, heads, dim)
    plan = [([1, 15, 16, 17, 0, 33], [0] * 6),
            ([15, 1, 1, 30, 5, 0], [0] * 6),
            ([3, 16, 31, 2, 11, 100], [0] * 6),
            ([45, 0, 16, 15, 48, 1], [0, 0, 0, 0, 0, -1])]
    for counts, empty in plan:
        first = [-1 if e else n for e, n in zip(empty, c.lengths())]
        k, v = c.random_rows(sum(counts))
        c.write(first, counts, k, v, pad)
        assert c.st() == 0
        check_contents(c)
    n = c.lengths()
    k, v = c.read([0] * 6, n, pad)
    at = 0
    for s in range(6):
        for got, rows in ((k, c.rows[s][0]), (v, c.rows[s][1])):
            assert np.array_equal(got[at:at + n[s]].astype(np.float64), model.seen(rows))
        at += n[s]
    # Parts: from inside a block to inside another, one row, none, the newest block only.
    first = [5, 16, max(n[2] - 1, 0), 0, (n[4] - 1) // 16 * 16, 31]
    counts = [n[0] - 9, 1, 1, 0, n[4] - first[4], 2]
    k, v = c.read(first, counts)
    at = 0
    for s in range(6):
        for got, rows in ((k, c.rows[s][0]), (v, c.rows[s][1])):
            assert np.array_equal(got[at:at + counts[s]].astype(np.float64),
                                  model.seen(rows)[first[s]:first[s] + counts[s]])
        at += counts[s]
    assert c.st() == 0


def test_one_row_a_stream_gives_the_bits_of_runs(cache):
    c = cache(3, 2, 64, positions=64)
    c.fill([0, 14, 31])
    for _ in range(33):
        k, v = c.random_rows(3)
        c.write(c.lengths(), [1, 1, 1], k, v, one=True)
    assert c.st() == 0
    check_contents(c)


def test_values_at_the_ends_of_the_range(cache):
    """Zero blocks, subnormal and very large values, every tie, and one value
    that is not finite: only its block is lost, and that is said."""
    c = cache(7, 1, 64, positions=40)
    k, v = [x.reshape(7, 40, 1, 64) for x in c.random_rows(280)]
    k[0, :16] = 0
    v[0, :16] = -0.0
    k[1, :16] *= np.float32(1e-42)
    v[1, :16] *= np.float32(3e-38)
    k[2, :16] = np.float32(3.4028234e38) * np.sign(k[2, :16])
    s = float(model.scale_of(k[3, :16].transpose(1, 0, 2))[0])
    ties = (np.arange(-126, 126) + 0.5) * s
    top = np.abs(k[3, :16]).max()
    k[3, 1:5] = np.concatenate([ties, [0] * 4]).reshape(4, 1, 64)
    k[3, 0, 0, 0] = top
    k, v = k.reshape(280, 1, 64), v.reshape(280, 1, 64)
    c.write([0] * 7, [40] * 7, k, v)
    assert c.st() == 0
    check_contents(c)
    back = c.read([0] * 7, [40] * 7)
    assert np.isfinite(back[0]).all() and np.isfinite(back[1]).all()
    bad_k, bad_v = c.random_rows(7)
    bad_k, bad_v = np.repeat(bad_k, 8, 0), np.repeat(bad_v, 8, 0)
    bad_k[3, 0, 5], bad_v[8 + 7, 0, 9], bad_k[16, 0, 0] = np.nan, np.inf, -np.inf
    c.write([40] * 7, [8] * 7, bad_k, bad_v)
    assert c.st() == 1
    values, scales, _ = c.raw()
    for st in range(7):
        nan = np.isnan(scales[1, c.table[st, 2], 0])
        assert list(nan) == [st in (0, 2), st == 1]
    # A row of an open block that is not finite is said at once.
    bad = c.random_rows(7)
    bad[1][2, 0, 0] = np.inf
    c.rows = [[x[:40] for x in r] for r in c.rows]
    c.write([40] * 7, [1] * 7, *bad)
    assert c.st() == 1


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("heads,group,dim", [(8, 1, 64), (2, 3, 128), (1, 16, 64)])
def test_rotated_rows(cache, pkg, lib, heads, group, dim, norm):
    """Queries are off the 64-bit result by at most an fp32 rounding; keys and
    values are stored as their fp32 values would be."""
    c = cache(5, heads, dim)
    rng = c.rng
    positions, eps, scale = 224, 1e-5, np.float32(0.125 * 1.1)
    angle = np.arange(positions)[:, None] * 10000.0 ** (-2 * np.arange(dim // 2) / dim)
    rope = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    weights = [(1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) if norm else None
               for _ in range(2)]
    dev = [c.up(w) if norm else None for w in weights]
    drope, pad = c.up(rope), 12
    width = heads * dim * (2 + group)
    for counts, one in (([1, 20, 0, 16, 47], False), ([1] * 5, True), ([17, 1, 31, 5, 90], False)):
        first = c.lengths()
        total = sum(counts)
        qkv = np.full((total, width + pad), np.nan, np.float32)
        qkv[:, :width] = rng.standard_normal((total, width)) * np.exp(rng.standard_normal(width))
        rows = c.call_rows(first, None if one else counts)
        mark = np.full((total + 2, heads * group * dim), 3.25, np.float32)
        dq, dx = c.up(mark), c.up(qkv)
        assert lib.pgpu_kv8_rotate_write(
            None, ctypes.byref(c.kv), 1, ctypes.byref(rows), dx.ptr, width + pad, group,
            dev[0] and dev[0].ptr, dev[1] and dev[1].ptr, eps, drope.ptr, positions,
            float(scale), dq.ptr, c.status.ptr), pkg.last_error(lib)
        assert c.st() == 0
        got = dq.download(mark.shape)
        assert (got[total:] == 3.25).all()
        at = np.concatenate([np.arange(f, f + n) for f, n in zip(first, counts)])
        x = qkv[:, :width].reshape(total, -1, dim)
        q = model.turn(x[:, :heads * group], weights[0], eps, rope[at]) * float(scale)
        assert (np.abs(got[:total].reshape(q.shape) - q) <= 2.0 ** -24 * np.abs(q) + 1e-44).all()
        k = model.turn(x[:, heads * group:heads * (group + 1)], weights[1], eps, rope[at])
        c.note(first, counts, k.astype(np.float32), x[:, heads * (group + 1):])
        check_contents(c)
    # A stream past the rope table is left out and flagged.
    rows = c.call_rows([positions - 1, -1, -1, -1, -1], [2, 0, 0, 0, 0])
    c.kv.slots = c.slots
    before = c.raw()
    assert lib.pgpu_kv8_rotate_write(None, ctypes.byref(c.kv), 1, ctypes.byref(rows), dx.ptr,
                                     width + pad, group, None, None, eps, drope.ptr, positions,
                                     1.0, dq.ptr, c.status.ptr)
    assert c.st() == 2
    assert all(np.array_equal(x, y) for x, y in zip(before, c.raw()))


@pytest.mark.parametrize("heads,dim", [(8, 64), (3, 128)])
def test_close_stores_full_slots_of_every_layer(cache, lib, heads, dim):
    c = cache(5, heads, dim, positions=64)
    positions = [15, 14, 63, 16, -1]
    d = c.up(np.asarray(positions, np.int32))
    assert lib.pgpu_kv8_close(None, ctypes.byref(c.kv), 0, 2, c.tables.ptr, c.stride, c.slotd.ptr,
                              d.ptr, 5, c.status.ptr)
    assert c.st() == 0
    values, scales, opened = c.raw()
    assert np.array_equal(opened, c.open0)
    want_v, want_s = c.values0.copy(), c.scales0.copy()
    for s in (0, 2):
        b = c.table[s, positions[s] // 16]
        for layer in range(2):
            q, sc = model.quantise(c.open0[layer, c.slot[s]])
            for h in range(heads):
                want_v[layer, b, h] = model.tile(q[h, 0], q[h, 1])
            want_s[layer, b] = sc
    assert np.array_equal(values, want_v) and np.array_equal(scales, want_s)
    # Past the table: flagged, nothing written.
    d = c.up(np.asarray([16 * c.stride + 15, -1, -1, -1, -1], np.int32))
    assert lib.pgpu_kv8_close(None, ctypes.byref(c.kv), 0, 2, c.tables.ptr, c.stride, c.slotd.ptr,
                              d.ptr, 5, c.status.ptr)
    assert c.st() == 2 and np.array_equal(c.raw()[0], values)


# ------------------------------------------------------------------ attention


class Attend:
    """One attention call over a cache: its buffers, the call, and the result."""

    def __init__(self, c, first, counts, group, most=None, pad=0, scale=None, seed=3):
        self.c, self.first, self.group, self.pad = c, first, group, pad
        self.counts = [1] * c.n if counts is None else counts
        self.total = sum(self.counts)
        self.scale = c.dim ** -0.5 if scale is None else scale
        self.width = c.heads * group * c.dim
        rng = np.random.default_rng(seed)
        self.q = rng.standard_normal((self.total, c.heads * group, c.dim)).astype(np.float32)
        wide = np.full((max(1, self.total), self.width + pad), np.nan, np.float32)
        wide[:self.total, :self.width] = self.q.reshape(self.total, -1)
        self.rows = c.call_rows(first, counts)
        self.most = most or max([f + n for f, n in zip(first, self.counts)] + [1])
        self.dq = c.up(wide)
        self.mark = np.full((self.total + 3, self.width + pad), 5.5, np.float32)
        self.dout = c.up(self.mark)
        self.bytes = c.lib.pgpu_kv8_attention_bytes(ctypes.byref(c.kv), ctypes.byref(self.rows),
                                                    group, self.most)
        # Whatever a workspace held before: here bits that are NaN as floats.
        self.work = c.up(np.full(max(16, self.bytes), 0xFF, np.uint8))

    def enqueue(self, stream=None):
        c = self.c
        return c.lib.pgpu_kv8_attention(
            stream, ctypes.byref(c.kv), 1, ctypes.byref(self.rows), self.dq.ptr,
            self.width + self.pad, self.group, self.scale, self.most, self.dout.ptr,
            self.width + self.pad, self.work.ptr, self.bytes, c.status.ptr)

    def result(self):
        x = self.dout.download(self.mark.shape)
        assert (x[self.total:] == 5.5).all() and (x[:, self.width:] == 5.5).all()
        return x[:self.total, :self.width].reshape(self.q.shape)

    def run(self):
        assert self.enqueue(), self.c.pkg.last_error(self.c.lib)
        return self.result()

    def check(self, got, near=2e-6):
        """Every element within the model's bound, and the whole within `near`
        (independent roundings: 2^-22 of the largest q element, of dim 64..128
        elements of N(0, 1), gives scores that are off by some 4e-7)."""
        c, at, off, norm = self.c, 0, 0.0, 0.0
        for s, n in enumerate(self.counts):
            if n and self.first[s] < 0:
                assert (got[at:at + n] == 0).all()
            elif n:
                length = self.first[s] + n
                k, v = (model.seen(x[:length]) for x in c.rows[s])
                want, bound = model.attention(self.q[at:at + n], k, v, self.first[s], self.scale)
                err = np.abs(got[at:at + n] - want)
                assert (err <= bound).all(), (s, self.first[s], n, float((err / bound).max()))
                off, norm = off + (err ** 2).sum(), norm + (want ** 2).sum()
            at += n
        assert off <= near ** 2 * norm, (off / norm) ** 0.5
        assert c.st() == 0


@pytest.mark.parametrize("heads,group,dim", [(8, 1, 64), (2, 2, 64), (3, 4, 128), (1, 5, 64),
                                             (2, 8, 128), (1, 16, 64)])
def test_attention_of_one_row_a_stream(cache, heads, group, dim):
    lengths = [1, 2, 15, 16, 17, 64, 65, 0, 255, 256, 257, 600]
    c = cache(len(lengths), heads, dim, positions=600)
    c.fill(lengths)
    first = [n - 1 for n in lengths]  # -1: the empty place
    a = Attend(c, first, None, group, pad=8)
    a.check(a.run())
    # A longer bound, and another scale.
    b = Attend(c, first, None, group, most=c.stride * 16, scale=0.6, seed=4)
    b.check(b.run(), near=1e-5)


@pytest.mark.parametrize("heads,group,dim", [(8, 1, 64), (2, 2, 64), (2, 4, 128), (1, 16, 64),
                                             (3, 3, 64)])
def test_attention_of_runs_of_rows(cache, heads, group, dim):
    """Runs from the first position and after held ones, across blocks, of one
    row and none, next to an empty place with rows."""
    before = [0, 0, 5, 16, 40, 131, 0, 200, 300]
    counts = [1, 16, 27, 16, 0, 90, 7, 33, 2]
    c = cache(len(before), heads, dim, positions=310)
    c.fill(before)
    k, v = c.random_rows(sum(counts))
    first = [-1 if i == 6 else f for i, f in enumerate(before)]
    c.write(first, counts, k, v)
    c.rows[6] = [np.zeros((0, heads, dim), np.float32)] * 2
    a = Attend(c, first, counts, group, pad=4)
    a.check(a.run())


@pytest.mark.parametrize("counts", [None, [1], [3], [16], [40], [130]])
def test_attention_over_a_long_context(cache, counts):
    """Few rows over thousands of keys: the keys are dealt to work-groups and joined."""
    n = 1 if counts is None else counts[0]
    c = cache(1, 2, 64, positions=5003)
    c.fill([5003 - n])
    c.write([5003 - n], [n], *c.random_rows(n))
    a = Attend(c, [5003 - n], counts, 2)
    a.check(a.run())


@pytest.mark.parametrize("rows", [None, [40, 40, 40]])
def test_attention_where_scales_and_scores_differ_widely(cache, rows):
    """Keys that take all the weight late or early, blocks whose values are
    2^30 times their neighbours', and scores in the hundreds."""
    c = cache(3, 2, 64, positions=300)
    for n in (260, 40):
        k, v = c.random_rows(3 * n)
        k, v = k.reshape(3, n, 2, 64), v.reshape(3, n, 2, 64)
        k[0] *= np.float32(40)
        v[1] *= np.float32(2.0) ** (30 * (np.arange(n) // 16 % 3 - 1))[:, None, None]
        k[2, ::37] *= np.float32(60)
        c.write(c.lengths(), [n] * 3, k.reshape(-1, 2, 64), v.reshape(-1, 2, 64))
    first = [299] * 3 if rows is None else [260] * 3
    a = Attend(c, first, rows, 1)
    # Scores in the hundreds lose 8 more bits: the elements' bounds say how much.
    a.check(a.run(), near=1e-3)


def test_rows_past_the_newest_position_are_not_read_as_keys(cache):
    """The open slot's rows and the blocks' bytes past a stream's length are
    NaN, infinite or another stream's; a row of one key returns its value."""
    c = cache(4, 2, 64, positions=100)
    c.fill([1, 18, 35, 90])
    opened = c.open.download(c.open0.shape)
    for s, n in enumerate(c.lengths()):
        opened[1, c.slot[s], :, :, (n - 1) % 16 + 1:] = [[np.nan] * 64, [np.inf] * 64][s % 2]
    c.open.upload(opened)
    scales = c.scales.download(c.scales0.shape)
    for s, n in enumerate(c.lengths()):
        scales[1, c.table[s, (n - 1) // 16:]] = np.nan
    c.scales.upload(scales)
    for counts in (None, [1, 3, 19, 40]):
        n = counts or [1] * 4
        first = [x - y for x, y in zip(c.lengths(), n)]
        a = Attend(c, first, counts, 2)
        got = a.run()
        a.check(got)
        assert np.array_equal(got[0], np.repeat(c.rows[0][1][0], 2, 0))


def test_attention_flags_what_it_cannot_cover(cache):
    c = cache(4, 2, 64, positions=100)
    c.fill([40, 33, 90, 17])
    good = Attend(c, [39, 32, 89, 16], None, 1)
    want = good.run()
    good.check(want)
    # Past max_positions: that stream's row is left alone, the others are whole.
    a = Attend(c, [39, 32, 89, 16], None, 1, most=64)
    got = a.run()
    assert c.st() == 2 and (got[2] == 5.5).all()
    assert np.allclose(got[[0, 1, 3]], want[[0, 1, 3]], rtol=0, atol=1e-5)
    # A block id and a slot outside the cache.
    table = c.table.copy()
    table[0, 1], table[3, 0] = c.blocks, -1
    c.tables.upload(table)
    got = good.run()
    assert c.st() == 2 and np.array_equal(got[1:3], want[1:3])
    c.tables.upload(c.table)
    slot = c.slot.copy()
    slot[1] = c.slots
    c.slotd.upload(slot)
    mark = good.mark
    good.dout.upload(mark)
    got = good.run()
    assert c.st() == 2 and (got[1] == 5.5).all() and np.array_equal(got[[0, 2, 3]], want[[0, 2, 3]])
    c.slotd.upload(c.slot)
    # A value that is not finite is said.
    opened = c.open.download(c.open0.shape)
    opened[1, c.slot[2], 0, 1, 0, 3] = np.inf
    c.open.upload(opened)
    good.run()
    assert c.st() == 1


def test_writes_flag_what_they_cannot_cover(cache):
    """Streams outside their table, slots or offsets, and block ids outside the
    cache: flagged and left out, the others written."""
    c = cache(4, 2, 64, positions=32)
    k, v = c.random_rows(40)
    before = c.raw()

    def go(first, counts, change=None):
        rows = c.call_rows(first, counts)
        if change:
            change(rows)
        dk, dv = c.up(k), c.up(v)
        assert c.lib.pgpu_kv8_write(None, ctypes.byref(c.kv), 1, ctypes.byref(rows), dk.ptr, dv.ptr,
                                    128, c.status.ptr)
        return c.st()
    assert go([30, -1, -1, -1], [3, 0, 0, 0]) == 2          # past the table
    assert go([0, -1, -1, -1], [20, 0, 0, 0], lambda r: setattr(r, "max_rows", 19)) == 2
    assert go([0, -1, -1, -1], [20, 0, 0, 0], lambda r: setattr(r, "rows", 19) or
              setattr(r, "max_rows", 19)) == 2
    bad = c.up(np.array([0, 5, 3, 2 ** 31 - 1, -4], np.int32))
    assert go([0] * 4, [5, 5, 5, 5], lambda r: setattr(r, "offsets", bad.ptr) or
              setattr(r, "first", c.up(np.array([-1, 0, 0, 0], np.int32)).ptr)) == 2
    assert go([2 ** 31 - 1, -1, -1, -1], [2, 0, 0, 0]) == 2
    assert all(np.array_equal(x, y) for x, y in zip(before, c.raw()))
    table = c.table.copy()
    table[0, 0] = c.blocks
    c.tables.upload(table)
    assert go([0, 0, -1, -1], [17, 16, 0, 0]) == 2           # block 0 of stream 0 lost
    c.note([0, 0, -1, -1], [17, 16, 0, 0], k, v)
    values, scales, opened = c.raw()
    q, s = model.quantise(c.rows[1][0].transpose(1, 0, 2))
    assert np.array_equal(scales[1, c.table[1, 0], :, 0], s)
    c.rows = c.rows[:2]
    c.check_slots(opened)


@pytest.mark.parametrize("counts", [None, [20, 3, 40]])
def test_attention_replays_from_a_graph(cache, counts):
    """Captured once in global mode (nothing is allocated), replayed with the
    program's own work between; the streams grow between replays, as the
    captured positions do."""
    c = cache(3, 2, 64, positions=400)
    lib, n = c.lib, counts or [1] * 3
    c.fill([150, 1, 300])
    c.write(c.lengths(), n, *c.random_rows(sum(n)))
    a = Attend(c, [150, 1, 300], counts, 1, most=400)
    stream, exec_ = ctypes.c_void_p(), ctypes.c_void_p()
    assert lib.pgpu_stream_create(ctypes.byref(stream))
    try:
        want = a.run()
        a.check(want)
        assert lib.pgpu_graph_begin_global(stream)
        enqueued = a.enqueue(stream)
        ended = lib.pgpu_graph_end(stream, ctypes.byref(exec_))
        assert enqueued and ended, c.pkg.last_error(lib)
        for replay in range(4):
            a.dout.upload(a.mark)
            assert lib.pgpu_graph_launch(exec_, stream) and lib.pgpu_stream_sync(stream)
            got = a.result()
            a.check(got)
            assert np.array_equal(got, a.run()), replay
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
    c.fill([700, 17, 1300])
    c.write(c.lengths(), n, *c.random_rows(sum(n)))
    a = Attend(c, [700, 17, 1300], counts, 1)
    want = a.run()
    for _ in range(5):
        assert np.array_equal(a.run(), want)


def test_a_prompt_then_frames_together(cache, lib):
    """The operators as a server uses them: prompts rotated, written and
    attended in two runs, then frames one at a time, every result against the
    model."""
    heads, group, dim = 2, 2, 64
    c = cache(3, heads, dim, positions=140)
    rng = c.rng
    angle = np.arange(160)[:, None] * 10000.0 ** (-2 * np.arange(dim // 2) / dim)
    rope = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    w = [(1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) for _ in range(2)]
    dw, drope = [c.up(x) for x in w], c.up(rope)
    width = heads * dim * (2 + group)
    for counts in ([50, 7, 0], [21, 60, 90], *[None] * 19):
        n = counts or [1] * 3
        first = c.lengths()
        qkv = rng.standard_normal((sum(n), width)).astype(np.float32)
        rows, a = c.call_rows(first, counts), Attend(c, first, counts, group)
        dx = c.up(qkv)
        assert lib.pgpu_kv8_rotate_write(None, ctypes.byref(c.kv), 1, ctypes.byref(rows), dx.ptr,
                                         width, group, dw[0].ptr, dw[1].ptr, 1e-5, drope.ptr, 160,
                                         1.0, a.dq.ptr, c.status.ptr)
        at = np.concatenate([np.arange(f, f + m) for f, m in zip(first, n)])
        x = qkv.reshape(len(qkv), -1, dim)
        k = model.turn(x[:, heads * group:-heads], w[1], 1e-5, rope[at]).astype(np.float32)
        c.note(first, n, k, x[:, -heads:])
        a.q = a.dq.download(a.q.shape)
        q = model.turn(x[:, :heads * group], w[0], 1e-5, rope[at])
        assert (np.abs(a.q - q) <= 2.0 ** -24 * np.abs(q) + 1e-44).all()
        a.check(a.run())


@pytest.mark.parametrize("streams,heads,group,dim,most", [
    (1, 8, 1, 64, 2000),     # whole streams, 16 waves, two steps
    (40, 8, 1, 64, 1500),    # 8 waves
    (100, 8, 1, 64, 700),    # 4 waves
    (12, 8, 1, 64, 2300),    # 16 waves, three steps
    (64, 8, 1, 64, 8192),    # dealt, three steps
    (3, 2, 1, 64, 8192),     # dealt, a step
    (30, 8, 4, 64, 900),     # four queries, 8 waves
    (100, 8, 2, 64, 500),    # four queries' places, two queries
    (9, 8, 3, 128, 8192),    # wide heads, dealt
    (20, 4, 1, 128, 800),    # wide heads, whole
    (3, 3, 9, 128, 1200),    # three passes over the queries
])
def test_attention_in_each_way_of_dealing_the_keys(cache, streams, heads, group, dim, most):
    """How the keys are dealt goes by max_positions and the batch; the contexts
    themselves are short, and of every offset in a block and a step."""
    c = cache(streams, heads, dim, positions=700, seed=streams)
    lengths = [1 + (s * 37 + s * s) % min(690, most - 1) if s % 9 else 1 for s in range(streams)]
    lengths[-1] = min(690, most - 1)
    c.fill(lengths)
    first = [-1 if s % 11 == 5 else n - 1 for s, n in enumerate(lengths)]
    a = Attend(c, first, None, group, most=most)
    got = a.run()
    keep = [s for s in range(streams) if s % max(1, streams // 8) == 0 or s == streams - 1]
    assert (got[[s for s in range(streams) if first[s] < 0]] == 0).all()
    assert c.st() == 0
    for s in keep:
        if first[s] < 0:
            continue
        k, v = (model.seen(x) for x in c.rows[s])
        want, bound = model.attention(a.q[s:s + 1], k, v, first[s], a.scale)
        assert (np.abs(got[s:s + 1] - want) <= bound).all(), s


@pytest.mark.parametrize("streams,heads,group,dim,most", [
    (12, 8, 1, 64, 4096),    # dealt, two steps of 4 waves
    (3, 3, 1, 128, 2000),    # wide heads, dealt, a step
    (26, 8, 1, 128, 4000),   # dealt, three steps
    (26, 8, 4, 128, 4000),
    (100, 8, 1, 128, 700),   # whole, 4 waves
    (40, 8, 2, 128, 1500),   # whole, 8 waves, three steps
])
def test_attention_of_wide_heads_and_dealt_steps(cache, streams, heads, group, dim, most):
    """Contexts that end in every block of a step, at its borders and in its first
    block: a step's last blocks are not there, and a wave may have no step."""
    c = cache(streams, heads, dim, positions=1300 if streams < 30 else 330)
    lengths = [(1, 16, 17, 63, 64, 65, 113, 255, 256, 257, 321, 511, 513, 767, 769, 1025, 1281)
               [s % 17] for s in range(streams)]
    lengths = [min(n, 1300 if streams < 30 else 330) for n in lengths]
    c.fill(lengths)
    a = Attend(c, [n - 1 for n in lengths], None, group, most=most)
    a.check(a.run())


@pytest.mark.parametrize("streams,heads,most", [(9, 8, 700), (9, 8, 1000), (2, 2, 1000), (2, 2, 380)])
def test_runs_dealt_by_their_number(cache, streams, heads, most):
    """More or fewer than 64 work-groups, with 11, 16 and 6 chunks of keys."""
    c = cache(streams, heads, 64, positions=380)
    before = [(0, 300, 129, 64)[s % 4] for s in range(streams)]
    counts = [(80, 5, 16, 37)[s % 4] for s in range(streams)]
    c.fill(before)
    c.write(before, counts, *c.random_rows(sum(counts)))
    a = Attend(c, before, counts, 1, most=most)
    a.check(a.run())


@pytest.mark.parametrize("most,heads,group,dim", [(4000, 2, 1, 64), (8192, 8, 2, 64),
                                                  (2000, 1, 5, 128), (120, 8, 1, 64)])
def test_runs_in_each_way_of_dealing_the_keys(cache, most, heads, group, dim):
    counts, before = [40, 1, 17, 3], [70, 0, 33, 100]
    c = cache(4, heads, dim, positions=120)
    c.fill(before)
    c.write(before, counts, *c.random_rows(sum(counts)))
    a = Attend(c, before, counts, group, most=most)
    a.check(a.run())


@pytest.mark.parametrize("scale", [-0.125, 0.0, 1e-30])
@pytest.mark.parametrize("counts", [None, [20, 33, 1]])
def test_attention_with_other_scales(cache, scale, counts):
    """A negative scale turns the order of the scores; with none every key weighs
    the same."""
    c = cache(3, 2, 64, positions=100)
    n = counts or [1] * 3
    c.fill([50, 0, 63])
    c.write([50, 0, 63], n, *c.random_rows(sum(n)))
    a = Attend(c, [50, 0, 63], counts, 2, scale=scale)
    a.check(a.run())


@pytest.mark.parametrize("counts", [None, [40, 3]])
def test_queries_of_zero_and_of_any_magnitude(cache, counts):
    c = cache(2, 2, 64, positions=120)
    n = counts or [1, 1]
    c.fill([70, 40])
    c.write([70, 40], n, *c.random_rows(sum(n)))
    for factor in (0.0, 1e-42, 1e-20, 1e20):
        a = Attend(c, [70, 40], counts, 2, scale=0.125 / max(factor, 1e-3) if factor > 1 else 0.125)
        a.q = (a.q * np.float32(factor)).astype(np.float32)
        a.dq.upload(a.q.reshape(a.total, -1))
        a.check(a.run())


def test_a_cache_past_32_bits(lib, pkg):
    """Blocks whose bytes start past 2^32, in layer 1 of 2."""
    heads, dim, blocks = 8, 64, 300000
    tile, slot = 2 * 16 * dim, 2 * 16 * dim
    assert blocks * heads * tile > 2 ** 32
    big = [pkg.DeviceBuffer(lib, n) for n in (2 * blocks * heads * tile, 2 * blocks * heads * 8,
                                              2 * 2 * heads * slot * 4)]
    try:
        kv = pkg.PgpuKv8(*(b.ptr for b in big), 2, heads, dim, blocks, 2)
        table = np.array([[blocks - 1, 5, blocks - 7, 262144], [blocks - 2, 1, 2, 3]], np.int32)
        n = [60, 33]
        rng = np.random.default_rng(8)
        k, v = (rng.standard_normal((sum(n), heads, dim)).astype(np.float32) for _ in range(2))
        host = dict(tables=table, slots=np.array([1, 0], np.int32), first=np.zeros(2, np.int32),
                    offsets=np.array([0, 60, 93], np.int32), status=np.zeros(1, np.int32),
                    lengths=np.array(n, np.int32), last=np.array(n, np.int32) - 1, k=k, v=v,
                    q=rng.standard_normal((2, heads, dim)).astype(np.float32))
        dev = {}
        for name, a in host.items():
            dev[name] = pkg.DeviceBuffer(lib, a.nbytes)
            dev[name].upload(a)
        out, bk, bv = (pkg.DeviceBuffer(lib, x) for x in (2 * 2048, k.nbytes, k.nbytes))
        rows = pkg.PgpuKv8Rows(dev["tables"].ptr, 4, dev["slots"].ptr, dev["first"].ptr,
                               dev["offsets"].ptr, 2, 93, 60)
        one = pkg.PgpuKv8Rows(dev["tables"].ptr, 4, dev["slots"].ptr, dev["last"].ptr, None, 2, 2, 1)
        kp = ctypes.byref(kv)
        assert lib.pgpu_kv8_write(None, kp, 1, ctypes.byref(rows), dev["k"].ptr, dev["v"].ptr, 512,
                                  dev["status"].ptr)
        assert lib.pgpu_kv8_read(None, kp, 1, ctypes.byref(rows), dev["lengths"].ptr, bk.ptr,
                                 bv.ptr, 512, dev["status"].ptr)
        assert lib.pgpu_kv8_attention(None, kp, 1, ctypes.byref(one), dev["q"].ptr, 512, 1, 0.125,
                                      64, out.ptr, 512, None, 0, dev["status"].ptr)
        assert dev["status"].download((1,), np.int32)[0] == 0
        gk, gv, go = bk.download(k.shape), bv.download(v.shape), out.download((2, heads, dim))
        for s, lo in ((0, 0), (1, 60)):
            wk, wv = model.seen(k[lo:lo + n[s]]), model.seen(v[lo:lo + n[s]])
            assert np.array_equal(gk[lo:lo + n[s]], wk) and np.array_equal(gv[lo:lo + n[s]], wv)
            want, bound = model.attention(host["q"][s:s + 1], wk, wv, n[s] - 1, 0.125)
            assert (np.abs(go[s:s + 1] - want) <= bound).all()
    finally:
        for b in big:
            b.free()


def test_two_streams_at_once(cache, lib):
    """Two calls on HIP streams of their own, each with its workspace, give the
    bits that they give alone."""
    c = cache(4, 8, 64, positions=2400)
    c.fill([2300, 5, 900, 60])
    c.write(c.lengths(), [30, 1, 70, 16], *c.random_rows(117))
    calls = [Attend(c, [2300, 5, 900, 60], [30, 1, 70, 16], 1),
             Attend(c, [n - 1 for n in c.lengths()], None, 2, most=8192, seed=9)]
    want = [a.run() for a in calls]
    streams = [ctypes.c_void_p(), ctypes.c_void_p()]
    for s in streams:
        assert lib.pgpu_stream_create(ctypes.byref(s))
    try:
        for _ in range(4):
            for a, s in zip(calls, streams):
                a.dout.upload(a.mark)
            for _ in range(3):
                for a, s in zip(calls, streams):
                    assert a.enqueue(s)
            for s in streams:
                assert lib.pgpu_stream_sync(s)
            for a, w in zip(calls, want):
                assert np.array_equal(a.result(), w)
    finally:
        for s in streams:
            lib.pgpu_stream_destroy(s)


def test_frames_from_one_graph(cache, lib):
    """A frame's rotated append, its attention and the advance of the positions
    captured once, and replayed over block borders with the program's own work
    between; the cache and every result against the model."""
    heads, group, dim, frames = 2, 2, 64, 40
    c = cache(3, heads, dim, positions=160)
    rng = c.rng
    angle = np.arange(160)[:, None] * 10000.0 ** (-2 * np.arange(dim // 2) / dim)
    rope = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    drope = c.up(rope)
    c.fill([100, 15, 0])
    width = heads * dim * (2 + group)
    a = Attend(c, [100, 15, 0], None, group, most=160)
    dx = c.up(np.zeros((3, width), np.float32))
    stream, exec_ = ctypes.c_void_p(), ctypes.c_void_p()
    assert lib.pgpu_stream_create(ctypes.byref(stream))
    try:
        assert lib.pgpu_graph_begin_global(stream)
        ok = lib.pgpu_kv8_rotate_write(stream, ctypes.byref(c.kv), 1, ctypes.byref(a.rows), dx.ptr,
                                       width, group, None, None, 0.0, drope.ptr, 160, 1.0,
                                       a.dq.ptr, c.status.ptr) and a.enqueue(stream) and \
            lib.pgpu_advance_positions(stream, a.rows.first, 3, 1)
        ended = lib.pgpu_graph_end(stream, ctypes.byref(exec_))
        assert ok and ended, c.pkg.last_error(lib)
        for frame in range(frames):
            first = c.lengths()
            qkv = rng.standard_normal((3, width)).astype(np.float32)
            dx.upload(qkv)
            assert lib.pgpu_graph_launch(exec_, stream) and lib.pgpu_stream_sync(stream)
            x = qkv.reshape(3, -1, dim)
            at = np.asarray(first)
            k = model.turn(x[:, heads * group:-heads], None, 0.0, rope[at]).astype(np.float32)
            c.note(first, [1] * 3, k, x[:, -heads:])
            a.first, a.q = first, a.dq.download(a.q.shape)
            a.check(a.result())
            if frame % 7 == 0:
                check_contents(c)
    finally:
        lib.pgpu_graph_destroy(exec_)
        lib.pgpu_stream_destroy(stream)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_is_not_finite_stays_with_the_rows_that_see_it(cache, which, bad):
    """A key or value of the newest block, and one of a stored block: rows of the
    same run before it come out whole, those that see it do not come out finite,
    and it is said."""
    c = cache(2, 2, 64, positions=120)
    c.fill([30, 0])
    k, v = c.random_rows(50 + 90)
    c.write([30, 0], [50, 90], k, v)
    assert c.st() == 0
    clean = [[x.copy() for x in r] for r in c.rows]
    opened = c.open.download(c.open0.shape)
    opened[1, c.slot[0], :, which, 75 - 64, 7] = bad            # newest block of stream 0
    opened[1, c.slot[1], :, which, 85 - 80, 7] = bad            # and of stream 1
    c.open.upload(opened)
    scales = c.scales.download(c.scales0.shape)
    scales[1, c.table[1, 40 // 16], :, which] = np.nan          # block 2 of stream 1
    c.scales.upload(scales)
    a = Attend(c, [30, 0], [50, 90], 2)
    got = a.run()
    assert c.st() == 1
    at = 0
    for s, (first, n, ends) in enumerate(((30, 50, 75), (0, 90, 32))):
        kk, vv = (model.seen(x) for x in clean[s])
        fine = ends - first
        want, bound = model.attention(a.q[at:at + fine], kk[:ends], vv[:ends], first, a.scale)
        assert (np.abs(got[at:at + fine] - want) <= bound).all()
        rest = np.isfinite(got[at + fine:at + n]).reshape(n - fine, -1)
        if s == 1 or which == 1 or np.isnan(bad):
            assert not rest.all(1).any()
        at += n


@pytest.mark.parametrize("group", [1, 3])
def test_a_stored_block_that_was_not_finite_reaches_its_stream_s_row_alone(cache, group):
    """A NaN scale of keys or values of a block at the front, inside a step and in
    a later step: that stream's row does not come out finite, the others do."""
    c = cache(4, 2, 64, positions=700)
    c.fill([600, 690, 650, 40])
    a = Attend(c, [n - 1 for n in c.lengths()], None, group)
    want = a.run()
    a.check(want)
    fine = c.scales.download(c.scales0.shape)
    for which in (0, 1):
        scales = fine.copy()
        for s, b in ((0, 0), (1, 41), (2, 7)):
            scales[1, c.table[s, b], :, which] = np.nan
        c.scales.upload(scales)
        got = a.run()
        assert c.st() == 1
        assert not np.isfinite(got[:3]).any()
        assert np.array_equal(got[3], want[3])
    c.scales.upload(fine)


def test_runs_flag_what_they_cannot_cover(cache):
    """Block ids outside the cache at the front and in a later chunk, a slot
    outside it, and rows past max_positions: said, and the other streams whole."""
    c = cache(3, 2, 64, positions=400)
    c.fill([300, 200, 100])
    counts = [20, 90, 33]
    c.write(c.lengths(), counts, *c.random_rows(sum(counts)))
    a = Attend(c, [300, 200, 100], counts, 2)
    want = a.run()
    a.check(want)
    for s, b in ((0, 0), (1, 7), (0, 13), (2, 5)):
        table = c.table.copy()
        table[s, b] = [c.blocks, -1][b % 2]
        c.tables.upload(table)
        got = a.run()
        assert c.st() == 2, (s, b)
        at = np.concatenate([[0], np.cumsum(counts)])
        for o in range(3):
            if o != s:
                assert np.array_equal(got[at[o]:at[o + 1]], want[at[o]:at[o + 1]])
    c.tables.upload(c.table)
    slot = c.slot.copy()
    slot[2] = -1
    c.slotd.upload(slot)
    a.dout.upload(a.mark)
    got = a.run()
    assert c.st() == 2 and (got[110:] == 5.5).all() and np.array_equal(got[:110], want[:110])
    c.slotd.upload(c.slot)
    b = Attend(c, [300, 200, 100], counts, 2, most=300)
    got = b.run()
    assert c.st() == 2 and (got[:20] == 5.5).all()
    assert np.allclose(got[20:], want[20:], rtol=0, atol=1e-5)
