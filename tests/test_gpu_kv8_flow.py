"""Decode steps and prefills of the Flow transformer over an 8-bit KV pool:
every layer against float64 on what the pool holds, and the pool against the
model of its stored values."""
import ctypes

import numpy as np
import pytest

import helpers
import kv8_model as model

pytestmark = pytest.mark.gpu
LAYERS, MOST = 2, 128
I32, F32 = ctypes.POINTER(ctypes.c_int32), ctypes.POINTER(ctypes.c_float)


def i32(a):
    return a.ctypes.data_as(I32)


def f32(a):
    return a.ctypes.data_as(F32)


def layer_over(w, x, keys, values, pos):
    """helpers.f64_layer with the row's own key and value as the pool holds them:
    the output, and the key and value in float64."""
    class Held:  # takes the row's key (value), gives the held ones
        def __init__(self, held):
            self.held, self.row = held, None

        def __setitem__(self, at, row):
            self.row = row

        def __getitem__(self, at):
            return self.held[at]

    k, v = Held(keys), Held(values)
    return helpers.f64_layer(w, x, k, v, pos), k.row, v.row


class Server:
    def __init__(self, lib, pkg, oracle, syn, streams, seed=3, max_streams=64):
        self.lib, self.pkg, self.n = lib, pkg, streams
        flow = helpers.scaled_model(syn, seed, LAYERS)
        self.weights = helpers.oracle_layers(oracle, flow)
        self.views = pkg.Views()
        self.model, self.pool, self.batch = (ctypes.c_void_p() for _ in range(3))
        layers = self.views.layers(flow)
        assert lib.phonon_flow_model_create(layers, LAYERS, ctypes.byref(self.model))
        self.stride = MOST // 16
        assert lib.phonon_kv_pool_create_q8(LAYERS, streams * self.stride + 3, streams + 2,
                                            ctypes.byref(self.pool))
        assert lib.phonon_flow_batch_create(self.model, self.pool, max_streams, MOST,
                                            ctypes.byref(self.batch))
        rng = np.random.default_rng(seed)
        ids = np.zeros(streams * self.stride, np.int32)
        assert lib.phonon_kv_pool_alloc(self.pool, ids.size, i32(ids))
        self.tables = np.ascontiguousarray(rng.permutation(ids).reshape(streams, -1))
        slots = np.zeros(streams + 2, np.int32)
        assert lib.phonon_kv_pool_alloc_slots(self.pool, slots.size, i32(slots))
        self.slots = np.ascontiguousarray(rng.permutation(slots)[:streams])
        self.lengths = np.zeros(streams, int)
        # What was written, fp32, [layer][stream] lists of rows.
        self.raw = np.zeros((2, LAYERS, streams, MOST, 512), np.float32)
        self.rng = rng

    def hold(self, lengths):
        """Random contexts through the host call, in two parts."""
        for s, n in enumerate(lengths):
            k, v = (self.rng.standard_normal((LAYERS, MOST, 512)).astype(np.float32)
                    for _ in range(2))
            self.raw[0, :, s, :n], self.raw[1, :, s, :n] = k[:, :n], v[:, :n]
            for lo, hi in ((0, n // 3), (n // 3, n)):
                if hi > lo:
                    assert self.lib.phonon_kv_pool_write_q8(
                        self.pool, i32(self.tables[s]), self.stride, int(self.slots[s]), lo,
                        hi - lo, f32(k), f32(v), MOST), self.pkg.last_error(self.lib)
            self.lengths[s] = n

    def held(self, s):
        """Keys and values of stream s as a read gives them, [layer][length][512]."""
        n = int(self.lengths[s])
        k, v = np.zeros((LAYERS, MOST, 512), np.float32), np.zeros((LAYERS, MOST, 512), np.float32)
        assert self.lib.phonon_kv_pool_read_q8(self.pool, i32(self.tables[s]), self.stride,
                                               int(self.slots[s]), n, 0, n, f32(k), f32(v), MOST)
        return k, v

    def set(self):
        pos = self.lengths.astype(np.uintp)
        assert self.lib.phonon_flow_batch_set_streams_q8(
            self.batch, self.n, pos.ctypes.data_as(ctypes.POINTER(ctypes.c_size_t)),
            i32(self.tables), self.stride, i32(self.slots)), self.pkg.last_error(self.lib)

    def step(self, x):
        y = np.zeros_like(x)
        assert self.lib.phonon_flow_batch_step(self.batch, f32(x), 10000.0, f32(y)), \
            self.pkg.last_error(self.lib)
        self.lengths += 1
        return y

    def check(self, s, first, x, y):
        """Rows y of stream s at positions first, ...: every layer in float64 over
        the pool's keys and values; the fp32 rows of the newest block against
        float64, the blocks before it against the rows that were written."""
        k, v = self.held(s)
        n, lo = int(self.lengths[s]), (int(self.lengths[s]) - 1) // 16 * 16
        for r in range(len(x)):
            want = x[r].astype(np.float64)
            for layer in range(LAYERS):
                want, *rows = layer_over(self.weights[layer], want, k[layer].astype(np.float64),
                                         v[layer].astype(np.float64), first + r)
                for i, (got, row) in enumerate(zip((k, v), rows)):
                    if first + r >= lo:
                        assert helpers.normwise(got[layer, first + r], row) <= 1e-4
                        self.raw[i, layer, s, first + r] = got[layer, first + r]
                    else:  # stored in 8 bits: within half a step and the fp32 rounding
                        q = got[layer, first + r].reshape(8, 64)
                        b = (first + r) // 16 * 16
                        step = np.abs(got[layer, b:b + 16].reshape(16, 8, 64)).max((0, 2)) / 126
                        far = np.abs(q - row.reshape(8, 64))
                        assert (far <= step[:, None] * 0.51).all()
            assert helpers.normwise(y[r], want) <= 2e-4, (s, first + r)

    def close(self):
        self.lib.phonon_flow_batch_destroy(self.batch)
        self.lib.phonon_kv_pool_destroy(self.pool)
        self.lib.phonon_flow_model_destroy(self.model)


@pytest.fixture
def server(lib, pkg, oracle, syn):
    made = []

    def make(*args, **kw):
        made.append(Server(lib, pkg, oracle, syn, *args, **kw))
        return made[-1]
    yield make
    for s in made:
        s.close()


@pytest.mark.parametrize("graph", [1, 0])
def test_decode_steps_over_an_8_bit_pool(server, graph):
    sv = server(5)
    assert sv.lib.phonon_flow_batch_set_graph(sv.batch, graph)
    sv.hold([0, 15, 31, 40, 64])
    sv.set()
    for n in range(19):
        x = sv.rng.standard_normal((5, 512)).astype(np.float32)
        y = sv.step(x)
        for s in range(5):
            if n < 3 or (sv.lengths[s] % 16) in (0, 1, 2):
                sv.check(s, int(sv.lengths[s]) - 1, x[s:s + 1], y[s:s + 1])
            else:  # the newest row, for the check of its block
                k, v = sv.held(s)
                p = int(sv.lengths[s]) - 1
                sv.raw[0, :, s, p], sv.raw[1, :, s, p] = k[:, p], v[:, p]
    # The blocks that steps filled hold their rows' model.
    for s in range(5):
        got = sv.held(s)
        n = int(sv.lengths[s])
        for i in range(2):
            for layer in range(LAYERS):
                want = model.seen(sv.raw[i, layer, s, :n].reshape(n, 8, 64)).reshape(n, 512)
                assert np.array_equal(got[i][layer, :n].astype(np.float64), want), (s, i, layer)


@pytest.mark.parametrize("exact", [0, 1])
def test_prefill_then_steps_over_an_8_bit_pool(server, exact):
    """Prompts in two calls, ragged, after held contexts and none; then steps."""
    sv = server(4)
    lib, pkg = sv.lib, sv.pkg
    assert lib.phonon_flow_batch_set_prefill_exact(sv.batch, exact)
    sv.hold([0, 5, 0, 33])
    for counts in ([20, 1, 16, 9], [3, 14, 2, 40]):
        first = sv.lengths.astype(np.uintp).copy()
        total = sum(counts)
        x = sv.rng.standard_normal((total, 512)).astype(np.float32)
        dx, dy = pkg.DeviceBuffer(lib, x.nbytes), pkg.DeviceBuffer(lib, x.nbytes)
        dx.upload(x)
        c = np.asarray(counts, np.uintp)
        assert lib.phonon_flow_batch_prefill_q8_device(
            sv.batch, 4, first.ctypes.data, c.ctypes.data, sv.tables.ctypes.data, sv.stride,
            sv.slots.ctypes.data, dx.ptr, 10000.0, dy.ptr), pkg.last_error(lib)
        assert lib.phonon_flow_batch_sync(sv.batch)
        y = dy.download(x.shape)
        sv.lengths += counts
        at = 0
        for s, n in enumerate(counts):
            sv.check(s, int(first[s]), x[at:at + n], y[at:at + n])
            at += n
    sv.set()
    for _ in range(18):
        x = sv.rng.standard_normal((4, 512)).astype(np.float32)
        y = sv.step(x)
    for s in range(4):
        sv.check(s, int(sv.lengths[s]) - 1, x[s:s + 1], y[s:s + 1])


def test_many_streams_step_together(server):
    """More streams than a tile, contexts at every offset of a block."""
    sv = server(40)
    sv.hold([n % 37 for n in range(40)])
    sv.set()
    for _ in range(2):
        x = sv.rng.standard_normal((40, 512)).astype(np.float32)
        y = sv.step(x)
    for s in range(0, 40, 3):
        sv.check(s, int(sv.lengths[s]) - 1, x[s:s + 1], y[s:s + 1])


def test_calls_refuse_the_other_kind_of_pool(server, lib, pkg):
    sv = server(2)
    sv.hold([3, 4])
    pos = np.zeros(2, np.uintp)
    szp = ctypes.POINTER(ctypes.c_size_t)
    buf = np.zeros((LAYERS, MOST, 512), np.float32)
    kv, k8 = pkg.PgpuPagedKv(), pkg.PgpuKv8()
    t = i32(sv.tables)
    assert not lib.phonon_flow_batch_set_streams(sv.batch, 2, pos.ctypes.data_as(szp), t, sv.stride)
    assert b"_q8" in lib.pgpu_last_error()
    assert not lib.phonon_kv_pool_fill_normal(sv.pool, 1)
    assert not lib.phonon_kv_pool_view(sv.pool, ctypes.byref(kv))
    assert lib.phonon_kv_pool_view_q8(sv.pool, ctypes.byref(k8)) and k8.heads == 8
    assert not lib.phonon_kv_pool_write(sv.pool, t, sv.stride, 0, 4, f32(buf), f32(buf), MOST)
    assert not lib.phonon_kv_pool_read(sv.pool, t, sv.stride, 0, 4, f32(buf), f32(buf), MOST)
    assert not lib.phonon_flow_batch_set_groups(sv.batch, 2)
    d = pkg.DeviceBuffer(lib, 4096)
    one = np.ones(1, np.uintp)
    assert not lib.phonon_flow_batch_prefill_device(sv.batch, 1, pos.ctypes.data, one.ctypes.data,
                                                    sv.tables.ctypes.data, sv.stride, d.ptr,
                                                    10000.0, d.ptr)
    # Slots outside the pool, and a length that its table does not reach.
    bad = np.array([0, sv.n + 2], np.int32)
    assert not lib.phonon_flow_batch_set_streams_q8(sv.batch, 2, pos.ctypes.data_as(szp), t,
                                                    sv.stride, i32(bad))
    both = np.array([sv.slots[0], sv.slots[0]], np.int32)  # one slot for two streams
    assert not lib.phonon_flow_batch_set_streams_q8(sv.batch, 2, pos.ctypes.data_as(szp), t,
                                                    sv.stride, i32(both))
    assert b"two streams" in lib.pgpu_last_error()
    two = np.ones(2, np.uintp)
    assert not lib.phonon_flow_batch_prefill_q8_device(
        sv.batch, 2, pos.ctypes.data, two.ctypes.data, sv.tables.ctypes.data, sv.stride,
        both.ctypes.data, d.ptr, 10000.0, d.ptr)
    assert not lib.phonon_kv_pool_write_q8(sv.pool, t, sv.stride, sv.n + 2, 0, 4, f32(buf),
                                           f32(buf), MOST)
    assert not lib.phonon_kv_pool_write_q8(sv.pool, t, 1, int(sv.slots[0]), 3, 14, f32(buf),
                                           f32(buf), MOST)
    assert not lib.phonon_kv_pool_read_q8(sv.pool, t, sv.stride, int(sv.slots[0]), 3, 0, 4,
                                          f32(buf), f32(buf), MOST)
    # An fp32 pool and its batch refuse the 8-bit forms.
    pool, batch = ctypes.c_void_p(), ctypes.c_void_p()
    assert lib.phonon_kv_pool_create(LAYERS, 16, ctypes.byref(pool))
    assert lib.phonon_flow_batch_create(sv.model, pool, 4, MOST, ctypes.byref(batch))
    try:
        assert not lib.phonon_flow_batch_set_streams_q8(batch, 2, pos.ctypes.data_as(szp), t,
                                                        sv.stride, i32(sv.slots))
        assert not lib.phonon_kv_pool_view_q8(pool, ctypes.byref(k8))
        assert not lib.phonon_kv_pool_write_q8(pool, t, sv.stride, 0, 0, 4, f32(buf), f32(buf),
                                               MOST)
        assert lib.phonon_kv_pool_free_slots(pool) == 0
    finally:
        lib.phonon_flow_batch_destroy(batch)
        lib.phonon_kv_pool_destroy(pool)
    # Ids: one given twice, or not in use, is refused whole.
    free = lib.phonon_kv_pool_free_slots(sv.pool)
    twice = np.array([sv.slots[0], sv.slots[0]], np.int32)
    assert not lib.phonon_kv_pool_release_slots(sv.pool, 2, i32(twice))
    assert lib.phonon_kv_pool_free_slots(sv.pool) == free
    assert lib.phonon_kv_pool_release_slots(sv.pool, 1, i32(twice))
    assert not lib.phonon_kv_pool_release_slots(sv.pool, 1, i32(twice))
    assert lib.phonon_kv_pool_free_slots(sv.pool) == free + 1


def test_a_step_after_a_prefill_needs_its_streams(server, lib, pkg):
    """The prefill's rows are the batch's streams until they are set: a step
    would write them again. It is refused, and what the pool holds stays."""
    sv = server(2)
    sv.hold([5, 16])
    counts = np.array([20, 3], np.uintp)
    x = sv.rng.standard_normal((23, 512)).astype(np.float32)
    d = pkg.DeviceBuffer(lib, x.nbytes)
    d.upload(x)
    out = pkg.DeviceBuffer(lib, x.nbytes)
    first = sv.lengths.astype(np.uintp)
    assert lib.phonon_flow_batch_prefill_q8_device(
        sv.batch, 2, first.ctypes.data, counts.ctypes.data, sv.tables.ctypes.data, sv.stride,
        sv.slots.ctypes.data, d.ptr, 10000.0, out.ptr), pkg.last_error(lib)
    assert lib.phonon_flow_batch_sync(sv.batch)
    sv.lengths += counts.astype(int)
    before = [sv.held(s) for s in range(2)]
    assert not lib.phonon_flow_batch_step_device(sv.batch, d.ptr, 10000.0, out.ptr)
    assert b"set the streams" in lib.pgpu_last_error()
    for s in range(2):
        for a, b in zip(before[s], sv.held(s)):
            assert np.array_equal(a, b)
    sv.set()
    y = sv.step(x[:2])
    assert np.isfinite(y).all()
