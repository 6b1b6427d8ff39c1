"""Device memory of a batch over an 8-bit KV pool."""
import ctypes

import numpy as np
import pytest

import helpers

pytestmark = pytest.mark.gpu
STREAMS, MOST = 2048, 8192


class Batch:
    """A batch of 2048 streams of up to 8192 positions over a small pool."""

    def __init__(self, lib, pkg, model, q8):
        self.lib, self.pkg, self.q8 = lib, pkg, q8
        self.pool, self.batch = ctypes.c_void_p(), ctypes.c_void_p()
        made = (lib.phonon_kv_pool_create_q8(1, 16, 2, ctypes.byref(self.pool)) if q8 else
                lib.phonon_kv_pool_create(1, 16, ctypes.byref(self.pool)))
        assert made, pkg.last_error(lib)
        before = used()
        assert lib.phonon_flow_batch_create(model, self.pool, STREAMS, MOST,
                                            ctypes.byref(self.batch)), pkg.last_error(lib)
        self.bytes = used() - before

    def prefill(self, count=20):
        lib = self.lib
        x = np.random.default_rng(3).standard_normal((count, 512)).astype(np.float32)
        d = [self.pkg.DeviceBuffer(lib, x.nbytes) for _ in range(2)]
        d[0].upload(x)
        first, counts = np.zeros(1, np.uintp), np.array([count], np.uintp)
        table, slot = np.zeros((1, MOST // 16), np.int32), np.zeros(1, np.int32)
        table[0, :2] = 3, 7
        if self.q8:
            assert lib.phonon_flow_batch_prefill_q8_device(
                self.batch, 1, first.ctypes.data, counts.ctypes.data, table.ctypes.data, MOST // 16,
                slot.ctypes.data, d[0].ptr, 10000.0, d[1].ptr), self.pkg.last_error(lib)
        else:
            assert lib.phonon_flow_batch_prefill_device(
                self.batch, 1, first.ctypes.data, counts.ctypes.data, table.ctypes.data, MOST // 16,
                d[0].ptr, 10000.0, d[1].ptr), self.pkg.last_error(lib)
        assert lib.phonon_flow_batch_sync(self.batch)
        y = d[1].download(x.shape)
        for b in d:
            b.free()
        return y

    def close(self):
        self.lib.phonon_flow_batch_destroy(self.batch)
        self.lib.phonon_kv_pool_destroy(self.pool)


def used():
    free, total = ctypes.c_size_t(), ctypes.c_size_t()
    hip = ctypes.CDLL("libamdhip64.so")
    assert hip.hipMemGetInfo(ctypes.byref(free), ctypes.byref(total)) == 0
    return total.value - free.value


@pytest.fixture
def model(lib, pkg, syn):
    flow = helpers.scaled_model(syn, 3, 1)
    views = pkg.Views()
    m = ctypes.c_void_p()
    assert lib.phonon_flow_model_create(views.layers(flow), 1, ctypes.byref(m))
    yield m
    lib.phonon_flow_model_destroy(m)


def test_a_batch_holds_the_attention_parts_of_its_kind_only(lib, pkg, model):
    """The parts of an fp32 attention are 138 MB here, those of an 8-bit one 48; the
    rest is alike but for the slots' tables and the attention's rows, 8 MB."""
    b = [Batch(lib, pkg, model, q8) for q8 in (False, True)]
    try:
        assert b[1].bytes <= b[0].bytes - (138 - 48 - 8 - 10) * 1000000
        y = [x.prefill() for x in b]  # both work
        assert helpers.normwise(y[1], y[0].astype(np.float64)) < 0.05
    finally:
        for x in b:
            x.close()


def test_the_first_prefill_takes_one_plane_of_projected_rows(lib, pkg, model):
    """12.6 MB of 2048 rows of queries, keys and values; the same prefill over an fp32
    pool takes the rest that this one takes."""
    b = [Batch(lib, pkg, model, q8) for q8 in (False, True)]
    try:
        taken = []
        for x in b:
            x.prefill()  # what the runtime takes for it
            x.close()
        for n, q8 in enumerate((False, True)):
            b[n] = Batch(lib, pkg, model, q8)
            before = used()
            b[n].prefill()
            taken.append(used() - before)
        assert taken[1] - taken[0] <= 2048 * 1536 * 4 + (4 << 20)
    finally:
        for x in b:
            x.close()
