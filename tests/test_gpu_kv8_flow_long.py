"""Steps and prefills over an 8-bit KV pool whose contexts are dealt to several
work-groups and joined: captured steps that outgrow their graph, prefills between
them, other streams in the batch, and what a step allocates."""
import ctypes

import numpy as np
import pytest

import test_gpu_kv8_flow as flow
from test_gpu_kv8_flow import LAYERS, i32, server  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture
def long_server(server, monkeypatch):
    def make(streams, most, **kw):
        monkeypatch.setattr(flow, "MOST", most)
        return server(streams, **kw)
    return make


def parts(sv, rows, most):
    """Bytes of the workspace that an attention call of these rows needs at least: 0
    where it takes every stream whole."""
    kv = sv.pkg.PgpuKv8()
    assert sv.lib.phonon_kv_pool_view_q8(sv.pool, ctypes.byref(kv))
    one = ctypes.c_int32(0)
    at = ctypes.addressof(one)
    r = sv.pkg.PgpuKv8Rows(at, most // 16, at, at, at if rows else None, sv.n,
                           sum(rows) if rows else sv.n, max(rows) if rows else 1)
    return sv.lib.pgpu_kv8_attention_bytes(ctypes.byref(kv), ctypes.byref(r), 1, most)


def prefill(sv, counts):
    lib, pkg = sv.lib, sv.pkg
    first = sv.lengths.astype(np.uintp).copy()
    x = sv.rng.standard_normal((sum(counts), 512)).astype(np.float32)
    dx, dy = pkg.DeviceBuffer(lib, x.nbytes), pkg.DeviceBuffer(lib, x.nbytes)
    dx.upload(x)
    c = np.asarray(counts, np.uintp)
    assert lib.phonon_flow_batch_prefill_q8_device(
        sv.batch, sv.n, first.ctypes.data, c.ctypes.data, sv.tables.ctypes.data, sv.stride,
        sv.slots.ctypes.data, dx.ptr, 10000.0, dy.ptr), pkg.last_error(lib)
    assert lib.phonon_flow_batch_sync(sv.batch)
    y = dy.download(x.shape)
    dx.free()
    dy.free()
    sv.lengths += counts
    return first, x, y


def step(sv):
    x = sv.rng.standard_normal((sv.n, 512)).astype(np.float32)
    return x, sv.step(x)


def check_step(sv, x, y, streams=None):
    for s in streams or range(sv.n):
        sv.check(s, int(sv.lengths[s]) - 1, x[s:s + 1], y[s:s + 1])


@pytest.mark.parametrize("graph", [1, 0])
def test_steps_over_dealt_contexts(long_server, graph):
    """Captured steps cross a border of 256 positions past their headroom and are
    captured again; a prefill of long contexts and a new set of streams come between.
    Every result against float64 over what the pool holds."""
    sv = long_server(3, 4096, max_streams=256)
    assert sv.lib.phonon_flow_batch_set_graph(sv.batch, graph)
    assert parts(sv, None, 3328) and parts(sv, [200, 20, 9], 3328)
    sv.hold([3060, 14, 255])
    sv.set()
    for n in range(275):  # to 3335 positions: past 3060 + 256 rounded up
        x, y = step(sv)
        if n in (0, 1, 2, 241, 266, 267, 268, 269, 274):
            check_step(sv, x, y, (0, 1) if n % 2 else (0, 2))
    first, x, y = prefill(sv, [120, 7, 40])
    at = 0
    for s, n in enumerate((120, 7, 40)):
        for r in (0, n // 2, n - 1):
            # The rows' own keys and values as the pool holds them are checked elsewhere.
            check_row(sv, s, int(first[s]) + r, x[at + r], y[at + r])
        at += n
    sv.set()
    for n in range(4):
        x, y = step(sv)
        check_step(sv, x, y)
    # Other streams: one long context alone, then the three again.
    keep = sv.lengths.copy()
    pos = np.array([keep[0]], np.uintp)
    szp = ctypes.POINTER(ctypes.c_size_t)
    assert sv.lib.phonon_flow_batch_set_streams_q8(
        sv.batch, 1, pos.ctypes.data_as(szp), i32(sv.tables), sv.stride, i32(sv.slots))
    x = sv.rng.standard_normal((1, 512)).astype(np.float32)
    y = np.zeros_like(x)
    assert sv.lib.phonon_flow_batch_step(sv.batch, flow.f32(x), 10000.0, flow.f32(y))
    sv.lengths[0] += 1
    sv.check(0, int(sv.lengths[0]) - 1, x, y)
    sv.set()
    x, y = step(sv)
    check_step(sv, x, y)


def check_row(sv, s, position, x, y):
    k, v = sv.held(s)
    want = x.astype(np.float64)
    for layer in range(LAYERS):
        want, _, _ = flow.layer_over(sv.weights[layer], want, k[layer].astype(np.float64),
                                     v[layer].astype(np.float64), position)
    assert flow.helpers.normwise(y, want) <= 2e-4, (s, position)


def test_steps_allocate_nothing(long_server, pkg, lib):
    """Over contexts that need the workspace after ones that do not, and fewer streams
    after more: the batch took what it needs when it was made."""
    hip = ctypes.CDLL("libamdhip64.so")

    def used():
        free, total = ctypes.c_size_t(), ctypes.c_size_t()
        assert hip.hipMemGetInfo(ctypes.byref(free), ctypes.byref(total)) == 0
        return total.value - free.value

    def run(sv, n, position):
        sv.n = n
        sv.lengths[:] = position  # the pool's zeros
        sv.set()
        x = sv.rng.standard_normal((n, 512)).astype(np.float32)
        y = np.zeros_like(x)
        assert lib.phonon_flow_batch_step(sv.batch, flow.f32(x), 10000.0, flow.f32(y))
        assert np.isfinite(y).all()

    # What the runtime itself takes for kernels and copies of these kinds.
    first = long_server(23, 8192, max_streams=48)
    sv = long_server(23, 8192, max_streams=48)
    for batch in (first, sv):
        assert lib.phonon_flow_batch_set_graph(batch.batch, 0)
    for n, position in ((23, 5), (23, 8000), (7, 8000)):
        run(first, n, position)
    run(sv, 23, 5)
    before = used()
    for n in (23, 7, 1, 20):
        run(sv, n, 8000)
        assert parts(sv, None, 8192) > 0 and used() == before, n


def test_one_launch_steps_are_refused(server, lib):
    """A mode that the pool's steps cannot have is not taken and then ignored."""
    sv = server(2)
    for mode in (0, 1):
        assert lib.phonon_flow_batch_set_pipeline(sv.batch, mode)
    assert not lib.phonon_flow_batch_set_pipeline(sv.batch, 2)
    assert b"8-bit" in lib.pgpu_last_error()
    sv.hold([5, 16])
    sv.set()
    x, y = step(sv)
    check_step(sv, x, y)
