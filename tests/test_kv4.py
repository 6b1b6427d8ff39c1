"""CPU checks of the 4-bit paged KV cache: the rules of its stored values, and what its
entry points refuse (no GPU is touched by a refused call)."""
import ctypes

import numpy as np
import pytest

import kv4_model as model


def test_the_quantisation_does_not_depend_on_the_precision_it_is_done_in():
    """q from fp32 division is q from 64-bit division, on random rows and on values at and
    one step beside every tie (n + 1/2) s; a stored value is off by half a step at most and
    is an fp16 number."""
    rng = np.random.default_rng(5)
    for spread in (1e-7, 1e-4, 1.0, 3e4):
        x = np.clip(rng.standard_normal((2000, 64)) * spread, -57000, 57000).astype(np.float32)
        s = model.scale_of(x)
        ties = ((np.arange(-8, 7) + 0.5)[None] * s[:, None]).astype(np.float32)
        assert (ties.astype(np.float64) == (np.arange(-8, 7) + 0.5) * s[:, None]).all()
        beside = np.stack([ties, np.nextafter(ties, np.float32(np.inf)),
                           np.nextafter(ties, np.float32(-np.inf))])
        for y in (x, *beside):
            s32 = s.astype(np.float32)[:, None]
            assert (np.rint(y / s32) == np.rint(y.astype(np.float64) / s[:, None])).all()
        q, s = model.quantise(x)
        assert q.min() >= -8 and q.max() <= 7
        if spread > 1e-5:
            assert ((q == 7).any(1) | (q == -8).any(1) | (np.abs(q) >= 6).any(1)).all()
        held = model.seen(x)
        assert (np.abs(held - x) <= s / 2 * (1 + 2.0 ** -20)).all()
        assert (held.astype(np.float16).astype(np.float64) == held).all()
    # The largest scale that fits, and the least.
    edge = np.array([8160 * 7.0, -8160 * 8.0, 0.0, 1e-9])
    x = np.zeros((4, 64), np.float32)
    x[:, 5] = edge
    q, s = model.quantise(x)
    assert list(s[:, 0]) == [8160, 8160, 2.0 ** -17, 2.0 ** -17] and list(q[:, 5]) == [7, -8, 0, 0]


@pytest.mark.parametrize("dim", [64, 128])
def test_the_byte_order_says_where_each_number_is(dim):
    rng = np.random.default_rng(dim)
    k, v = rng.integers(-8, 8, (2, 16, dim))
    t = model.tile(k, v)
    for p, d in ((0, 0), (5, 3), (15, dim - 1), (8, 21), (12, 44)):
        for which, at, i in ((0, p * 32 + d % 64 // 16 * 8, d % 16), (1, d % 64 * 8, p)):
            byte = int(t[which, d // 64, at + i // 8 * 4 + i % 4])
            n = byte >> (i // 4 % 2 * 4) & 15
            assert (n ^ 8) - 8 == (k, v)[which][p, d]


class Args:
    """Arguments of every call that would be accepted, with host addresses that nothing
    reads."""

    def __init__(self, pkg, rows=5, streams=2):
        self.buf = np.zeros(1 << 12, np.float32)
        a = (self.buf.ctypes.data + 255) // 256 * 256
        self.ptr = a
        self.kv = pkg.PgpuKv4(a, a, 2, 8, 64, 10)
        self.rows = pkg.PgpuKv4Rows(a, 4, a, a, streams, rows, min(rows, 3))
        self.sums = pkg.PgpuKv4Sums(a, a, 64, 3)
        self.values = dict(kv=self.kv, layer=0, rows=self.rows, k=a, v=a, q=a, out=a,
                           stride=512 * 3, group=1, scale=0.125, lengths=a, max_positions=64,
                           sums=self.sums, work=a, work_bytes=1 << 30, status=a, layers=2,
                           to_tables=a, keep=8, first=2, newest=3, weighed=a, to_sums=a,
                           sums_stride=64, kept=a)


def call(lib, name, a, **changed):
    v = {**a.values, **changed}
    kv, rows, sums = (ctypes.byref(v[n]) if v[n] is not None else None
                      for n in ("kv", "rows", "sums"))
    if name == "write":
        return lib.pgpu_kv4_write(None, kv, v["layer"], rows, v["k"], v["v"], v["stride"],
                                  v["status"])
    if name == "read":
        return lib.pgpu_kv4_read(None, kv, v["layer"], rows, v["lengths"], v["k"], v["v"],
                                 v["stride"], v["status"])
    if name == "evict":
        r = v["rows"]
        return lib.pgpu_kv4_evict(None, kv, v["layer"], v["layers"], r.tables, v["to_tables"],
                                  r.table_stride, v["lengths"], r.streams, v["keep"], v["first"],
                                  v["newest"], v["weighed"], v["to_sums"], v["sums_stride"],
                                  v["kept"], v["status"])
    return lib.pgpu_kv4_attention(None, kv, v["layer"], rows, v["q"], v["stride"], v["group"],
                                  v["scale"], v["max_positions"], v["out"], v["stride"], sums,
                                  v["work"], v["work_bytes"], v["status"])


NAMES = ("write", "read", "attention", "evict")


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("field,value", [
    ("values", None), ("scales", None), ("values", 8), ("scales", 8), ("layers", 0),
    ("heads", 0), ("heads", 257), ("head_dim", 32), ("head_dim", 96), ("blocks", 0),
    ("blocks", 1 << 31)])
def test_calls_refuse_a_bad_cache(pkg, name, field, value):
    a = Args(pkg)
    if value == 8:
        value = a.ptr + 8
    setattr(a.kv, field, value)
    lib = pkg.load()
    lib.pgpu_record_error(b"")
    assert not call(lib, name, a)
    assert b"invalid arguments" in lib.pgpu_last_error()


@pytest.mark.parametrize("name", [n for n in NAMES if n != "evict"])
@pytest.mark.parametrize("field,value", [
    ("tables", None), ("table_stride", 0), ("first", None), ("streams", 0), ("streams", 65536),
    ("rows", -1), ("max_rows", 0), ("max_rows", 6), ("max_rows", -1), ("offsets", None)])
def test_calls_refuse_bad_rows(pkg, name, field, value):
    a = Args(pkg)  # offsets NULL: five rows are not one for each of two streams
    setattr(a.rows, field, value)
    assert not call(pkg.load(), name, a)


@pytest.mark.parametrize("name,changed", [
    *[(n, {"layer": -1}) for n in NAMES], *[(n, {"layer": 2}) for n in NAMES],
    *[(n, {"status": None}) for n in NAMES], *[(n, {"kv": None}) for n in NAMES],
    *[(n, {"rows": None}) for n in NAMES if n != "evict"],
    *[(n, {k: None}) for n in ("write", "read") for k in "kv"],
    *[(n, {k: "odd"}) for n in ("write", "read") for k in "kv"],
    *[(n, {"stride": s}) for n in ("write", "read") for s in (508, 514)],
    ("read", {"lengths": None}),
    ("attention", {"q": None}), ("attention", {"q": "odd"}), ("attention", {"out": None}),
    ("attention", {"out": "odd"}), ("attention", {"group": 0}), ("attention", {"group": 17}),
    ("attention", {"stride": 508}), ("attention", {"stride": 514}),
    ("attention", {"max_positions": 0}), ("attention", {"scale": float("nan")}),
    ("attention", {"scale": 2.4e38}), ("attention", {"group": 4}),
    ("attention", {"max_positions": 65}),  # past the sums
    ("attention", {"work": None}), ("attention", {"work": "odd"}),
    ("attention", {"work_bytes": 15}),
    ("evict", {"layer": 1}), ("evict", {"layers": 0}), ("evict", {"layers": -1}),
    ("evict", {"lengths": None}), ("evict", {"keep": 0}), ("evict", {"first": -1}),
    ("evict", {"newest": -1}), ("evict", {"first": 6}), ("evict", {"newest": 2 ** 31 - 1}),
    ("evict", {"weighed": None}), ("evict", {"to_sums": None}), ("evict", {"sums_stride": 0}),
    ("evict", {"kept": None})])
def test_calls_refuse_bad_arguments(pkg, name, changed):
    a = Args(pkg)
    changed = {k: a.ptr + 4 if v == "odd" else v for k, v in changed.items()}
    lib = pkg.load()
    lib.pgpu_record_error(b"")
    assert not call(lib, name, a, **changed)
    assert b"invalid arguments" in lib.pgpu_last_error() or b"workspace" in lib.pgpu_last_error()


@pytest.mark.parametrize("field,value", [("after", None), ("stride", 63), ("rows", 0), ("rows", -2)])
def test_attention_refuses_bad_sums(pkg, field, value):
    a = Args(pkg)
    setattr(a.sums, field, value)
    assert not call(pkg.load(), "attention", a)


@pytest.mark.parametrize("field,value", [("tables", None), ("table_stride", 0), ("streams", 0),
                                         ("streams", 65536)])
def test_evict_refuses_bad_streams(pkg, field, value):
    a = Args(pkg)
    setattr(a.rows, field, value)
    assert not call(pkg.load(), "evict", a)


@pytest.mark.parametrize("name", ("write", "read", "attention"))
def test_a_call_of_no_rows_does_nothing(pkg, name):
    assert call(pkg.load(), name, Args(pkg, rows=0)) == 1


def test_attention_refuses_more_positions_than_it_can_count(pkg):
    """2^30 of a stream; with runs' sums, 2^28 over the heads."""
    lib = pkg.load()
    for sums, offsets, most in ((False, True, 2 ** 30 + 1), (False, False, 2 ** 30 + 1),
                                (True, True, 2 ** 28 // 8), (True, False, 2 ** 30 + 1)):
        a = Args(pkg, *(() if offsets else (2, 2)))
        if not offsets:
            a.rows.offsets, a.rows.max_rows = None, 1
        a.sums.stride = 2 ** 31
        assert not call(lib, "attention", a, max_positions=most, work_bytes=1 << 62,
                        **({} if sums else {"sums": None}))
        assert b"invalid arguments" in lib.pgpu_last_error()
        if most > 2 ** 30:
            assert lib.pgpu_kv4_attention_bytes(ctypes.byref(a.kv), ctypes.byref(a.rows), 1, most, sums) == 0


def test_evict_refuses_to_keep_more_rows_than_it_can_count(pkg):
    a = Args(pkg)
    for keep in (2 ** 30 + 1, 2 ** 31 - 1):
        assert not call(pkg.load(), "evict", a, keep=keep)
