"""CPU checks of the 8-bit paged KV cache: the rules of its stored values, and
what its entry points refuse (no GPU is touched by a refused call)."""
import ctypes

import numpy as np
import pytest

import kv8_model as model


def test_the_quantisation_does_not_depend_on_the_precision_it_is_done_in():
    """q from fp32 division is q from 64-bit division, on random blocks and on
    values at and one step beside every tie (n + 1/2) s."""
    rng = np.random.default_rng(5)
    for spread in (1e-30, 1.0, 3e4, 1e30):
        x = (rng.standard_normal((200, 16, 64)) * spread).astype(np.float32)
        s = model.scale_of(x)
        ties = ((np.arange(-126, 126) + 0.5)[None] * s[:, None]).astype(np.float32)
        assert (ties.astype(np.float64) == (np.arange(-126, 126) + 0.5) * s[:, None]).all()
        beside = np.stack([ties, np.nextafter(ties, np.float32(np.inf)),
                           np.nextafter(ties, np.float32(-np.inf))])
        for y in (x.reshape(200, -1), *beside):
            s32 = s.astype(np.float32)[:, None]
            assert (np.rint(y / s32) == np.rint(y.astype(np.float64) / s[:, None])).all()
        q, _ = model.quantise(x)
        assert np.abs(q).max() == 127 and (np.abs(q).max((1, 2)) >= 126).all()
        # Half a step: s is at most max/127 (1 + 2^-11) (1 + 2^-24).
        top = np.abs(x.astype(np.float64)).max((1, 2))[:, None, None]
        assert (np.abs(q * s[:, None, None] - x) <= top / 254 * (1 + 2.0 ** -10)).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_the_value_order_is_a_permutation(dim):
    assert sorted(model.value_order(dim).reshape(-1)) == list(range(16 * dim))


class Args:
    """Arguments of every call that would be accepted, with host addresses
    that nothing reads."""

    def __init__(self, pkg, rows=5, streams=2):
        self.buf = np.zeros(1 << 12, np.float32)
        a = (self.buf.ctypes.data + 255) // 256 * 256
        self.ptr = a
        self.kv = pkg.PgpuKv8(a, a, a, 2, 8, 64, 10, 4)
        self.rows = pkg.PgpuKv8Rows(a, 4, a, a, a, streams, rows, min(rows, 3))
        self.values = dict(stream=None, kv=self.kv, layer=0, rows=self.rows, k=a, v=a, qkv=a, q=a,
                           out=a, stride=512 * 3, group=1, weight=a, epsilon=1e-5, rope=a,
                           rope_positions=64, scale=0.125, lengths=a, max_positions=64, work=a,
                           work_bytes=1 << 30, status=a, layers=2)


def call(lib, name, a, **changed):
    v = {**a.values, **changed}
    kv = ctypes.byref(v["kv"]) if v["kv"] is not None else None
    rows = ctypes.byref(v["rows"]) if v["rows"] is not None else None
    if name == "write":
        return lib.pgpu_kv8_write(None, kv, v["layer"], rows, v["k"], v["v"], v["stride"],
                                  v["status"])
    if name == "rotate":
        return lib.pgpu_kv8_rotate_write(None, kv, v["layer"], rows, v["qkv"], v["stride"],
                                         v["group"], v["weight"], v["weight"], v["epsilon"],
                                         v["rope"], v["rope_positions"], v["scale"], v["out"],
                                         v["status"])
    if name == "read":
        return lib.pgpu_kv8_read(None, kv, v["layer"], rows, v["lengths"], v["k"], v["v"],
                                 v["stride"], v["status"])
    if name == "close":
        return lib.pgpu_kv8_close(None, kv, v["layer"], v["layers"], v["rows"].tables,
                                  v["rows"].table_stride, v["rows"].slots, v["lengths"],
                                  v["rows"].streams, v["status"])
    return lib.pgpu_kv8_attention(None, kv, v["layer"], rows, v["q"], v["stride"], v["group"],
                                  v["scale"], v["max_positions"], v["out"], v["stride"],
                                  v["work"], v["work_bytes"], v["status"])


NAMES = ("write", "rotate", "read", "close", "attention")


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("field,value", [
    ("values", None), ("scales", None), ("open", None), ("values", 8), ("scales", 4),
    ("open", 4), ("layers", 0), ("heads", 0), ("heads", 257), ("head_dim", 32),
    ("head_dim", 96), ("blocks", 0), ("blocks", 1 << 31), ("slots", 0), ("slots", 1 << 31)])
def test_calls_refuse_a_bad_cache(pkg, name, field, value):
    a = Args(pkg)
    if value in (4, 8) and field in ("values", "scales", "open"):
        value = a.ptr + value if field != "scales" else a.ptr + 4
    setattr(a.kv, field, value)
    lib = pkg.load()
    assert not call(lib, name, a)
    assert b"invalid arguments" in lib.pgpu_last_error()


@pytest.mark.parametrize("name", [n for n in NAMES if n != "close"])
@pytest.mark.parametrize("field,value", [
    ("tables", None), ("table_stride", 0), ("slots", None), ("first", None), ("streams", 0),
    ("streams", 65536), ("rows", -1), ("max_rows", 0), ("max_rows", 6), ("max_rows", -1),
    ("offsets", None)])
def test_calls_refuse_bad_rows(pkg, name, field, value):
    a = Args(pkg)  # offsets NULL: five rows are not one for each of two streams
    setattr(a.rows, field, value)
    assert not call(pkg.load(), name, a)


@pytest.mark.parametrize("name,changed", [
    *[(n, {"layer": -1}) for n in NAMES], *[(n, {"layer": 2}) for n in NAMES],
    *[(n, {"status": None}) for n in NAMES], *[(n, {"kv": None}) for n in NAMES],
    *[(n, {"rows": None}) for n in NAMES if n != "close"],
    ("close", {"layer": 1}), ("close", {"layers": 0}), ("close", {"lengths": None}),
    *[(n, {k: None}) for n in ("write", "read") for k in "kv"],
    *[(n, {k: "odd"}) for n in ("write", "read") for k in "kv"],
    *[(n, {"stride": s}) for n in ("write", "read") for s in (508, 514)],
    ("read", {"lengths": None}),
    ("rotate", {"qkv": None}), ("rotate", {"qkv": "odd"}), ("rotate", {"rope": None}),
    ("rotate", {"rope": "odd"}), ("rotate", {"out": None}), ("rotate", {"out": "odd"}),
    ("rotate", {"weight": "odd"}), ("rotate", {"group": 0}), ("rotate", {"group": 17}),
    ("rotate", {"stride": 1532}), ("rotate", {"stride": 1538}), ("rotate", {"epsilon": -1.0}),
    ("rotate", {"epsilon": float("nan")}), ("rotate", {"scale": float("inf")}),
    ("rotate", {"rope_positions": 0}),
    ("attention", {"q": None}), ("attention", {"q": "odd"}), ("attention", {"out": None}),
    ("attention", {"out": "odd"}), ("attention", {"group": 0}), ("attention", {"group": 17}),
    ("attention", {"stride": 508}), ("attention", {"stride": 514}),
    ("attention", {"max_positions": 0}), ("attention", {"scale": float("nan")}),
    ("attention", {"group": 4})])
def test_calls_refuse_bad_arguments(pkg, name, changed):
    a = Args(pkg)
    changed = {k: a.ptr + 4 if v == "odd" else v for k, v in changed.items()}
    lib = pkg.load()
    lib.pgpu_record_error(b"")
    assert not call(lib, name, a, **changed)
    assert b"invalid arguments" in lib.pgpu_last_error()


@pytest.mark.parametrize("name", ("write", "rotate", "read", "attention"))
def test_a_call_of_no_rows_does_nothing(pkg, name):
    a = Args(pkg, rows=0)
    assert call(pkg.load(), name, a) == 1
