"""The attention of the 8-bit cache: its workspace (what holds a full batch holds every
smaller one), and a scale that it cannot take."""
import ctypes

import pytest

from test_kv8 import Args, call


def size(lib, pkg, heads, dim, group, streams, most, max_rows=None):
    a = Args(pkg)
    a.kv.heads, a.kv.head_dim = heads, dim
    rows = pkg.PgpuKv8Rows(a.ptr, 4, a.ptr, a.ptr, a.ptr if max_rows else None, streams,
                           streams * (max_rows or 1), max_rows or 1)
    return lib.pgpu_kv8_attention_bytes(ctypes.byref(a.kv), ctypes.byref(rows), group, most)


SHAPES = [(8, 64, 1), (8, 64, 4), (2, 128, 1), (4, 128, 9), (1, 64, 16), (256, 64, 1)]


@pytest.mark.parametrize("heads,dim,group", SHAPES)
def test_one_row_a_stream(pkg, heads, dim, group):
    lib = pkg.load()
    for most in (16, 700, 3136, 8192, 131072):
        last = 0
        for streams in (*range(1, 70), 95, 96, 97, 191, 192, 193, 300, 4096, 65535):
            n = size(lib, pkg, heads, dim, group, streams, most)
            assert n >= last, (most, streams)
            assert n >= size(lib, pkg, heads, dim, group, streams, max(1, most // 3))
            last = n


@pytest.mark.parametrize("heads,dim,group", SHAPES)
def test_runs(pkg, heads, dim, group):
    lib = pkg.load()
    for most in (16, 300, 700, 3136, 131072):
        for streams in (1, 2, 3, 7, 16, 63, 64, 200):
            for rows in (1, 5, 16, 17, 100, 300, 4096):
                n = size(lib, pkg, heads, dim, group, streams, most, rows)
                assert n <= 1024 * 64 * (dim + 2) * 4
                for s, r, p in ((1, rows, most), (streams, 1, most), ((streams + 1) // 2, rows, most),
                                (streams, (rows + 1) // 2, most), (streams, rows, most // 2 + 1),
                                (max(1, streams - 1), max(1, rows - 1), most)):
                    assert n >= size(lib, pkg, heads, dim, group, s, p, r), (most, streams, rows, s, r)


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38])
def test_a_scale_that_is_not_finite_in_units_of_log_2(pkg, scale):
    lib = pkg.load()
    lib.pgpu_record_error(b"")
    assert not call(lib, "attention", Args(pkg), scale=scale)
    assert b"invalid arguments" in lib.pgpu_last_error()
