"""The workspace of the 4-bit cache's attention: what holds a full batch holds every smaller
one, and with sums what their scores need."""
import ctypes

import pytest

from test_kv4 import Args


def size(lib, pkg, heads, dim, group, streams, most, max_rows=None, sums=0):
    a = Args(pkg)
    a.kv.heads, a.kv.head_dim = heads, dim
    rows = pkg.PgpuKv4Rows(a.ptr, 4, a.ptr, a.ptr if max_rows else None, streams,
                           streams * (max_rows or 1), max_rows or 1)
    return lib.pgpu_kv4_attention_bytes(ctypes.byref(a.kv), ctypes.byref(rows), group, most, sums)


SHAPES = [(8, 64, 1), (8, 64, 4), (2, 128, 1), (4, 128, 9), (1, 64, 16), (256, 64, 1), (8, 128, 2)]


@pytest.mark.parametrize("sums", [0, 1])
@pytest.mark.parametrize("heads,dim,group", SHAPES)
def test_one_row_a_stream(pkg, heads, dim, group, sums):
    lib = pkg.load()
    for most in (16, 700, 1600, 3136, 6200, 8192, 131072):
        last = 0
        for streams in (*range(1, 70), 95, 96, 97, 191, 192, 193, 300, 511, 512, 4096, 65535):
            n = size(lib, pkg, heads, dim, group, streams, most, sums=sums)
            assert n >= last, (most, streams)
            assert n >= size(lib, pkg, heads, dim, group, streams, max(1, most // 3), sums=sums)
            assert n >= sums * streams * heads * group * (most + 1) * 4
            last = n


@pytest.mark.parametrize("sums", [0, 1])
@pytest.mark.parametrize("heads,dim,group", SHAPES)
def test_runs(pkg, heads, dim, group, sums):
    lib = pkg.load()
    for most in (16, 300, 700, 3136, 131072):
        for streams in (1, 2, 3, 7, 16, 63, 64, 200):
            for rows in (1, 5, 16, 17, 100, 300, 4096):
                n = size(lib, pkg, heads, dim, group, streams, most, rows, sums)
                # Parts of 64 rows by 1024 work-groups; with sums, the queries as operands, a
                # factor and a log sum for each, by tiles of 16 rows.
                kept = sums * heads * group * streams * ((rows + 16) * (dim + 1) + rows) + 4
                assert n <= (1024 * 64 * (dim + 2) + kept) * 4
                for s, r, p in ((1, rows, most), (streams, 1, most), ((streams + 1) // 2, rows, most),
                                (streams, (rows + 1) // 2, most), (streams, rows, most // 2 + 1),
                                (max(1, streams - 1), max(1, rows - 1), most)):
                    assert n >= size(lib, pkg, heads, dim, group, s, p, r, sums), (most, streams, rows, s, r)
