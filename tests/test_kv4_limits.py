"""CPU checks of the 4-bit cache attention's limits: one bound of positions for every batch,
known to both entry points, and sizes of the largest ragged batches."""
import ctypes

import pytest

from test_kv4 import Args, call

MOST_ONE = 65535 * 256  # positions, one row a stream


def batch(pkg, streams, group=1, heads=8, dim=64):
    a = Args(pkg, streams, streams)
    a.kv.heads, a.kv.head_dim = heads, dim
    a.rows.offsets, a.rows.max_rows = None, 1
    a.sums.stride = 1 << 40
    a.values.update(group=group, stride=heads * dim * group)
    return a


@pytest.mark.parametrize("sums", [0, 1])
@pytest.mark.parametrize("streams,group,heads,dim", [(1, 1, 8, 64), (2, 1, 8, 64), (20, 4, 8, 128),
                                                     (300, 1, 8, 64), (65535, 16, 256, 128)])
def test_one_row_a_stream_has_one_bound_of_positions(pkg, streams, group, heads, dim, sums):
    """A size, and a call that only lacks its workspace, up to the bound; past it neither,
    however many streams there are."""
    lib = pkg.load()
    a = batch(pkg, streams, group, heads, dim)
    kv, rows = ctypes.byref(a.kv), ctypes.byref(a.rows)
    without = {} if sums else {"sums": None}
    for most in (MOST_ONE - 1, MOST_ONE):
        n = lib.pgpu_kv4_attention_bytes(kv, rows, group, most, sums)
        assert n > 0
        lib.pgpu_record_error(b"")
        assert not call(lib, "attention", a, max_positions=most, work=None, **without)
        assert b"workspace" in lib.pgpu_last_error()
    for most in (MOST_ONE + 1, 2 ** 24 - 1, 2 ** 24, 2 ** 26, 2 ** 30):
        assert lib.pgpu_kv4_attention_bytes(kv, rows, group, most, sums) == 0
        lib.pgpu_record_error(b"")
        assert not call(lib, "attention", a, max_positions=most, work_bytes=1 << 62, **without)
        assert b"invalid arguments" in lib.pgpu_last_error()
        assert b"workspace" not in lib.pgpu_last_error()


@pytest.mark.parametrize("heads", [1, 3, 8, 256])
def test_runs_with_sums_have_one_bound_of_positions(pkg, heads):
    lib = pkg.load()
    a = Args(pkg)
    a.kv.heads = heads
    a.sums.stride = 1 << 40
    a.values.update(stride=heads * 64)
    kv, rows = ctypes.byref(a.kv), ctypes.byref(a.rows)
    most = min(((1 << 22) - 1) // heads * 64, 1 << 30)
    assert lib.pgpu_kv4_attention_bytes(kv, rows, 1, most, 1) > 0
    assert not call(lib, "attention", a, max_positions=most, work=None)
    assert b"workspace" in lib.pgpu_last_error()
    assert lib.pgpu_kv4_attention_bytes(kv, rows, 1, most + 1, 1) == 0
    lib.pgpu_record_error(b"")
    assert not call(lib, "attention", a, max_positions=most + 1, work_bytes=1 << 62)
    assert b"workspace" not in lib.pgpu_last_error()
    assert b"invalid arguments" in lib.pgpu_last_error()


@pytest.mark.parametrize("sums", [0, 1])
@pytest.mark.parametrize("heads,dim,group", [(1, 64, 1), (8, 64, 2), (256, 128, 16)])
@pytest.mark.parametrize("streams,max_rows", [(65535, 65535), (65535, 40000), (32768, 65535)])
def test_the_workspace_of_the_largest_ragged_batches(pkg, streams, max_rows, heads, dim, group, sums):
    """streams * max_rows past 2^31: parts of 64 rows by 1024 work-groups, or none where the
    work-groups are always many, and with sums what `rows` rows need."""
    lib, rows = pkg.load(), 2 ** 31 - 1
    a = Args(pkg)
    a.kv.heads, a.kv.head_dim = heads, dim
    r = pkg.PgpuKv4Rows(a.ptr, 4, a.ptr, a.ptr, streams, rows, max_rows)
    n = lib.pgpu_kv4_attention_bytes(ctypes.byref(a.kv), ctypes.byref(r), group, 131072, sums)
    wide = heads * group
    parts = 1024 * 64 if 1024 // (heads * ((group + 3) // 4)) > 1 else 0
    kept = sums * ((rows + 16 * streams) * wide * (dim + 1) + rows * wide + 4)
    assert n == (parts * (dim + 2) + kept) * 4
