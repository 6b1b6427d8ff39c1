"""The 4-bit paged KV cache's attention where magnitudes meet, against 64 bits: scores past
what fp32 counts in ones, spans of a head whose values differ in size, one large value among
many ordinary ones, the precision that one row a stream is held to; values, not only
finiteness, and the sums of weights with them."""
import numpy as np
import pytest

import kv4_bounds as bounds
import kv4_model as model
from test_gpu_kv4 import Attend, cache  # noqa: F401

pytestmark = pytest.mark.gpu
U = model.U


def attend(c, q, counts, group, **kw):
    """The last rows of every stream, with these queries -> Attend, its output."""
    n = counts or [1] * c.n
    a = Attend(c, [m - x for m, x in zip(c.lengths(), n)], counts, group, **kw)
    a.q = q.astype(np.float32)
    a.dq.upload(a.q.reshape(a.total, -1))
    return a, a.run()


def streams_of(c, a):
    """(stream, its rows of the call, keys and values as held, its first row's index)."""
    at = 0
    for s, n in enumerate(a.n):
        yield s, slice(at, at + n), [model.seen(x) for x in c.rows[s]], a.first[s]
        at += n


def check_sums(c, a, s, w, rel):
    """A stream's sums against weights [rows][q heads][keys] that may be off by rel."""
    keys = w.shape[-1]
    w = w[max(0, len(w) - a.counted):].reshape(-1, c.heads, a.group, keys).sum((0, 2))
    want = np.zeros((c.heads, keys))
    want[:, :a.first[s]] = a.before0[s, :, :a.first[s]]
    count = min(a.n[s], a.counted) * a.group
    miss = np.abs(a.added()[s, :, :keys] - want - w) - rel * w - (count + 2) * U * (want + w) - 1e-37
    assert (miss <= 0).all(), (s, miss.max())


def two_kinds(c, counts, group, size, large):
    """Keys of a stream and head that are all the same, or half of that, at the places that
    `half` says: any two scores are equal, also when they are rounded, or far apart. Queries
    along them, every second head against them. `size`: of the scores in units of log 2."""
    rng, dim = c.rng, c.dim
    lengths = [1, 1, 40, 70, 300, 17, 130]
    sign = np.where(rng.integers(0, 2, (c.n, c.heads, dim)), 1.0, -1.0)
    half = [np.zeros(n, bool) for n in lengths]
    half[2][:] = True
    half[2][20] = False      # one of full size among halves, in the middle, late, last
    half[4][:] = True
    half[4][250] = False
    half[5][:] = True
    half[5][16] = False
    half[6][100:] = True     # halves at the end
    k = np.concatenate([np.where(h, 0.5, 1.0)[:, None, None] * sign[s][None] * large
                        for s, h in enumerate(half)])
    v = rng.standard_normal((sum(lengths), c.heads, dim))
    v *= np.exp2(rng.integers(-12, 13, (len(v), c.heads, 1)))
    v[0] *= 57000 / np.abs(v[0]).max()
    v[1] *= 2.0 ** -17 / np.abs(v[1]).max()
    c.write([0] * c.n, lengths, k.astype(np.float32), np.clip(v, -57000, 57000).astype(np.float32))
    assert c.st() == 0
    n = counts or [1] * c.n
    held = np.abs(model.seen(np.float32(large) * np.ones(64, np.float32)))[0]
    q = rng.uniform(1.0, 2.0, (sum(n), c.heads * group, dim))
    along = np.repeat(np.concatenate([np.repeat(sign[s][None], m, 0) for s, m in enumerate(n)]),
                      group, 1)
    flip = np.where(np.arange(c.heads * group) % 2, -1.0, 1.0)[:, None]
    return along * flip * q * (size / 1.4427 / (c.dim ** -0.5 * 1.5 * dim * held))


@pytest.mark.parametrize("most", [None, 8192])
@pytest.mark.parametrize("size,large", [(2.0 ** 18, 1.0), (1.3e7, 1e4), (3e8, 1.0), (1.15e9, 1e4),
                                        (2.0 ** 41, 1e4), (1e30, 1.0)])
@pytest.mark.parametrize("heads,dim,group", [(2, 64, 1), (2, 64, 3), (1, 128, 2), (2, 128, 1)])
@pytest.mark.parametrize("counts", [None, [1, 1, 25, 60, 55, 17, 40]], ids=["one", "runs"])
def test_scores_of_any_size(cache, counts, heads, dim, group, large, size, most):
    """Rows see one key, some that weigh the same, or some that weigh nothing beside others;
    their values differ by 2^24 and more. A key alone weighs 1, whatever its score is."""
    c = cache(7, heads, dim, positions=300)
    q = two_kinds(c, counts, group, size, large)
    a, got = attend(c, q, counts, group, most=most)
    assert c.st() == 0
    one = counts is None
    for s, rows, (k, v), first in streams_of(c, a):
        x, w = bounds.weights(a.q[rows], k, first, a.scale)
        assert (np.abs(x[np.isfinite(x)]).max() * 1.4427 > size / 4)
        out, off = bounds.output(w, v, np.zeros((len(w), heads * group, 1)), one)
        miss = np.abs(got[rows] - out) - off
        assert (miss <= 0).all(), (s, miss.max())


@pytest.mark.parametrize("most", [None, 8192])
@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 18, 1.3e7, 3e8, 1.15e9, 2.0 ** 41, 1e30])
@pytest.mark.parametrize("heads,dim,group", [(2, 64, 1), (2, 64, 3), (1, 128, 2), (1, 128, 8)])
@pytest.mark.parametrize("counts", [None, [1, 1, 25, 60, 55, 17, 40]], ids=["one", "runs"])
def test_sums_of_weights_of_scores_of_any_size(cache, counts, heads, dim, group, size, most):
    """The same keys' weights: 1, or one part of as many as weigh the same. Runs hold a row's
    sum of weights to 2^-23, or to 2^-16 where the scores pass 2^23."""
    c = cache(7, heads, dim, positions=300)
    q = two_kinds(c, counts, group, size, 1.0)
    a, _ = attend(c, q, counts, group, most=most, sums=30)
    assert c.st() == 0
    for s, rows, (k, _), first in streams_of(c, a):
        x, w = bounds.weights(a.q[rows], k, first, a.scale)
        if size < 2000:  # halves weigh something: only rows that see one kind are exact
            w = np.where(w < 2.0 ** -100, 0, w)
        # exp2 twice and a logarithm or a division: 16 roundings; a row's sum: one for
        # every key, and in runs two truncated terms of each weight.
        rel = (w.shape[-1] + 16) * U + (0 if counts is None else
                                        2.0 ** -20 if size < 2.0 ** 22 else 2.0 ** -15)
        check_sums(c, a, s, w, rel)


@pytest.mark.parametrize("most", [None, 8192])
@pytest.mark.parametrize("apart", [0, 10, 20, 25, -10, -20, -25])
@pytest.mark.parametrize("heads,group", [(2, 1), (1, 4), (3, 2)])
@pytest.mark.parametrize("counts", [None, [40, 33, 150]], ids=["one", "runs"])
def test_spans_whose_values_differ_in_size(cache, counts, heads, group, apart, most):
    """A head of 128 whose last 64 dims are 2^apart times its first: each span is held to
    its own largest weighted value."""
    c = cache(3, heads, 128, positions=300)
    k, v = c.random_rows(800)
    v = c.rng.standard_normal(v.shape) * np.where(np.arange(128) < 64, 1.0, 2.0 ** apart)
    v *= 2.0 ** (-12 if apart > 0 else 12 if apart < -20 else 5 if apart < -10 else 0)
    c.write([0] * 3, [300, 201, 299], k, np.clip(v, -5e4, 5e4).astype(np.float32))
    assert c.st() == 0
    n = sum(counts or [1] * 3)
    a, got = attend(c, c.rng.standard_normal((n, heads * group, 128)), counts, group, most=most)
    assert c.st() == 0
    check_rows(c, a, got, counts is None)


def check_rows(c, a, got, one):
    for s, rows, (k, v), first in streams_of(c, a):
        x, w = bounds.weights(a.q[rows], k, first, a.scale)
        ds = bounds.score_error(a.q[rows], k, x, a.scale, one)
        # exp2 and its argument, of a score and of the maximum.
        spread = np.where(np.isfinite(x), x.max(-1, keepdims=True) - x, 0).max(-1, keepdims=True)
        rel = 2 * ds + 8 * U + 4 * U * spread
        out, off = bounds.output(w, v, rel, one)
        miss = np.abs(got[rows] - out) - off
        assert (miss <= 0).all(), (s, miss.max(), (np.abs(got[rows] - out) / off).max())
        if a.sums:
            # And the weight by itself: relative to the row's sum.
            check_sums(c, a, s, w, 2 * rel.max() + (w.shape[-1] + 16) * U + (0 if one else 2.0 ** -20))


@pytest.mark.parametrize("heads,dim,group", [(2, 64, 1), (1, 64, 4), (2, 128, 1), (1, 128, 3)])
@pytest.mark.parametrize("most", [None, 8192])
def test_one_row_a_stream_is_held_to_2_to_the_minus_29(cache, heads, dim, group, most):
    """Queries and values whose elements differ by 2^20, in one span or the other."""
    c = cache(4, heads, dim, positions=900)
    k, v = c.random_rows(1700)
    v *= np.exp2(c.rng.integers(-11, 10, (len(v), heads, 1))).astype(np.float32)
    c.write([0] * 4, [899, 1, 500, 300], k, np.clip(v, -5e4, 5e4))
    q = c.rng.standard_normal((4, heads * group, dim))
    q *= np.exp2(c.rng.integers(-20, 1, q.shape))
    a, got = attend(c, q, None, group, most=most, sums=1)
    assert c.st() == 0
    check_rows(c, a, got, True)


CALLS = {"one": (None, 2, 2, [2100, 1300]), "runs": ([40, 100], 2, 2, [2100, 1300]),
         # So many work-groups that each has all of its rows' keys.
         "whole": ([512, 500], 8, 4, [900, 1000])}


@pytest.mark.parametrize("above", [0.0, 8.0])
@pytest.mark.parametrize("larger", [12, 20, 28])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("call", CALLS)
def test_one_large_value_among_ordinary_ones(cache, call, dim, larger, above):
    """One key with values 2^larger times the others' and a score `above` the others' (in
    units of log 2): it raises what the products are held to, not what the row's sum of
    weights is. All of a row's weights together are 1."""
    counts, heads, group, lengths = CALLS[call]
    c = cache(2, heads, dim, positions=max(lengths))
    rng = c.rng
    at, n = [70, 133], counts or [1, 1]
    k, v = c.random_rows(sum(lengths))
    v = rng.standard_normal(v.shape) * 2.0 ** (-14 if larger > 12 else 0)
    way = rng.standard_normal((2, heads, dim))  # queries and the large keys lie along it
    way /= np.sqrt((way ** 2).sum(-1, keepdims=True))
    for s in range(2):
        row = at[s] + (lengths[0] if s else 0)
        v[row] *= 2.0 ** larger
        if above:
            k[row] = way[s] * (above / 1.4427 * dim ** 0.5)
    c.write([0, 0], lengths, k.astype(np.float32), np.clip(v, -5e4, 5e4).astype(np.float32))
    assert c.st() == 0
    q = np.concatenate([np.repeat(np.repeat(way[s][None], m, 0), group, 1) for s, m in enumerate(n)])
    q = q + 0.02 * rng.standard_normal(q.shape)
    a, got = attend(c, q, counts, group, sums=1)
    assert c.st() == 0
    check_rows(c, a, got, counts is None)
    # With before all zeros: the weights of the last row's queries.
    a.before.upload(np.zeros_like(a.before0))
    a.run()
    total = a.added()
    for s in range(2):
        # 16 roundings of a weight. The row's sum of weights: of one row a stream a lane adds
        # 16, then 6 and 8 levels; in runs each of 33 chunks takes 4 products, of weights in
        # two truncated terms.
        t = total[s, :, :lengths[s]].astype(np.float64).sum(-1) / group
        off = 48 * U if counts is None else 2.0 ** -21 + 150 * U
        assert (np.abs(t - 1) <= off).all(), (s, t - 1)


@pytest.mark.parametrize("heads,dim,group", [(2, 64, 1), (1, 64, 3), (2, 128, 2)])
def test_ordinary_rows_after_large_ones(cache, heads, dim, group):
    """Blocks of large and of ordinary values in turn, scores that rise and fall along the
    keys: what the products are held to rises with the ones and falls behind the others."""
    c = cache(3, heads, dim, positions=1000)
    k, v = c.random_rows(2600)
    v = c.rng.standard_normal(v.shape)
    place = np.arange(2600)
    v *= np.exp2(np.where(place // 48 % 3 == 1, 12.0, np.where(place // 48 % 3 == 2, -8.0, 0.0)))[:, None, None]
    k *= np.float32(0.3) + (np.abs(place % 400 - 200) / 200).astype(np.float32)[:, None, None]
    c.write([0] * 3, [1000, 700, 900], k, np.clip(v, -5e4, 5e4).astype(np.float32))
    for counts in (None, [100, 700, 60]):
        n = sum(counts or [1] * 3)
        for most in (None, 8192):
            a, got = attend(c, 2 * c.rng.standard_normal((n, heads * group, dim)), counts, group,
                            most=most, sums=50)
            assert c.st() == 0
            check_rows(c, a, got, counts is None)


@pytest.mark.parametrize("size", [3e6, 3e8, 2e9])
@pytest.mark.parametrize("heads,dim,group", [(2, 64, 1), (2, 64, 3), (1, 128, 1), (2, 128, 4)])
@pytest.mark.parametrize("counts", [None, [130, 70, 33, 200, 100]], ids=["one", "runs"])
def test_scores_that_pass_what_is_counted_and_come_back(cache, counts, heads, dim, group, size):
    """Keys of three sizes, all of one size the same, in runs along the context: ordinary
    scores before and behind vast ones, of both signs; some blocks are not in the cache, and
    values differ by 2^24."""
    c = cache(5, heads, dim, positions=1100)
    rng = c.rng
    lengths = [1100, 900, 1000, 600, 700]
    kinds = [np.r_[np.zeros(600), np.full(300, 2), np.zeros(200)],          # ordinary, vast, ordinary
             np.r_[np.full(300, 2), np.zeros(600)],                         # vast first
             np.arange(1000) // 70 % 3,                                     # in turn
             np.r_[np.zeros(590), np.full(10, 1)],                          # vast at the end
             np.r_[np.full(40, 1), np.zeros(400), np.full(260, 2)]]
    sign = np.where(rng.integers(0, 2, (5, heads, dim)), 1.0, -1.0)
    large = 1e4
    k = np.concatenate([np.array([2.0 ** -20, 0.5, 1.0])[x.astype(int)][:, None, None] * sign[s][None] * large
                        for s, x in enumerate(kinds)])
    v = rng.standard_normal(k.shape) * np.exp2(rng.integers(-12, 13, (len(k), heads, 1)))
    c.write([0] * 5, lengths, k.astype(np.float32), np.clip(v, -5e4, 5e4).astype(np.float32))
    assert c.st() == 0
    table = c.table.copy()
    lost = [[], [3, 40], [7], [], [1, 2, 30]]
    for s, blocks in enumerate(lost):
        table[s, blocks] = c.blocks + s
    n = counts or [1] * 5
    q = rng.uniform(1.0, 2.0, (sum(n), heads * group, dim))
    q *= np.repeat(np.concatenate([np.repeat(sign[s][None], m, 0) for s, m in enumerate(n)]), group, 1)
    q *= np.where(np.arange(heads * group) % 2, -1.0, 1.0)[:, None]
    q *= size / 1.4427 / (dim ** -0.5 * 1.5 * dim * large)
    for tables, missing in ((c.table, [[]] * 5), (table, lost)):
        c.tables.upload(tables)
        a, got = attend(c, q, counts, group, sums=50)
        assert c.st() == (2 if tables is table else 0)
        for s, rows, (kk, vv), first in streams_of(c, a):
            there = np.ones(len(kk), bool)
            for b in missing[s]:
                there[b * 16:b * 16 + 16] = False
            x, _ = bounds.weights(a.q[rows], kk, first, a.scale)
            x = np.where(there, x, -np.inf)
            w = np.exp(x - x.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            # Keys of a size weigh the same, to the roundings of a weight.
            out, off = bounds.output(w, vv, np.zeros((len(w), heads * group, 1)), counts is None)
            miss = np.abs(got[rows] - out) - off
            assert (miss <= 0).all(), (s, miss.max())
            check_sums(c, a, s, w, (w.shape[-1] + 16) * U + (0 if counts is None else 2.0 ** -15))
