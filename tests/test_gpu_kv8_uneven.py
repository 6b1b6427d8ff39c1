"""Attention over the 8-bit cache where magnitudes are uneven: blocks, dims and
queries that differ by many powers of two. Every element against 64 bits, within
a bound of its own dim: what an fp32 computation of it loses, and of the largest
weighted scale of the row as little as phonon_gpu.h says."""
import numpy as np
import pytest

import kv8_model as model
from test_gpu_kv8 import BLOCK, Attend, cache  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def want_by_dim(q, k, v, first, scale, held, lost=()):
    """q [rows][q heads][dim] at positions first, ...; k, v [length][heads][dim] as
    model.seen gives them; held [blocks][heads]: the value scales of the blocks
    before the newest; lost: blocks that weigh nothing. -> the output and each
    element's bound."""
    n, qh, dim = q.shape
    group, u = qh // k.shape[1], 2.0 ** -24
    out, bound = np.zeros((n, qh, dim)), np.zeros((n, qh, dim))
    for h in range(qh):
        kk, vv, sv = k[:, h // group], np.abs(v[:, h // group]), held[:, h // group]
        sv = np.repeat(sv, BLOCK)
        sv = np.concatenate([sv, np.zeros(len(kk) - len(sv))])  # the newest block: fp32
        whole = np.where(sv[:, None] > 0, vv / np.where(sv > 0, sv, 1)[:, None], 0)
        for r in range(n):
            keys = first + r + 1
            x = q[r, h].astype(np.float64)
            s = scale * (kk[:keys] @ x)
            on = ~np.isin(np.arange(keys) // BLOCK, lost)
            if not on.any():
                continue  # zeros
            s[~on] = s[on].min()
            p = np.exp(s - s.max()) * on
            l = p.sum()
            out[r, h] = p @ v[:keys, h // group] / l
            # A score: a query in two truncated fp16 terms (2^-21 of an element), or
            # to 2^-30 of its largest one; the fp32 sum of both terms' products, and
            # its scaling. Its exponential: the subtraction of the maximum, 1 ulp.
            ds = abs(scale) * ((2.0 ** -21 + (2 * dim + 8) * u) * (np.abs(kk[:keys]) @ np.abs(x))
                               + 2.0 ** -30 * np.abs(x).max() * np.abs(kk[:keys]).sum(1))
            rel = ds + 4 * u * (s.max() - s) + 8 * u
            # A weight times its block's scale: two terms again, and 2^-28 of the
            # largest of them; the sums of both terms, and of the weights.
            rel = rel + 2.0 ** -21 + 2 * keys * u
            mass = p @ vv[:keys] / l
            bound[r, h] = 1.1 * ((p * rel) @ vv[:keys] / l + (p @ rel) / l * mass) + \
                2.0 ** -28 * (p * sv[:keys]).max() / l * whole[:keys].sum(0) + 8 * u * mass
    return out, bound


def check(c, a, got, lost=(), status=0):
    """lost[s]: blocks of stream s that weigh nothing."""
    at = 0
    for s, n in enumerate(a.counts):
        length = a.first[s] + n
        k, v = (model.seen(x[:length]) for x in c.rows[s])
        closed = (length - 1) // BLOCK
        held = np.array([model.scale_of(c.rows[s][1][b * BLOCK:(b + 1) * BLOCK].transpose(1, 0, 2))
                         for b in range(closed)]).reshape(closed, c.heads)
        want, bound = want_by_dim(a.q[at:at + n], k, v, a.first[s], a.scale, held,
                                  lost[s] if lost else ())
        far = np.abs(got[at:at + n] - want) > bound
        assert not far.any(), (s, np.argwhere(far)[:3], got[at:at + n][far][:3], want[far][:3],
                               bound[far][:3])
        at += n
    assert c.st() == status


GROWTH = {
    "up": lambda b: 30 * b - 60,           # each block 2^30 times the one before
    "down": lambda b: 60 - 30 * b,
    "one": lambda b: 40 * (b == 1),        # one block above all others
    "first": lambda b: 40 * (b == 0),
    "steps": lambda b: 5 * (b % 3),        # just past what shares one exponent
    "near": lambda b: 4 * (b % 2),
}


@pytest.mark.parametrize("growth", GROWTH)
@pytest.mark.parametrize("heads,group,dim", [(2, 1, 64), (1, 3, 128)])
def test_runs_over_blocks_of_uneven_values(cache, growth, heads, group, dim):
    """Rows of a run from position 0, whose blocks of values differ by up to 2^120: a
    row takes its bits from what it sees, whatever stands behind it."""
    c = cache(2, heads, dim, positions=190)
    for n in (70, 85):
        k, v = (x.reshape(2, n, heads, dim) for x in c.random_rows(2 * n))
        at = np.stack([len(r[0]) + np.arange(n) for r in c.rows])
        power = np.array([[GROWTH[growth](p // BLOCK % 5) for p in r] for r in at])
        v = v * np.float32(2.0) ** power[..., None, None].astype(np.float32)
        c.write(c.lengths(), [n, n], k.reshape(-1, heads, dim), v.reshape(-1, heads, dim))
    for first, counts in (([0, 0], [155, 155]), ([16, 150], [139, 5])):
        a = Attend(c, first, counts, group)
        check(c, a, a.run())
    # The same rows with their keys dealt to several work-groups and joined.
    a = Attend(c, [120, 140], [35, 15], group, most=c.stride * BLOCK + 2000)
    check(c, a, a.run())


@pytest.mark.parametrize("behind", [0.0, 21.0, 60.0, 250.0])
def test_a_large_block_with_a_small_weight(cache, behind):
    """A block of values 2^40 above the others whose keys score `behind` below
    them: it weighs e^-behind, and the others keep their bits."""
    c = cache(1, 2, 64, positions=200)
    k, v = c.random_rows(200)
    k *= np.float32(0.1)
    k[32:48, :, 0] = -2 * behind
    v[32:48] *= np.float32(2.0 ** 40)
    c.write([0], [200], k, v)
    a = Attend(c, [0], [200], 1)
    a.q[:, :, 0] = 4.0
    a.dq.upload(a.q.reshape(a.total, -1))
    check(c, a, a.run())


@pytest.mark.parametrize("behind", [0.0, 5.0, 21.0, 250.0])
@pytest.mark.parametrize("heads,group,dim", [(2, 1, 64), (1, 4, 128)])
def test_one_row_beside_a_large_block_of_little_weight(cache, behind, heads, group, dim):
    c = cache(1, heads, dim, positions=400)
    k, v = c.random_rows(400)
    k *= np.float32(0.1)
    k[32:48, :, 0] = -2 * behind
    v[32:48] *= np.float32(2.0 ** 40)
    c.write([0], [400], k, v)
    for most in (400, 8192):  # whole, and dealt
        a = Attend(c, [399], None, group, most=most)
        a.q[:, :, 0] = 0.5 * dim ** 0.5
        a.dq.upload(a.q.reshape(a.total, -1))
        check(c, a, a.run())


@pytest.mark.parametrize("power", [4, 10, 14, 17])
@pytest.mark.parametrize("heads,group,dim", [(2, 1, 64), (1, 4, 128)])
@pytest.mark.parametrize("runs", [False, True])
def test_dims_beside_a_far_larger_one(cache, power, heads, group, dim, runs):
    """One element of the values, and one of the queries over a key channel of next to
    nothing, 2^power above the others: the other dims are held by their own size."""
    c = cache(2, heads, dim, positions=300)
    k, v = (x.reshape(2, 300, heads, dim) for x in c.random_rows(600))
    v[0, 40::64, :, 5] = 2.0 ** power
    k[1, :, :, 7] *= np.float32(2.0 ** -power)
    c.write([0, 0], [300, 300], k.reshape(-1, heads, dim), v.reshape(-1, heads, dim))
    first, counts = ([0, 200], [300, 100]) if runs else ([299, 299], None)
    a = Attend(c, first, counts, group)
    a.q[counts[0] if runs else 1:, :, 7] = 2.0 ** power
    a.dq.upload(a.q.reshape(a.total, -1))
    check(c, a, a.run())
