"""The 8-bit paged KV cache's attention at scores past what fp32 counts in ones, against 64
bits: values, not only finiteness."""
import numpy as np
import pytest

import kv8_model as model
from test_gpu_kv8 import Attend, cache  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("most", [None, 8192])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("size,large", [(2.0 ** 18, 1.0), (1.3e7, 1e4), (3e8, 1.0), (1.15e9, 1e4),
                                        (2.0 ** 41, 1e4), (1e30, 1.0)])
@pytest.mark.parametrize("heads,dim,group", [(2, 64, 1), (1, 64, 3), (2, 128, 1), (1, 128, 2)])
@pytest.mark.parametrize("counts", [None, [1, 15, 40, 100]], ids=["one", "runs"])
def test_scores_of_any_size(cache, counts, heads, dim, group, size, large, sign, most):
    """One key has a score that is half of the others', or the others' half of its: it weighs
    1, whatever the scores are, and rows come out as its values."""
    lengths, at = [1, 40, 300, 130], [0, 20, 250, 3]
    c = cache(4, heads, dim, positions=320)
    rng = c.rng
    way = np.where(rng.integers(0, 2, (4, heads, dim)), 1.0, -1.0)
    k = np.concatenate([np.repeat(way[s][None] * large * (0.5 if sign > 0 else 1.0), n, 0)
                        for s, n in enumerate(lengths)])
    _, v = c.random_rows(sum(lengths))
    rows = np.asarray(at) + np.concatenate([[0], np.cumsum(lengths)[:-1]])
    k[rows] *= 2.0 if sign > 0 else 0.5
    v *= np.exp2(rng.integers(-12, 13, (len(v) // 16 + 1, heads, 1))).repeat(16, 0)[:len(v)].astype(np.float32)
    c.write([0] * 4, lengths, k.astype(np.float32), v)
    assert c.st() == 0
    n = counts or [1] * 4
    a = Attend(c, [m - x for m, x in zip(lengths, n)], counts, group, most=most)
    q = rng.uniform(1.0, 2.0, a.q.shape) * sign
    q *= np.repeat(np.concatenate([np.repeat(way[s][None], m, 0) for s, m in enumerate(n)]), group, 1)
    a.q = (q * (size / 1.4427 / (abs(a.scale) * 1.5 * dim * large))).astype(np.float32)
    a.dq.upload(a.q.reshape(len(a.q), -1))
    got = a.run()
    assert c.st() == 0
    here = 0
    for s, m in enumerate(n):
        held = np.repeat(model.seen(c.rows[s][1])[at[s]], group, 0)
        # Two truncated fp16 terms of the weight, some roundings: 2^-20 of the largest.
        off = 2.0 ** -20 * np.abs(held).max(-1, keepdims=True)
        miss = np.abs(got[here:here + m] - held) - off
        assert (miss <= 0).all(), (s, miss.max())
        here += m
