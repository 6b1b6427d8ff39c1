"""A plain model of the 8-bit paged KV cache in numpy, in 64 bits: what a cache
holds after rows were written to it, and the attention over that."""
import numpy as np

BLOCK = 16


def scale_of(x):
    """The scale of blocks [..., 16, dim]."""
    t = (np.abs(np.asarray(x, np.float64)).max((-2, -1)) / 127.0).astype(np.float32)
    bits = (t.view(np.uint32).astype(np.uint64) + 0xFFF) // 0x1000 * 0x1000
    s = bits.astype(np.uint32).view(np.float32).astype(np.float64)
    return np.clip(s, 2.0 ** -126, (1 + 16 / 2048) * 2.0 ** 121)


def quantise(x):
    """Blocks [..., 16, dim] -> whole numbers and scales (both float64)."""
    s = scale_of(x)
    return np.rint(np.asarray(x, np.float64) / s[..., None, None]), s


def value_order(dim):
    """Byte of value (position, dim) within a block's values, [16][dim]."""
    p, d = np.arange(BLOCK)[:, None], np.arange(dim)[None]
    return ((p // 4 * 16 + d % 16) * (dim // 16) + d // 16) * 4 + p % 4


def tile(k, v):
    """Whole numbers [16][dim] of keys and values -> the bytes of a (block, head)."""
    out = np.zeros((2, k.size), np.int8)
    out[0] = k.reshape(-1)
    out[1, value_order(k.shape[1]).reshape(-1)] = v.reshape(-1)
    return out


def seen(rows):
    """Rows [length][heads][dim] of one stream's keys or values -> what a read
    of the cache gives: full blocks before the newest as stored, the rest fp32."""
    length = len(rows)
    out = np.asarray(rows, np.float64).copy()
    for b in range(0, (length - 1) // BLOCK * BLOCK, BLOCK):
        q, s = quantise(out[b:b + BLOCK].transpose(1, 0, 2))
        out[b:b + BLOCK] = (q * s[:, None, None]).transpose(1, 0, 2)
    return out


def attention(q, k, v, first, scale):
    """q [rows][q heads][dim] at positions first, first + 1, ...; k, v as `seen`.
    -> the output and a bound on the error of an fp32 computation of it."""
    n, qh, dim = q.shape
    group = qh // k.shape[1]
    out = np.zeros((n, qh, dim))
    bound = np.zeros((n, qh, dim))
    u = 2.0 ** -24
    for h in range(qh):
        kk, vv = k[:, h // group], v[:, h // group]
        for r in range(n):
            keys = first + r + 1
            x = q[r, h].astype(np.float64)
            s = scale * (kk[:keys] @ x)
            p = np.exp(s - s.max())
            l = p.sum()
            out[r, h] = p @ vv[:keys] / l
            # A score: q held to 22 bits below its largest element, and dim + 8
            # fp32 roundings of its terms. exp, the maximum's subtraction and
            # the sums of l: 8 roundings, and one for each unit of the exponent.
            ds = abs(scale) * (2.0 ** -22 * np.abs(x).max() * np.abs(kk[:keys]).sum(1)
                               + (dim + 8) * u * (np.abs(kk[:keys]) @ np.abs(x))).max()
            rel = 2 * ds + 8 * u + 4 * u * (s.max() - s.min())
            # The weights: 22 bits below the largest weighted value, for every
            # key; the sums, one rounding for every key.
            top = (p * np.abs(vv[:keys]).max(1)).max()
            bound[r, h] = (rel * 2 + keys * u) * (p @ np.abs(vv[:keys])) / l + \
                keys * 2.0 ** -22 * top / l + 4 * u * np.abs(out[r, h])
    return out, bound


def turn(x, weight, epsilon, rope):
    """Heads [rows][heads][dim], normalised (weight or None) and turned by
    rope [rows][dim / 2][2], in 64 bits."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + epsilon) * weight
    a, b = x[..., 0::2], x[..., 1::2]
    c, s = rope[:, None, :, 0].astype(np.float64), rope[:, None, :, 1].astype(np.float64)
    return np.stack((a * c - b * s, a * s + b * c), -1).reshape(x.shape)
