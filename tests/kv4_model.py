"""A plain model of the 4-bit paged KV cache in numpy, in 64 bits: what a cache holds
after rows were written to it, the attention over that with the sums of its weights, and
what an eviction keeps."""
import numpy as np

BLOCK, SPAN = 16, 64
U = 2.0 ** -24  # half a step of fp32, relative


def scale_of(x):
    """The scale of rows [..., 64], float64."""
    x = np.asarray(x, np.float32)
    t = np.maximum((x.max(-1) / np.float32(7)).astype(np.float32),
                   (-x.min(-1) / np.float32(8)).astype(np.float32))
    t = np.maximum(t, np.float32(0))
    bits = (t.view(np.uint32).astype(np.uint64) + 0xFFFF) // 0x10000 * 0x10000
    return np.maximum(bits.astype(np.uint32).view(np.float32).astype(np.float64), 2.0 ** -17)


def quantise(x):
    """Rows [..., dim] -> whole numbers [..., dim] and scales [..., dim / 64], float64."""
    y = np.asarray(x, np.float64).reshape(*x.shape[:-1], x.shape[-1] // SPAN, SPAN)
    s = scale_of(np.asarray(x, np.float32).reshape(y.shape))
    return np.rint(y / s[..., None]).reshape(x.shape), s


def seen(x):
    """Rows [..., dim] -> what a read of the cache gives."""
    q, s = quantise(x)
    return (q.reshape(*s.shape, SPAN) * s[..., None]).reshape(x.shape)


def pack(n):
    """Whole numbers [..., 16 k] -> bytes [..., 8 k]."""
    n = n.astype(np.int64).reshape(*n.shape[:-1], -1, 16) & 15
    out = np.zeros((*n.shape[:-1], 8), np.uint8)
    for i in range(16):
        out[..., i // 8 * 4 + i % 4] |= (n[..., i] << (i // 4 % 2 * 4)).astype(np.uint8)
    return out.reshape(*out.shape[:-2], -1)


def tile(k, v):
    """Whole numbers [16][dim] of a block's keys and values -> [keys, values][dim / 64][512]."""
    dim = k.shape[1]
    keys = pack(k.reshape(BLOCK, dim // SPAN, SPAN)).transpose(1, 0, 2).reshape(-1, 512)
    values = pack(v.T.reshape(dim // SPAN, SPAN, BLOCK)).reshape(-1, 512)
    return np.stack([keys, values])


def attention(q, k, v, first, scale, seen_keys=None):
    """q [rows][q heads][dim] at cache rows first, first + 1, ...; k, v [keys][heads][dim] as
    held (float64); seen_keys [keys]: False for keys that weigh nothing.
    -> the output, a bound on the error of an fp32 computation of it, the weights
    [rows][q heads][keys], and a bound on theirs."""
    n, qh, dim = q.shape
    group = qh // k.shape[1]
    q = q.astype(np.float64)
    there = np.ones(len(k), bool) if seen_keys is None else np.asarray(seen_keys)
    last = first + np.arange(n)
    mask = (np.arange(len(k))[None] <= last[:, None]) & there
    out, bound = np.zeros((n, qh, dim)), np.zeros((n, qh, dim))
    weights, off = np.zeros((n, qh, len(k))), np.zeros((n, qh, len(k)))
    for h in range(qh):
        kk, vv = k[:, h // group], v[:, h // group]
        x = q[:, h]
        s = np.where(mask, scale * (x @ kk.T), -np.inf)
        top = s.max(1, keepdims=True)
        top[~np.isfinite(top)] = 0
        p = np.where(mask, np.exp(s - top), 0.0)
        l = p.sum(1, keepdims=True)
        l[l == 0] = 1
        weights[:, h] = p / l
        out[:, h] = weights[:, h] @ vv
        # A score: q held to 22 bits below its largest element (two fp16 terms, each
        # truncated), and dim + 8 fp32 roundings of its terms. exp, the maximum's
        # subtraction and the sums of l: 8 roundings, and one for each unit of the exponent.
        ds = abs(scale) * (2.0 ** -21 * np.abs(x).max(1)[:, None] * np.abs(kk).sum(1)[None] +
                           (dim + 8) * U * (np.abs(x) @ np.abs(kk).T))
        ds = np.where(mask, ds, 0).max(1, keepdims=True)
        low = np.where(mask, s, top).min(1, keepdims=True)
        rel = 2 * ds + 8 * U + 4 * U * (top - low)
        # The weights: 21 bits of themselves, or 27 of the largest weighted value of the row;
        # the sums, one rounding for every key.
        count = mask.sum(1, keepdims=True)
        most = (weights[:, h] * np.abs(vv).max(1)[None]).max(1, keepdims=True)
        bound[:, h] = (rel * 2 + 2.0 ** -21 + count * U) * (weights[:, h] @ np.abs(vv)) + \
            count * 2.0 ** -27 * most + 4 * U * np.abs(out[:, h])
        # A weight by itself: 2^(score - log2 of the sum), each rounded once more.
        lse = np.abs(top + np.log(l)) * 1.4427
        off[:, h] = weights[:, h] * (rel * 2 + (count + 8) * U + U * (lse + np.abs(np.where(mask, s, 0)) * 1.4427))
    return out, bound, weights, off


def sums(before, weights, off, first, rows, heads):
    """before [heads][>= keys] or None, and attention's weights of a stream's rows -> what the
    sums of its keys are after the call, [heads][keys], and a bound on an fp32 sum's error."""
    n, qh, keys = weights.shape
    late = slice(max(0, n - rows), n)
    w = weights[late].reshape(-1, heads, qh // heads, keys)
    e = off[late].reshape(w.shape)
    start = np.zeros((heads, keys))
    if before is not None:
        start[:, :first] = before[:, :first]
    total = start + w.sum((0, 2))
    count = w.shape[0] * w.shape[2] + 1
    return total, e.sum((0, 2)) + (count + 2) * U * total + 1e-37


def keep(sums, n, keep, first, newest):
    """The rows that a head with these sums keeps of n."""
    got = np.arange(n)
    if n <= keep:
        return got
    w = np.where(np.isnan(sums[:n]), 0, sums[:n]).astype(np.float64)
    middle = got[first:n - newest]
    best = middle[np.lexsort((middle, -w[middle]))][:keep - first - newest]
    return np.sort(np.concatenate([got[:first], best, got[n - newest:]]))
