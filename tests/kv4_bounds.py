"""What the 4-bit cache's attention may be off by, against a model in 64 bits, span by span:
the 64 dims that share a scale are held to their own largest weighted value."""
import numpy as np

from kv4_model import SPAN, U


def weights(q, k, first, scale):
    """q [rows][q heads][dim], k [keys][heads][dim] as held -> scores and softmax weights
    [rows][q heads][keys] in 64 bits."""
    group = q.shape[1] // k.shape[1]
    s = scale * np.stack([q[:, h].astype(np.float64) @ k[:, h // group].T
                          for h in range(q.shape[1])], 1)
    seen = np.arange(len(k))[None] <= first + np.arange(len(q))[:, None]
    s = np.where(seen[:, None], s, -np.inf)
    with np.errstate(over="ignore"):
        p = np.exp(s - s.max(-1, keepdims=True))
    return s, p / p.sum(-1, keepdims=True)


def score_error(q, k, s, scale, one):
    """A bound on a score's error, [rows][q heads][1]. One row a stream: q to 2^-29 of its
    largest element, products and sums of 64 exact, 8 roundings of a span's sum. Runs: q in
    two truncated fp16 terms, 2^-21 of each element and 2^-25 of the largest, dim + 8
    roundings of the terms."""
    group = q.shape[1] // k.shape[1]
    out = np.zeros((len(q), q.shape[1], 1))
    for h in range(q.shape[1]):
        x, kk = np.abs(q[:, h].astype(np.float64)), np.abs(k[:, h // group])
        top = x.max(1)[:, None]
        if one:
            spans = sum(np.abs(q[:, h, n:n + SPAN].astype(np.float64) @ k[:, h // group, n:n + SPAN].T)
                        for n in range(0, q.shape[2], SPAN))
            e = 2.0 ** -29 * top * kk.sum(1)[None] + 8 * U * spans
        else:
            e = (2.0 ** -21 + (q.shape[2] + 8) * U) * (x @ kk.T) + 2.0 ** -25 * top * kk.sum(1)[None]
        e = abs(scale) * e
        out[:, h, 0] = np.where(np.isfinite(s[:, h]), e, 0).max(1)
    return out


def output(w, v, rel, one):
    """weights, v [keys][heads][dim] as held, the weights' relative error [rows][q heads][1] ->
    the output in 64 bits and a bound. The weights times their values: 2^-29 of a span's
    largest for each key with one row a stream; in runs 2^-21 of themselves, or 2^-25 of the
    span's largest. A rounding for every key of a sum."""
    rows, heads, keys = w.shape
    group = heads // v.shape[1]
    out, bound = np.zeros((2, rows, heads, v.shape[2]))
    for h in range(heads):
        for n in range(0, v.shape[2], SPAN):
            x = v[:, h // group, n:n + SPAN]
            out[:, h, n:n + SPAN] = o = w[:, h] @ x
            count = (w[:, h] > 0).sum(1, keepdims=True)
            most = (w[:, h] * np.abs(x).max(1)[None]).max(1, keepdims=True)
            part = 2.0 ** -29 if one else 2.0 ** -25
            bound[:, h, n:n + SPAN] = (
                (2 * rel[:, h] + (0 if one else 2.0 ** -20) + (count + 16) * U) * (w[:, h] @ np.abs(x)) +
                count * part * most + 4 * U * np.abs(o))
    return out, bound
