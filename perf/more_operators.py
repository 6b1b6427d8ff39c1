"""Operators of the 4-bit paged KV cache and of eviction from it: plain forms, and the library's calls.

A server with more or longer requests than an 8-bit cache has room for holds their keys and
values in 4 bits. Each row (one position of one head) has a scale of its own for every 64
dims of its key and of its value, so that a row is quantised once, when it is written, and
moved as it is. The attention reads the cache one query a stream (a frame) or in runs of
rows (a prompt); it can add what each position weighed to that position's sum. Where a
stream outgrows its budget, each head keeps its first and newest positions and those with
the largest sums, closed up in order.

  own        False: the plain forms, in torch; True: the library's entry points
  listed()   the cases that are reported by name
  draw(rng)  one more case of the same ranges
  prepare / run / work / exact   see each function
"""
import ctypes
import importlib.util
import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BLOCK = 16           # positions of a block
SPAN = 64            # dims of a scale
LEAST, MOST = 2.0 ** -17, 8160.0  # scales


# ------------------------------------------------------------------ the cases


def listed():
    return [
        # The first frame of a lone request: one key. The smallest call.
        {"name": "attend_1_first", "kind": "attend", "streams": 1, "idle": 0, "low": 1, "high": 1,
         "heads": 8, "group": 1, "dim": 64, "sums": 0},
        # 64 requests somewhere in their lives; three slots of the batch are empty.
        {"name": "attend_64", "kind": "attend", "streams": 64, "idle": 3, "low": 1, "high": 2048,
         "heads": 8, "group": 1, "dim": 64, "sums": 0},
        # A full server with long contexts.
        {"name": "attend_256_long", "kind": "attend", "streams": 256, "idle": 0, "low": 256,
         "high": 8187, "heads": 8, "group": 1, "dim": 64, "sums": 0},
        # Four query heads to a key head, wider heads.
        {"name": "attend_48_grouped", "kind": "attend", "streams": 48, "idle": 0, "low": 1,
         "high": 4096, "heads": 8, "group": 4, "dim": 128, "sums": 0},
        # A frame of 64 requests that are near their budget: what each key weighed is kept.
        {"name": "weigh_64", "kind": "attend", "streams": 64, "idle": 3, "low": 1, "high": 2048,
         "heads": 8, "group": 1, "dim": 64, "sums": 1},
        # Prompts of newly admitted requests that continue a prefix already held, ragged.
        {"name": "prompt_3_ragged", "kind": "prompt", "streams": 3, "low": 37, "high": 300,
         "prefix": 200, "heads": 8, "group": 1, "dim": 64, "sums": 0},
        # One prompt as long as a stream may be: the largest call.
        {"name": "prompt_1_long", "kind": "prompt", "streams": 1, "low": 8187, "high": 8187,
         "prefix": 0, "heads": 8, "group": 1, "dim": 64, "sums": 0},
        # Prompts over their budget at once: every row's weights are summed.
        {"name": "weigh_5_prompts", "kind": "prompt", "streams": 5, "low": 300, "high": 1777,
         "prefix": 0, "heads": 8, "group": 2, "dim": 64, "sums": 1777},
        # A request's rows into the cache and out again, of an odd length and from inside a
        # block; and a whole server's, handed over to another process.
        {"name": "store_1x211", "kind": "store", "streams": 1, "low": 211, "high": 211,
         "heads": 8, "dim": 64},
        {"name": "store_64", "kind": "store", "streams": 64, "low": 1, "high": 2048, "heads": 8,
         "dim": 64},
        # A lone request shrunk to a quarter; a server's requests shrunk to half of what the
        # longest hold (the shorter ones stay whole).
        {"name": "evict_1", "kind": "evict", "streams": 1, "low": 2011, "high": 2011, "keep": 500,
         "first": 4, "newest": 128, "heads": 8, "dim": 64},
        {"name": "evict_64", "kind": "evict", "streams": 64, "low": 600, "high": 2048,
         "keep": 1024, "first": 4, "newest": 256, "heads": 8, "dim": 64},
    ]


def _between(rng, low, high):
    """A whole number in [low, high], even over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "prompt", "prompt", "store", "evict", "evict"))
    heads, dim = rng.choice(((8, 64), (8, 64), (4, 128), (8, 128), (6, 64)))
    group = rng.choice((1, 1, 2, 3, 4, 8))
    if kind == "attend":
        high = _between(rng, 1, 8187)
        most = 256 * 4200 * 512 // (high * heads * dim)
        streams = _between(rng, 1, min(256, most))
        return {"kind": kind, "streams": streams, "idle": rng.choice((0, streams // 7)),
                "low": rng.randint(1, high), "high": high, "heads": heads, "group": group,
                "dim": dim, "sums": rng.choice((0, 0, 1))}
    if kind == "prompt":
        streams = _between(rng, 1, 16)
        most = int(math.sqrt(8 * 8187 * 8187 // (streams * heads * group))) // 2
        high = _between(rng, 5, min(4000, most))
        return {"kind": kind, "streams": streams, "low": rng.randint(1, high), "high": high,
                "prefix": rng.choice((0, rng.randint(1, min(700, most)))), "heads": heads,
                "group": group, "dim": dim, "sums": rng.choice((0, 0, 64, high))}
    high = _between(rng, 16, 2048)
    streams = _between(rng, 1, 64 * 2048 // high)
    low = rng.randint(1, high)
    if kind == "store":
        return {"kind": kind, "streams": streams, "low": low, "high": high, "heads": heads,
                "dim": min(dim, 4096 // (8 * heads))}
    high = _between(rng, 64, 8000)
    streams = _between(rng, 1, min(256, 64 * 2048 * 512 // (high * heads * dim)))
    keep = rng.randint(high // 8, high * 3 // 4)
    return {"kind": kind, "streams": streams, "low": rng.randint(high // 4, high), "high": high,
            "keep": keep, "first": min(keep // 4, rng.choice((0, 4, 17))),
            "newest": rng.randint(0, keep // 2), "heads": heads, "dim": dim}


def _plan(case):
    """Per stream: the index of its first row in this call (-1: an empty place of the batch)
    and the number of rows (evict: of positions). The same for every seed."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    s = case["streams"]
    lengths = [rng.randint(case["low"], case["high"]) for _ in range(s)]
    lengths[rng.randrange(s)] = case["high"]
    if case["kind"] == "attend":  # one row a stream, the last of its length
        first = [n - 1 for n in lengths]
        for i in rng.sample(range(s), case["idle"]):
            first[i] = -1
        return first, [1] * s
    if case["kind"] == "prompt":
        return [case["prefix"] if i % 3 != 1 else case["prefix"] // 2 for i in range(s)], lengths
    if case["kind"] == "store":  # after rows that the stream holds already, also inside a block
        return [11 * (i % 3) for i in range(1, s + 1)], lengths
    return [0] * s, lengths


def work(case):
    first, count = _plan(case)
    heads, dim = case["heads"], case["dim"]
    width = heads * dim
    row = heads * (dim + 4 * (dim // SPAN))  # bytes of a position's keys, values and scales
    if case["kind"] == "evict":
        kept = sum(min(n, case["keep"]) for n in count)
        # Sums in, rows, sums and their indexes out; and the rows read back.
        return {"bytes": kept * (3 * row + 2 * width * 4) + heads * (4 * sum(count) + 8 * kept),
                "flops": heads * sum(count)}
    live = [(f, n) for f, n in zip(first, count) if f >= 0]
    rows = sum(n for _, n in live)
    if case["kind"] == "store":  # rows in, the cache out, and back
        return {"bytes": 2 * rows * (2 * width * 4 + row), "flops": 6 * rows * 2 * width}
    held = sum(f + n for f, n in live)
    keys = sum(n * f + n * (n + 1) // 2 for f, n in live)
    return {"bytes": held * row + rows * 2 * width * case["group"] * 4 +
            (8 * heads * held if case["sums"] else 0), "flops": 4 * keys * width * case["group"]}


# ------------------------------------------------------------ the cache's form


def _pack(x):
    """Whole numbers [..., 16 k] -> bytes [..., 8 k]: of 16, number 8 a + b is the low half of
    byte 4 a + b, number 8 a + 4 + b its high half."""
    n = x.to(torch.int32).reshape(*x.shape[:-1], -1, 2, 2, 4)
    n = (n[..., 0, :] & 15) | ((n[..., 1, :] & 15) << 4)
    return n.to(torch.uint8).reshape(*x.shape[:-1], -1)


def _unpack(x):
    """The inverse of _pack, in fp32."""
    n = x.to(torch.int32).reshape(*x.shape[:-1], -1, 2, 1, 4)
    n = torch.cat((n & 15, n >> 4), -2).reshape(*x.shape[:-1], -1)
    return torch.where(n > 7, n - 16, n).float()


def _tiles(q, s):
    """Whole numbers [blocks, heads, 2, 16, dim] and scales [blocks, heads, 2, 16, dim / 64] ->
    the cache's bytes [blocks, heads, 2, dim / 64, 512] and scales [blocks, heads, dim / 64, 16, 2]:
    keys by position, values by dim."""
    b, h, _, _, dim = q.shape
    q = q.reshape(b, h, 2, BLOCK, -1, SPAN).transpose(3, 4)
    k = _pack(q[:, :, 0]).reshape(b, h, -1, 512)
    v = _pack(q[:, :, 1].transpose(-1, -2).contiguous()).reshape(b, h, -1, 512)
    return torch.stack((k, v), 2), s.permute(0, 1, 4, 3, 2).half()


def _rows(values, scales):
    """The inverse of _tiles, multiplied out, in fp32: [..., heads, 2, 16, dim]."""
    lead = values.shape[:-3]
    n = len(lead)
    k = _unpack(values[..., 0, :, :].reshape(*lead, -1, BLOCK, SPAN // 2))
    v = _unpack(values[..., 1, :, :].reshape(*lead, -1, SPAN, BLOCK // 2)).transpose(-1, -2)
    x = torch.stack((k, v), n) * scales.float().permute(*range(n), n + 2, n, n + 1)[..., None]
    return x.transpose(-2, -3).reshape(*lead, 2, BLOCK, -1)


def _quantise(x):
    """fp32 [..., dim] -> whole numbers in [-8, 7] and scales [..., dim / 64]: the larger of
    max / 7 and -min / 8, to 8 significant bits, upwards. In 64 bits: x is next to a border
    here and there."""
    y = x.double().reshape(*x.shape[:-1], -1, SPAN)
    t = torch.maximum((y.amax(-1) / 7).float(), (-y.amin(-1) / 8).float())
    s = ((t.view(torch.int32) + 0xFFFF) & ~0xFFFF).view(torch.float32).clamp_min(LEAST)
    return torch.round(y / s.double()[..., None]).float().reshape(x.shape), s


# ------------------------------------------------------------------- requests


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _int32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    """The cache, its block tables, the rows of the call, room for its results."""
    g = torch.Generator("cuda").manual_seed(seed)
    first, count = _plan(case)
    s, heads, dim, group = case["streams"], case["heads"], case["dim"], case.get("group", 1)
    held = [f + n if f >= 0 else 0 for f, n in zip(first, count)]
    need = [-(-n // BLOCK) for n in held]
    blocks, stride = sum(need) + 3, -(-max(max(held), 1) // BLOCK)
    ids = torch.randperm(blocks, generator=g, device="cuda").int()
    before = _int32(np.concatenate(([0], np.cumsum(need)[:-1])))
    at = torch.arange(stride, device="cuda")
    inside = at[None] < _int32(need)[:, None]
    tables = torch.where(inside, ids[(before[:, None] + at[None]).clamp_max(blocks - 1).long()], 0)
    st = {"case": case, "tables": tables.int().contiguous(), "first": _int32(first),
          "offsets": _int32(np.concatenate(([0], np.cumsum(count)))), "rows": sum(count),
          "max_rows": max(count), "max_positions": max(held), "stride": stride,
          "lengths": _int32(held), "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
    # For each row of the call: its stream and its place in the stream's run.
    st["stream"] = torch.repeat_interleave(torch.arange(s, device="cuda"), _int32(count).long())
    st["place"] = torch.arange(st["rows"], device="cuda") - st["offsets"][:-1].long()[st["stream"]]
    # Dims of a head differ in size, and so do positions.
    gain = torch.exp(0.3 * _normal(g, heads, 2, 1, dim))
    more = blocks if case["kind"] == "evict" else 0  # and as many blocks for what is kept
    st["values"] = torch.empty(1, blocks + more, heads, 2, dim // SPAN, 512, dtype=torch.uint8,
                               device="cuda")
    st["scales"] = torch.empty(1, blocks + more, heads, dim // SPAN, BLOCK, 2, dtype=torch.half,
                               device="cuda")
    for b in range(0, blocks + more, 4096):
        n = min(4096, blocks + more - b)
        x = _normal(g, n, heads, 2, BLOCK, dim) * gain * torch.exp(0.2 * _normal(g, n, heads, 2, BLOCK, 1))
        st["values"][0, b:b + n], st["scales"][0, b:b + n] = _tiles(*_quantise(x))
    if case["kind"] in ("attend", "prompt"):
        st["q"] = _normal(g, st["rows"], heads * group * dim)
        st["out"] = torch.zeros_like(st["q"])
        st["before"] = st["after"] = None
        if case["sums"]:  # what the positions weighed before
            st["before"] = torch.exp(2.0 * _normal(g, s, heads, stride * BLOCK))
            st["after"] = torch.zeros_like(st["before"])
        return st
    if case["kind"] == "store":
        st["k"] = (_normal(g, st["rows"], heads, dim) * gain[:, 0].reshape(1, heads, dim)).reshape(st["rows"], -1)
        st["v"] = (_normal(g, st["rows"], heads, dim) * gain[:, 1].reshape(1, heads, dim)).reshape(st["rows"], -1)
        st["back_k"], st["back_v"] = torch.zeros_like(st["k"]), torch.zeros_like(st["v"])
        return st
    # Sums: a few positions weigh much, many the same little.
    sums = torch.exp(2.0 * _normal(g, s, heads, stride * BLOCK))
    st["sums"] = torch.where(sums < 0.3, torch.round(sums * 16) / 16, sums)
    st["to_sums"] = torch.zeros_like(st["sums"])
    st["to_tables"] = (st["tables"] + blocks).contiguous()
    st["kept"] = torch.zeros(s, heads, case["keep"], dtype=torch.int32, device="cuda")
    # What is read back: all that each stream kept.
    kept = [min(n, case["keep"]) for n in held]
    st["kept_lengths"], st["kept_rows"], st["kept_max"] = _int32(kept), sum(kept), max(kept)
    st["kept_offsets"] = _int32(np.concatenate(([0], np.cumsum(kept))))
    st["kept_stream"] = torch.repeat_interleave(torch.arange(s, device="cuda"), _int32(kept).long())
    st["kept_place"] = (torch.arange(st["kept_rows"], device="cuda") -
                        st["kept_offsets"][:-1].long()[st["kept_stream"]])
    return st


# ---------------------------------------------------------------- plain forms


def _plain_attention(st):
    case = st["case"]
    s, heads, group, dim, r = (case["streams"], case["heads"], case["group"], case["dim"],
                               st["max_rows"])
    ids = st["tables"].long()
    x = _rows(st["values"][0][ids], st["scales"][0][ids])  # [s, blocks, heads, 2, 16, dim]
    k, v = x.permute(3, 0, 2, 1, 4, 5).reshape(2, s, heads, -1, dim)
    key = torch.arange(k.shape[2], device="cuda")
    at = (st["offsets"][:-1].long()[:, None] + torch.arange(r, device="cuda")).clamp_max(
        st["rows"] - 1)
    q = st["q"][at].reshape(s, r, heads, group, dim).permute(0, 2, 3, 1, 4)
    q = q.reshape(s, heads, group * r, dim) * dim ** -0.5
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()).reshape(s, heads, group, r, -1)
    last = st["first"][:, None] + torch.arange(r, device="cuda")
    seen = (key[None, None] <= last[..., None])[:, None, None]
    score = torch.where(seen, score, -torch.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(score - top), 0.0)
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.reshape(s, heads, group * r, -1), v).reshape(s, heads, group, r, dim)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(s, r, -1)
    st["out"].copy_(o[st["stream"], st["place"]])
    if not case["sums"]:
        return st["out"]
    count = (st["offsets"][1:] - st["offsets"][:-1])[:, None]
    row = torch.arange(r, device="cuda")
    counts = (row < count) & (row >= count - case["sums"]) & (st["first"][:, None] >= 0)
    w = torch.where(counts[:, None, None, :, None] & (total > 0), e / total, 0.0).sum((2, 3))
    old = torch.where(key < st["first"][:, None, None], st["before"], 0.0)
    held = key < st["lengths"][:, None, None]
    st["after"].copy_(torch.where(held, old + w, st["after"]))
    return {"out": st["out"], "sums": st["after"]}


def _plain_store(st):
    case = st["case"]
    heads, dim = case["heads"], case["dim"]
    position = st["first"].long()[st["stream"]] + st["place"]
    ids = st["tables"].long()[st["stream"], position // BLOCK]
    q, s = _quantise(torch.stack((st["k"], st["v"]), 1).reshape(-1, 2, heads, dim))
    at = position % BLOCK
    # Keys: a position's 32 bytes of 64 dims; values: its half of every dim's byte.
    n = q.reshape(-1, 2, heads, dim // SPAN, SPAN)
    k = st["values"][0].view(-1, heads, 2, dim // SPAN, BLOCK, SPAN // 2)
    k[ids, :, 0, :, at] = _pack(n[:, 0])
    v = st["values"][0].view(-1, heads, 2, dim // SPAN, SPAN, BLOCK // 2)[:, :, 1]
    full = torch.zeros(v.shape[0], BLOCK, dtype=torch.bool, device="cuda")
    full[ids, at] = True
    rows = torch.zeros(v.shape[0], BLOCK, heads, dim // SPAN, SPAN, device="cuda")
    rows[ids, at] = n[:, 1]
    mine = full[:, None, None, None]
    v.copy_(_pack(torch.where(mine, rows.permute(0, 2, 3, 4, 1), _unpack(v))))
    st["scales"][0][ids, :, :, at] = s.permute(0, 2, 3, 1).half()
    x = _rows(st["values"][0], st["scales"][0])[ids, :, :, at]
    st["back_k"].copy_(x[:, :, 0].reshape(st["rows"], -1))
    st["back_v"].copy_(x[:, :, 1].reshape(st["rows"], -1))
    return {"k": st["back_k"], "v": st["back_v"], "scales": st["scales"]}


def _plain_evict(st):
    case = st["case"]
    s, heads, keep = case["streams"], case["heads"], case["keep"]
    n = st["lengths"].long()[:, None, None]
    key = torch.arange(st["sums"].shape[-1], device="cuda")
    sums = torch.where((key < case["first"]) | (key >= n - case["newest"]), torch.inf, st["sums"])
    sums = torch.where(key < n, sums, -1.0)
    order = torch.sort(sums, dim=-1, descending=True, stable=True).indices[..., :keep]
    place = torch.arange(keep, device="cuda")
    got = torch.where(place < n, order, key.numel()).sort(-1).values  # what is kept, in order
    there = got < key.numel()
    st["kept"].copy_(torch.where(there, got, -1))
    got = got.clamp_max(key.numel() - 1)
    kept = torch.nn.functional.pad(torch.where(there, st["sums"].gather(-1, got), 0.0),
                                   (0, key.numel() - keep))
    st["to_sums"].copy_(torch.where(key < n.clamp_max(keep), kept, st["to_sums"]))
    # The rows as they are: [s, heads, 2, keep, dim] whole numbers, and scales.
    ids = st["tables"].long().gather(1, (got // BLOCK).reshape(s, -1)).reshape(got.shape)
    head = torch.arange(heads, device="cuda")[None, :, None]
    at = got % BLOCK
    v = st["values"][0].view(-1, heads, 2, case["dim"] // SPAN, 512)
    k_rows = v[:, :, 0].reshape(v.shape[0], heads, -1, BLOCK, SPAN // 2)[ids, head, :, at]
    dims = v[:, :, 1].reshape(v.shape[0], heads, -1, SPAN, BLOCK // 2)
    byte = dims[ids, head, :, :, (at // 8 * 4 + at % 4)]
    v_rows = torch.where((at // 4 % 2 == 1)[..., None, None], byte >> 4, byte & 15)
    scales = st["scales"][0][ids, head, :, at]
    # Into the blocks that hold them from now on.
    to, b = st["to_tables"].long(), -(-keep // BLOCK)
    pad = b * BLOCK - keep
    full = torch.nn.functional.pad(there, (0, pad)).reshape(s, heads, b, BLOCK)

    def blocks(x):
        return torch.nn.functional.pad(x, (0, 0) * (x.dim() - 3) + (0, pad)).reshape(
            s, heads, b, BLOCK, *x.shape[3:]).transpose(1, 2)

    mine = full.transpose(1, 2)
    to = to[:, :b]
    old_k = v[:, :, 0].reshape(v.shape[0], heads, -1, BLOCK, SPAN // 2)[to].transpose(3, 4)
    old_v = _unpack(v[:, :, 1].reshape(v.shape[0], heads, -1, SPAN, BLOCK // 2)[to])
    old_v = old_v.permute(0, 1, 2, 5, 3, 4)
    new_k = torch.where(mine[..., None, None], blocks(k_rows), old_k).transpose(3, 4)
    new_v = torch.where(mine[..., None, None], blocks(v_rows).float(), old_v).permute(0, 1, 2, 4, 5, 3)
    old_s = st["scales"][0][to].transpose(3, 4)
    new_s = torch.where(mine[..., None, None], blocks(scales), old_s).transpose(3, 4)
    live = (torch.arange(b, device="cuda") * BLOCK < st["lengths"][:, None]).nonzero(as_tuple=True)
    st["values"][0][to[live], :, 0] = new_k[live].reshape(-1, heads, case["dim"] // SPAN, 512)
    st["values"][0][to[live], :, 1] = _pack(new_v[live].contiguous()).reshape(
        -1, heads, case["dim"] // SPAN, 512)
    st["scales"][0][to[live]] = new_s[live]
    return _kept(st)


def _kept(st):
    """What the streams hold after an eviction, as rows."""
    x = _rows(st["values"][0], st["scales"][0])
    ids = st["to_tables"].long()[st["kept_stream"], st["kept_place"] // BLOCK]
    x = x[ids, :, :, st["kept_place"] % BLOCK].reshape(
        st["kept_rows"], -1, 2, st["case"]["dim"])
    return {"kept": st["kept"], "sums": st["to_sums"], "k": x[:, :, 0], "v": x[:, :, 1]}


# -------------------------------------------------------------- library calls


def _package():
    if "speech_mac_amd" not in sys.modules:
        home = os.path.join(ROOT, "speech-mac_amd")
        spec = importlib.util.spec_from_file_location(
            "speech_mac_amd", os.path.join(home, "__init__.py"), submodule_search_locations=[home])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["speech_mac_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["speech_mac_amd"]


def _check(ok, lib):
    if not ok:
        raise RuntimeError(_package().last_error(lib) or "the call was refused")


def _hold(st):
    """The descriptions of the cache and of the call's rows, and the workspace, which a program
    makes once for its batch."""
    if "held" in st:
        return st["held"]
    pkg, case = _package(), st["case"]
    lib = pkg.load()
    _check(lib.pgpu_device_init(), lib)
    kv = pkg.PgpuKv4(st["values"].data_ptr(), st["scales"].data_ptr(), 1, case["heads"],
                     case["dim"], st["values"].shape[1])

    def rows(tables, first, offsets, count, most):
        return pkg.PgpuKv4Rows(tables.data_ptr(), st["stride"], first.data_ptr(),
                               None if offsets is None else offsets.data_ptr(), case["streams"],
                               count, most)

    held = {"lib": lib, "kv": ctypes.byref(kv), "keep": [kv]}
    if case["kind"] == "evict":
        held["zero"] = torch.zeros_like(st["first"])
        held["rows"] = rows(st["to_tables"], held["zero"], st["kept_offsets"], st["kept_rows"],
                            st["kept_max"])
        held["k"] = torch.empty(st["kept_rows"], case["heads"], case["dim"], device="cuda")
        held["v"] = torch.empty_like(held["k"])
    else:
        held["rows"] = rows(st["tables"], st["first"],
                            None if case["kind"] == "attend" else st["offsets"], st["rows"],
                            st["max_rows"])
    if "out" in st:
        held["sums"] = None
        if case["sums"]:
            sums = pkg.PgpuKv4Sums(st["before"].data_ptr(), st["after"].data_ptr(),
                                   st["after"].shape[-1], case["sums"])
            held["sums"] = ctypes.byref(sums)
            held["keep"].append(sums)
        held["bytes"] = lib.pgpu_kv4_attention_bytes(held["kv"], ctypes.byref(held["rows"]),
                                                     case["group"], st["max_positions"],
                                                     1 if case["sums"] else 0)
        held["work"] = torch.empty(max(held["bytes"], 16), dtype=torch.uint8, device="cuda")
    st["held"] = held
    return held


def _own(st):
    h, case = _hold(st), st["case"]
    lib, width = h["lib"], case["heads"] * case["dim"]
    stream = torch.cuda.current_stream().cuda_stream
    rows, status = ctypes.byref(h["rows"]), st["status"].data_ptr()
    if case["kind"] in ("attend", "prompt"):
        wide = width * case["group"]
        _check(lib.pgpu_kv4_attention(
            stream, h["kv"], 0, rows, st["q"].data_ptr(), wide, case["group"],
            case["dim"] ** -0.5, st["max_positions"], st["out"].data_ptr(), wide, h["sums"],
            h["work"].data_ptr(), h["bytes"], status), lib)
        return {"out": st["out"], "sums": st["after"]} if case["sums"] else st["out"]
    if case["kind"] == "store":
        _check(lib.pgpu_kv4_write(stream, h["kv"], 0, rows, st["k"].data_ptr(),
                                  st["v"].data_ptr(), width, status), lib)
        _check(lib.pgpu_kv4_read(stream, h["kv"], 0, rows, st["lengths"].data_ptr(),
                                 st["back_k"].data_ptr(), st["back_v"].data_ptr(), width, status),
               lib)
        return {"k": st["back_k"], "v": st["back_v"], "scales": st["scales"]}
    _check(lib.pgpu_kv4_evict(
        stream, h["kv"], 0, 1, st["tables"].data_ptr(), st["to_tables"].data_ptr(), st["stride"],
        st["lengths"].data_ptr(), case["streams"], case["keep"], case["first"], case["newest"],
        st["sums"].data_ptr(), st["to_sums"].data_ptr(), st["sums"].shape[-1],
        st["kept"].data_ptr(), status), lib)
    _check(lib.pgpu_kv4_read(stream, h["kv"], 0, rows, st["kept_lengths"].data_ptr(),
                             h["k"].data_ptr(), h["v"].data_ptr(), width, status), lib)
    return {"kept": st["kept"], "sums": st["to_sums"], "k": h["k"], "v": h["v"]}


def run(st):
    """One pass: attention rows, and the positions' sums where they are kept; rows written and
    read back, with the scales; or an eviction, and what is held after it read back."""
    if own:
        return _own(st)
    kind = st["case"]["kind"]
    if kind == "store":
        return _plain_store(st)
    return _plain_evict(st) if kind == "evict" else _plain_attention(st)


# ------------------------------------------------------------------ in 64 bits


def _nibbles(x):
    """Bytes [..., 8 k] -> signed numbers [..., 16 k], in 64 bits, by each number's place."""
    n = np.arange(16)
    byte, high = n // 8 * 4 + n % 4, n // 4 % 2
    x = x.reshape(*x.shape[:-1], -1, 8)[..., byte].astype(np.int64) >> (4 * high) & 15
    return np.where(x > 7, x - 16, x).reshape(*x.shape[:-2], -1).astype(np.float64)


def _exact_rows(values, scales):
    """Bytes and scales of one head's blocks, on the host -> keys, values [positions][dim]."""
    blocks = values.shape[0]
    k = _nibbles(values[:, 0].reshape(blocks, -1, BLOCK, 32)).transpose(0, 2, 1, 3)
    v = _nibbles(values[:, 1].reshape(blocks, -1, SPAN, 8)).transpose(0, 3, 1, 2)
    scale = scales.astype(np.float64).transpose(3, 0, 2, 1)[..., None]
    return [(x * f).reshape(blocks * BLOCK, -1) for x, f in zip((k, v), scale)]


def _exact_attention(st, case):
    heads, group, dim = case["heads"], case["group"], case["dim"]
    first, count = _plan(case)
    order = torch.tensor(np.stack((np.arange(16) // 8 * 4 + np.arange(16) % 4,
                                   np.arange(16) // 4 % 2 * 4)), device="cuda")

    def numbers(x):  # [..., 8 k] -> [..., 16 k]
        n = x.reshape(*x.shape[:-1], -1, 8).long()[..., order[0]] >> order[1] & 15
        return (n - (n > 7) * 16).reshape(*x.shape[:-1], -1).double()

    out = torch.zeros(st["rows"], heads, group, dim, dtype=torch.float64, device="cuda")
    sums = st["after"].double() if case["sums"] else None
    at = 0
    for s, (f, n) in enumerate(zip(first, count)):
        if f >= 0:
            length = f + n
            ids = st["tables"][s, :-(-length // BLOCK)].long()
            k, v = st["values"][0, ids].unbind(2)  # [blocks, heads, dim / 64, 512]
            scale = st["scales"][0, ids].double()
            k = numbers(k.reshape(*k.shape[:3], BLOCK, 32)) * scale[..., 0, None]
            v = numbers(v.reshape(*v.shape[:3], SPAN, 8)).transpose(-1, -2) * scale[..., 1, None]
            k, v = (x.permute(1, 0, 3, 2, 4).reshape(heads, -1, dim)[:, :length] for x in (k, v))
            key = torch.arange(length, device="cuda")
            if sums is not None:
                sums[s, :, :length] = torch.where(key < f, st["before"][s, :, :length].double(), 0.0)
            for r in range(0, n, 512):
                m = min(512, n - r)
                q = st["q"][at + r:at + r + m].double().reshape(m, heads, group, dim)
                w = torch.einsum("mhgd,hkd->mhgk", q, k) / math.sqrt(dim)
                hide = key[None] > f + r + torch.arange(m, device="cuda")[:, None]
                w = torch.softmax(w.masked_fill(hide[:, None, None], -math.inf), -1)
                out[at + r:at + r + m] = torch.einsum("mhgk,hkd->mhgd", w, v)
                if sums is not None:
                    late = max(0, min(m, n - case["sums"] - r))  # rows before these do not count
                    sums[s, :, :length] += w[late:].sum((0, 2))
        at += n
    out = out.reshape(st["rows"], -1)
    return out if sums is None else {"out": out, "sums": sums}


def exact(case, seed):
    """run()'s outputs from the definition, in 64 bits."""
    st = prepare(case, seed)
    heads, dim = case["heads"], case["dim"]
    if case["kind"] in ("attend", "prompt"):
        return _exact_attention(st, case)
    first, count = _plan(case)
    if sum(count) * heads * dim > 50_000_000:
        return None  # taken on the host
    host = {k: v.cpu().numpy() for k, v in st.items() if isinstance(v, torch.Tensor)}
    if case["kind"] == "store":
        scales = host["scales"][0].astype(np.float64)
        back, at = [[], []], 0
        for s, (f, n) in enumerate(zip(first, count)):
            p = np.arange(f, f + n)
            for i, name in enumerate("kv"):
                x = host[name][at:at + n].astype(np.float64).reshape(n, heads, -1, SPAN)
                t = np.maximum((x.max(-1) / 7).astype(np.float32), (-x.min(-1) / 8).astype(np.float32))
                e = np.floor(np.log2(np.maximum(t, 1e-30).astype(np.float64))) - 7
                scale = np.maximum(np.ceil(t / 2.0 ** e) * 2.0 ** e, LEAST)
                back[i].append((np.rint(x / scale[..., None]) * scale[..., None]).reshape(n, -1))
                scales[host["tables"][s, p // BLOCK], :, :, p % BLOCK, i] = scale
            at += n
        return {"k": np.concatenate(back[0]), "v": np.concatenate(back[1]), "scales": scales[None]}
    keep, newest = case["keep"], case["newest"]
    kept = np.full((len(count), heads, keep), -1, np.int32)
    sums = host["to_sums"].astype(np.float64)
    k = np.zeros((st["kept_rows"], heads, dim))
    v = np.zeros_like(k)
    at = 0
    for s, n in enumerate(count):
        m = min(n, keep)
        ids = host["tables"][s, :-(-n // BLOCK)]
        for h in range(heads):
            w = host["sums"][s, h, :n].astype(np.float64)
            got = np.arange(n)
            if n > keep:
                middle = got[case["first"]:n - newest]
                best = middle[np.lexsort((middle, -w[middle]))][:keep - case["first"] - newest]
                got = np.sort(np.concatenate((got[:case["first"]], best, got[n - newest:])))
            kept[s, h, :m] = got
            sums[s, h, :m] = w[got]
            rows = _exact_rows(host["values"][0][ids, h], host["scales"][0][ids, h])
            k[at:at + m, h], v[at:at + m, h] = rows[0][got], rows[1][got]
        at += m
    return {"kept": kept, "sums": sums, "k": k, "v": v}
