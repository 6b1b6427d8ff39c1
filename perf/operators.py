"""Operators of the 8-bit paged KV cache: its plain forms, and the library's calls.

A server that holds its requests' keys and values in 8 bits quantises them as they are
written (prompts in runs of rows, frames one row a stream), hands blocks on to another
process by reading them back, and attends to the cache: one query a stream for a frame, runs
of rows for a prompt. One scale goes to the 16 positions of a block, for each head and for
keys and values apart; the block that a stream is still writing stays in fp32 in the stream's
open slot.

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
MAX_POSITIONS = 8192
THETA, EPSILON = 10000.0, 1e-5


# ------------------------------------------------------------------ the cases


def listed():
    return [
        # The first frame of a lone request: one key. The smallest call.
        {"name": "attend_1_first", "kind": "attend", "streams": 1, "idle": 0, "low": 1, "high": 1,
         "heads": 8, "group": 1, "dim": 64},
        # A lone request late in its life.
        {"name": "attend_1_late", "kind": "attend", "streams": 1, "idle": 0, "low": 2011,
         "high": 2011, "heads": 8, "group": 1, "dim": 64},
        # 64 requests somewhere in their lives; three slots of the batch are empty.
        {"name": "attend_64", "kind": "attend", "streams": 64, "idle": 3, "low": 1, "high": 2048,
         "heads": 8, "group": 1, "dim": 64},
        # A full server with long contexts.
        {"name": "attend_256_long", "kind": "attend", "streams": 256, "idle": 0, "low": 256,
         "high": 8187, "heads": 8, "group": 1, "dim": 64},
        # Four query heads to a key head, wider heads.
        {"name": "attend_48_grouped", "kind": "attend", "streams": 48, "idle": 0, "low": 1,
         "high": 4096, "heads": 8, "group": 4, "dim": 128},
        # Prompts of newly admitted requests that continue a prefix already held, ragged.
        {"name": "prompt_3_ragged", "kind": "prompt", "streams": 3, "low": 37, "high": 300,
         "prefix": 200, "heads": 8, "group": 1, "dim": 64},
        # A full admission round.
        {"name": "prompt_16x256", "kind": "prompt", "streams": 16, "low": 256, "high": 256,
         "prefix": 0, "heads": 8, "group": 1, "dim": 64},
        # One prompt as long as a stream may be: the largest call.
        {"name": "prompt_1_long", "kind": "prompt", "streams": 1, "low": 8187, "high": 8187,
         "prefix": 0, "heads": 8, "group": 1, "dim": 64},
        # A request's rows into the cache and out again, of an odd length; and a whole server's,
        # handed over to another process.
        {"name": "store_1x211", "kind": "store", "streams": 1, "low": 211, "high": 211,
         "heads": 8, "dim": 64},
        {"name": "store_64", "kind": "store", "streams": 64, "low": 1, "high": 2048, "heads": 8,
         "dim": 64},
        # One frame of 64 requests: rotated and appended, the newest block read back.
        {"name": "rotate_64", "kind": "rotate", "streams": 64, "low": 1, "high": 2048, "rows": 1,
         "heads": 8, "group": 1, "dim": 64, "norm": False},
        # Prompts with normalised queries and keys, two query heads to a key head.
        {"name": "rotate_16_norm", "kind": "rotate", "streams": 16, "low": 31, "high": 501,
         "rows": 0, "heads": 8, "group": 2, "dim": 128, "norm": True},
    ]


def _between(rng, low, high):
    """A whole number in [low, high], even over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "prompt", "prompt", "store", "rotate"))
    heads, dim = rng.choice(((8, 64), (8, 64), (4, 128), (8, 128), (6, 64)))
    group = rng.choice((1, 1, 2, 3, 4, 8))
    if kind == "attend":
        high = _between(rng, 1, 8187)
        most = 256 * 4200 * 512 // (high * heads * dim)
        streams = _between(rng, 1, min(256, most))
        return {"kind": kind, "streams": streams, "idle": rng.choice((0, streams // 7)),
                "low": rng.randint(1, high), "high": high, "heads": heads, "group": group,
                "dim": dim}
    if kind == "prompt":
        streams = _between(rng, 1, 16)
        most = int(math.sqrt(8 * 8187 * 8187 // (streams * heads * group))) // 2
        high = _between(rng, 5, min(4000, most))
        return {"kind": kind, "streams": streams, "low": rng.randint(1, high), "high": high,
                "prefix": rng.choice((0, rng.randint(1, min(700, most)))), "heads": heads,
                "group": group, "dim": dim}
    high = _between(rng, 16, 2048)
    streams = _between(rng, 1, 64 * 2048 // high)
    if kind == "store":
        return {"kind": kind, "streams": streams, "low": rng.randint(1, high), "high": high,
                "heads": heads, "dim": min(dim, 4096 // (8 * heads))}
    if rng.random() < 0.5:
        return {"kind": kind, "streams": _between(rng, 1, 256), "low": 1,
                "high": _between(rng, 16, 8000), "rows": 1, "heads": heads, "group": group,
                "dim": dim, "norm": rng.random() < 0.5}
    high = _between(rng, 16, 600)
    return {"kind": kind, "streams": _between(rng, 1, 16), "low": rng.randint(1, high),
            "high": high, "rows": 0, "heads": heads, "group": min(group, 4), "dim": dim,
            "norm": rng.random() < 0.5}


def _plan(case):
    """Per stream: the position of its first row in this call (-1: an empty slot of the batch)
    and the number of rows. The same for every seed."""
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
    if case["kind"] == "rotate" and case["rows"]:
        return [n - 1 for n in lengths], [1] * s
    # New rows after none, or after a prefix of whole blocks that other requests hold too.
    return [BLOCK * (i % 3) for i in range(s)], lengths


def work(case):
    first, count = _plan(case)
    heads, dim = case["heads"], case["dim"]
    width = heads * dim
    live = [(f, n) for f, n in zip(first, count) if f >= 0]
    tile = heads * (2 * BLOCK * dim + 8)
    rows = sum(n for _, n in live)
    if case["kind"] in ("attend", "prompt"):
        held = [f + n for f, n in live]
        cache = sum((n - 1) // BLOCK * tile + ((n - 1) % BLOCK + 1) * 2 * width * 4 for n in held)
        keys = sum(n * f + n * (n + 1) // 2 for f, n in live)
        return {"bytes": cache + rows * 2 * width * case["group"] * 4,
                "flops": 4 * keys * width * case["group"]}
    full = sum((f + n) // BLOCK - f // BLOCK for f, n in live)
    tails = sum((f + n - 1) % BLOCK + 1 for f, n in live)
    read = rows * 2 * width * 4
    if case["kind"] == "store":  # rows in, blocks and open rows out, and back
        return {"bytes": 2 * read + full * tile + tails * 2 * width * 4, "flops": 6 * rows * 2 * width}
    q = rows * width * case["group"] * 4
    back = sum((f + n - 1) % BLOCK + 1 if case["rows"] else n for f, n in live) * 2 * width * 4
    return {"bytes": read + 2 * q + full * tile + tails * 2 * width * 4 + back,
            "flops": 10 * rows * width * (2 + case["group"])}


# ------------------------------------------------------------ the cache's form


def _pack(x):
    """Whole numbers [..., 2, 16, dim] (keys, values) -> the bytes of a block's head: keys in
    rows of positions; values [position / 4][dim % 16][dim / 16][position % 4]."""
    *lead, _, _, dim = x.shape
    k = x[..., 0, :, :].reshape(*lead, BLOCK * dim)
    v = x[..., 1, :, :].reshape(*lead, 4, 4, dim // 16, 16)
    n = len(lead)
    v = v.permute(*range(n), n, n + 3, n + 2, n + 1).reshape(*lead, BLOCK * dim)
    return torch.stack((k, v), -2).to(torch.int8)


def _unpack(x, dim):
    """The inverse of _pack, in fp32."""
    *lead, _, _ = x.shape
    n = len(lead)
    k = x[..., 0, :].reshape(*lead, BLOCK, dim)
    v = x[..., 1, :].reshape(*lead, 4, 16, dim // 16, 4)
    v = v.permute(*range(n), n, n + 3, n + 2, n + 1).reshape(*lead, BLOCK, dim)
    return torch.stack((k, v), -3).float()


def _quantise(x):
    """fp32 [..., 16, dim] -> whole numbers and scales: max/127 to 12 significant bits, upwards."""
    t = x.abs().amax((-2, -1)) / 127
    s = ((t.view(torch.int32) + 0xFFF) & ~0xFFF).view(torch.float32).clamp_min(2.0 ** -126)
    return torch.round(x / s[..., None, None]), s


# ------------------------------------------------------------------- requests


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _int32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    """The cache, its block tables and slots, the rows of the call, room for its results."""
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
          "slots": torch.randperm(s, generator=g, device="cuda").int(),
          "offsets": _int32(np.concatenate(([0], np.cumsum(count)))), "rows": sum(count),
          "max_rows": max(count), "max_positions": max(held), "stride": stride,
          "lengths": _int32(held), "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
    # For each row of the call: its stream and its place in the stream's run.
    st["stream"] = torch.repeat_interleave(torch.arange(s, device="cuda"), _int32(count).long())
    st["place"] = torch.arange(st["rows"], device="cuda") - st["offsets"][:-1].long()[st["stream"]]
    gain = torch.exp(0.3 * _normal(g, heads, 2, 1, dim))
    st["open"] = _normal(g, 1, s, heads, 2, BLOCK, dim) * gain
    if case["kind"] in ("attend", "prompt"):
        q, scales = _quantise(_normal(g, 1, blocks, heads, 2, BLOCK, dim) * gain)
        st["values"], st["scales"] = _pack(q), scales
        st["q"] = _normal(g, st["rows"], heads * group * dim)
        st["out"] = torch.zeros_like(st["q"])
        return st
    st["values"] = torch.zeros(1, blocks, heads, 2, BLOCK * dim, dtype=torch.int8, device="cuda")
    st["scales"] = torch.zeros(1, blocks, heads, 2, device="cuda")
    # What is read back: the rows of the call, or the newest block of each stream.
    newest = case["kind"] == "rotate" and case["rows"]
    back = [(n - 1) // BLOCK * BLOCK for n in held] if newest else first
    many = [n - b for n, b in zip(held, back)]
    st["back_first"], st["back_rows"], st["back_max"] = _int32(back), sum(many), max(many)
    st["back_offsets"] = _int32(np.concatenate(([0], np.cumsum(many))))
    st["back_stream"] = torch.repeat_interleave(torch.arange(s, device="cuda"), _int32(many).long())
    st["back_place"] = (torch.arange(st["back_rows"], device="cuda") -
                        st["back_offsets"][:-1].long()[st["back_stream"]])
    st["back_k"] = torch.zeros(st["back_rows"], heads * dim, device="cuda")
    st["back_v"] = torch.zeros_like(st["back_k"])
    width = (heads * dim) * (2 + group)
    if case["kind"] == "store":
        st["k"] = _normal(g, st["rows"], heads * dim) * gain[:, 0].reshape(1, -1)
        st["v"] = _normal(g, st["rows"], heads * dim) * gain[:, 1].reshape(1, -1)
        return st
    st["qkv"] = _normal(g, st["rows"], width)
    st["q_weight"] = 1 + 0.1 * _normal(g, dim) if case["norm"] else None
    st["k_weight"] = 1 + 0.1 * _normal(g, dim) if case["norm"] else None
    inverse = THETA ** (-2.0 * torch.arange(dim // 2, dtype=torch.float64, device="cuda") / dim)
    angle = torch.arange(MAX_POSITIONS, dtype=torch.float64, device="cuda")[:, None] * inverse
    st["rope"] = torch.stack((angle.cos(), angle.sin()), -1).float().contiguous()
    st["q_out"] = torch.zeros(st["rows"], heads * group * dim, device="cuda")
    return st


# ---------------------------------------------------------------- plain forms


def _context(st):
    """Keys and values [stream, head, position, dim] of every stream, from the blocks and the
    open slots, zero past a stream's length."""
    case = st["case"]
    dim, s = case["dim"], case["streams"]
    ids = st["tables"].long()
    x = _unpack(st["values"][0][ids], dim) * st["scales"][0][ids][..., None, None]
    newest = ((st["lengths"].long() - 1).clamp_min(0)) // BLOCK
    x[torch.arange(s, device="cuda"), newest] = st["open"][0][st["slots"].long()]
    x = x.permute(3, 0, 2, 1, 4, 5).reshape(2, s, case["heads"], -1, dim)
    at = torch.arange(x.shape[3], device="cuda")
    live = at[None] < st["lengths"][:, None]
    return torch.where(live[None, :, None, :, None], x, torch.zeros((), device="cuda"))


def _plain_attention(st):
    case = st["case"]
    s, heads, group, dim, r = (case["streams"], case["heads"], case["group"], case["dim"],
                               st["max_rows"])
    k, v = _context(st)
    at = (st["offsets"][:-1].long()[:, None] + torch.arange(r, device="cuda")).clamp_max(
        st["rows"] - 1)
    q = st["q"][at].reshape(s, r, heads, group, dim).permute(0, 2, 3, 1, 4)
    q = q.reshape(s, heads, group * r, dim) * dim ** -0.5
    score = torch.matmul(q, k.transpose(-1, -2)).reshape(s, heads, group, r, -1)
    last = st["first"][:, None] + torch.arange(r, device="cuda")
    key = torch.arange(k.shape[2], device="cuda")
    seen = (key[None, None] <= last[..., None])[:, None, None]
    score = torch.where(seen, score, -torch.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(score - top), 0.0)
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.reshape(s, heads, group * r, -1), v).reshape(s, heads, group, r, dim)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(s, r, -1)
    st["out"].copy_(o[st["stream"], st["place"]])
    return st["out"]


def _plain_write(st, k, v):
    """Rows [rows, heads * dim] into the blocks and the open slots."""
    case = st["case"]
    s, heads, dim = case["streams"], case["heads"], case["dim"]
    first, lengths = st["first"].long(), st["lengths"].long()
    position = first[st["stream"]] + st["place"]
    block0 = first // BLOCK
    tiles = (st["max_rows"] + 2 * BLOCK - 2) // BLOCK
    x = torch.zeros(s, tiles, heads, 2, BLOCK, dim, device="cuda")
    slots = st["slots"].long()
    x[:, 0] = st["open"][0][slots]  # the rows that the first block had before
    rows = torch.stack((k, v), 1).reshape(-1, 2, heads, dim).transpose(1, 2)
    x[st["stream"], position // BLOCK - block0[st["stream"]], :, :, position % BLOCK] = rows
    # Full blocks into the cache.
    tile = block0[:, None] + torch.arange(tiles, device="cuda")
    full = ((tile + 1) * BLOCK <= lengths[:, None]).reshape(-1).nonzero()[:, 0]
    q, scales = _quantise(x.reshape(-1, heads, 2, BLOCK, dim)[full])
    ids = st["tables"].long().gather(1, tile.clamp_max(st["stride"] - 1)).reshape(-1)[full]
    st["values"][0][ids] = _pack(q)
    st["scales"][0][ids] = scales
    # The newest block's new rows into the open slot.
    newest = (lengths - 1) // BLOCK
    mine = position // BLOCK == newest[st["stream"]]
    at, place = slots[st["stream"]][mine], (position % BLOCK)[mine]
    st["open"][0][at, :, :, place] = rows[mine]


def _plain_read(st):
    case = st["case"]
    position = st["back_first"].long()[st["back_stream"]] + st["back_place"]
    block, newest = position // BLOCK, (st["lengths"].long() - 1) // BLOCK
    ids = st["tables"].long()[st["back_stream"], block]
    x = _unpack(st["values"][0], case["dim"]) * st["scales"][0][..., None, None]
    x = x[ids, :, :, position % BLOCK]
    fresh = st["open"][0][st["slots"].long()[st["back_stream"]], :, :, position % BLOCK]
    x = torch.where((block == newest[st["back_stream"]])[:, None, None, None], fresh, x)
    st["back_k"].copy_(x[:, :, 0].reshape(st["back_rows"], -1))
    st["back_v"].copy_(x[:, :, 1].reshape(st["back_rows"], -1))


def _plain_rotate(st):
    """q for the attention, k, v: each head normalised where there are weights, its pairs turned
    by their position's angle. In 64 bits: k is next to a border of 8 bits here and there."""
    case = st["case"]
    heads, group, dim = case["heads"], case["group"], case["dim"]
    n = st["rows"]
    x = st["qkv"].double()
    turn = st["rope"][st["first"].long()[st["stream"]] + st["place"]].double()[:, None]

    def one(y, weight):
        y = y.reshape(n, -1, dim)
        if weight is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPSILON) * weight.double()
        a, b = y[..., 0::2], y[..., 1::2]
        c, d = turn[..., 0], turn[..., 1]
        return torch.stack((a * c - b * d, a * d + b * c), -1).reshape(n, -1)

    split = heads * group * dim
    st["q_out"].copy_((one(x[:, :split], st["q_weight"]) * dim ** -0.5).float())
    k = one(x[:, split:split + heads * dim], st["k_weight"]).float()
    return k, st["qkv"][:, split + heads * dim:]


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
    """The descriptions of the cache and of the call's rows, and the attention's workspace,
    which a program makes once for its batch."""
    if "held" in st:
        return st["held"]
    pkg, case = _package(), st["case"]
    lib = pkg.load()
    _check(lib.pgpu_device_init(), lib)
    one_row = case["kind"] == "attend" or (case["kind"] == "rotate" and case["rows"])
    kv = pkg.PgpuKv8(st["values"].data_ptr(), st["scales"].data_ptr(), st["open"].data_ptr(), 1,
                     case["heads"], case["dim"], st["values"].shape[1], case["streams"])

    def rows(first, offsets, count, most):
        return pkg.PgpuKv8Rows(st["tables"].data_ptr(), st["stride"], st["slots"].data_ptr(),
                               first.data_ptr(), offsets, case["streams"], count, most)

    held = {"lib": lib, "kv": ctypes.byref(kv), "keep": [kv], "rows": rows(
        st["first"], None if one_row else st["offsets"].data_ptr(), st["rows"], st["max_rows"])}
    if "back_first" in st:
        held["back"] = rows(st["back_first"], st["back_offsets"].data_ptr(), st["back_rows"],
                            st["back_max"])
    if "out" in st:
        held["bytes"] = lib.pgpu_kv8_attention_bytes(held["kv"], ctypes.byref(held["rows"]),
                                                     case["group"], st["max_positions"])
        held["work"] = torch.empty(max(held["bytes"], 16), dtype=torch.uint8, device="cuda")
    st["held"] = held
    return held


def _own(st):
    h, case = _hold(st), st["case"]
    lib, width = h["lib"], case["heads"] * case["dim"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["kind"] in ("attend", "prompt"):
        wide = width * case["group"]
        _check(lib.pgpu_kv8_attention(
            stream, h["kv"], 0, ctypes.byref(h["rows"]), st["q"].data_ptr(), wide, case["group"],
            case["dim"] ** -0.5, st["max_positions"], st["out"].data_ptr(), wide,
            h["work"].data_ptr(), h["bytes"], st["status"].data_ptr()), lib)
        return st["out"]
    if case["kind"] == "store":
        _check(lib.pgpu_kv8_write(stream, h["kv"], 0, ctypes.byref(h["rows"]), st["k"].data_ptr(),
                                  st["v"].data_ptr(), width, st["status"].data_ptr()), lib)
    else:
        _check(lib.pgpu_kv8_rotate_write(
            stream, h["kv"], 0, ctypes.byref(h["rows"]), st["qkv"].data_ptr(),
            width * (2 + case["group"]), case["group"],
            st["q_weight"].data_ptr() if case["norm"] else None,
            st["k_weight"].data_ptr() if case["norm"] else None, EPSILON, st["rope"].data_ptr(),
            MAX_POSITIONS, case["dim"] ** -0.5, st["q_out"].data_ptr(), st["status"].data_ptr()),
            lib)
    _check(lib.pgpu_kv8_read(stream, h["kv"], 0, ctypes.byref(h["back"]),
                             st["lengths"].data_ptr(), st["back_k"].data_ptr(),
                             st["back_v"].data_ptr(), width, st["status"].data_ptr()), lib)
    return None


def run(st):
    """One pass: attention rows; or rows written and read back, with the cache's scales and open
    rows (the 8-bit values are returned as what they stand for, by reading them back)."""
    case = st["case"]
    if own:
        out = _own(st)
        if out is not None:
            return out
    elif case["kind"] in ("attend", "prompt"):
        return _plain_attention(st)
    else:
        k, v = (st["k"], st["v"]) if case["kind"] == "store" else _plain_rotate(st)
        _plain_write(st, k, v)
        _plain_read(st)
    out = {"k": st["back_k"], "v": st["back_v"], "scales": st["scales"], "open": st["open"]}
    if case["kind"] == "rotate":
        out["q"] = st["q_out"]
    return out


# ------------------------------------------------------------------ in 64 bits


def _exact_blocks(x):
    """64-bit rows [..., 16, dim] of blocks -> what is stored for them, and their scales."""
    t = (np.abs(x).max((-2, -1)) / 127.0).astype(np.float32)
    bits = (t.view(np.uint32).astype(np.uint64) + 0xFFF) // 0x1000 * 0x1000
    s = np.maximum(bits.astype(np.uint32).view(np.float32).astype(np.float64), 2.0 ** -126)
    return np.rint(x / s[..., None, None]) * s[..., None, None], s


def _exact_attention(st, case):
    heads, group, dim = case["heads"], case["group"], case["dim"]
    first, count = _plan(case)
    values = st["values"][0].reshape(-1, heads, 2, BLOCK * dim)
    # Where value (position, dim) of a block lies among its bytes.
    p, d = np.arange(BLOCK)[:, None], np.arange(dim)[None]
    where = torch.tensor((((p // 4) * 16 + d % 16) * (dim // 16) + d // 16) * 4 + p % 4,
                         device="cuda")
    out = torch.zeros(st["rows"], heads, group, dim, dtype=torch.float64, device="cuda")
    at = 0
    for s, (f, n) in enumerate(zip(first, count)):
        if f >= 0:
            length = f + n
            closed = (length - 1) // BLOCK
            ids = st["tables"][s, :closed].long()
            scale = st["scales"][0, ids].double()
            k = values[ids, :, 0].double().reshape(closed, heads, BLOCK, dim)
            v = values[ids, :, 1].double()[:, :, where.reshape(-1)].reshape(closed, heads, BLOCK, dim)
            k, v = k * scale[:, :, 0, None, None], v * scale[:, :, 1, None, None]
            slot = st["open"][0, int(st["slots"][s])].double()
            k = torch.cat((k.transpose(0, 1).reshape(heads, -1, dim), slot[:, 0]), 1)[:, :length]
            v = torch.cat((v.transpose(0, 1).reshape(heads, -1, dim), slot[:, 1]), 1)[:, :length]
            key = torch.arange(length, device="cuda")
            for r in range(0, n, 1024):
                m = min(1024, n - r)
                q = st["q"][at + r:at + r + m].double().reshape(m, heads, group, dim)
                w = torch.einsum("mhgd,hkd->mhgk", q, k) / math.sqrt(dim)
                hide = key[None] > f + r + torch.arange(m, device="cuda")[:, None]
                w = torch.softmax(w.masked_fill(hide[:, None, None], -math.inf), -1)
                out[at + r:at + r + m] = torch.einsum("mhgk,hkd->mhgd", w, v)
        at += n
    return out.reshape(st["rows"], -1)


def exact(case, seed):
    """run()'s outputs from the definition, in 64 bits."""
    st = prepare(case, seed)
    heads, dim = case["heads"], case["dim"]
    if case["kind"] in ("attend", "prompt"):
        return _exact_attention(st, case)
    first, count = _plan(case)
    if sum(count) > 150000:
        return None  # taken on the host
    host = {k: v.cpu().numpy() for k, v in st.items() if isinstance(v, torch.Tensor)}
    group = case.get("group", 1)
    if case["kind"] == "store":
        k, v, q = host["k"].astype(np.float64), host["v"].astype(np.float64), None
    else:
        x = host["qkv"].astype(np.float64).reshape(-1, heads * (group + 2), dim)
        position = np.concatenate([np.arange(f, f + n) for f, n in zip(first, count)])
        turn = host["rope"].astype(np.float64)[position]
        turn = (turn[..., 0] + 1j * turn[..., 1])[:, None]

        def one(y, weight):
            if case["norm"]:
                y = y / np.sqrt((y * y).mean(-1, keepdims=True) + EPSILON) * host[weight]
            z = (y[..., 0::2] + 1j * y[..., 1::2]) * turn
            return np.stack((z.real, z.imag), -1).reshape(y.shape)

        q = one(x[:, :heads * group], "q_weight").reshape(len(x), -1) / math.sqrt(dim)
        # A key is held as fp32 before it is quantised.
        k = one(x[:, heads * group:heads * (group + 1)], "k_weight")
        k = k.reshape(len(x), -1).astype(np.float32).astype(np.float64)
        v = x[:, heads * (group + 1):].reshape(len(x), -1)
    scales, opened = host["scales"].astype(np.float64), host["open"].astype(np.float64)
    back_k, back_v = [], []
    at = 0
    for s, (f, n) in enumerate(zip(first, count)):
        slot, length = host["slots"][s], f + n
        lo = f // BLOCK * BLOCK
        rows = np.zeros((2, heads, -(-length // BLOCK) * BLOCK - lo, dim))
        rows[:, :, :BLOCK] = opened[0, slot].transpose(1, 0, 2, 3)
        rows[0, :, f - lo:f - lo + n] = k[at:at + n].reshape(n, heads, dim).transpose(1, 0, 2)
        rows[1, :, f - lo:f - lo + n] = v[at:at + n].reshape(n, heads, dim).transpose(1, 0, 2)
        last = (length - 1) // BLOCK * BLOCK
        fresh = max(f, last)
        opened[0, slot][:, :, fresh - last:length - last] = (
            rows[:, :, fresh - lo:length - lo].transpose(1, 0, 2, 3))
        full = length // BLOCK - lo // BLOCK
        x, scale = _exact_blocks(rows[:, :, :full * BLOCK].reshape(2, heads, full, BLOCK, dim))
        ids = host["tables"][s, lo // BLOCK:lo // BLOCK + full]
        scales[0, ids] = scale.transpose(2, 1, 0)
        rows[:, :, :last - lo] = x.reshape(2, heads, -1, dim)[:, :, :last - lo]
        start = int(host["back_first"][s])
        back_k.append(rows[0, :, start - lo:length - lo].transpose(1, 0, 2).reshape(length - start, -1))
        back_v.append(rows[1, :, start - lo:length - lo].transpose(1, 0, 2).reshape(length - start, -1))
        at += n
    out = {"k": np.concatenate(back_k), "v": np.concatenate(back_v), "scales": scales,
           "open": opened}
    if q is not None:
        out["q"] = q
    return out
