"""Workloads of the 8-bit key/value cache: what a program that serves a decoder
(or attends from it to an encoder's states) has the library do with one layer's
cache.

The cache holds, for each sequence and kv head, blocks of 64 tokens. A full
block of keys (or of values) is held as int8 codes with one f32 scale: with a
the largest |x| of the block's 64 rows (x rounded to f16), scale = a / 127 and
code = 127 x / a rounded to the nearest whole number, ties to even. The tokens
of the last, partial block are held in f16 until it fills.

A case is a dict of plain values whose "op" selects the work:

  append  a prompt's keys and values into an empty cache, which is then read
          back as the values it holds
  attend  attention of the last n tokens of each sequence over the cache,
          optionally adding every token's attention weight to an accumulator
  step    n new tokens: append, attention of their queries, and the cache taken
          back to its length (what a verification of drafted tokens does when
          it rejects them; a plain decode step is n = 1)
  evict   each kv head keeps `keep` tokens of its cache, the first and the
          most recent ones and otherwise those of largest accumulated weight,
          moved into another cache, which is then read back

Ragged cases have sequences of other lengths, and padded query rows and new
tokens at the end of their batch rows.
"""
import math

import torch

own = False

BLOCK = 64
DTYPE = {"f16": torch.float16, "f32": torch.float32}
SIZE = {"f16": 2, "f32": 4}
TYPESTR = {"f16": "<f2", "f32": "<f4", "u32": "<i4"}
NOWHERE = 1 << 40         # the position of a key that does not exist


# ---- the cases ------------------------------------------------------------------

def listed():
    return [
        # one decode step of a small decoder (9 query heads on 3 kv heads of 64)
        # a sentence into its answer: nothing to stream, latency alone
        {"name": "step_small", "op": "step", "dtype": "f16", "batch": 1, "heads": 9, "kv_heads": 3,
         "dim": 64, "vdim": 64, "length": 200, "n": 1, "ragged": False},
        # four drafted tokens verified for each of six sequences of other lengths
        {"name": "step_draft", "op": "step", "dtype": "f16", "batch": 6, "heads": 32, "kv_heads": 8,
         "dim": 128, "vdim": 128, "length": 2500, "n": 4, "ragged": True},
        # a long prompt enters an empty cache
        {"name": "append_prompt", "op": "append", "dtype": "f16", "batch": 1, "kv_heads": 8, "dim": 128,
         "vdim": 128, "n": 16400, "ragged": False},
        # a padded batch of f32 keys and values of odd length
        {"name": "append_ragged_f32", "op": "append", "dtype": "f32", "batch": 6, "kv_heads": 12, "dim": 72,
         "vdim": 72, "n": 777, "ragged": True},
        # one decode step of eight sequences over their caches
        {"name": "attend_decode", "op": "attend", "dtype": "f16", "batch": 8, "heads": 32, "kv_heads": 8,
         "dim": 128, "vdim": 128, "length": 4096, "n": 1, "causal": True, "ragged": False, "weights": False},
        # the same with the weights that an eviction goes by
        {"name": "attend_weights", "op": "attend", "dtype": "f16", "batch": 8, "heads": 32, "kv_heads": 8,
         "dim": 128, "vdim": 128, "length": 4090, "n": 1, "causal": True, "ragged": True, "weights": True},
        # one sequence with a very long cache
        {"name": "attend_long", "op": "attend", "dtype": "f16", "batch": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "vdim": 128, "length": 131000, "n": 1, "causal": True, "ragged": False, "weights": False},
        # f32 text queries over a vision encoder's states of another length (a
        # class token makes it odd), every state visible to every query
        {"name": "attend_cross_f32", "op": "attend", "dtype": "f32", "batch": 4, "heads": 16, "kv_heads": 16,
         "dim": 80, "vdim": 80, "length": 1025, "n": 48, "causal": False, "ragged": True, "weights": False},
        # a chunk of a long prompt over the chunks before it
        {"name": "attend_prompt", "op": "attend", "dtype": "f16", "batch": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "vdim": 128, "length": 8192, "n": 2048, "causal": True, "ragged": False, "weights": False},
        # a prompt whose tokens' weights are wanted
        {"name": "attend_prompt_weights", "op": "attend", "dtype": "f16", "batch": 2, "heads": 15,
         "kv_heads": 5, "dim": 64, "vdim": 64, "length": 1500, "n": 1500, "causal": True, "ragged": False,
         "weights": True},
        # a small decoder's cache cut to its budget
        {"name": "evict_small", "op": "evict", "batch": 1, "kv_heads": 3, "dim": 64, "vdim": 64,
         "length": 1100, "keep": 500, "first": 4, "recent": 64, "ragged": False},
        # the caches of eight sequences cut to half
        {"name": "evict_large", "op": "evict", "batch": 8, "kv_heads": 8, "dim": 128, "vdim": 128,
         "length": 8200, "keep": 4096, "first": 4, "recent": 256, "ragged": True},
    ]


def _log(rng, low, high):
    """An integer of [low, high], uniform in its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "attend", "step", "step", "evict", "evict"])
    dim = rng.choice([64, 64, 64, 128, 128, 128, 32, 72, 80, 96, 256, 100])
    c = {"op": op, "dim": dim, "vdim": dim if rng.random() < 0.8 else rng.choice([64, 96, 128])}
    kv = rng.choice([1, 2, 3, 4, 5, 8, 12])
    c["kv_heads"] = kv
    c["ragged"] = rng.random() < 0.5
    if op == "append":
        c["dtype"] = rng.choice(["f16", "f16", "f32"])
        c["n"] = _log(rng, 1, 16000)
        c["batch"] = _log(rng, 1, max(1, min(32, (16 << 20) // (c["n"] * kv * dim))))
        return c
    if op == "evict":
        c["length"] = _log(rng, 100, 16000)
        c["batch"] = _log(rng, 1, max(1, min(16, (32 << 20) // (c["length"] * kv * dim))))
        c["keep"] = max(2, int(c["length"] * rng.uniform(0.25, 1.1)))
        c["first"] = min(rng.choice([0, 4]), c["keep"] // 2)
        c["recent"] = min(_log(rng, 1, 512), c["keep"] // 2)
        return c
    c["dtype"] = rng.choice(["f16", "f16", "f16", "f32"])
    c["heads"] = kv * rng.choice([1, 1, 2, 3, 4, 7, 8])
    if op == "step":
        c["n"] = rng.choice([1, 1, 1, 2, 4, 7])
        c["length"] = _log(rng, 1, 16000)
        c["batch"] = _log(rng, 1, max(1, min(48, (96 << 20) // (c["length"] * kv * dim))))
        return c
    c["causal"] = rng.random() < 0.75
    c["weights"] = rng.random() < 0.3
    form = rng.choice(["decode", "decode", "chunk", "prompt"])
    c["length"] = _log(rng, 64, 32000 if form == "decode" else 4000)
    c["n"] = 1 if form == "decode" else _log(rng, 2, 64) if form == "chunk" else c["length"]
    c["n"] = min(c["n"], c["length"])
    most = min((96 << 20) // (c["length"] * kv * dim), (256 << 20) // (c["length"] * c["n"] * c["heads"]), 48)
    c["batch"] = _log(rng, 1, max(1, most))
    while c["batch"] * c["heads"] * c["n"] * c["length"] * dim > 32 << 30:
        c["length"] = c["length"] * 3 // 4
        c["n"] = c["length"] if form == "prompt" else c["n"]
    return c


def _lengths(c):
    """Tokens of each sequence before the call (append: none)."""
    b, n = c["batch"], c.get("length", 0)
    return [n - n * i // (2 * b) if c["ragged"] else n for i in range(b)]


def _counts(c):
    """Query rows and new tokens of each sequence; a padded batch's last one has
    hardly any."""
    b, n = c["batch"], c["n"]
    counts = [n - n * i // (2 * b) if c["ragged"] else n for i in range(b)]
    if c["ragged"] and b > 3:
        counts[-1] = min(1, n - 1)
    return counts


# ---- inputs ---------------------------------------------------------------------

def _inputs(c, seed):
    """Name -> torch tensor on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 29)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    b, h, d, e = c["batch"], c["kv_heads"], c["dim"], c["vdim"]
    dtype = DTYPE[c.get("dtype", "f16")]
    # keys have a few channels that are several times the others; values are even
    channel = torch.exp(0.6 * normal(1, h, 1, d))

    def keys(n):
        return normal(b, h, n, d) * channel

    out = {}
    if c["op"] in ("attend", "step", "evict"):
        out["k"] = keys(c["length"]).to(torch.float16)
        out["v"] = normal(b, h, c["length"], e).to(torch.float16)
    if c["op"] in ("append", "step"):
        out["new_k"] = keys(c["n"]).to(dtype)
        out["new_v"] = normal(b, h, c["n"], e).to(dtype)
    if c["op"] in ("attend", "step"):
        out["q"] = normal(b, c["heads"], c["n"], d).to(dtype)
    if c.get("weights") or c["op"] == "evict":
        # what earlier calls have added up: many small, a few large
        out["w"] = torch.exp(2.0 * normal(b, h, c["length"]) - 2.0)
    return out


# ---- the plain form of the cache ---------------------------------------------------

def _hold(x, lengths):
    """The cache of rows x [B, H, T, D] (f32 or f64, exact), of which sequence b
    has lengths[b]: codes and scales of every whole block, and the rows of each
    sequence's last block in f16."""
    b, h, t, d = x.shape
    blocks = -(-t // BLOCK)
    x = torch.nn.functional.pad(x, (0, 0, 0, blocks * BLOCK - t))
    # borders between two codes are decided in 64 bits
    tiles = x.double().reshape(b, h, blocks, BLOCK, d)
    largest = tiles.abs().amax((3, 4))
    step = largest[..., None, None]
    codes = torch.where(step > 0, torch.round(127.0 * tiles / step), torch.zeros_like(tiles)).to(torch.int8)
    scale = (largest / 127.0).float()
    rows = (lengths // BLOCK * BLOCK)[:, None] + torch.arange(BLOCK, device=x.device)
    open_rows = x.gather(2, rows.clamp(max=max(blocks * BLOCK - 1, 0))[:, None, :, None].expand(b, h, BLOCK, d))
    return {"codes": codes, "scale": scale, "open": open_rows.to(torch.float16)}


def _closed(held, dtype=torch.float32):
    """The values of the whole blocks, [B, H, blocks * 64, D]."""
    return (held["codes"].to(dtype) * held["scale"][..., None, None].to(dtype)).flatten(2, 3)


def _positions(held, lengths):
    """Position of each row of _closed() and of the open block; NOWHERE for rows
    that are not there."""
    blocks = held["codes"].shape[2]
    first = lengths // BLOCK * BLOCK
    t = torch.arange(blocks * BLOCK, device=lengths.device)[None, :]
    w = torch.arange(BLOCK, device=lengths.device)[None, :]
    closed = torch.where(t < first[:, None], t, NOWHERE)
    return closed, torch.where(w < (lengths - first)[:, None], first[:, None] + w, NOWHERE)


def _whole(held, lengths, rows, dtype):
    """Rows 0 .. rows - 1 of the cache in their order; zeros where there are none."""
    b, h, d = held["open"].shape[0], held["open"].shape[1], held["open"].shape[3]
    closed, opened = _positions(held, lengths)
    at = torch.cat([closed, opened], 1)
    values = torch.cat([_closed(held, dtype), held["open"].to(dtype)], 2)
    values = torch.where((at < NOWHERE)[:, None, :, None], values, torch.zeros_like(values))
    out = torch.zeros((b, h, rows + 1, d), device=values.device, dtype=dtype)
    out.scatter_(2, at.clamp(max=rows)[:, None, :, None].expand(b, h, at.shape[1], d), values)
    return out[:, :, :rows]


def _attend(c, q, keys, values, at, lengths, counts):
    """Attention of q [B, Hq, n, D] (f32) over keys and values [B, H, T, ..] at
    positions at [B, T]; also p [B, H, group * n, T]."""
    b, hq, n, d = q.shape
    h = keys.shape[1]
    i = torch.arange(n, device=q.device)
    # how many keys query row i sees
    seen = (lengths - counts)[:, None] + i + 1 if c.get("causal", True) else lengths[:, None] + 0 * i
    seen = torch.where(i < counts[:, None], seen, 0 * seen)
    seen = seen[:, None, :].expand(b, hq // h, n).reshape(b, 1, -1, 1)
    s = torch.matmul(q.reshape(b, h, hq // h * n, d), keys.transpose(2, 3).contiguous()) * d ** -0.5
    s = s.masked_fill(at[:, None, None, :] >= seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    return torch.matmul(p, values).reshape(b, hq, n, -1), p


def _plain_append(c, s):
    lengths = s["lengths"]
    rows = c["n"]
    out = {}
    for name in ("k", "v"):
        x = s["new_" + name].to(torch.float16).float()
        out[name] = _whole(_hold(x, lengths), lengths, rows, torch.float32).to(DTYPE[c["dtype"]])
    return out


def _plain_attend(c, s):
    lengths = s["lengths"]
    closed, opened = _positions(s["held_k"], lengths)
    at = torch.cat([closed, opened], 1)
    kv = [torch.cat([_closed(s[n]), s[n]["open"].float()], 2) for n in ("held_k", "held_v")]
    kv[1] = torch.where((at < NOWHERE)[:, None, :, None], kv[1], torch.zeros_like(kv[1]))
    out, p = _attend(c, s["q"].float(), kv[0], kv[1], at, lengths, s["counts"])
    # padded rows are left as they were
    s["out"].copy_(torch.where(s["live"], out, s["out"].float()))
    got = {"out": s["out"]}
    if c["weights"]:
        b, h, t = s["w"].shape
        add = p.sum(2)
        s["w"].scatter_add_(2, at.clamp(max=t - 1)[:, None, :].expand(b, h, at.shape[1]), add)
        got["w"] = s["w"]
    return got


def _plain_step(c, s):
    lengths, counts = s["lengths"], s["counts"]
    first = lengths // BLOCK * BLOCK
    # the open block's rows and the new ones behind them, held anew
    window = -(-(BLOCK - 1 + c["n"]) // BLOCK) * BLOCK
    inside = lengths - first
    w = torch.arange(window, device=lengths.device)[None, :]
    source = torch.where(w < inside[:, None], w, BLOCK + w - inside[:, None]).clamp(max=BLOCK + c["n"] - 1)
    closed, _ = _positions(s["held_k"], lengths)
    ends = inside + counts
    parts = []
    for name in ("k", "v"):
        rows = torch.cat([s["held_" + name]["open"], s["new_" + name].to(torch.float16)], 2).float()
        rows = rows.gather(2, source[:, None, :, None].expand(-1, rows.shape[1], -1, rows.shape[3]))
        rows = torch.where((w < ends[:, None])[:, None, :, None], rows, torch.zeros_like(rows))
        rows = _whole(_hold(rows, ends), ends, window, torch.float32)
        parts.append(torch.cat([_closed(s["held_" + name]), rows], 2))
    at = torch.cat([closed, torch.where(w < ends[:, None], first[:, None] + w, NOWHERE)], 1)
    out, _ = _attend(c, s["q"].float(), parts[0], parts[1], at, lengths + counts, counts)
    s["out"].copy_(torch.where(s["live"], out, s["out"].float()))
    return {"out": s["out"]}


def _plain_evict(c, s):
    lengths = s["lengths"]
    b, h, t = s["w"].shape
    kept = lengths.clamp(max=c["keep"])
    i = torch.arange(t, device=lengths.device)[None, :]
    there = i < lengths[:, None]
    always = there & ((i < c["first"]) | (i >= (lengths - c["recent"])[:, None]))
    rank = torch.where(always[:, None], math.inf, torch.where(there[:, None], s["w"], -math.inf))
    best = torch.argsort(rank, dim=-1, descending=True, stable=True)[..., :c["keep"]]
    slot = torch.arange(best.shape[-1], device=lengths.device)[None, :]
    live = (slot < kept[:, None])[:, None].expand(b, h, -1)
    best = torch.sort(torch.where(live, best, t), dim=-1).values
    index = best.clamp(max=t - 1)
    got = {"w": torch.where(live, s["w"].gather(2, index), torch.zeros((), device=best.device)),
           "kept": torch.where(live, best, torch.zeros_like(best)).int()}
    for name in ("k", "v"):
        rows = _whole(s["held_" + name], lengths, t, torch.float64)
        rows = rows.gather(2, index[..., None].expand(-1, -1, -1, rows.shape[3]))
        rows = torch.where(live[..., None], rows, torch.zeros_like(rows))
        got[name] = _whole(_hold(rows, kept), kept, best.shape[-1], torch.float32).half()
    return got


# ---- state ------------------------------------------------------------------------

class _Memory:
    """A library tensor's device memory for torch.as_tensor (no copy)."""

    def __init__(self, tensor):
        self.tensor = tensor
        self.__cuda_array_interface__ = {
            "shape": tensor.shape, "typestr": TYPESTR[tensor.dtype],
            "data": (tensor.device_ptr(), False), "version": 2}


_library = None


def _sdk():
    global _library
    if _library is None:
        from inference_c_amd import Sdk
        _library = Sdk()
        _library.require_device()
    return _library


def _tensor(dtype, value):
    """(library tensor, torch view of it) that holds `value`."""
    tensor = _sdk().tensor(dtype, tuple(value.shape))
    view = torch.as_tensor(_Memory(tensor), device="cuda")
    view.copy_(value)
    return tensor, view


def _rows_kept(c):
    return min(c["keep"], c["length"])


def _prepare_own(c, a, state):
    """The handle with its tokens, and the operands and outputs as library tensors."""
    import ctypes
    lib, b = _sdk(), c["batch"]
    name = {torch.float16: "f16", torch.float32: "f32"}
    t, views = {}, {}
    for key, value in a.items():
        t[key], views[key] = _tensor(name[value.dtype], value)
    before = _lengths(c) if c["op"] != "append" else [0] * b
    state["before"] = (ctypes.c_uint32 * b)(*before)
    state["rows"] = (ctypes.c_uint32 * b)(*_counts(c)) if c["op"] != "evict" and c["ragged"] else None
    capacity = max(before) + (c["n"] if c["op"] in ("append", "step") else 0)
    cache = lib.kv_cache(b, c["kv_heads"], capacity, c["dim"], c["vdim"])
    out = {}
    if c["op"] in ("append", "evict"):
        rows = c["n"] if c["op"] == "append" else _rows_kept(c)
        for key, width in (("k", c["dim"]), ("v", c["vdim"])):
            zeros = torch.zeros((b, c["kv_heads"], rows, width), device="cuda")
            t["out_" + key], out[key] = _tensor(c.get("dtype", "f16"), zeros)
    if c["op"] in ("attend", "step"):
        zeros = torch.zeros((b, c["heads"], c["n"], c["vdim"]), device="cuda")
        t["out"], out["out"] = _tensor(c["dtype"], zeros)
    if c.get("weights"):
        out["w"] = views["w"]
    if c["op"] == "evict":
        state["target"] = lib.kv_cache(b, c["kv_heads"], _rows_kept(c), c["dim"], c["vdim"])
        zeros = torch.zeros((b, c["kv_heads"], _rows_kept(c)), device="cuda")
        t["out_w"], out["w"] = _tensor("f32", zeros)
        t["kept"], out["kept"] = _tensor("u32", zeros.int())
    torch.cuda.synchronize()   # torch fills on its own stream, the library reads on another
    if c["op"] != "append":
        lib.call("tensor_kv_cache_append_f16", cache, t["k"], t["v"], state["before"])
    lib.synchronize()
    state.update(cache=cache, t=t, result=out)


def prepare(case, seed):
    c = case
    a = _inputs(c, seed)
    state = {"case": c}
    if own:
        _prepare_own(c, a, state)
        return state
    tell = torch.tensor
    lengths = _lengths(c) if c["op"] != "append" else _counts(c)
    state["lengths"] = tell(lengths, device="cuda")
    state.update({n: x for n, x in a.items() if n not in ("k", "v")})
    if "k" in a:
        state["held_k"] = _hold(a["k"].float(), state["lengths"])
        state["held_v"] = _hold(a["v"].float(), state["lengths"])
    if "q" in a:
        counts = _counts(c)
        state["counts"] = tell(counts, device="cuda")
        i = torch.arange(c["n"], device="cuda")
        state["live"] = (i < state["counts"][:, None])[:, None, :, None]
        state["out"] = torch.zeros((c["batch"], c["heads"], c["n"], c["vdim"]), device="cuda",
                                   dtype=DTYPE[c["dtype"]])
    torch.cuda.synchronize()
    return state


def _run_own(c, s):
    call, cache, t = _sdk().call, s["cache"], s["t"]
    op, d, rows = c["op"], c.get("dtype", "f16"), s["rows"]
    if op == "append":
        call("tensor_kv_cache_truncate", cache, None)
        call(f"tensor_kv_cache_append_{d}", cache, t["new_k"], t["new_v"], rows)
        call(f"tensor_kv_cache_read_{d}", cache, t["out_k"], t["out_v"])
    elif op == "attend":
        call(f"tensor_kv_cache_attention_{d}", cache, t["q"], rows, c["dim"] ** -0.5, int(c["causal"]),
             t["w"] if c["weights"] else None, t["out"])
    elif op == "step":
        call(f"tensor_kv_cache_append_{d}", cache, t["new_k"], t["new_v"], rows)
        call(f"tensor_kv_cache_attention_{d}", cache, t["q"], rows, c["dim"] ** -0.5, 1, None, t["out"])
        call("tensor_kv_cache_truncate", cache, s["before"])
    else:
        call("tensor_kv_cache_evict", cache, t["w"], c["first"], c["recent"], c["keep"], s["target"],
             t["out_w"], t["kept"])
        call("tensor_kv_cache_read_f16", s["target"], t["out_k"], t["out_v"])
    return s["result"]


def run(state):
    c = state["case"]
    if own:
        return _run_own(c, state)
    return {"append": _plain_append, "attend": _plain_attend, "step": _plain_step,
            "evict": _plain_evict}[c["op"]](c, state)


# ---- what a pass cannot do without ---------------------------------------------------

def work(case):
    c, op = case, case["op"]
    h, d, e = c["kv_heads"], c["dim"], c["vdim"]
    if op == "append":     # rows in, codes out; codes in, rows out
        tokens = sum(_counts(c)) * h
        return {"bytes": tokens * (d + e) * 2 * (SIZE[c["dtype"]] + 1), "flops": 0}
    if op == "evict":      # every weight, and of the kept tokens codes in and out, then rows out
        kept = sum(min(c["keep"], n) for n in _lengths(c)) * h
        return {"bytes": 4 * h * sum(_lengths(c)) + kept * ((d + e) * (1 + 1 + 1 + 2) + 8), "flops": 0}
    lengths, counts = _lengths(c), _counts(c)
    if op == "step":
        lengths = [x + y for x, y in zip(lengths, counts)]
    causal = c.get("causal", True)
    group = c["heads"] // h
    pairs = seen = 0
    for length, n in zip(lengths, counts):
        if n == 0:
            continue
        # row i sees length - n + i + 1 keys (none where that is not positive)
        start = max(0, length - n)
        live = min(n, length)
        pairs += group * (n * length if not causal else live * start + live * (live + 1) // 2)
        seen += length
    size = SIZE[c["dtype"]]
    tokens = sum(counts)
    moved = seen * h * (d + e) + tokens * c["heads"] * (d + e) * size
    if op == "step":
        moved += tokens * h * (d + e) * size
    if c.get("weights"):
        moved += 8 * seen * h
    return {"bytes": moved, "flops": 2 * pairs * h * (d + e)}


# ---- the same in 64 bits ---------------------------------------------------------------

def _held_values(x):
    """What a cache of x [H, T, D] (f64) gives back: whole blocks through their
    codes, the rest rounded to f16."""
    h, t, d = x.shape
    n = t // BLOCK * BLOCK
    tiles = x[:, :n].reshape(h, -1, BLOCK * d)
    big = tiles.abs().max(-1, keepdim=True).values if n else tiles
    codes = torch.round(tiles * 127.0 / torch.where(big == 0, 1.0, big))
    scale = (big / 127.0).float().double()      # the scale is held in f32
    return torch.cat([(codes * scale).reshape(h, n, d), x[:, n:].half().double()], 1)


def _softmax_rows(c, q, k, v, n):
    """Outputs and summed weights of the n rows per head that end the sequence."""
    h, t = k.shape[0], k.shape[1]
    group = c["heads"] // h
    out = torch.zeros((c["heads"], n, v.shape[2]), device=q.device, dtype=torch.float64)
    weight = torch.zeros((h, t), device=q.device, dtype=torch.float64)
    hidden = None
    if c.get("causal", True):
        hidden = torch.arange(t, device=q.device)[None, :] > torch.arange(n, device=q.device)[:, None] + t - n
    for j in range(c["heads"]):
        s = q[j] @ k[j // group].t().contiguous() / math.sqrt(c["dim"])
        if hidden is not None:
            s = s.masked_fill(hidden, -math.inf)
        p = torch.softmax(s, -1).nan_to_num(0.0)     # a row that sees nothing is zero
        out[j] = p @ v[j // group]
        weight[j // group] += p.sum(0)
    return out, weight


def exact(case, seed):
    c = case
    a = {n: x.double() for n, x in _inputs(c, seed).items()}
    b, h = c["batch"], c["kv_heads"]
    half = {n: a[n].half().double() for n in ("new_k", "new_v") if n in a}
    if c["op"] == "append":
        out = {n: torch.zeros_like(a["new_" + n]) for n in ("k", "v")}
        for i, n in enumerate(_counts(c)):
            for name in out:
                out[name][i, :, :n] = _held_values(half["new_" + name][i, :, :n])
        return out
    if c["op"] == "evict":
        rows = _rows_kept(c)
        out = {"w": torch.zeros((b, h, rows), device="cuda", dtype=torch.float64),
               "kept": torch.zeros((b, h, rows), device="cuda", dtype=torch.int32)}
        for name, width in (("k", c["dim"]), ("v", c["vdim"])):
            out[name] = torch.zeros((b, h, rows, width), device="cuda", dtype=torch.float64)
        for i, length in enumerate(_lengths(c)):
            w = a["w"][i, :, :length].clone()
            n = min(c["keep"], length)
            w[:, :c["first"]] = math.inf
            w[:, max(0, length - c["recent"]):] = math.inf
            # the n largest, the earlier of two equal ones first
            order = torch.sort(-w, dim=-1, stable=True).indices[:, :n].sort(-1).values
            out["kept"][i, :, :n] = order.int()
            out["w"][i, :, :n] = a["w"][i].gather(1, order)
            for name in ("k", "v"):
                x = _held_values(a[name][i, :, :length])
                out[name][i, :, :n] = _held_values(x.gather(1, order[..., None].expand(-1, -1, x.shape[2])))
        return out
    out = torch.zeros((b, c["heads"], c["n"], c["vdim"]), device="cuda", dtype=torch.float64)
    weights = a["w"].clone() if c.get("weights") else None
    for i, (length, n) in enumerate(zip(_lengths(c), _counts(c))):
        kv = []
        for name in ("k", "v"):
            x = a[name][i, :, :length]
            if c["op"] == "step":
                # the blocks that were whole are held as they were; the others anew
                x = torch.cat([x, half["new_" + name][i, :, :n]], 1)
            kv.append(_held_values(x))
        if n:
            out[i, :, :n], add = _softmax_rows(c, a["q"][i, :, :n], kv[0], kv[1], n)
            if weights is not None:
                weights[i, :, :add.shape[1]] += add
    return {"out": out} if weights is None else {"out": out, "w": weights}
