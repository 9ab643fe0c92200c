"""Workloads of beam search and of batches that share a prompt: what a program
that serves a decoder has the library do between and inside its steps, beside the
8-bit key/value cache (perf/operators.py says how that holds its tokens).

A case is a dict of plain values whose "op" selects the work:

  select   one step's choice over beams and vocabulary: of each group of beams the
           `keep` candidates (beam, token) of the largest score[beam] +
           log softmax(logits[beam])[token], in that order; a beam that has ended
           has one candidate, the end token at its own score
  reorder  the beams' caches follow the choice: within each group sequence b goes
           on as a copy of sequence parents[b]; the cache is then read back
  copy     sequences of a cache copied into another one (a prompt into its beams,
           the sequences that are still running into a smaller batch), which is
           then read back
  shared   attention of each sequence's last n tokens over a prompt that is held
           once for all sequences of its group, followed by the sequence's own
           tokens

Ragged cases have prompts and sequences of other lengths, groups of other sizes
and padded query rows.
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
        # four beams of one sentence: two launches, latency alone
        {"name": "select_small", "op": "select", "dtype": "f32", "groups": 1, "beams": 4, "vocab": 49152,
         "keep": 4, "ended": False, "masked": False},
        # a batch of sentences, f16 logits of an odd vocabulary, as many candidates again
        # as beams (those that end leave room), some beams at their end
        {"name": "select_batch", "op": "select", "dtype": "f16", "groups": 16, "beams": 8, "vocab": 32003,
         "keep": 16, "ended": True, "masked": False},
        # a large batch over a large vocabulary, streamed from memory
        {"name": "select_large", "op": "select", "dtype": "f32", "groups": 32, "beams": 8, "vocab": 128256,
         "keep": 8, "ended": False, "masked": False},
        # the caches of four beams of a small decoder
        {"name": "reorder_small", "op": "reorder", "groups": 1, "beams": 4, "kv_heads": 3, "dim": 64, "vdim": 64,
         "length": 300, "ragged": False},
        # those of sixteen sentences with eight beams each
        {"name": "reorder_large", "op": "reorder", "groups": 16, "beams": 8, "kv_heads": 8, "dim": 128, "vdim": 128,
         "length": 1100, "ragged": True},
        # four prompts, each into its eight beams
        {"name": "copy_fork", "op": "copy", "batch": 4, "target": 32, "kv_heads": 8, "dim": 128, "vdim": 128,
         "length": 2000, "ragged": False},
        # a batch closed up: nine of sixteen sequences still run
        {"name": "copy_compact", "op": "copy", "batch": 16, "target": 9, "kv_heads": 5, "dim": 72, "vdim": 72,
         "length": 777, "ragged": True},
        # a decode step of four beams on one short prompt
        {"name": "shared_small", "op": "shared", "dtype": "f16", "prompts": 1, "batch": 4, "heads": 9, "kv_heads": 3,
         "dim": 64, "vdim": 64, "prompt": 200, "length": 20, "n": 1, "causal": True, "ragged": False},
        # a decode step of eight sentences with eight beams each
        {"name": "shared_beams", "op": "shared", "dtype": "f16", "prompts": 8, "batch": 64, "heads": 32, "kv_heads": 8,
         "dim": 128, "vdim": 128, "prompt": 2000, "length": 100, "n": 1, "causal": True, "ragged": False},
        # a decode step of 64 conversations that begin with the same instructions
        {"name": "shared_system", "op": "shared", "dtype": "f16", "prompts": 1, "batch": 64, "heads": 32, "kv_heads": 8,
         "dim": 128, "vdim": 128, "prompt": 16000, "length": 500, "n": 1, "causal": True, "ragged": True},
        # drafted tokens of f32 sequences on three prompts of other lengths
        {"name": "shared_draft_f32", "op": "shared", "dtype": "f32", "prompts": 3, "batch": 14, "heads": 16,
         "kv_heads": 4, "dim": 80, "vdim": 80, "prompt": 1500, "length": 130, "n": 4, "causal": True, "ragged": True},
        # questions about one long document, a chunk of each at once
        {"name": "shared_chunk", "op": "shared", "dtype": "f16", "prompts": 1, "batch": 4, "heads": 32, "kv_heads": 8,
         "dim": 128, "vdim": 128, "prompt": 8000, "length": 512, "n": 512, "causal": True, "ragged": False},
    ]


def _log(rng, low, high):
    """An integer of [low, high], uniform in its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["select", "select", "select", "reorder", "copy", "shared", "shared", "shared", "shared"])
    c = {"op": op}
    if op == "select":
        c["dtype"] = rng.choice(["f16", "f32"])
        c["vocab"] = _log(rng, 1000, 150000)
        c["beams"] = rng.choice([1, 2, 3, 4, 4, 5, 8, 8, 10, 16])
        c["groups"] = _log(rng, 1, max(1, min(64, (32 << 20) // (c["vocab"] * c["beams"]))))
        c["keep"] = rng.choice([c["beams"], c["beams"], 2 * c["beams"], 2 * c["beams"] + 1, rng.randint(1, 64)])
        c["ended"] = rng.random() < 0.4
        c["masked"] = rng.random() < 0.25
        return c
    dim = rng.choice([64, 64, 64, 128, 128, 128, 32, 72, 80, 96, 256, 100])
    c["dim"], c["vdim"] = dim, dim if rng.random() < 0.8 else rng.choice([64, 96, 128])
    kv = c["kv_heads"] = rng.choice([1, 2, 3, 4, 5, 8, 12])
    c["ragged"] = rng.random() < 0.5
    if op in ("reorder", "copy"):
        c["length"] = _log(rng, 1, 4000)
        most = max(2, min(128, (16 << 20) // (c["length"] * kv * dim)))
        if op == "reorder":
            c["beams"] = min(rng.choice([2, 3, 4, 4, 5, 8, 8, 16]), most)
            c["groups"] = _log(rng, 1, max(1, most // c["beams"]))
        else:
            c["batch"] = _log(rng, 1, most)
            c["target"] = _log(rng, 1, most)
        return c
    c["dtype"] = rng.choice(["f16", "f16", "f16", "f32"])
    c["heads"] = kv * rng.choice([1, 1, 2, 3, 4, 7, 8])
    c["causal"] = rng.random() < 0.8
    form = rng.choice(["decode", "decode", "decode", "draft", "chunk"])
    c["n"] = 1 if form == "decode" else rng.randint(2, 8) if form == "draft" else _log(rng, 9, 512)
    c["length"] = c["n"] + _log(rng, 1, 1000) - 1
    c["prompt"] = _log(rng, 1, 16000)
    rows = c["heads"] * c["n"] * (c["prompt"] + c["length"])
    most = min((48 << 20) // (c["length"] * kv * dim), (160 << 20) // rows, (24 << 30) // (rows * dim), 96)
    c["batch"] = _log(rng, 1, max(1, most))
    c["prompts"] = _log(rng, 1, max(1, min(c["batch"], (48 << 20) // (c["prompt"] * kv * dim))))
    return c


def _shorter(n, parts, ragged):
    """`parts` lengths of up to n; ragged ones go down to the half of it."""
    return [n - n * i // (2 * parts) if ragged else n for i in range(parts)]


def _lengths(c):
    """Tokens of each sequence of the cache (shared: of its own)."""
    if c["op"] == "reorder":
        return [n for n in _shorter(c["length"], c["groups"], c["ragged"]) for _ in range(c["beams"])]
    return _shorter(c["length"], c["batch"], c["ragged"])


def _members(c):
    """Sequences on each prompt; ragged groups are of other sizes."""
    p, b = c["prompts"], c["batch"]
    if not c["ragged"]:
        return [b * (i + 1) // p - b * i // p for i in range(p)]
    ends = [int(b * ((i + 1) / p) ** 1.5 + 0.5) for i in range(p)]
    ends = [max(e, i + 1) for i, e in enumerate(ends)]
    return [e - s for s, e in zip([0] + ends, ends)]


def _counts(c):
    """Query rows of each sequence; a padded batch's last one has hardly any."""
    counts = _shorter(c["n"], c["batch"], c["ragged"])
    if c["ragged"] and c["batch"] > 3:
        counts[-1] = min(1, c["n"] - 1)
    return counts


def _sources(c):
    """The sequence that each of the target's is a copy of: spread over the batch."""
    return [i * c["batch"] // c["target"] for i in range(c["target"])]


# ---- inputs ---------------------------------------------------------------------

def _inputs(c, seed):
    """Name -> torch tensor on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 31)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda", dtype=torch.float32)

    out = {}
    if c["op"] == "select":
        rows = (c["groups"], c["beams"])
        x = 2.5 * normal(*rows, c["vocab"])
        if c["masked"]:          # what a grammar does not allow
            x = x.masked_fill(uniform(*rows, c["vocab"]) < 0.98, -math.inf)
        out["logits"] = x.to(DTYPE[c["dtype"]])
        # sums of the log probabilities of the tokens so far, the best beam first
        out["scores"] = torch.sort(-8.0 - 2.0 * normal(*rows).abs(), descending=True).values
        if c["ended"]:
            out["ended"] = (uniform(*rows) < 0.25).int()
        return out
    h, d, e = c["kv_heads"], c["dim"], c["vdim"]
    # keys have a few channels that are several times the others; values are even
    channel = torch.exp(0.6 * normal(1, h, 1, d))
    b = c["groups"] * c["beams"] if c["op"] == "reorder" else c["batch"]
    out["k"] = (normal(b, h, c["length"], d) * channel).to(torch.float16)
    out["v"] = normal(b, h, c["length"], e).to(torch.float16)
    if c["op"] == "reorder":
        # the beams whose continuations win keep their places, the others take copies of
        # them (so a pass over its own result is the same work again)
        wins = uniform(c["groups"], c["beams"]) < 0.4
        wins[:, 0] = True
        i = torch.arange(c["beams"], device="cuda")[None, :]
        last = torch.cummax(torch.where(wins, i, torch.zeros_like(i)), 1).values
        out["parents"] = torch.where(wins, i, last).int()
    if c["op"] == "shared":
        out["prompt_k"] = (normal(c["prompts"], h, c["prompt"], d) * channel).to(torch.float16)
        out["prompt_v"] = normal(c["prompts"], h, c["prompt"], e).to(torch.float16)
        out["q"] = normal(c["batch"], c["heads"], c["n"], d).to(DTYPE[c["dtype"]])
    return out


# ---- the plain form --------------------------------------------------------------

def _hold(x, lengths):
    """The cache of f16 rows x [B, H, T, D], of which sequence b has lengths[b]:
    codes and scales of every whole block, and the rows of each sequence's last
    block in f16."""
    b, h, t, d = x.shape
    blocks = -(-t // BLOCK)
    x = torch.nn.functional.pad(x, (0, 0, 0, blocks * BLOCK - t))
    # borders between two codes are decided in 64 bits
    tiles = x.double().reshape(b, h, blocks, BLOCK, d)
    largest = tiles.abs().amax((3, 4))
    step = largest[..., None, None]
    codes = torch.where(step > 0, torch.round(127.0 * tiles / step), torch.zeros_like(tiles)).to(torch.int8)
    rows = (lengths // BLOCK * BLOCK)[:, None] + torch.arange(BLOCK, device=x.device)
    at = rows.clamp(max=blocks * BLOCK - 1)[:, None, :, None].expand(b, h, BLOCK, d)
    return {"codes": codes, "scale": (largest / 127.0).float(), "open": x.gather(2, at)}


def _rows(held, lengths):
    """Every row of a cache in f32, the open block's behind the others', and each
    one's position (NOWHERE where there is none); values of such rows are zeros."""
    values = (held["codes"].float() * held["scale"][..., None, None]).flatten(2, 3)
    first = lengths // BLOCK * BLOCK
    t = torch.arange(values.shape[2], device=lengths.device)[None, :]
    w = torch.arange(BLOCK, device=lengths.device)[None, :]
    at = torch.cat([torch.where(t < first[:, None], t, NOWHERE),
                    torch.where(w < (lengths - first)[:, None], first[:, None] + w, NOWHERE)], 1)
    values = torch.cat([values, held["open"].float()], 2)
    return torch.where((at < NOWHERE)[:, None, :, None], values, torch.zeros_like(values)), at


def _read(held, lengths, rows):
    """Rows 0 .. rows - 1 of the cache in their order, in f16; zeros where there are none."""
    values, at = _rows(held, lengths)
    b, h, t, d = values.shape
    out = torch.zeros((b, h, rows + 1, d), device=values.device)
    out.scatter_(2, at.clamp(max=rows)[:, None, :, None].expand(b, h, t, d), values)
    return out[:, :, :rows].half()


def _plain_select(c, s):
    g, k, v, keep = c["groups"], c["beams"], c["vocab"], c["keep"]
    # two candidates' scores may lie closer than 32 bits tell apart
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    score = s["scores"].double()[..., None] + (x - top - torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    if c["ended"]:
        token = torch.arange(v, device=x.device)
        alone = torch.where(token == s["end"], s["scores"].double()[..., None], -math.inf)
        score = torch.where(s["ended"][..., None] != 0, alone, score)
    score = score.reshape(g, k * v)
    # all above the last kept score, and of those equal to it the first ones
    least = torch.topk(score, keep).values[:, -1:]
    place = torch.arange(k * v, device=x.device)[None, :]
    rank = torch.where(score > least, place - k * v, torch.where(score == least, place, 2 * k * v))
    place = torch.sort(torch.topk(rank, keep, largest=False).values % (k * v)).values
    best, order = torch.sort(score.gather(1, place), descending=True, stable=True)
    place = place.gather(1, order)
    there = best > -math.inf
    parents = torch.where(there, place // v, torch.zeros_like(place))
    tokens = torch.where(there, place % v, s["end"] + torch.zeros_like(place))
    return {"parents": parents.int(), "tokens": tokens.int(), "scores": best.float(),
            "ended": (tokens == s["end"]).int()}


def _plain_reorder(c, s):
    first = torch.arange(c["groups"], device="cuda")[:, None] * c["beams"]
    source = (first + s["parents"]).reshape(-1)
    s.update({name: {part: x.index_select(0, source) for part, x in s[name].items()} for name in ("held_k", "held_v")})
    return {name: _read(s["held_" + name], s["lengths"], c["length"]) for name in ("k", "v")}


def _plain_copy(c, s):
    lengths = s["lengths"].index_select(0, s["source"])
    held = {name: {part: x.index_select(0, s["source"]) for part, x in s["held_" + name].items()} for name in ("k", "v")}
    return {name: _read(x, lengths, c["length"]) for name, x in held.items()}


def _plain_shared(c, s):
    b, hq, n, d = s["q"].shape
    h, p = c["kv_heads"], c["prompts"]
    q = s["q"].float()
    # scores of the prompt, the members of a group side by side as rows of one product
    # (`place`: the sequences of each prompt, `back`: where each sequence is there)
    keys, at = _rows(s["prompt_k"], s["prompt_lengths"])
    values, _ = _rows(s["prompt_v"], s["prompt_lengths"])
    together = q.index_select(0, s["place"].reshape(-1)).reshape(p, -1, h, hq // h * n, d).transpose(1, 2)
    x = torch.matmul(together.reshape(p, h, -1, d), keys.transpose(2, 3).contiguous()) * d ** -0.5
    x = x.masked_fill(at[:, None, None, :] == NOWHERE, -math.inf)
    most = s["place"].shape[1]
    there = x.reshape(p, h, most, hq // h * n, -1).transpose(1, 2).reshape(p * most, h, hq // h * n, -1)
    there = there.index_select(0, s["back"])
    # scores of the own tokens
    own_keys, own_at = _rows(s["held_k"], s["lengths"])
    own_values, _ = _rows(s["held_v"], s["lengths"])
    i = torch.arange(n, device=q.device)
    seen = (s["lengths"] - s["counts"])[:, None] + i + 1 if c["causal"] else s["lengths"][:, None] + 0 * i
    seen = seen[:, None, :].expand(b, hq // h, n).reshape(b, 1, -1, 1)
    x = torch.matmul(q.reshape(b, h, hq // h * n, d), own_keys.transpose(2, 3).contiguous()) * d ** -0.5
    x = x.masked_fill(own_at[:, None, None, :] >= seen, -math.inf)
    # one softmax over both
    top = torch.maximum(there.amax(-1, keepdim=True), x.amax(-1, keepdim=True))
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    there, x = torch.exp(there - top), torch.exp(x - top)
    total = there.sum(-1, keepdim=True) + x.sum(-1, keepdim=True)
    together = there.index_select(0, s["place"].reshape(-1)).reshape(p, most, h, hq // h * n, -1).transpose(1, 2)
    out = torch.matmul(together.reshape(p, h, most * (hq // h) * n, -1), values)
    out = out.reshape(p, h, most, hq // h * n, -1).transpose(1, 2).reshape(p * most, h, hq // h * n, -1)
    out = out.index_select(0, s["back"]) + torch.matmul(x, own_values)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    # padded rows are left as they were
    s["out"].copy_(torch.where(s["live"], out.reshape(b, hq, n, -1), s["out"].float()))
    return {"out": s["out"]}


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


def _end(c):
    return c["vocab"] - 1 if c["vocab"] % 2 else 2


def _prepare_own(c, a, state):
    """The handles with their tokens, and the operands and outputs as library tensors."""
    import ctypes
    lib = _sdk()
    name = {torch.float16: "f16", torch.float32: "f32", torch.int32: "u32"}
    t, out = {}, {}
    for key, value in a.items():
        t[key] = _tensor(name[value.dtype], value)[0]

    def output(key, dtype, *shape):
        t["out_" + key], out[key] = _tensor(dtype, torch.zeros(shape, device="cuda", dtype=torch.float32))

    def array(values):
        return (ctypes.c_uint32 * len(values))(*values)

    if c["op"] == "select":
        for key, dtype in (("parents", "u32"), ("tokens", "u32"), ("scores", "f32"), ("ended", "u32")):
            output(key, dtype, c["groups"], c["keep"])
    else:
        lengths = _lengths(c)
        state["cache"] = lib.kv_cache(len(lengths), c["kv_heads"], c["length"], c["dim"], c["vdim"])
    if c["op"] in ("reorder", "copy"):
        for key in ("k", "v"):
            output(key, "f16", c.get("target", len(lengths)), c["kv_heads"], c["length"], c[{"k": "dim", "v": "vdim"}[key]])
    if c["op"] == "copy":
        state["source"] = array(_sources(c))
        state["target"] = lib.kv_cache(c["target"], c["kv_heads"], c["length"], c["dim"], c["vdim"])
    if c["op"] == "shared":
        output("out", c["dtype"], c["batch"], c["heads"], c["n"], c["vdim"])
        state["members"] = array(_members(c)) if c["ragged"] or c["batch"] % c["prompts"] else None
        state["counts"] = array(_counts(c)) if c["ragged"] else None
        state["prompt"] = lib.kv_cache(c["prompts"], c["kv_heads"], c["prompt"], c["dim"], c["vdim"])
    torch.cuda.synchronize()   # torch fills on its own stream, the library reads on another
    if c["op"] != "select":
        lib.call("tensor_kv_cache_append_f16", state["cache"], t["k"], t["v"], array(lengths))
    if c["op"] == "shared":
        lib.call("tensor_kv_cache_append_f16", state["prompt"], t["prompt_k"], t["prompt_v"],
                 array(_shorter(c["prompt"], c["prompts"], c["ragged"])))
    lib.synchronize()
    state.update(t=t, result=out)


def prepare(case, seed):
    c = case
    a = _inputs(c, seed)
    state = {"case": c}
    if own:
        _prepare_own(c, a, state)
        return state

    def tell(values):
        return torch.tensor(values, device="cuda")

    if c["op"] == "select":
        state.update(a, end=tell(_end(c)))
        return state
    state["lengths"] = tell(_lengths(c))
    for name in ("k", "v"):
        state["held_" + name] = _hold(a[name], state["lengths"])
    if c["op"] == "reorder":
        state["parents"] = a["parents"].long()
    if c["op"] == "copy":
        state["source"] = tell(_sources(c))
    if c["op"] == "shared":
        state["prompt_lengths"] = tell(_shorter(c["prompt"], c["prompts"], c["ragged"]))
        for name in ("prompt_k", "prompt_v"):
            state[name] = _hold(a[name], state["prompt_lengths"])
        members, first = _members(c), 0
        place, back = [], []
        for i, m in enumerate(members):
            place.append([first + min(j, m - 1) for j in range(max(members))])
            back += [i * max(members) + j for j in range(m)]
            first += m
        state["place"], state["back"] = tell(place), tell(back)
        state["q"], state["counts"] = a["q"], tell(_counts(c))
        i = torch.arange(c["n"], device="cuda")
        state["live"] = (i < state["counts"][:, None])[:, None, :, None]
        state["out"] = torch.zeros((c["batch"], c["heads"], c["n"], c["vdim"]), device="cuda", dtype=DTYPE[c["dtype"]])
    torch.cuda.synchronize()
    return state


def _run_own(c, s):
    call, t, op = _sdk().call, s["t"], c["op"]
    if op == "select":
        call(f"tensor_beam_select_{c['dtype']}", t["logits"], t["scores"], t.get("ended"), _end(c), t["out_parents"],
             t["out_tokens"], t["out_scores"], t["out_ended"])
    elif op == "reorder":
        call("tensor_kv_cache_reorder", s["cache"], t["parents"])
        call("tensor_kv_cache_read_f16", s["cache"], t["out_k"], t["out_v"])
    elif op == "copy":
        call("tensor_kv_cache_copy", s["cache"], s["source"], s["target"])
        call("tensor_kv_cache_read_f16", s["target"], t["out_k"], t["out_v"])
    else:
        call(f"tensor_kv_cache_attention_shared_{c['dtype']}", s["prompt"], s["cache"], t["q"], s["members"],
             s["counts"], c["dim"] ** -0.5, int(c["causal"]), t["out_out"])
    return s["result"]


def run(state):
    c = state["case"]
    if own:
        return _run_own(c, state)
    return {"select": _plain_select, "reorder": _plain_reorder, "copy": _plain_copy,
            "shared": _plain_shared}[c["op"]](c, state)


# ---- what a pass cannot do without ---------------------------------------------------

def work(case):
    c, op = case, case["op"]
    if op == "select":     # every logit (of ended beams none); what is chosen is next to nothing
        live = c["groups"] * c["beams"] * (0.75 if c["ended"] else 1.0)
        return {"bytes": int(live * c["vocab"] * SIZE[c["dtype"]]) + c["groups"] * (8 * c["beams"] + 16 * c["keep"]),
                "flops": 0}
    h, d, e = c["kv_heads"], c["dim"], c["vdim"]
    lengths = _lengths(c)
    if op == "reorder":    # codes of three in five sequences in and out; then all codes in, rows out
        moved = sum(lengths) * 0.6 * (c["beams"] - 1) / c["beams"]
        return {"bytes": int((2 * moved + 3 * sum(lengths)) * h * (d + e)), "flops": 0}
    if op == "copy":       # codes of the sources in, of the target out; then codes in, rows out
        sources = _sources(c)
        read = sum(lengths[i] for i in set(sources))
        written = sum(lengths[i] for i in sources)
        return {"bytes": (read + 4 * written) * h * (d + e), "flops": 0}
    prompts = _shorter(c["prompt"], c["prompts"], c["ragged"])
    counts = _counts(c)
    pairs = 0
    on = [p for p, m in zip(prompts, _members(c)) for _ in range(m)]
    for prompt, length, n in zip(on, lengths, counts):
        # row i sees the prompt and length - n + i + 1 own tokens
        pairs += n * (prompt + length) - (n * (n - 1) // 2 if c["causal"] else 0)
    moved = (sum(prompts) + sum(lengths)) * h * (d + e) + sum(counts) * c["heads"] * (d + e) * SIZE[c["dtype"]]
    return {"bytes": moved, "flops": 2 * pairs * c["heads"] * (d + e)}


# ---- the same in 64 bits ---------------------------------------------------------------

def _held_values(x):
    """What a cache of x [H, T, D] (f64) gives back: whole blocks through their
    codes, the rest as it is."""
    h, t, d = x.shape
    n = t // BLOCK * BLOCK
    tiles = x[:, :n].reshape(h, -1, BLOCK * d)
    big = tiles.abs().max(-1, keepdim=True).values if n else tiles
    codes = torch.round(tiles * 127.0 / torch.where(big == 0, 1.0, big))
    scale = (big / 127.0).float().double()      # the scale is held in f32
    return torch.cat([(codes * scale).reshape(h, n, d), x[:, n:]], 1)


def exact(case, seed):
    c = case
    a = {n: x.double() for n, x in _inputs(c, seed).items()}
    if c["op"] == "select":
        shape = (c["groups"], c["keep"])
        out = {"scores": torch.full(shape, -math.inf, device="cuda", dtype=torch.float64)}
        for name, value in (("parents", 0), ("tokens", _end(c)), ("ended", 1)):
            out[name] = torch.full(shape, value, device="cuda", dtype=torch.int32)
        for g in range(c["groups"]):
            table = torch.log_softmax(a["logits"][g], -1) + a["scores"][g][:, None]
            if c["ended"]:
                over = a["ended"][g] != 0
                table[over] = -math.inf
                table[over, _end(c)] = a["scores"][g][over]
            score, place = torch.sort(table.reshape(-1), descending=True, stable=True)
            n = min(c["keep"], int((score > -math.inf).sum()))
            out["scores"][g, :n] = score[:n]
            out["parents"][g, :n] = (place[:n] // c["vocab"]).int()
            out["tokens"][g, :n] = (place[:n] % c["vocab"]).int()
            out["ended"][g, :n] = (place[:n] % c["vocab"] == _end(c)).int()
        return out
    lengths = _lengths(c)
    if c["op"] in ("reorder", "copy"):
        if c["op"] == "copy":
            source = _sources(c)
        else:
            source = [g * c["beams"] + int(p) for g, row in enumerate(a["parents"].tolist()) for p in row]
        out = {}
        for name, width in (("k", c["dim"]), ("v", c["vdim"])):
            out[name] = torch.zeros((len(source), c["kv_heads"], c["length"], width), device="cuda", dtype=torch.float64)
            for i, s in enumerate(source):
                out[name][i, :, :lengths[s]] = _held_values(a[name][s, :, :lengths[s]])
        return out
    out = torch.zeros((c["batch"], c["heads"], c["n"], c["vdim"]), device="cuda", dtype=torch.float64)
    group, seq = c["heads"] // c["kv_heads"], 0
    for p, (prompt, members) in enumerate(zip(_shorter(c["prompt"], c["prompts"], c["ragged"]), _members(c))):
        before = [_held_values(a["prompt_" + name][p, :, :prompt]) for name in ("k", "v")]
        for seq in range(seq, seq + members):
            length, n = lengths[seq], _counts(c)[seq]
            k, v = (torch.cat([x, _held_values(a[name][seq, :, :length])], 1) for name, x in zip(("k", "v"), before))
            hidden = torch.arange(prompt + length, device="cuda")[None, :] > \
                torch.arange(n, device="cuda")[:, None] + prompt + length - n
            for j in range(c["kv_heads"]):
                x = a["q"][seq, group * j:group * (j + 1), :n] @ k[j].t().contiguous() / math.sqrt(c["dim"])
                if c["causal"]:
                    x = x.masked_fill(hidden, -math.inf)
                out[seq, group * j:group * (j + 1), :n] = torch.softmax(x, -1) @ v[j]
        seq += 1
    return {"out": out}
