"""The 8-bit key/value cache: what it holds after appends, cuts and evictions,
against the plain model (bit for bit: codes are decided exactly)."""
import ctypes

import numpy as np
import pytest

from tests.helpers import assert_bits_equal
from tests.kv_model import BLOCK, Model, u32s

pytestmark = pytest.mark.gpu

DTYPES = {"f16": np.float16, "f32": np.float32}


def rows_of(rng, shape, dtype, scale=1.0):
    """Rows with a few channels several times the others."""
    channel = np.exp(0.6 * rng.standard_normal((1, 1, 1, shape[3])))
    return (rng.standard_normal(shape) * channel * scale).astype(DTYPES[dtype])


def check_read(sdk, cache, model, what=""):
    batch, heads, dim, vdim = model.shape
    longest = max(model.length(b) for b in range(batch))
    assert cache.lengths == [model.length(b) for b in range(batch)], what
    for dtype, extra in (("f32", 0), ("f16", 3)):
        rows = longest + extra
        if rows == 0:
            continue
        k0 = np.full((batch, heads, rows, dim), 7, DTYPES[dtype])
        v0 = np.full((batch, heads, rows, vdim), -7, DTYPES[dtype])
        k, v = sdk.from_numpy(k0), sdk.from_numpy(v0)
        sdk.call(f"tensor_kv_cache_read_{dtype}", cache, k, v)
        want_k, want_v = model.read(DTYPES[dtype], rows, k0, v0)
        assert_bits_equal(k.download(), want_k, f"{what} keys {dtype}")
        assert_bits_equal(v.download(), want_v, f"{what} values {dtype}")


class Pair:
    """A cache and its model, fed alike."""

    def __init__(self, sdk, batch, heads, capacity, dim, vdim, seed=0):
        self.sdk, self.rng = sdk, np.random.default_rng(seed)
        self.cache = sdk.kv_cache(batch, heads, capacity, dim, vdim)
        self.model = Model(batch, heads, dim, vdim)

    def append(self, n, dtype="f16", counts=None, key=None, value=None):
        batch, heads, dim, vdim = self.model.shape
        key = rows_of(self.rng, (batch, heads, n, dim), dtype) if key is None else key
        value = rows_of(self.rng, (batch, heads, n, vdim), dtype) if value is None else value
        dtype = "f16" if key.dtype == np.float16 else "f32"
        self.sdk.call(f"tensor_kv_cache_append_{dtype}", self.cache, self.sdk.from_numpy(key),
                      self.sdk.from_numpy(value), None if counts is None else u32s(counts))
        self.model.append(key, value, counts)

    def truncate(self, lengths):
        self.sdk.call("tensor_kv_cache_truncate", self.cache, u32s(lengths))
        self.model.truncate(lengths)

    def check(self, what=""):
        check_read(self.sdk, self.cache, self.model, what)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("dims", [(1, 1), (16, 16), (33, 7), (64, 64), (72, 80), (100, 36), (128, 128), (192, 64),
                                  (250, 256), (256, 256)])
def test_append_and_read(sdk, dims, dtype):
    """Tokens of every kind of split: into an empty cache, within a block, up to
    its end, over several, and the same tokens one by one."""
    pair = Pair(sdk, 2, 3, 400, *dims, seed=sum(dims))
    for n in (5, 1, 58, 1, 63, 130, 6, 64):
        pair.append(n, dtype)
    pair.check(f"{dims}")


def test_append_one_by_one(sdk):
    pair, whole = Pair(sdk, 1, 2, 130, 40, 48, 1), Pair(sdk, 1, 2, 130, 40, 48, 1)
    k, v = rows_of(pair.rng, (1, 2, 130, 40), "f16"), rows_of(pair.rng, (1, 2, 130, 48), "f16")
    for t in range(130):
        pair.append(1, key=k[:, :, t:t + 1], value=v[:, :, t:t + 1])
    pair.check()
    whole.append(130, key=k, value=v)
    whole.check()
    assert pair.cache.lengths == [130]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_ragged_append(sdk, dtype):
    """Counts per sequence, none among them; the padding holds NaN and is not read."""
    pair = Pair(sdk, 5, 2, 300, 24, 40, 3)
    for counts in ([0, 1, 64, 65, 100], [100, 63, 0, 64, 27], [1, 0, 0, 0, 0], [0, 0, 0, 0, 0], [70, 64, 1, 63, 100]):
        k, v = (rows_of(pair.rng, (5, 2, 100, d), dtype) for d in (24, 40))
        for b, n in enumerate(counts):
            k[b, :, n:] = np.nan
            v[b, :, n:] = np.inf
        pair.append(100, counts=counts, key=k, value=v)
        pair.check(str(counts))


def test_many_sequences(sdk):
    """More sequences than one launch takes."""
    pair = Pair(sdk, 300, 1, 70, 16, 16, 4)
    counts = [(7 * b) % 71 for b in range(300)]
    pair.append(70, counts=counts)
    pair.check()
    pair.truncate([n // 2 for n in counts])
    pair.check()


@pytest.mark.parametrize("largest", [127.0, 126.0, 254.0, 1.0, 63.5, 65504.0, 2.0 ** -24, 127 * 2.0 ** -24, 0.0])
def test_codes_at_borders(sdk, largest):
    """Elements on and next to the borders between codes: ties go to even ones."""
    pair = Pair(sdk, 1, 1, 64, 256, 256, 5)
    with np.errstate(over="ignore"):
        n = np.arange(-127, 128)[:, None] + np.array([0.5, 0.0])
        ties = (n.reshape(-1) * largest / 127.0).astype(np.float16)
    near = np.concatenate([ties, np.nextafter(ties, np.float16(9)), np.nextafter(ties, np.float16(-9))])
    near = near[np.abs(near) <= largest] if largest else near[:1] * 0
    k = np.resize(near, (1, 1, 64, 256)).astype(np.float16)
    k[0, 0, 17, 3] = largest
    pair.append(64, key=k, value=-k[:, :, ::-1].copy())
    pair.check(str(largest))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_marked_tokens(sdk, dtype):
    """A token with an element that is no finite f16, in its key or its value, is
    marked in that head alone and leaves its block's scales as they are."""
    pair = Pair(sdk, 1, 2, 300, 20, 33, 6)
    k, v = rows_of(pair.rng, (1, 2, 200, 20), dtype), rows_of(pair.rng, (1, 2, 200, 33), dtype)
    k[0, 0, 3, 19] = np.nan
    k[0, 1, 63, 0] = np.inf
    v[0, 0, 64, 32] = -np.inf
    v[0, 1, 150, 1] = np.nan
    k[0, 0, 199, 5] = v[0, 0, 199, 5] = np.nan
    if dtype == "f32":
        k[0, 0, 70, 1] = 65520.0      # rounds to infinity
        v[0, 1, 71, 1] = 65519.0      # rounds to 65504
    pair.append(70, key=k[:, :, :70], value=v[:, :, :70])
    pair.append(130, key=k[:, :, 70:], value=v[:, :, 70:])
    pair.check()
    assert pair.model.marked[0][0].sum() == (4 if dtype == "f32" else 3)
    pair.truncate([195])
    pair.append(69, dtype)
    pair.check("cut behind a mark and filled again")
    pair.truncate([3])
    pair.append(61, dtype)
    pair.check("the marked token gone")


def test_truncate(sdk):
    pair = Pair(sdk, 3, 2, 400, 64, 48, 7)
    pair.append(390, counts=[390, 200, 64])
    for lengths in ([389, 200, 64], [384, 193, 63], [320, 130, 0], [319, 128, 0], [65, 1, 0]):
        pair.truncate(lengths)
        pair.check(str(lengths))
    pair.append(150, counts=[150, 63, 150])
    pair.check("appended behind the cut")
    pair.sdk.call("tensor_kv_cache_truncate", pair.cache, None)
    pair.model.truncate([0, 0, 0])
    pair.append(65)
    pair.check("emptied")


EVICTIONS = [   # lengths, first, recent, keep
    ([100, 64, 1, 0], 4, 16, 40), ([300, 129, 200, 63], 0, 0, 64), ([300, 129, 200, 63], 4, 60, 64),
    ([300, 299, 298, 128], 3, 10, 128), ([700, 650, 513, 300], 0, 1, 299), ([130, 70, 5, 2], 1, 0, 1),
    ([500, 400, 300, 200], 200, 100, 300), ([128, 128, 127, 64], 0, 64, 1000),
]


@pytest.mark.parametrize("case", EVICTIONS, ids=str)
@pytest.mark.parametrize("dims", [(64, 64), (40, 100), (128, 128), (256, 17)], ids=str)
def test_evict(sdk, case, dims):
    lengths, first, recent, keep = case
    batch, heads = len(lengths), 2
    pair = Pair(sdk, batch, heads, 800, *dims, seed=keep)
    k, v = (rows_of(pair.rng, (batch, heads, max(lengths), d), "f16") for d in dims)
    k[:, 0, max(lengths) // 3] = np.nan
    pair.append(max(lengths), counts=lengths, key=k, value=v)
    w = np.exp(2 * pair.rng.standard_normal((batch, heads, max(lengths) + 5))).astype(np.float32)
    w[0, 0] = np.rint(w[0, 0])                     # many equal ones
    w[0, 1, ::3], w[0, 1, 1::7], w[0, 1, 2::5], w[0, 1, ::11] = -0.0, 0.0, -1.0, -np.inf
    w[1, 0, ::2], w[1, 0, 1::6] = np.nan, np.inf
    w[2, 1] = 0.25                                  # all equal: the earliest
    tw = sdk.from_numpy(w)
    slots = min(keep, max(lengths)) + 2
    target = sdk.kv_cache(batch, heads, max(keep, 10), *dims)
    filler = Pair(sdk, batch, heads, 10, *dims)     # what the target held is dropped
    sdk.call("tensor_kv_cache_append_f16", target, sdk.from_numpy(rows_of(filler.rng, (batch, heads, 9, dims[0]), "f16")),
             sdk.from_numpy(rows_of(filler.rng, (batch, heads, 9, dims[1]), "f16")), None)
    for weights in (tw, None):
        kept0 = np.full((batch, heads, slots), 12345, np.uint32)
        w0 = np.full((batch, heads, slots), -5, np.float32)
        kept, out_w = sdk.from_numpy(kept0), sdk.from_numpy(w0)
        sdk.call("tensor_kv_cache_evict", pair.cache, weights, first, recent, keep, target,
                 out_w if weights is not None else None, kept)
        model, index = pair.model.evict(None if weights is None else w, first, recent, keep)
        for b in range(batch):
            for h in range(heads):
                kept0[b, h, :len(index[b][h])] = index[b][h]
                if weights is not None:
                    w0[b, h, :len(index[b][h])] = w[b, h, index[b][h]]
        assert_bits_equal(kept.download(), kept0, "kept")
        assert_bits_equal(out_w.download(), w0, "weights")
        check_read(sdk, target, model, f"{case} {dims}")
    pair.check("the source stays")
    # the target goes on as a cache of its own
    sdk.call("tensor_kv_cache_truncate", target, u32s([n // 2 for n in target.lengths]))
    model.truncate([model.length(b) // 2 for b in range(batch)])
    check_read(sdk, target, model, "target cut")


@pytest.mark.parametrize("dims", [(8, 8), (72, 72), (24, 120), (200, 136), (136, 64)], ids=str)
def test_evict_of_odd_groups(sdk, dims):
    """Rows of whole groups of 8 but not of 16: what is held past them is no value."""
    pair = Pair(sdk, 2, 2, 500, *dims, seed=31)
    pair.append(400, counts=[400, 333])
    w = np.exp(pair.rng.standard_normal((2, 2, 400))).astype(np.float32)
    target = sdk.kv_cache(2, 2, 200, *dims)
    sdk.call("tensor_kv_cache_evict", pair.cache, sdk.from_numpy(w), 3, 20, 200, target, None, None)
    pair.model, _ = pair.model.evict(w, 3, 20, 200)
    pair.cache = target
    pair.check(str(dims))
    pair.truncate([150, 100])
    pair.append(30)
    pair.check("cut and appended to")


def test_more_rows_than_an_int_are_refused(sdk):
    cache = sdk.kv_cache(1, 1, 10, 1)
    rows = sdk.tensor("f16", (1, 1, 2 ** 31, 1))
    ok, message = sdk.try_call("tensor_kv_cache_append_f16", cache, rows, rows, u32s([1]))
    assert ok == 0 and message == "cache append: too many tokens"
    ok, message = sdk.try_call("tensor_kv_cache_read_f16", cache, rows, None)
    assert ok == 0 and message == "cache read: too many rows"
    rows.free()


@pytest.mark.parametrize("length", [32768, 32769, 70001])
def test_evict_of_long_sequences(sdk, length):
    """Around the length up to which the weights stay in registers."""
    pair = Pair(sdk, 1, 1, length, 4, 4, 30)
    pair.append(length)
    w = np.rint(pair.rng.exponential(50, (1, 1, length))).astype(np.float32)     # many equal ones
    target = sdk.kv_cache(1, 1, 5000, 4, 4)
    for first, recent, keep in ((4, 100, 5000), (0, 0, 1), (7, 0, 4097)):
        kept = sdk.tensor("u32", (1, 1, keep))
        sdk.call("tensor_kv_cache_evict", pair.cache, sdk.from_numpy(w), first, recent, keep, target, None, kept)
        model, index = pair.model.evict(w, first, recent, keep)
        assert np.array_equal(kept.download()[0, 0], index[0][0])
        check_read(sdk, target, model)


def test_evict_of_equal_scales_keeps_codes(sdk):
    """Values that lie on the borders of the new codes (all blocks of one scale,
    the largest code gone): exact ties, decided for the even code."""
    pair = Pair(sdk, 1, 1, 256, 16, 16, 9)
    k = pair.rng.integers(-126, 127, (1, 1, 256, 16)).astype(np.float16)
    k[0, 0, ::64, 0] = 127           # each block's largest, at its first token
    pair.append(256, key=k, value=(k / 4).astype(np.float16))
    w = np.ones((1, 1, 256), np.float32)
    w[0, 0, ::64] = 0                # ... which goes
    target = sdk.kv_cache(1, 1, 252, 16, 16)
    sdk.call("tensor_kv_cache_evict", pair.cache, sdk.from_numpy(w), 0, 0, 252, target, None, None)
    model, index = pair.model.evict(w, 0, 0, 252)
    assert 0 not in index[0][0]
    check_read(sdk, target, model)
    # half of the largest remaining code: 63 of 126 is a tie
    k = np.where(pair.rng.random((1, 1, 128, 16)) < 0.5, 63, 126).astype(np.float16)
    k[0, 0, ::64, 0] = 127
    pair = Pair(sdk, 1, 1, 128, 16, 16, 9)
    pair.append(128, key=k, value=(-k * 3).astype(np.float16))
    target = sdk.kv_cache(1, 1, 126, 16, 16)
    sdk.call("tensor_kv_cache_evict", pair.cache, sdk.from_numpy(w[..., :128].copy()), 0, 0, 126, target, None, None)
    model, _ = pair.model.evict(w[..., :128], 0, 0, 126)
    assert (np.abs(model.k[0][0].blocks[0][0]) == 64).any()
    check_read(sdk, target, model)


def test_refusals(sdk):
    cache, other = sdk.kv_cache(2, 2, 100, 32, 48), sdk.kv_cache(2, 2, 50, 32, 48)
    f16 = lambda *shape: sdk.tensor("f16", shape)      # noqa: E731
    f32 = lambda *shape: sdk.tensor("f32", shape)      # noqa: E731
    k, v, q, o = f16(2, 2, 60, 32), f16(2, 2, 60, 48), f16(2, 4, 3, 32), f16(2, 4, 3, 48)
    sdk.call("tensor_kv_cache_append_f16", cache, k.upload(np.zeros(k.shape, np.float16)),
             v.upload(np.zeros(v.shape, np.float16)), None)
    host = sdk.tensor("f16", (2, 2, 60, 32), device=False)
    bad = [
        ("append", (cache, host, v, None), "rank-4 F16 device tensors"),
        ("append", (cache, k, f32(2, 2, 60, 48), None), "rank-4 F16 device tensors"),
        ("append", (cache, v, v, None), "must be [batch, kv_heads, tokens, dim]"),
        ("append", (cache, k, f16(2, 2, 59, 48), None), "must be [batch, kv_heads, tokens, dim]"),
        ("append", (cache, f16(2, 1, 60, 32), v, None), "must be [batch, kv_heads, tokens, dim]"),
        ("append", (cache, k, v, u32s([61, 0])), "a count exceeds"),
        ("append", (cache, k, v, None), "sequence 0 holds 60 of 100 tokens, no room for 60"),
        ("append", (cache, k, v, u32s([40, 41])), "sequence 1 holds 60 of 100 tokens, no room for 41"),
        ("read", (cache, None, None), "one for each output"),
        ("read", (cache, k, k), "one for each output"),
        ("read", (cache, f16(2, 2, 59, 32), None), "fewer rows than the longest"),
        ("read", (cache, k, f16(2, 2, 61, 48)), "must be [batch, kv_heads, rows, dim]"),
        ("attention", (cache, host, None, 1.0, 1, None, o), "cache attention requires rank-4 F16"),
        ("attention", (cache, q, None, float("nan"), 1, None, o), "finite scale"),
        ("attention", (cache, q, None, 1.0, 2, None, o), "causal 0 or 1"),
        ("attention", (cache, q, None, 1.0, 1, f32(2, 2, 59), o), "room for the longest"),
        ("attention", (cache, q, None, 1.0, 1, f32(2, 4, 60), o), "weights must be"),
        ("attention", (cache, q, None, 1.0, 1, f16(2, 2, 60), o), "rank-3 F32 device weights"),
        ("attention", (cache, f16(2, 3, 3, 32), None, 1.0, 1, None, f16(2, 3, 3, 48)), "a multiple of its kv_heads"),
        ("attention", (cache, q, None, 1.0, 1, None, f16(2, 4, 3, 32)), "query and output must be"),
        ("attention", (cache, q, u32s([3, 4]), 1.0, 1, None, o), "a count exceeds"),
    ]
    for op, args, message in bad:
        ok, text = sdk.try_call(f"tensor_kv_cache_{op}_f16", *args)
        assert ok == 0 and message in text, (op, message, text)
    same = sdk.kv_cache(2, 2, 100, 32, 32)
    qq = f16(2, 2, 1, 32)
    assert "an output of its own" in sdk.try_call("tensor_kv_cache_attention_f16", same, qq, None, 1.0, 1, None, qq)[1]
    for lengths in ([61, 0], [0, 61]):
        ok, text = sdk.try_call("tensor_kv_cache_truncate", cache, u32s(lengths))
        assert ok == 0 and "holds 60 tokens, not 61" in text
    w, u = f32(2, 2, 60), sdk.tensor("u32", (2, 2, 60))
    evictions = [
        ((cache, None, 0, 0, 10, cache, None, None), "another one as its target"),
        ((cache, None, 0, 0, 10, same, None, None), "must be the cache's"),
        ((cache, None, 0, 0, 0, other, None, None), "keep must be positive"),
        ((cache, None, 0, 0, 51, other, None, None), "within the target's capacity"),
        ((cache, None, 5, 6, 10, other, None, None), "no less than first + recent"),
        ((cache, None, 11, 0, 10, other, None, None), "no less than first + recent"),
        ((cache, None, 2 ** 63, 2 ** 63, 10, other, None, None), "no less than first + recent"),
        ((cache, f32(2, 2, 59), 0, 0, 10, other, None, None), "a weight for every token"),
        ((cache, u, 0, 0, 10, other, None, None), "rank-3 F32"),
        ((cache, w, 0, 0, 10, other, w, None), "distinct"),
        ((cache, None, 0, 0, 10, other, w, None), "target weights need weights"),
        ((cache, w, 0, 0, 10, other, None, w), "rank-3 U32"),
        ((cache, w, 0, 0, 10, other, None, sdk.tensor("u32", (2, 2, 9))), "a slot for every kept token"),
        ((cache, w, 0, 0, 10, other, f32(2, 2, 11), sdk.tensor("u32", (2, 2, 10))), "a slot for every kept token"),
    ]
    for args, message in evictions:
        ok, text = sdk.try_call("tensor_kv_cache_evict", *args)
        assert ok == 0 and message in text, (message, text)
    assert cache.lengths == [60, 60] and other.lengths == [0, 0]
    # empty calls do nothing and succeed
    sdk.call("tensor_kv_cache_append_f16", cache, f16(2, 2, 0, 32), f16(2, 2, 0, 48), None)
    sdk.call("tensor_kv_cache_attention_f16", cache, f16(2, 4, 0, 32), None, 1.0, 1, None, f16(2, 4, 0, 48))
    sdk.call("tensor_kv_cache_append_f16", cache, k, v, u32s([0, 0]))
    assert cache.lengths == [60, 60]


def test_calls_that_change_lengths_are_not_recorded(sdk):
    hip = sdk.lib
    hip.tensor_device_hip_stream.restype = ctypes.c_void_p
    stream = ctypes.c_void_p(hip.tensor_device_hip_stream())
    cache, other = sdk.kv_cache(1, 1, 100, 32), sdk.kv_cache(1, 1, 100, 32)
    k = sdk.from_numpy(np.ones((1, 1, 30, 32), np.float16))
    sdk.call("tensor_kv_cache_append_f16", cache, k, k, None)
    sdk.synchronize()
    graph = ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    try:
        answers = [sdk.try_call("tensor_kv_cache_append_f16", cache, k, k, None),
                   sdk.try_call("tensor_kv_cache_truncate", cache, u32s([3])),
                   sdk.try_call("tensor_kv_cache_evict", cache, None, 0, 0, 5, other, None, None)]
        with pytest.raises(Exception, match="cannot be created while a graph is recorded"):
            sdk.kv_cache(1, 1, 10, 16)
    finally:
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    if graph.value:
        assert hip.hipGraphDestroy(graph) == 0
    assert all(ok == 0 and "cannot be recorded into a graph" in text for ok, text in answers), answers
    assert cache.lengths == [30] and other.lengths == [0]


def test_offsets_past_32_bits(sdk):
    """The last heads' codes lie more than 2^32 bytes into the arrays."""
    pair = Pair(sdk, 2, 12, 1 << 20, 256, 256, 11)
    assert pair.cache.nbytes > 12 << 30
    pair.append(70, counts=[3, 70])
    pair.append(70, counts=[0, 70])
    pair.check()
    target = sdk.kv_cache(2, 12, 100, 256, 256)
    sdk.call("tensor_kv_cache_evict", pair.cache, None, 4, 10, 90, target, None, None)
    check_read(sdk, target, pair.model.evict(None, 4, 10, 90)[0])


@pytest.mark.parametrize("shape", [(65535, 1), (1, 4096), (300, 257)], ids=str)
def test_the_most_sequences_and_heads(sdk, shape):
    """Every entry point at the largest batch and head count, over three tokens."""
    batch, kv, dim = *shape, 8
    rng = np.random.default_rng(47)
    k, v = (rng.standard_normal((batch, kv, 3, dim)).astype(np.float16) for _ in range(2))
    cache, target = sdk.kv_cache(batch, kv, 64, dim), sdk.kv_cache(batch, kv, 64, dim)
    tk, tv = sdk.from_numpy(k), sdk.from_numpy(v)
    sdk.call("tensor_kv_cache_append_f16", cache, tk, tv, None)
    sdk.call("tensor_kv_cache_append_f16", cache, tk, tv, None)
    sdk.call("tensor_kv_cache_truncate", cache, u32s([3] * batch))
    out_k, out_v = sdk.tensor("f16", k.shape), sdk.tensor("f16", v.shape)
    sdk.call("tensor_kv_cache_read_f16", cache, out_k, out_v)
    assert_bits_equal(out_k.download(), k, "keys")
    assert_bits_equal(out_v.download(), v, "values")
    q = rng.standard_normal((batch, kv, 1, dim)).astype(np.float32)
    s = np.einsum("bhqd,bhtd->bht", q.astype(np.float64), k.astype(np.float64))
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    w, out = sdk.from_numpy(np.zeros((batch, kv, 3), np.float32)), sdk.tensor("f32", q.shape)
    sdk.call("tensor_kv_cache_attention_f32", cache, sdk.from_numpy(q), None, 1.0, 1, w, out)
    # scores of 8 products of up to 25 or so, and a few roundings of what is no larger than 5
    assert np.abs(out.download()[:, :, 0] - np.einsum("bht,bhtd->bhd", p, v.astype(np.float64))).max() < 2.0 ** -15
    got_w = w.download()
    assert np.abs(got_w - p).max() < 2.0 ** -17
    kept = sdk.tensor("u32", (batch, kv, 2))
    sdk.call("tensor_kv_cache_evict", cache, w, 0, 0, 2, target, None, kept)
    index = np.sort(np.argsort(-got_w.astype(np.float64), axis=-1, kind="stable")[..., :2], axis=-1)
    assert np.array_equal(kept.download(), index)
    out_k, out_v = sdk.tensor("f16", (batch, kv, 2, dim)), sdk.tensor("f16", (batch, kv, 2, dim))
    sdk.call("tensor_kv_cache_read_f16", target, out_k, out_v)
    assert_bits_equal(out_k.download(), np.take_along_axis(k, index[..., None], 2), "kept keys")
    assert_bits_equal(out_v.download(), np.take_along_axis(v, index[..., None], 2), "kept values")
    assert target.lengths == [2] * batch
