"""Attention over a prefix that sequences share and their own tokens, against the
plain model's attention over both as one sequence: outputs within the roundings that
tests/kv_model.py counts, special rows exactly."""
import ctypes
import threading

import numpy as np
import pytest

from tests import beam_model
from tests.kv_model import u32s
from tests.test_gpu_kv_attention import compare
from tests.test_gpu_kv_cache import DTYPES, Pair, rows_of
from tests.test_gpu_kv_sequences import copied

pytestmark = pytest.mark.gpu


def pair_of(sdk, heads, dims, lengths, seed, spread=1.0, capacity=None):
    pair = Pair(sdk, len(lengths), heads, capacity or max(max(lengths), 1), *dims, seed=seed)
    n = max(max(lengths), 1)
    k, v = (rows_of(pair.rng, (len(lengths), heads, n, d), "f16", spread) for d in dims)
    pair.append(n, counts=lengths, key=k, value=v)
    return pair


def equal(prefix, own):
    return [own.model.shape[0] // prefix.model.shape[0]] * prefix.model.shape[0]


def attend(prefix, own, q, members, scale, causal, counts):
    dtype = "f16" if q.dtype == np.float16 else "f32"
    sdk = own.sdk
    out = sdk.from_numpy(np.full(q.shape[:3] + (own.model.shape[3],), 99, q.dtype))
    sdk.call(f"tensor_kv_cache_attention_shared_{dtype}", prefix.cache, own.cache, sdk.from_numpy(q),
             None if members is None else u32s(members), None if counts is None else u32s(counts), scale, int(causal), out)
    return out.download()


def run(prefix, own, dtype, heads, n, members=None, causal=True, counts=None, scale=None, spread=1.0, what=""):
    batch, _, dim, _ = own.model.shape
    q = (own.rng.standard_normal((batch, heads, n, dim)) * spread).astype(DTYPES[dtype])
    if counts is not None:
        for b, c in enumerate(counts):
            q[b, :, c:] = np.nan       # padding
    scale = dim ** -0.5 if scale is None else scale
    got = attend(prefix, own, q, members, scale, causal, counts)
    model = beam_model.joined(prefix.model, own.model, equal(prefix, own) if members is None else members)
    compare(model, q, scale, causal, counts, got, what=what)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("before,length", [(1, 1), (64, 1), (63, 64), (130, 65), (1000, 5), (1, 700), (500, 129)])
def test_one_token(sdk, before, length, dtype):
    prefix = pair_of(sdk, 2, (64, 64), [before, max(1, before // 2)], 1)
    own = pair_of(sdk, 2, (64, 64), [length, length, max(1, length - 3), 1, length, max(1, length // 2)], 2)
    run(prefix, own, dtype, 8, 1, what=f"{before} {length}")
    run(prefix, own, dtype, 2, 1, causal=False, what=f"{before} {length} all seen")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("dims", [(1, 1), (8, 24), (33, 7), (32, 32), (72, 72), (96, 64), (100, 36), (128, 128), (64, 128),
                                  (192, 128), (200, 250), (256, 256)], ids=str)
def test_head_dims(sdk, dims, dtype):
    prefix = pair_of(sdk, 2, dims, [333], 3)
    own = pair_of(sdk, 2, dims, [40, 70, 33], 4)
    run(prefix, own, dtype, 6, 1, what=f"{dims} decode")
    run(prefix, own, dtype, 4, 30, what=f"{dims} chunk")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("members", [[0, 5, 1], [6, 0, 0], [0, 0, 6], [2, 2, 2], [1, 0, 5]], ids=str)
def test_groups_of_other_sizes(sdk, members, dtype):
    prefix = pair_of(sdk, 3, (64, 32), [200, 65, 128], 5)
    own = pair_of(sdk, 3, (64, 32), [10, 64, 3, 90, 1, 65], 6)
    run(prefix, own, dtype, 6, 1, members, what="decode")
    run(prefix, own, dtype, 3, 7, members, counts=[7, 3, 3, 0, 1, 7], what="ragged")
    run(prefix, own, dtype, 3, 20, members, causal=False, counts=[20, 0, 5, 20, 1, 19], what="all seen")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_many_rows(sdk, dtype):
    """Products enough for tiles over the prefix, over the own tokens, and over both."""
    prefix = pair_of(sdk, 4, (128, 128), [2500], 7)
    own = pair_of(sdk, 4, (128, 128), [150 + i for i in range(10)], 8)
    run(prefix, own, dtype, 16, 75, counts=[75, 75, 20, 75, 0, 75, 75, 1, 75, 75], what="prefix")
    prefix = pair_of(sdk, 4, (128, 128), [70, 1], 9)
    own = pair_of(sdk, 4, (128, 128), [1500, 1300], 10)
    run(prefix, own, dtype, 16, 1300, counts=[1300, 1299], what="own")
    prefix = pair_of(sdk, 4, (128, 128), [2000, 1777], 11)
    run(prefix, own, dtype, 16, 900, members=[0, 2], what="both")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_nothing_held(sdk, dtype):
    """Empty prefixes and empty sequences; a row that sees nothing is zeros."""
    prefix = pair_of(sdk, 2, (32, 32), [0, 70], 12)
    own = pair_of(sdk, 2, (32, 32), [0, 5, 0, 66], 13, capacity=70)
    run(prefix, own, dtype, 4, 1, causal=False, what="one")
    run(prefix, own, dtype, 4, 5, causal=False, what="five")
    run(prefix, own, dtype, 4, 5, counts=[0, 5, 0, 5], what="causal")
    nothing = pair_of(sdk, 2, (32, 32), [0], 14, capacity=64)
    run(nothing, own, dtype, 4, 1, causal=False, what="no prefix")
    run(prefix, pair_of(sdk, 2, (32, 32), [0, 0], 15, capacity=3), dtype, 4, 3, causal=False, what="no own tokens")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_more_rows_than_own_tokens(sdk, dtype):
    """Causal rows before a sequence's first token see the prefix alone."""
    prefix = pair_of(sdk, 2, (48, 16), [150], 16)
    own = pair_of(sdk, 2, (48, 16), [3, 0], 17, capacity=8)
    q = own.rng.standard_normal((2, 4, 8, 48)).astype(DTYPES[dtype])
    got = attend(prefix, own, q, None, 0.2, True, [8, 6])
    both = beam_model.joined(prefix.model, own.model, [2])
    # the last three rows of the first sequence see own tokens
    seen = [np.full_like(got, 99), np.full_like(got, 99)]
    seen[0][0, :, :3] = got[0, :, 5:]
    last = np.zeros_like(q)
    last[:, :, :3] = q[:, :, 5:]
    compare(both, last, 0.2, True, [3, 0], seen[0], what="own rows")
    alone = beam_model.joined(prefix.model, pair_of(sdk, 2, (48, 16), [0, 0], 18, capacity=8).model, [2])
    seen[1][0, :, :5], seen[1][1, :, :6] = got[0, :, :5], got[1, :, :6]
    compare(alone, q, 0.2, False, [5, 6], seen[1], what="prefix rows")
    assert (got[1, :, 6:] == 99).all()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_special_rows(sdk, dtype):
    """Marked tokens in the prefix or among the own tokens make the rows that see
    them NaN; queries that are not finite, zeros."""
    prefix, own = Pair(sdk, 2, 2, 100, 32, 32, 19), Pair(sdk, 4, 2, 70, 32, 32, 20)
    k, v = (rows_of(prefix.rng, (2, 2, 100, 32), "f16") for _ in range(2))
    k[1, 0, 37, 5] = np.nan
    prefix.append(100, key=k, value=v)
    k, v = (rows_of(own.rng, (4, 2, 66, 32), "f16") for _ in range(2))
    v[0, 1, 64, 3] = np.inf
    own.append(66, key=k, value=v)
    run(prefix, own, dtype, 4, 1, what="one")
    run(prefix, own, dtype, 4, 40, what="many")
    run(prefix, own, dtype, 4, 2, scale=0.0, what="scale 0")
    run(prefix, own, dtype, 4, 2, scale=-0.7, what="scale below 0")
    q = own.rng.standard_normal((4, 2, 3, 32)).astype(DTYPES[dtype])
    q[0, 0, 0, 0], q[1, 1, 1, 4] = np.inf, np.nan
    got = attend(prefix, own, q, None, 0.3, False, None)
    model = beam_model.joined(prefix.model, own.model, [2, 2])
    want, tol, _, _ = model.attention(q, 0.3, False)
    there = np.ones((4, 2, 3), bool)
    there[0, 0, 0] = there[1, 1, 1] = False
    g, w, t = (np.nan_to_num(x[there].astype(np.float64)) for x in (got, want, tol))
    assert (np.abs(g - w) <= t).all()
    # what attention over the same tokens in one cache gives
    one = Pair(sdk, 4, 2, 200, 32, 32, 21)
    for b in range(4):
        one.model.k[b] = model.k[b]
    sdk.call("tensor_kv_cache_copy", prefix.cache, u32s([0, 0, 1, 1]), one.cache)
    sdk.call("tensor_kv_cache_append_f16", one.cache, sdk.from_numpy(k), sdk.from_numpy(v), None)
    out = sdk.tensor(dtype, (4, 2, 3, 32))
    sdk.call(f"tensor_kv_cache_attention_{dtype}", one.cache, sdk.from_numpy(q), None, 0.3, 0, None, out)
    alike = out.download()
    assert np.array_equal(np.isnan(got[~there]), np.isnan(alike[~there]))
    assert np.array_equal(np.nan_to_num(got[~there]), np.nan_to_num(alike[~there]))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("spreads", [(1.0, 60.0), (60.0, 1.0), (0.001, 30.0), (30.0, 0.001)], ids=str)
def test_maxima_in_either(sdk, spreads, dtype):
    """The largest scores, and the largest values, in the prefix or in the own tokens."""
    prefix = pair_of(sdk, 2, (64, 64), [300], 22, spreads[0])
    own = pair_of(sdk, 2, (64, 64), [200, 100], 23, spreads[1])
    run(prefix, own, dtype, 4, 3, spread=2.0, what=f"{spreads}")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_many_sequences(sdk, dtype):
    """More prefixes, and more sequences, than one launch takes."""
    rng = np.random.default_rng(24)
    prefix = pair_of(sdk, 1, (16, 16), [int(n) for n in rng.integers(0, 80, 270)], 25)
    members = [int(m) for m in rng.integers(0, 3, 270)]
    members[0] += max(0, 300 - sum(members))
    own = pair_of(sdk, 1, (16, 16), [int(n) for n in rng.integers(1, 70, sum(members))], 26)
    run(prefix, own, dtype, 2, 1, members)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("dims", [(1, 1), (8, 24), (33, 7), (32, 32), (72, 72), (96, 64), (100, 36), (128, 128), (64, 128),
                                  (192, 128), (200, 250), (256, 256)], ids=str)
def test_head_dims_on_a_longer_prefix(sdk, dims, dtype):
    prefix = pair_of(sdk, 2, dims, [1400, 130], 60)
    own = pair_of(sdk, 2, dims, [40, 70, 33, 128], 61)
    run(prefix, own, dtype, 6, 1, what=f"{dims} decode")
    run(prefix, own, dtype, 4, 19, members=[3, 1], counts=[19, 5, 0, 18], what=f"{dims} chunk")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_many_short_sequences(sdk, dtype):
    """More sequences than one launch takes, of few tokens, on prefixes of several and none."""
    rng = np.random.default_rng(62)
    prefix = pair_of(sdk, 1, (16, 32), [int(n) for n in rng.integers(0, 200, 40)], 63)
    members = [p % 2 * 13 for p in range(40)]
    members[7] += 30
    own = pair_of(sdk, 1, (16, 32), [int(n) for n in rng.integers(0, 70, 290)], 64)
    run(prefix, own, dtype, 3, 1, members, causal=False)
    run(prefix, own, dtype, 2, 3, members, causal=False, counts=[int(c) for c in rng.integers(0, 4, 290)])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("before,room", [([900, 650], (1000, 400)), ([250, 100], (330, 300))], ids=str)
def test_recorded(sdk, before, room, dtype):
    """Two recorded calls share nothing: replays follow the caches while eager calls
    take scratch memory in between."""
    hip, stream = sdk.lib, ctypes.c_void_p(sdk.stream())
    prefix = pair_of(sdk, 2, (64, 64), before, 27, capacity=room[0])
    own = pair_of(sdk, 2, (64, 64), [30, 20, 64, 1], 28, capacity=room[1])
    rng = np.random.default_rng(29)
    qs = [rng.standard_normal((4, 4, n, 64)).astype(DTYPES[dtype]) for n in (1, 5)]
    outs, runs = [], []
    for q in qs:
        out = sdk.from_numpy(np.full(q.shape, 99, q.dtype))
        call = (f"tensor_kv_cache_attention_shared_{dtype}", prefix.cache, own.cache, sdk.from_numpy(q), None, None,
                0.125, 1, out)
        sdk.call(*call)
        sdk.synchronize()
        graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
        assert hip.hipStreamBeginCapture(stream, 2) == 0
        try:
            sdk.call(*call)
        finally:
            assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
        assert hip.hipGraphDestroy(graph) == 0
        outs.append(out)
        runs.append((exe, call))
    for replay in range(3):
        own.append(70)
        prefix.append(20)
        for out in outs:
            out.upload(np.full(out.shape, 99, DTYPES[dtype]))
        for exe, _ in runs:
            assert hip.hipGraphLaunch(exe, stream) == 0
        run(prefix, own, dtype, 8, 3, what="eager")
        model = beam_model.joined(prefix.model, own.model, [2, 2])
        for q, out in zip(qs, outs):
            compare(model, q, 0.125, True, None, out.download(), what=f"replay {replay}")
    sdk.synchronize()
    for exe, _ in runs:
        assert hip.hipGraphExecDestroy(exe) == 0


def remembered(prefix):
    """The prefix's model with its exact values worked out once."""
    for heads in prefix.model.k + prefix.model.v:
        for head in heads:
            exact = head.held()
            head.held = lambda exact=exact: exact


@pytest.mark.parametrize("dims,tokens,dtype", [((128, 96), 16300, "f16"), ((64, 64), 32800, "f16"), ((200, 256), 8100, "f16"),
                                               ((64, 128), 22000, "f32")], ids=str)
def test_many_rows_on_a_long_prefix(sdk, dims, tokens, dtype):
    """Products enough for tiles over the prefix beside few rows over own tokens."""
    prefix = pair_of(sdk, 1, dims, [tokens], 34)
    remembered(prefix)
    own = pair_of(sdk, 1, dims, [(37 * b) % 200 for b in range(40)], 35)
    run(prefix, own, dtype, 2, 16, causal=False, counts=[16 if b % 5 else b % 17 for b in range(40)])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("dims", [(64, 64), (40, 33)], ids=str)
def test_few_rows_on_a_long_prefix(sdk, dims, dtype):
    """Many parts of few rows, and of more rows."""
    prefix = pair_of(sdk, 1, dims, [30000], 36)
    remembered(prefix)
    own = pair_of(sdk, 1, dims, [300, 20, 0, 64], 37)
    run(prefix, own, dtype, 4, 1, causal=False, counts=[1, 1, 0, 1], what="few")
    own = pair_of(sdk, 1, dims, [300 + i for i in range(20)], 38)
    run(prefix, own, dtype, 2, 13, counts=[13 - i % 4 for i in range(20)], what="more")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("dims", [(33, 7), (64, 64), (72, 96), (128, 128), (160, 192), (256, 256)], ids=str)
def test_short_own_tokens_of_many(sdk, dims, dtype):
    """Sequences enough to fill the chip, of 0 to 512 own tokens each."""
    rng = np.random.default_rng(39)
    prefix = pair_of(sdk, 4, dims, [100, 1, 65], 40)
    own = pair_of(sdk, 4, dims, [0, 512] + [int(n) for n in rng.integers(0, 513, 68)], 41)
    members = [30, 0, 40]
    run(prefix, own, dtype, 12, 1, members, causal=False, what="one")
    counts = [int(c) for c in rng.integers(0, 7, 70)]
    own = pair_of(sdk, 4, dims, [int(n) for n in rng.integers(6, 513, 70)], 42)
    run(prefix, own, dtype, 16, 6, members, counts=counts, what="six")


def test_codes_past_the_caches(sdk):
    """Lengths for which codes are read as a stream."""
    dims = (128, 128)
    some = pair_of(sdk, 1, dims, [4000, 70, 1, 64], 43)
    own = Pair(sdk, 200, 1, 4000, *dims, seed=44)
    source = [0] + [1 + b % 3 for b in range(199)]
    sdk.call("tensor_kv_cache_copy", some.cache, u32s(source), own.cache)
    own.model = copied(some.model, source, own.model)
    prefix = pair_of(sdk, 1, dims, [150, 3], 45)
    for dtype in ("f16", "f32"):
        run(prefix, own, dtype, 2, 1, [150, 50], what=dtype)


def test_threads_share_a_prefix(sdk):
    prefix = pair_of(sdk, 2, (64, 64), [200, 90], 46)
    errors = []

    def work(seed):
        try:
            own = pair_of(sdk, 2, (64, 64), [60, 3, 64, 5], seed, capacity=100)
            for i in range(5):
                own.append(1)
                run(prefix, own, ("f16", "f32")[i % 2], 4, 1 + i % 3, what=f"thread {seed}")
        except BaseException as e:      # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(50 + s,)) for s in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]


def test_refusals(sdk):
    prefix = pair_of(sdk, 2, (16, 32), [10, 20], 30)
    own = pair_of(sdk, 2, (16, 32), [5, 6, 7, 8], 31)
    q, out = sdk.tensor("f16", (4, 4, 2, 16)), sdk.tensor("f16", (4, 4, 2, 32))
    host = sdk.tensor("f16", (4, 4, 2, 16), device=False)

    def refuse(what, p=prefix, c=own, q=q, members=None, counts=None, scale=1.0, causal=1, out=out, dtype="f16"):
        ok, message = sdk.try_call(f"tensor_kv_cache_attention_shared_{dtype}", p and p.cache, c and c.cache, q, members,
                                   counts, scale, causal, out)
        assert ok == 0 and message.startswith(what), message

    first = "shared attention requires a prefix and another cache"
    refuse(first, p=None)
    refuse(first, c=None)
    refuse(first, p=own)
    kinds = "shared attention requires rank-4 F16 device tensors"
    refuse(kinds, q=None)
    refuse(kinds, q=host)
    refuse(kinds, out=None)
    refuse(kinds, q=sdk.tensor("f16", (4, 4, 32)))
    refuse(kinds, scale=float("nan"))
    refuse(kinds, causal=2)
    refuse("shared attention requires rank-4 F32 device tensors", dtype="f32")
    refuse("shared attention: the prefix's heads", p=pair_of(sdk, 1, (16, 32), [3], 32))
    refuse("shared attention: the prefix's heads", p=pair_of(sdk, 2, (17, 32), [3], 32))
    refuse("shared attention: the prefix's heads", p=pair_of(sdk, 2, (16, 31), [3], 32))
    shapes = "shared attention: query and output must be"
    refuse(shapes, q=sdk.tensor("f16", (4, 3, 2, 16)))
    refuse(shapes, q=sdk.tensor("f16", (3, 4, 2, 16)))
    refuse(shapes, q=sdk.tensor("f16", (4, 4, 3, 16)))
    refuse(shapes, out=sdk.tensor("f16", (4, 4, 2, 16)))
    refuse("shared attention: a count exceeds", counts=u32s([0, 1, 2, 3]))
    refuse("shared attention: 5 sequences on the prefixes, the cache has 4", members=u32s([2, 3]))
    refuse("shared attention: 4294967299 sequences on the prefixes", members=u32s([4, 2 ** 32 - 1]))
    refuse("shared attention: 3 sequences in equal groups", p=pair_of(sdk, 2, (16, 32), [1, 1, 1], 33))
    none = sdk.tensor("f16", (4, 4, 0, 16)), sdk.tensor("f16", (4, 4, 0, 32))
    sdk.call("tensor_kv_cache_attention_shared_f16", prefix.cache, own.cache, none[0], None, None, 1.0, 1, none[1])
    prefix.check()
    own.check()
