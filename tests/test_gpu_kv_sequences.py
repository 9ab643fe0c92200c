"""Sequences of the 8-bit key/value cache copied and reordered: what the caches then
hold, bit for bit, and what goes on from there."""
import copy
import ctypes
import threading

import numpy as np
import pytest

from tests.kv_model import Model, u32s
from tests.test_gpu_kv_attention import run as attend_like_the_model
from tests.test_gpu_kv_cache import Pair, rows_of

pytestmark = pytest.mark.gpu

KEEP = 2 ** 32 - 1


def copied(model, source, target):
    """The target's model after a copy."""
    new = copy.deepcopy(target)
    for b, s in enumerate(source):
        if s == KEEP:
            continue
        for part in ("k", "v", "marked"):
            getattr(new, part)[b] = copy.deepcopy(getattr(model, part)[s])
    return new


def filled(sdk, batch, heads, capacity, dims, lengths, seed=0, marks=False):
    pair = Pair(sdk, batch, heads, capacity, *dims, seed=seed)
    n = max(max(lengths), 1)
    k, v = (rows_of(pair.rng, (batch, heads, n, d), "f16") for d in dims)
    if marks:
        k[pair.rng.random(k.shape) < 0.002] = np.nan
        v[pair.rng.random(v.shape) < 0.002] = np.inf
    pair.append(n, counts=lengths, key=k, value=v)
    return pair


@pytest.mark.parametrize("dims", [(1, 1), (16, 16), (33, 7), (64, 64), (72, 80), (128, 128), (250, 256)], ids=str)
def test_copies(sdk, dims):
    """Lengths from none to several blocks, into places that held more, less or
    nothing; the rest stays."""
    lengths = [0, 1, 63, 64, 65, 130, 256, 300]
    a = filled(sdk, 8, 3, 300, dims, lengths, 1, marks=True)
    b = filled(sdk, 6, 3, 420, dims, [300, 0, 70, 64, 129, 10], 2, marks=True)
    for source in ([7, 6, KEEP, 5, 5, 0], [KEEP, KEEP, 3, 4, 2, 1], [KEEP] * 6, [1] * 6):
        sdk.call("tensor_kv_cache_copy", a.cache, u32s(source), b.cache)
        b.model = copied(a.model, source, b.model)
        b.check(str(source))
    a.check("the source")
    # both go on by themselves
    for pair in (a, b):
        pair.append(70, counts=[min(70, pair.cache.sdk.lib.tensor_kv_cache_capacity(pair.cache.handle) - n)
                                for n in pair.cache.lengths])
        pair.check("appended")
        pair.truncate([n // 2 for n in pair.cache.lengths])
        pair.check("cut")


def test_copies_within_a_cache(sdk):
    pair = filled(sdk, 7, 2, 200, (24, 40), [130, 7, 64, 0, 199, 20, 65], 3, marks=True)
    for source in ([KEEP, 0, KEEP, 0, KEEP, KEEP, 0], [KEEP, KEEP, 2, KEEP, 2, 5, KEEP], [4, 4, 4, 4, 4, 4, 4]):
        sdk.call("tensor_kv_cache_copy", pair.cache, u32s(source), pair.cache)
        pair.model = copied(pair.model, source, pair.model)
        pair.check(str(source))
    pair.append(1)
    pair.check()


def test_copies_of_many_sequences(sdk):
    """More sequences than one launch takes, and launches with nothing to do."""
    lengths = [(11 * b) % 140 for b in range(300)]
    a = filled(sdk, 300, 1, 140, (16, 16), lengths, 4)
    b = filled(sdk, 600, 1, 141, (16, 16), [(7 * b) % 90 for b in range(600)], 5)
    source = [(13 * b) % 300 if b % 3 else KEEP for b in range(256)] + [KEEP] * 256 + [b % 300 for b in range(88)]
    sdk.call("tensor_kv_cache_copy", a.cache, u32s(source), b.cache)
    b.model = copied(a.model, source, b.model)
    b.check()


def reordered(model, parents):
    groups, beams = parents.shape
    source = [g * beams + (int(p) if p < beams else i) for g in range(groups) for i, p in enumerate(parents[g])]
    return copied(model, source, model)


@pytest.mark.parametrize("dims", [(1, 1), (16, 48), (33, 7), (64, 64), (128, 128), (250, 256)], ids=str)
@pytest.mark.parametrize("length", [1, 63, 64, 65, 200])
def test_reorders(sdk, length, dims):
    """Copies, exchanges, cycles and chains, in groups of other lengths."""
    lengths = [length] * 5 + [0] * 5 + [length // 2] * 5
    pair = filled(sdk, 15, 2, 210, dims, lengths, length, marks=True)
    for order in ([0, 0, 0, 0, 0], [1, 0, 2, 4, 3], [1, 2, 3, 4, 0], [4, 4, 1, 0, 2], [0, 1, 2, 3, 4], [2, 1, KEEP, 5, 9]):
        parents = np.array([order, order[::-1], np.roll(order, 2)], np.uint32)
        sdk.call("tensor_kv_cache_reorder", pair.cache, sdk.from_numpy(parents))
        pair.model = reordered(pair.model, parents)
        pair.check(str(order))
    pair.append(3)
    pair.check("appended")


@pytest.mark.parametrize("beams", [1, 2, 3, 4, 7, 8, 9, 16, 17, 31, 32, 33, 63, 64])
def test_reorders_of_many_beams(sdk, beams):
    groups = 3
    pair = filled(sdk, groups * beams, 1, 100, (32, 16), [100] * beams + [37] * beams + [64] * beams, beams)
    rng = np.random.default_rng(beams)
    for parents in (rng.integers(0, beams, (groups, beams)), np.stack([rng.permutation(beams) for _ in range(groups)])):
        parents = parents.astype(np.uint32)
        sdk.call("tensor_kv_cache_reorder", pair.cache, sdk.from_numpy(parents))
        pair.model = reordered(pair.model, parents)
        pair.check()


def test_reorder_of_many_groups(sdk):
    pair = filled(sdk, 1200, 1, 70, (16, 16), [70] * 600 + [3] * 600, 6)
    parents = np.random.default_rng(6).integers(0, 4, (300, 4)).astype(np.uint32)
    sdk.call("tensor_kv_cache_reorder", pair.cache, sdk.from_numpy(parents))
    pair.model = reordered(pair.model, parents)
    pair.check()


def test_recorded_reorder(sdk):
    """Replays follow the parents and the lengths; eager calls lie in between."""
    hip, stream = sdk.lib, ctypes.c_void_p(sdk.stream())
    pair = filled(sdk, 8, 2, 300, (64, 32), [60] * 8, 7)
    rng = np.random.default_rng(8)
    parents = sdk.from_numpy(np.zeros((2, 4), np.uint32))
    call = ("tensor_kv_cache_reorder", pair.cache, parents)
    orders = rng.integers(0, 4, (5, 2, 4)).astype(np.uint32)
    parents.upload(orders[4])
    sdk.call(*call)
    pair.model = reordered(pair.model, orders[4])
    graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    try:
        sdk.call(*call)
        ok, message = sdk.try_call("tensor_kv_cache_copy", pair.cache, u32s([0] + [KEEP] * 7), pair.cache)
        assert ok == 1      # (the sequence itself: nothing to do)
        ok, message = sdk.try_call("tensor_kv_cache_copy", pair.cache, u32s([1] + [KEEP] * 7), pair.cache)
        assert ok == 0 and message.startswith("cache copy changes the cache's lengths")
    finally:
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
    pair.check("recorded")
    for replay in range(4):
        parents.upload(orders[replay])
        assert hip.hipGraphLaunch(exe, stream) == 0
        pair.model = reordered(pair.model, orders[replay])
        pair.check(f"replay {replay}")
        pair.append(50)
        attend_like_the_model(pair, "f16", 4, 1, what=f"replay {replay}")
    sdk.synchronize()
    assert hip.hipGraphExecDestroy(exe) == 0
    assert hip.hipGraphDestroy(graph) == 0


def test_refusals_leave_the_caches(sdk):
    a = filled(sdk, 3, 2, 100, (16, 32), [100, 40, 40], 9)
    b = filled(sdk, 4, 2, 90, (16, 32), [10, 20, 30, 40], 10)
    other = [filled(sdk, 4, *s, [1] * 4, 11) for s in ((1, 100, (16, 32)), (2, 100, (17, 32)), (2, 100, (16, 31)))]
    for call, what in (
            (("tensor_kv_cache_copy", a.cache, None, b.cache), "cache copy requires a cache, source sequences"),
            (("tensor_kv_cache_copy", a.cache, u32s([3, 0, 0, 0]), b.cache), "cache copy: sequence 3 of 3"),
            (("tensor_kv_cache_copy", a.cache, u32s([1, 1, 2, 0]), b.cache),
             "cache copy: sequence 0 holds 100 tokens, the target has room for 90"),
            (("tensor_kv_cache_copy", a.cache, u32s([1, 2, KEEP]), a.cache),
             "cache copy: sequence 1 is copied from and to within one cache"),
            (("tensor_kv_cache_reorder", a.cache, sdk.from_numpy(np.zeros((1, 3), np.uint32))),
             "cache reorder: the sequences of group 0 are not of one length"),
            (("tensor_kv_cache_reorder", a.cache, sdk.from_numpy(np.zeros((1, 3), np.int32))),
             "cache reorder requires rank-2 U32 device parents"),
            (("tensor_kv_cache_reorder", a.cache, sdk.from_numpy(np.zeros(3, np.uint32))),
             "cache reorder requires rank-2 U32 device parents"),
            (("tensor_kv_cache_reorder", a.cache, sdk.from_numpy(np.zeros((1, 3), np.uint32), device=False)),
             "cache reorder requires rank-2 U32 device parents"),
            (("tensor_kv_cache_reorder", a.cache, sdk.from_numpy(np.zeros((1, 2), np.uint32))),
             "cache reorder: parents must be"),
            (("tensor_kv_cache_reorder", a.cache, sdk.from_numpy(np.zeros((0, 3), np.uint32))),
             "cache reorder: parents must be")):
        ok, message = sdk.try_call(*call)
        assert ok == 0 and message.startswith(what), message
    for c in other:
        ok, message = sdk.try_call("tensor_kv_cache_copy", a.cache, u32s([1] * 4), c.cache)
        assert ok == 0 and message.startswith("cache copy: the target's heads and dimensions"), message
        c.check()
    a.check()
    b.check()


def test_copy_past_the_caches(sdk):
    """More than 96 MB of codes: what the target's sequences hold is what the sources do."""
    a = Pair(sdk, 2, 1, 8300, 256, 256, 12)
    a.append(8300, counts=[8300, 8211])
    target = sdk.kv_cache(26, 1, 8320, 256, 256)
    source = [b % 2 for b in range(25)] + [KEEP]
    sdk.call("tensor_kv_cache_copy", a.cache, u32s(source), target)
    assert target.lengths == [(8300, 8211)[s] if s != KEEP else 0 for s in source]
    held = []
    for cache, batch in ((a.cache, 2), (target, 26)):
        k, v = (sdk.from_numpy(np.full((batch, 1, 8300, 256), 7, np.float16)) for _ in range(2))
        sdk.call("tensor_kv_cache_read_f16", cache, k, v)
        held.append([x.download().view(np.uint16) for x in (k, v)])
    for of, to in zip(*held):
        for b, s in enumerate(source[:25]):
            assert np.array_equal(to[b], of[s]), b
        assert (to[25].view(np.float16) == 7).all()


def test_threads(sdk):
    """Copies between two caches in both directions at once, reorders and reads among
    them: all end, and of sequences alike every one stays what it is."""
    pairs = [filled(sdk, 4, 2, 200, (64, 32), [130] * 4, 13) for _ in range(2)]
    first = [KEEP, 0, KEEP, 0]
    for pair in pairs:
        sdk.call("tensor_kv_cache_copy", pair.cache, u32s([KEEP, 0, 0, 0]), pair.cache)
        pair.model = copied(pair.model, [KEEP, 0, 0, 0], pair.model)
    errors = []

    def work(i):
        try:
            a, b = pairs[i % 2], pairs[1 - i % 2]
            parents = sdk.from_numpy(np.array([[3, 2, 1, 0]], np.uint32))
            for _ in range(40):
                sdk.call("tensor_kv_cache_copy", a.cache, u32s(first), b.cache)
                sdk.call("tensor_kv_cache_reorder", b.cache, parents)
            a.check(f"thread {i}")
        except BaseException as e:      # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
    for pair in pairs:
        pair.check()
