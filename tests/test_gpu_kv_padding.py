"""Padded query rows of attention over the cache and over a shared prefix: what they
hold has no effect on any bit of the rows that are there, nor on the weights."""
import ctypes

import numpy as np
import pytest

from tests import beam_model
from tests.kv_model import u32s
from tests.test_gpu_kv_attention import attend as attend_plain, compare
from tests.test_gpu_kv_cache import DTYPES
from tests.test_gpu_kv_shared import attend, pair_of, run

pytestmark = pytest.mark.gpu


def paddings(rng, q, counts):
    """The rows q with padding of several kinds."""
    there = np.arange(q.shape[2]) < np.array(counts)[:, None]
    where = np.broadcast_to(there[:, None, :, None], q.shape)
    for kind in (0.0, 30.0, 1000.0, np.nan, np.inf):
        with np.errstate(over="ignore", invalid="ignore"):
            yield kind, np.where(where, q, (kind * rng.standard_normal(q.shape)).astype(q.dtype))


def same(results):
    (_, first), *others = results
    for kind, other in others:
        for a, b in zip(first, other):
            assert (a is None and b is None) or np.array_equal(a.view(np.uint8), b.view(np.uint8)), f"padding of {kind}"


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("before,lengths,heads,n,counts", [
    (100, [40, 30, 3, 20], 4, 3, [3, 1, 0, 2]),                    # one workgroup for both
    (1500, [300, 200, 400, 100], 8, 5, [5, 2, 0, 1]),              # rows in parts
    (2500, [150] * 10, 16, 75, [75, 75, 20, 1, 0, 75, 3, 40, 75, 75]),    # tiles over the prefix
    (2000, [1500, 1300], 16, 900, [333, 900])], ids=["close", "rows", "mixed", "tiles"])
def test_over_a_prefix(sdk, before, lengths, heads, n, counts, dtype):
    kv = 2 if heads < 16 else 4
    prefix, own = pair_of(sdk, kv, (128, 128), [before], 1), pair_of(sdk, kv, (128, 128), lengths, 2)
    q = own.rng.standard_normal((len(lengths), heads, n, 128)).astype(DTYPES[dtype])
    same([(kind, [attend(prefix, own, x, None, 0.3, True, counts)]) for kind, x in paddings(own.rng, q, counts)])


@pytest.mark.parametrize("weighted", [False, True], ids=["", "weights"])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("lengths,heads,n,counts", [
    ([40, 30, 3, 20], 8, 3, [3, 1, 0, 2]), ([900, 700, 800, 100], 8, 11, [11, 2, 0, 7]),
    ([3000, 2900], 16, 700, [333, 700])], ids=["few", "rows", "tiles"])
def test_over_own_tokens(sdk, lengths, heads, n, counts, dtype, weighted):
    own = pair_of(sdk, 4, (128, 128), lengths, 3)
    q = own.rng.standard_normal((len(lengths), heads, n, 128)).astype(DTYPES[dtype])
    w0 = np.zeros((len(lengths), 4, max(lengths)), np.float32) if weighted else None
    same([(kind, attend_plain(sdk, own.cache, x, 0.3, True, counts, w0, 128)) for kind, x in paddings(own.rng, q, counts)])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_more_sequences_than_one_launch_takes(sdk, dtype):
    """Padding of other sequences than a launch's own tokens are of; whole sequences,
    groups and tiles of padding."""
    rng = np.random.default_rng(4)
    members = [0, 290, 3, 30, 0, 1]
    prefix = pair_of(sdk, 1, (32, 32), [5, 700, 64, 130, 9, 0], 5)
    own = pair_of(sdk, 1, (32, 32), [int(n) for n in rng.integers(0, 70, sum(members))], 6)
    counts = [int(c) for c in rng.integers(0, 5, sum(members))]
    counts[20:60] = [0] * 40
    counts[290:293] = [0] * 3
    run(prefix, own, dtype, 2, 4, members, causal=False, counts=counts, what="few rows")
    q = own.rng.standard_normal((sum(members), 2, 4, 32)).astype(DTYPES[dtype])
    same([(kind, [attend(prefix, own, x, members, 0.3, True, counts)]) for kind, x in paddings(own.rng, q, counts)])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_tiles_of_padding(sdk, dtype):
    """Packed tiles, and waves of them, without a row that is there, in 300 sequences."""
    rng = np.random.default_rng(7)
    prefix, own = pair_of(sdk, 2, (64, 64), [1900], 8), pair_of(sdk, 2, (64, 64), [30 + b % 5 for b in range(300)], 9)
    counts = [0 if b % 60 < 40 else int(c) for b, c in enumerate(rng.integers(0, 25, 300))]
    counts[299] = 24
    run(prefix, own, dtype, 2, 24, counts=counts, what="tiles")
    q = own.rng.standard_normal((300, 2, 24, 64)).astype(DTYPES[dtype])
    same([(kind, [attend(prefix, own, x, None, 0.3, True, counts)]) for kind, x in paddings(own.rng, q, counts)])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("batch", [40, 300])
def test_recorded(sdk, batch, dtype):
    """Two recorded calls with other paddings: each keeps its own, whatever eager calls
    with others do between the replays."""
    hip, stream = sdk.lib, ctypes.c_void_p(sdk.stream())
    rng = np.random.default_rng(10)
    prefix = pair_of(sdk, 1, (32, 32), [900], 11, capacity=1200)
    own = pair_of(sdk, 1, (32, 32), [int(n) for n in rng.integers(5, 40, batch)], 12, capacity=200)
    q = rng.standard_normal((batch, 2, 5, 32)).astype(DTYPES[dtype])
    given, runs = sdk.from_numpy(q), []
    for _ in range(2):
        counts = [int(c) for c in rng.integers(0, 6, batch)]
        out = sdk.from_numpy(np.full(q.shape, 99, q.dtype))
        call = (f"tensor_kv_cache_attention_shared_{dtype}", prefix.cache, own.cache, given, None, u32s(counts), 0.2, 0, out)
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
        runs.append((exe, counts, out))
    for replay in range(3):
        own.append(20)
        for _, _, out in runs:
            out.upload(np.full(q.shape, 99, q.dtype))
        for exe, _, _ in runs:
            assert hip.hipGraphLaunch(exe, stream) == 0
        attend(prefix, own, q, None, 0.2, False, [(b + replay) % 6 for b in range(batch)])
        model = beam_model.joined(prefix.model, own.model, [batch])
        for _, counts, out in runs:
            compare(model, q, 0.2, False, counts, out.download(), what=f"replay {replay}")
    sdk.synchronize()
    for exe, _, _ in runs:
        assert hip.hipGraphExecDestroy(exe) == 0
