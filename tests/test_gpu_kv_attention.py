"""Attention over the 8-bit key/value cache against the plain model: outputs
within the roundings that tests/kv_model.py counts, special rows exactly."""
import ctypes
import threading

import numpy as np
import pytest

from tests.kv_model import Model, u32s
from tests.test_gpu_kv_cache import DTYPES, Pair, check_read, rows_of

pytestmark = pytest.mark.gpu


def attend(sdk, cache, q, scale, causal, counts=None, weights=None, vdim=None):
    """(out with 99 where it was not written, weights)."""
    dtype = "f16" if q.dtype == np.float16 else "f32"
    out = sdk.from_numpy(np.full(q.shape[:3] + (vdim,), 99, q.dtype))
    w = None if weights is None else sdk.from_numpy(weights)
    sdk.call(f"tensor_kv_cache_attention_{dtype}", cache, sdk.from_numpy(q),
             None if counts is None else u32s(counts), scale, int(causal), w, out)
    return out.download(), None if w is None else w.download()


def compare(model, q, scale, causal, counts, got, w0=None, got_w=None, what=""):
    want, tol, add, add_tol = model.attention(q, scale, causal, counts)
    batch, n = q.shape[0], q.shape[2]
    got = got.astype(np.float64)
    for b in range(batch):
        count = n if counts is None else counts[b]
        assert (got[b, :, count:] == 99).all(), f"{what}: padded rows of {b} were written"
        g, w, t = got[b, :, :count], want[b, :, :count], tol[b, :, :count]
        assert np.array_equal(np.isnan(g), np.isnan(w)), f"{what}: NaN rows of {b}"
        g, w = np.nan_to_num(g), np.nan_to_num(w)
        over = np.abs(g - w) > t
        assert not over.any(), (f"{what}: {over.sum()} outputs of {b} off, worst "
                                f"{(np.abs(g - w) / np.maximum(t, 1e-300)).max():.3g} of the bound")
    if got_w is not None:
        t = add.shape[2]
        off = np.abs(got_w[..., :t] - (w0[..., :t] + add))
        bound = add_tol + 2.0 ** -23 * (np.abs(w0[..., :t]) + add) + 1e-30
        assert (off <= bound).all(), f"{what}: weights off, worst {(off / bound).max():.3g} of the bound"
        assert np.array_equal(got_w[..., t:], w0[..., t:]), f"{what}: weights behind the tokens"
        for b in range(batch):
            n_b = model.length(b)
            assert np.array_equal(got_w[b, :, n_b:], w0[b, :, n_b:]), f"{what}: weights behind sequence {b}"


def run(pair, dtype, heads, n, causal=True, counts=None, weighted=False, scale=None, what="", spread=1.0):
    batch, kv, dim, vdim = pair.model.shape
    q = (pair.rng.standard_normal((batch, heads, n, dim)) * spread).astype(DTYPES[dtype])
    scale = dim ** -0.5 if scale is None else scale
    w0 = None
    if weighted:
        longest = max(pair.model.length(b) for b in range(batch))
        w0 = pair.rng.random((batch, kv, longest + 2)).astype(np.float32)
    got, got_w = attend(pair.sdk, pair.cache, q, scale, causal, counts, w0, vdim)
    compare(pair.model, q, scale, causal, counts, got, w0, got_w, what)


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("length", [1, 2, 63, 64, 65, 128, 130, 577, 1000])
def test_one_token(sdk, length, dtype, weighted):
    pair = Pair(sdk, 2, 2, 1000, 64, 64, length)
    pair.append(length, counts=[length, max(1, length // 3)])
    run(pair, dtype, 8, 1, weighted=weighted, what=f"{length}")
    run(pair, dtype, 2, 1, causal=False, weighted=weighted, what=f"{length} all seen")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("dims", [(1, 1), (8, 24), (16, 16), (33, 7), (32, 32), (72, 72), (80, 80), (96, 64), (100, 36),
                                  (128, 128), (64, 128), (192, 128), (200, 250), (256, 256)], ids=str)
def test_head_dims(sdk, dims, dtype):
    pair = Pair(sdk, 1, 2, 400, *dims, seed=sum(dims))
    pair.append(333)
    run(pair, dtype, 6, 1, weighted=True, what=f"{dims} decode")
    run(pair, dtype, 6, 45, weighted=True, what=f"{dims} chunk")
    run(pair, dtype, 2, 150, causal=False, weighted=True, what=f"{dims} all seen")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("shape", [   # kv heads, query heads, length, n
    (1, 1, 40, 40), (1, 7, 100, 3), (2, 16, 300, 5), (3, 3, 190, 64), (2, 6, 257, 257), (1, 4, 520, 130),
    (4, 4, 129, 17), (1, 32, 700, 2), (2, 4, 33, 50), (1, 3, 5, 200), (1, 2, 700, 260)], ids=str)
def test_chunks(sdk, shape, dtype):
    """Rows that end a sequence, among them more rows than tokens (the first see
    nothing and are zeros)."""
    kv, heads, length, n = shape
    pair = Pair(sdk, 1, kv, length, 64, 80, n)
    pair.append(length)
    run(pair, dtype, heads, n, weighted=True, what="causal")
    run(pair, dtype, heads, n, causal=False, what="all seen")


# kv heads, query heads, length, n, dim, value dim: enough products for the kernel
# of 128-row tiles, in few row groups (parts of the keys) and in many (none)
TILES = [(1, 2, 17000, 600, 128, 128), (1, 3, 16448, 470, 120, 100), (2, 2, 21000, 1000, 64, 64),
         (1, 1, 41000, 1000, 64, 40), (1, 2, 50001, 830, 20, 32), (1, 2, 20010, 700, 80, 96),
         (1, 1, 21000, 650, 192, 160), (1, 2, 9000, 601, 256, 200), (64, 64, 1300, 512, 32, 32),
         (32, 64, 641, 641, 64, 64), (8, 16, 2100, 2100, 33, 50)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", TILES, ids=str)
def test_tiles(sdk, shape, causal):
    kv, heads, length, n, dim, vdim = shape
    pair = Pair(sdk, 2 if kv == 64 else 1, kv, length, dim, vdim, n)
    pair.append(length)
    run(pair, "f16", heads, n, causal=causal, weighted=True, what="f16")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", TILES[:3] + TILES[4:8] + TILES[9:], ids=str)
def test_tiles_without_weights(sdk, shape, causal):
    kv, heads, length, n, dim, vdim = shape
    pair = Pair(sdk, 1, kv, length, dim, vdim, n + 1)
    pair.append(length)
    run(pair, "f16", heads, n, causal=causal, what="f16")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", [(1, 2, 30000, 1001, 128, 128), (1, 2, 40010, 1000, 80, 96), (2, 2, 50000, 1150, 64, 60),
                                   (1, 4, 64000, 1000, 30, 17), (64, 64, 1700, 1024, 32, 32)], ids=str)
def test_tiles_f32(sdk, shape, causal):
    kv, heads, length, n, dim, vdim = shape
    pair = Pair(sdk, 2 if kv == 64 else 1, kv, length, dim, vdim, n)
    pair.append(length)
    run(pair, "f32", heads, n, causal=causal, weighted=True, what="f32")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_tiles_ragged(sdk, dtype):
    """Sequences of other lengths and row counts in one call, one empty, one whose
    rows are more than its tokens, with marked tokens, zero and far value scales and
    query rows that are not finite."""
    long = 70000 if dtype == "f32" else 30000
    pair = Pair(sdk, 4, 1, long, 64, 64, 31)
    k = rows_of(pair.rng, (4, 1, long, 64), "f16")
    v = rows_of(pair.rng, (4, 1, long, 64), "f16")
    v[:, :, 128:192] = 0
    v[:, :, 640:704] *= np.float16(2.0 ** -12)
    v[:, :, 704:768] *= np.float16(64.0)
    lengths = [long, 6400, 0, 300]
    k[0, 0, long - 700, 3] = np.nan       # the first rows do not see it
    v[1, 0, 6399, 0] = np.inf             # the last row's own token
    k[3, 0, 299, 9] = np.nan
    pair.append(long, counts=lengths, key=k, value=v)
    n, counts = 1000, [1000, 700, 5, 900]
    run(pair, dtype, 3, n, counts=counts, weighted=True, what="causal")
    run(pair, dtype, 3, n, counts=counts, causal=False, what="all seen")
    q = pair.rng.standard_normal((4, 3, n, 64)).astype(DTYPES[dtype])
    q[0, 0, 0, 3], q[1, 1, 100, 0], q[3, 2, 899, 39] = np.nan, np.inf, -np.inf
    got, _ = attend(sdk, pair.cache, q, 0.2, True, counts, None, 64)
    assert (got[0, 0, 0] == 0).all() and (got[1, 1, 100] == 0).all() and (got[3, 2, 899] == 0).all()
    good = np.isfinite(q).all(-1)
    clean = np.where(np.isfinite(q), q, 0)
    want, tol, _, _ = pair.model.attention(clean, 0.2, True, counts)
    good &= ~np.isnan(want).any(-1)
    assert (np.abs(got.astype(np.float64) - want) <= tol)[good].all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_tiles_scales(sdk, scale):
    pair = Pair(sdk, 1, 1, 30000, 64, 64, 32)
    pair.append(29000)
    run(pair, "f16", 2, 900, scale=scale, weighted=True)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("n", [1, 4, 40, 130])
def test_ragged_batch(sdk, n, dtype):
    """Sequences of other lengths, one empty, with other numbers of rows."""
    pair = Pair(sdk, 5, 2, 600, 72, 64, n)
    pair.append(590, counts=[590, 64, 0, 321, 100])
    counts = [n, n // 2, n, 0, max(1, n - 1)]
    run(pair, dtype, 4, n, counts=counts, weighted=True, what="causal")
    run(pair, dtype, 4, n, counts=counts, causal=False, weighted=True, what="all seen")


def test_many_sequences(sdk):
    pair = Pair(sdk, 300, 1, 90, 32, 32, 4)
    pair.append(90, counts=[(11 * b) % 91 for b in range(300)])
    run(pair, "f16", 2, 2, counts=[b % 3 for b in range(300)], weighted=True)


@pytest.mark.parametrize("n", [1, 100])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_value_scales_apart(sdk, dtype, n):
    """Blocks whose values are zeros, tiny or huge, in an order that moves the
    output's unit both ways, with rows that look at the tiny ones alone."""
    pair = Pair(sdk, 1, 1, 700, 64, 64, 12)
    for scale in (1.0, 2.0 ** -14, 0.0, 1000.0, 2.0 ** -10, 1.0, 2.0 ** -14, 8000.0, 3.0):
        v = (pair.rng.standard_normal((1, 1, 64, 64)) * scale).astype(np.float16)
        pair.append(64, value=v)
    pair.append(70)
    run(pair, dtype, 4, n, what="mild")
    run(pair, dtype, 4, n, what="sharp", spread=25.0)     # nearly all weight on one token
    # every block in turn takes nearly all the weight
    k = np.zeros((1, 1, 576, 64), np.float16)
    for j in range(9):
        k[0, 0, 64 * j:64 * j + 64, j] = 8.0
    pair2 = Pair(sdk, 1, 1, 700, 64, 64, 13)
    v = pair.rng.standard_normal((1, 1, 576, 64)) * np.repeat(2.0 ** np.array([0, -14, 9, -14, 3, -10, 12, -14, 0]), 64)[:, None]
    pair2.append(576, key=k, value=v.astype(np.float16))
    q = np.zeros((1, 9 * 4, n, 64), DTYPES[dtype])
    for j in range(36):
        q[0, j, :, j % 9] = 40.0
    got, _ = attend(sdk, pair2.cache, q, 0.125, False, vdim=64)
    compare(pair2.model, q, 0.125, False, None, got, what="one block each")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("n", [1, 3, 90])
def test_marked_tokens(sdk, dtype, n):
    """Rows that see a marked token are NaN (zeros where they see nothing else);
    those before it are as if it were not there, and add their weights."""
    for length, at in ((200, (150,)), (200, (0, 1)), (130, (129,)), (130, (128, 64)), (90, (89,)), (300, (299,))):
        pair = Pair(sdk, 1, 2, 300, 64, 64, length)
        k, v = (rows_of(pair.rng, (1, 2, length, 64), "f16") for _ in range(2))
        for i, t in enumerate(at):
            (k if i == 0 else v)[0, 0, t, 5 + i] = np.nan if i else np.inf
        pair.append(length, key=k, value=v)
        run(pair, dtype, 4, n, weighted=True, what=f"{length} {at}")
        run(pair, dtype, 4, n, causal=False, weighted=True, what=f"{length} {at} all seen")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("n", [2, 66])
def test_query_rows_that_are_not_finite(sdk, dtype, n):
    """No score of such a row is finite: it is zeros, and its neighbours are not
    touched."""
    pair = Pair(sdk, 1, 1, 300, 40, 40, 15)
    pair.append(200)
    q = pair.rng.standard_normal((1, 3, n, 40)).astype(DTYPES[dtype])
    q[0, 0, 0, 3], q[0, 1, n - 1, 0], q[0, 2, 1, 39] = np.nan, np.inf, -np.inf
    w0 = np.zeros((1, 1, 200), np.float32)
    got, got_w = attend(sdk, pair.cache, q, 0.2, True, None, w0, 40)
    for j, i in ((0, 0), (1, n - 1), (2, 1)):
        assert (got[0, j, i] == 0).all()
    clean = np.where(np.isfinite(q), q, 0)
    want, tol, _, _ = pair.model.attention(clean, 0.2, True)
    good = np.isfinite(q).all(-1)
    assert (np.abs(got.astype(np.float64) - want) <= tol)[good].all()
    assert np.isfinite(got_w).all() and abs(float(got_w.sum()) - good.sum()) < 2e-3 * good.sum()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 12.0])
def test_scales(sdk, dtype, scale):
    pair = Pair(sdk, 1, 2, 300, 64, 64, 16)
    pair.append(270)
    run(pair, dtype, 4, 1, scale=scale, weighted=True, what="decode")
    run(pair, dtype, 4, 70, scale=scale, weighted=True, what="chunk")


def test_f32_queries_of_any_size(sdk):
    """f32 queries far outside f16's range, compensated by the scale."""
    for factor in (2.0 ** 40, 2.0 ** -60):
        pair = Pair(sdk, 1, 1, 200, 64, 64, 17)
        pair.append(150)
        for n in (1, 70):
            run(pair, "f32", 2, n, scale=0.125 / factor, spread=factor, what=f"{factor} {n}")


def test_scores_that_overflow(sdk):
    """Scores past f32: a row whose largest is +inf is zeros."""
    pair = Pair(sdk, 1, 1, 200, 16, 16, 18)
    pair.append(150)
    q = np.full((1, 1, 2, 16), 3e38, np.float32)
    q[0, 0, 1] = 1e-3
    got, _ = attend(sdk, pair.cache, q, 1e6, False, vdim=16)
    assert (got[0, 0, 0] == 0).all() and np.isfinite(got).all() and got[0, 0, 1].any()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_weights_of_a_long_causal_prompt(sdk, dtype):
    """Blocks enough to fill the chip, and the first seen by many more rows than the
    last: their rows are shared by more workgroups than that takes."""
    pair = Pair(sdk, 1, 40, 1600, 16, 24, 12)
    pair.append(1600)
    run(pair, dtype, 80, 1600, weighted=True)


@pytest.mark.parametrize("n", [1, 20])
@pytest.mark.parametrize("dims", [(72, 72), (40, 24), (100, 33)], ids=str)
def test_the_largest_keys_cut(sdk, dims, n):
    """A cut block goes on in f16: columns past the dims stay zeros at any scale."""
    pair = Pair(sdk, 1, 2, 200, *dims, seed=5)
    k = pair.rng.uniform(-65504, 65504, (1, 2, 130, dims[0])).astype(np.float16)
    k[0, :, 3, 0] = 65504
    k[0, :, 70, 1] = -65504
    v = pair.rng.uniform(-65504, 65504, (1, 2, 130, dims[1])).astype(np.float16)
    v[0, :, 70, 0] = 65504
    pair.append(130, key=k, value=v)
    pair.truncate([100])
    run(pair, "f32", 4, n, scale=1e-5, weighted=True)
    run(pair, "f16", 4, n, scale=1e-5, weighted=True)


def test_long_cache(sdk):
    """Enough blocks for many parts, in both types, one row and a few."""
    pair = Pair(sdk, 1, 1, 20000, 128, 128, 19)
    pair.append(19999)
    for dtype in ("f16", "f32"):
        run(pair, dtype, 4, 1, weighted=True, what=dtype)
        run(pair, dtype, 2, 9, weighted=True, what=dtype)


def test_calls_give_the_same_bits(sdk):
    """No sum depends on the order in which workgroups end."""
    pair = Pair(sdk, 2, 2, 3000, 64, 64, 20)
    pair.append(2900)
    for n in (1, 70, 1800):
        q = pair.rng.standard_normal((2, 6, n, 64)).astype(np.float16)
        w0 = np.zeros((2, 2, 2900), np.float32)
        first = attend(sdk, pair.cache, q, 0.125, True, None, w0, 64)
        for _ in range(3):
            again = attend(sdk, pair.cache, q, 0.125, True, None, w0, 64)
            assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(first, again))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("shape", [(4, 1), (4, 40), (8, 900)], ids=str)
def test_recorded_attention_follows_the_cache(sdk, shape, dtype):
    """A replay attends to what the cache then holds: after appends (tokens of
    the open block have become codes), cuts and eager calls in between."""
    hip = sdk.lib
    hip.tensor_device_hip_stream.restype = ctypes.c_void_p
    stream = ctypes.c_void_p(hip.tensor_device_hip_stream())
    heads, n = shape
    pair = Pair(sdk, 2, 2, 2000, 64, 48, 21)
    pair.append(100, counts=[100, 70])
    q = pair.rng.standard_normal((2, heads, n, 64)).astype(DTYPES[dtype])
    tq, out = sdk.from_numpy(q), sdk.tensor(dtype, (2, heads, n, 48))
    w = sdk.tensor("f32", (2, 2, 1500))      # less room than the cache's capacity
    kr, vr = sdk.tensor("f32", (2, 2, 1500, 64)), sdk.tensor("f32", (2, 2, 1500, 48))
    calls = [(f"tensor_kv_cache_attention_{dtype}", pair.cache, tq, None, 0.125, 1, w, out),
             ("tensor_kv_cache_read_f32", pair.cache, kr, vr)]
    graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
    for call in calls:
        sdk.call(*call)
    sdk.synchronize()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    try:
        for call in calls:
            sdk.call(*call)
    finally:
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
    for change in (None, "append", "append", "cut", "append", "eager"):
        if change == "append":
            pair.append(450, counts=[450, 200])
        elif change == "cut":
            pair.truncate([500, 90])
        elif change == "eager":
            attend(sdk, pair.cache, q, 0.3, False, vdim=48)
        w0 = pair.rng.random((2, 2, 1500)).astype(np.float32)
        w.upload(w0)
        out.upload(np.full(out.shape, 99, DTYPES[dtype]))
        kr.upload(np.zeros(kr.shape, np.float32))
        vr.upload(np.zeros(vr.shape, np.float32))
        sdk.synchronize()
        assert hip.hipGraphLaunch(exe, stream) == 0
        got, got_w = out.download(), w.download()
        compare(pair.model, q, 0.125, True, None, got, w0, got_w, str(change))
        want_k, want_v = pair.model.read(np.float32, 1500, np.zeros(kr.shape, np.float32), np.zeros(vr.shape, np.float32))
        assert np.array_equal(kr.download(), want_k) and np.array_equal(vr.download(), want_v)
    assert hip.hipGraphExecDestroy(exe) == 0
    assert hip.hipGraphDestroy(graph) == 0


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_serving_loop(sdk, dtype):
    """As a decoder uses it: a prompt, single tokens, drafted tokens of which some
    are rejected, the cache thinned by its accumulated weights and moved, and on."""
    batch, kv, heads, dim = 2, 2, 6, 64
    pair = Pair(sdk, batch, kv, 400, dim, dim, 22)
    weights = sdk.from_numpy(np.zeros((batch, kv, 400), np.float32))

    def step(n, counts=None):
        q = pair.rng.standard_normal((batch, heads, n, dim)).astype(DTYPES[dtype])
        out = sdk.from_numpy(np.full((batch, heads, n, dim), 99, DTYPES[dtype]))
        w0 = weights.download()
        sdk.call(f"tensor_kv_cache_attention_{dtype}", pair.cache, sdk.from_numpy(q),
                 None if counts is None else u32s(counts), 0.125, 1, weights, out)
        compare(pair.model, q, 0.125, True, counts, out.download(), w0, weights.download(), f"{n} rows")

    pair.append(150, dtype, counts=[150, 97])
    step(150, [150, 97])
    for _ in range(3):
        for _ in range(12):
            pair.append(1, dtype)
            step(1)
        pair.append(5, dtype)
        step(5)
        pair.truncate([n - 3 for n in pair.cache.lengths])
        step(2)
        w = weights.download()
        target = sdk.kv_cache(batch, kv, 400, dim, dim)
        moved = sdk.from_numpy(np.zeros((batch, kv, 400), np.float32))
        sdk.call("tensor_kv_cache_evict", pair.cache, weights, 4, 16, 100, target, moved, None)
        pair.model, index = pair.model.evict(w, 4, 16, 100)
        pair.cache, weights = target, moved
        check_read(sdk, pair.cache, pair.model, "moved")
        want = np.zeros((batch, kv, 400), np.float32)
        for b in range(batch):
            for h in range(kv):
                want[b, h, :len(index[b][h])] = w[b, h, index[b][h]]
        assert np.array_equal(weights.download(), want)
        step(1)


def test_threads_with_a_cache_each(sdk):
    errors = []

    def work(seed):
        try:
            pair = Pair(sdk, 1, 2, 300, 64, 64, seed)
            for n in (70, 1, 60, 1, 1):
                pair.append(n)
                run(pair, "f16", 4, 1, weighted=True, what=f"thread {seed}")
        except BaseException as e:      # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]


def test_threads_share_a_cache(sdk):
    """Appends and reads of one cache from several threads: each call sees a whole
    number of appends."""
    cache = sdk.kv_cache(1, 1, 4 * 30 * 3, 16)
    ones = sdk.from_numpy(np.ones((1, 1, 3, 16), np.float16))
    q, errors = np.ones((1, 1, 1, 16), np.float16), []

    def work():
        try:
            for _ in range(30):
                sdk.call("tensor_kv_cache_append_f16", cache, ones, ones, None)
                got, _ = attend(sdk, cache, q, 0.25, False, vdim=16)
                assert (got == 1).all()
        except BaseException as e:      # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
    assert cache.lengths == [360]


@pytest.mark.gpu
def test_model_is_its_own_check():
    """The plain model against direct sums on a small case."""
    model = Model(1, 1, 4, 4)
    rng = np.random.default_rng(0)
    k, v = rng.standard_normal((2, 1, 1, 70, 4)).astype(np.float16)
    model.append(k, v)
    a = np.abs(k[0, 0, :64].astype(np.float64)).max()
    held = model.k[0][0].held()
    assert np.abs(held[:64] - k[0, 0, :64]).max() <= a / 254 * (1 + 1e-6) and np.array_equal(held[64:], k[0, 0, 64:])
