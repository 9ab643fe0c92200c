"""Attention over the 8-bit key/value cache at the limits of its range: few query
rows over very many keys, queries far from 1, and how large errors typically are."""
import ctypes

import numpy as np
import pytest

from tests.kv_model import u32s
from tests.test_gpu_kv_attention import attend, compare, run
from tests.test_gpu_kv_cache import DTYPES, Pair, rows_of

pytestmark = pytest.mark.gpu


def one_long(sdk, batch, kv, length, dim, vdim, seed):
    """A batch whose first sequence has `length` tokens (its keys and values come
    four times) and whose others have a few: as many keys to plan for as if all
    were long."""
    pair = Pair(sdk, batch, kv, length, dim, vdim, seed)
    n = length // 4
    k, v = np.zeros((batch, kv, n, dim), np.float16), np.zeros((batch, kv, n, vdim), np.float16)
    short = [(7 * b) % 23 + 1 for b in range(batch)]
    few = max(short)
    for x in (k, v):
        x[0] = pair.rng.standard_normal(x[0].shape)
        x[1:, :, :few] = pair.rng.standard_normal(x[1:, :, :few].shape)
    tk, tv = sdk.from_numpy(k), sdk.from_numpy(v)
    for turn in range(4):
        counts = [n] + [m if turn == 2 else 0 for m in short[1:]]
        sdk.call("tensor_kv_cache_append_f16", pair.cache, tk, tv, u32s(counts))
        pair.model.append(k[:, :, :max(counts)], v[:, :, :max(counts)], counts)
    return pair


# batch, kv heads, query heads, rows, tokens of the longest, dim, value dim: at most
# 16 packed rows per kv head, and more products (sequences x kv heads x rows x tokens
# x the wider dim) than the tile kernel is used from for prompts; key parts (few
# sequences and heads) and none (many)
FEW = [("f16", 64, 4, 16, 1, 10400, 16, 256), ("f16", 64, 4, 64, 1, 2600, 16, 256), ("f16", 32, 8, 64, 2, 2600, 256, 16),
       ("f16", 16, 2, 32, 1, 20800, 16, 256), ("f32", 64, 4, 64, 1, 6800, 16, 128), ("f32", 16, 2, 16, 2, 54400, 16, 128)]


@pytest.mark.parametrize("shape", FEW, ids=str)
def test_weights_of_few_rows_over_many_keys(sdk, shape):
    dtype, batch, kv, heads, n, length, dim, vdim = shape
    pair = one_long(sdk, batch, kv, length, dim, vdim, n)
    run(pair, dtype, heads, n, weighted=True, what="causal")
    run(pair, dtype, heads, n, causal=False, weighted=True, what="all seen")
    run(pair, dtype, heads, n, what="no weights")


# around the packed rows from which so many products go to the tile kernel
MORE = [("f16", 64, 4, 68, 1, 2600, 16, 256), ("f16", 64, 4, 32, 4, 2600, 256, 16), ("f16", 64, 4, 44, 3, 1600, 16, 256),
        ("f16", 64, 8, 128, 4, 5200, 16, 32), ("f16", 64, 8, 104, 5, 5200, 16, 32), ("f32", 64, 4, 64, 3, 2400, 16, 128),
        ("f32", 64, 4, 128, 2, 1720, 16, 128), ("f32", 64, 4, 52, 5, 1720, 16, 128), ("f32", 64, 4, 68, 2, 3600, 16, 200)]


@pytest.mark.parametrize("shape", MORE, ids=str)
def test_some_rows_over_many_keys(sdk, shape):
    dtype, batch, kv, heads, n, length, dim, vdim = shape
    pair = one_long(sdk, batch, kv, length, dim, vdim, heads)
    run(pair, dtype, heads, n, weighted=True, what="causal")
    run(pair, dtype, heads, n, causal=False, what="no weights")


# capacity instead of tokens: what a recorded call is planned for
CAPACITIES = [("f16", 4, 2, 8, 1, 330000, 16, 256), ("f16", 64, 4, 16, 1, 10400, 16, 256), ("f16", 2, 2, 8, 4, 165000, 256, 16),
              ("f32", 64, 4, 64, 1, 6800, 16, 128), ("f32", 4, 2, 8, 3, 290000, 16, 128)]


@pytest.mark.parametrize("shape", CAPACITIES, ids=str)
def test_recorded_weights_of_few_rows_in_a_large_cache(sdk, shape):
    check_replays(sdk, shape)


# as many rows and so large a capacity that the tile kernel is recorded, in key parts
# that the cache does not reach and in one
@pytest.mark.parametrize("shape", [("f16", 4, 2, 8, 20, 40000, 16, 256), ("f32", 4, 2, 8, 30, 40000, 16, 128),
                                   ("f16", 64, 4, 8, 150, 2600, 32, 32), ("f16", 2, 2, 4, 200, 60000, 64, 64)], ids=str)
def test_recorded_tiles_in_a_large_cache(sdk, shape):
    check_replays(sdk, shape)


def check_replays(sdk, shape):
    """A call recorded at a hundred tokens, replayed as the cache grows."""
    dtype, batch, kv, heads, n, capacity, dim, vdim = shape
    hip = sdk.lib
    hip.tensor_device_hip_stream.restype = ctypes.c_void_p
    stream = ctypes.c_void_p(hip.tensor_device_hip_stream())
    pair = Pair(sdk, batch, kv, capacity, dim, vdim, 41)
    pair.append(100, counts=[100 - b % 90 for b in range(batch)])
    q = pair.rng.standard_normal((batch, heads, n, dim)).astype(DTYPES[dtype])
    tq, out = sdk.from_numpy(q), sdk.tensor(dtype, (batch, heads, n, vdim))
    w = sdk.tensor("f32", (batch, kv, 400))
    call = (f"tensor_kv_cache_attention_{dtype}", pair.cache, tq, None, 0.25, 1, w, out)
    sdk.call(*call)
    sdk.synchronize()
    graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    try:
        sdk.call(*call)
    finally:
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
    for change in (None, "append", "eager", "append"):
        if change == "append":
            pair.append(130, counts=[130 - b % 3 for b in range(batch)])
        elif change == "eager":
            attend(sdk, pair.cache, q, 0.3, False, vdim=vdim)
        w0 = pair.rng.random(w.shape).astype(np.float32)
        w.upload(w0)
        out.upload(np.full(out.shape, 99, DTYPES[dtype]))
        sdk.synchronize()
        assert hip.hipGraphLaunch(exe, stream) == 0
        compare(pair.model, q, 0.25, True, None, out.download(), w0, w.download(), str(change))
    assert hip.hipGraphExecDestroy(exe) == 0
    assert hip.hipGraphDestroy(graph) == 0


@pytest.mark.parametrize("keys", [1.0, 2.0 ** -12])
@pytest.mark.parametrize("size", [1e-30, 1e-37, 1e-40, 1e-44])
def test_tiny_f32_queries(sdk, size, keys):
    """Rows whose scores come to nothing see their tokens alike, and no others, and
    add their weights, on every kernel."""
    pair = Pair(sdk, 1, 2, 200, 64, 64, 42)
    k, v = (rows_of(pair.rng, (1, 2, 150, 64), "f16", s) for s in (keys, 1.0))
    pair.append(150, key=k, value=v)
    for n in (1, 9, 70):
        for scale in (0.125, -1e-4):
            run(pair, "f32", 4, n, scale=scale, spread=size, weighted=True, what=f"{n} rows, {scale}")
    run(pair, "f32", 4, 70, scale=0.125, spread=size, causal=False, weighted=True, what="all seen")


def test_tiny_f32_queries_in_tiles(sdk):
    pair = Pair(sdk, 2, 64, 1200, 64, 64, 43)
    pair.append(1200)
    for size in (1e-36, 1e-44):
        run(pair, "f32", 64, 512, scale=0.125, spread=size, weighted=True, what=f"{size}")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_zero_queries_at_any_scale(sdk, dtype):
    """Products of 0 are scores of 0, also where scale and keys together pass f32."""
    pair = Pair(sdk, 1, 2, 200, 64, 64, 44)
    k, v = (rows_of(pair.rng, (1, 2, 150, 64), "f16", s) for s in (1000.0, 1.0))
    k[0, 1, 64:128] = 0
    pair.append(150, key=k, value=v)
    for n in (1, 9, 70):
        for scale in (3e38, -3e38):
            run(pair, dtype, 4, n, scale=scale, spread=0.0, weighted=True, what=f"{n} rows, {scale}")


def test_tiny_f32_queries_at_large_scales(sdk):
    """Rows below the smallest power of two whose reciprocal f32 holds, with scales
    that bring their scores back."""
    pair = Pair(sdk, 1, 2, 200, 64, 64, 45)
    k, v = (rows_of(pair.rng, (1, 2, 150, 64), "f16", s) for s in (30.0, 1.0))
    pair.append(150, key=k, value=v)
    for size, scale in ((1e-37, 1e35), (1e-40, 1e38), (1e-42, 3e38)):
        for n in (1, 9, 70):
            run(pair, "f32", 4, n, scale=scale, spread=size, weighted=True, what=f"{size}: {n} rows")


def leaning(pair, heads, n, dtype, lean):
    """Causal query rows that each give one token they see about the weight `lean`
    (0: none in particular)."""
    batch, kv, dim, _ = pair.model.shape
    q = pair.rng.standard_normal((batch, heads, n, dim)) * 0.5
    for b, j in np.ndindex(batch, heads):
        k = pair.model.k[b][j // (heads // kv)].held()
        seen = len(k) - n + 1 + np.arange(n)
        if lean:
            to = k[(pair.rng.random(n) * seen).astype(np.int64)]
            score = np.log(seen * lean / (1 - lean))
            q[b, j] += to * (score * dim ** 0.5 / (to * to).sum(-1))[:, None]
    return q.astype(DTYPES[dtype])


@pytest.mark.parametrize("lean", [0.0, 0.9])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("shape", [(1, 2, 4, 5), (1, 2, 4, 70), (2, 64, 64, 512)], ids=["rows", "more rows", "tiles"])
def test_typical_errors(sdk, shape, dtype, lean):
    """Root mean squares of the errors, relative to those of what they are errors of;
    the bounds of the other tests are worst cases, and grow with the keys.

    f32 outputs, in units of u = 2^-24, 1200 keys of 64 dims. Scores (13 in log2 units
    where a row leans on a token) add up in four steps or so, each off by u of them:
    36 u of that token's weight, which comes to 0.9 * 0.1 of that in the output, 3 u.
    19 blocks' sums and outputs are added one by one: 19^0.5 u / 2, 2 u each. A block's
    products add up in eight steps, each off by u of the largest: 3 u. P is a pair, and
    its exponential is off by u. Together (3^2 + 2^2 + 2^2 + 3^2 + 1 + 1)^0.5, 5 u: less
    than 16.
    Weights: 36 u of the scores at most, and of those again 0.1 in their sum; the
    factor's rounding 9 u, likewise; at most 22 additions in a row, 3 u: less than 32.
    f16 outputs: P and the output rounded, each off by 2^-11 / 3^0.5 at most: 2^-11."""
    batch, kv, heads, n = shape
    pair = Pair(sdk, batch, kv, 1200, 64, 64, 46)
    pair.append(1200)
    q = leaning(pair, heads, n, dtype, lean)
    got, got_w = attend(sdk, pair.cache, q, 0.125, True, None, np.zeros((batch, kv, 1200), np.float32), 64)
    want, _, want_w, _ = pair.model.attention(q, 0.125, True)
    plain, _ = attend(sdk, pair.cache, q, 0.125, True, None, None, 64)

    def error(x, y):
        return float(np.sqrt(np.square(x.astype(np.float64) - y).mean() / np.square(y).mean()))

    most = 2.0 ** -11 if dtype == "f16" else 2.0 ** -20
    assert error(got, want) < most and error(plain, want) < most, (error(got, want), error(plain, want))
    assert error(got_w, want_w) < 2.0 ** -19, error(got_w, want_w)
    print(f"{shape} {dtype} {lean}: outputs {error(got, want):.2e}, weights {error(got_w, want_w):.2e}")
