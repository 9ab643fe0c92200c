"""The 8-bit key/value cache without a GPU: what creation refuses, and that a
missing cache is refused, before any device work."""
import ctypes
import math

import numpy as np
import pytest

from tests.kv_model import Model, u32s


def create(lib, *sizes):
    handle, err = ctypes.c_void_p(1), ctypes.create_string_buffer(512)
    ok = lib.tensor_kv_cache_create(*sizes, ctypes.byref(handle), err, 512)
    return ok, handle.value, err.value.decode()


@pytest.mark.parametrize("sizes", [(0, 1, 1, 1, 1), (65536, 1, 1, 1, 1), (1, 0, 1, 1, 1), (1, 4097, 1, 1, 1),
                                   (1, 1, 0, 1, 1), (1, 1, 2 ** 29 + 1, 1, 1), (1, 1, 1, 0, 1), (1, 1, 1, 257, 1),
                                   (1, 1, 1, 1, 0), (1, 1, 1, 1, 257), (2 ** 63, 2 ** 63, 2 ** 63, 64, 64)])
def test_create_refuses_sizes(lib, sizes):
    ok, handle, message = create(lib, *sizes)
    assert ok == 0 and handle is None
    assert message.startswith("cache requires a result pointer, 1 to 65535 sequences")


def test_create_refuses_a_missing_result(lib):
    err = ctypes.create_string_buffer(512)
    assert lib.tensor_kv_cache_create(1, 1, 1, 1, 1, None, err, 512) == 0
    assert err.value.startswith(b"cache requires a result pointer")
    assert lib.tensor_kv_cache_create(1, 1, 1, 1, 1, None, None, 0) == 0


def test_create_without_device_fails_loudly(lib):
    if lib.tensor_device_available():
        pytest.skip("a HIP device is present")
    ok, handle, message = create(lib, 1, 2, 100, 64, 64)
    assert ok == 0 and handle is None and message.startswith("HIP device unavailable")


def test_a_missing_cache_is_refused(lib):
    from inference_c_amd import Sdk
    sdk = Sdk()
    t = sdk.tensor("f16", (1, 1, 2, 4), device=False)
    for call, what in (
            (("tensor_kv_cache_append_f16", None, t, t, None), "cache append requires a cache"),
            (("tensor_kv_cache_append_f32", None, t, t, u32s([1])), "cache append requires a cache"),
            (("tensor_kv_cache_truncate", None, None), "cache truncate requires a cache"),
            (("tensor_kv_cache_read_f16", None, t, t), "cache read requires a cache"),
            (("tensor_kv_cache_attention_f32", None, t, None, 1.0, 1, None, t), "cache attention requires a cache"),
            (("tensor_kv_cache_evict", None, None, 0, 0, 1, None, None, None),
             "cache evict requires a cache and another one as its target")):
        ok, message = sdk.try_call(*call)
        assert ok == 0 and message == what
    assert lib.tensor_kv_cache_length(None, 0) == 0
    assert lib.tensor_kv_cache_capacity(None) == 0
    assert lib.tensor_kv_cache_byte_length(None) == 0
    lib.tensor_kv_cache_free(None)


@pytest.mark.parametrize("sizes", [(1, 1, 2 ** 27 + 1, 1, 1), (1, 17, 2 ** 27, 1, 1), (65535, 4096, 64, 1, 1),
                                   (65535, 513, 1, 256, 256)])
def test_create_refuses_too_many_tokens(lib, sizes):
    ok, handle, message = create(lib, *sizes)
    assert ok == 0 and handle is None
    assert message.startswith("cache requires a result pointer" if sizes[2] > 2 ** 27 else
                              "cache requires at most 2^31 tokens")


def direct(q, k, v, scale, seen):
    """One row's output and token weights by loops over the tokens it sees, and
    None for a row whose output is NaN."""
    scores = [scale * sum(float(a) * float(b) for a, b in zip(q, k[t])) if k[t] is not None else math.nan
              for t in range(seen)]
    finite = [s for s in scores if not math.isnan(s)]
    if not finite:
        return [0.0] * len(v[-1]), {}
    if len(finite) < len(scores):
        return None, {}
    top = max(scores)
    total = math.fsum(math.exp(s - top) for s in scores)
    p = [math.exp(s - top) / total for s in scores]
    return [math.fsum(p[t] * float(v[t][d]) for t in range(seen)) for d in range(len(v[-1]))], dict(enumerate(p))


@pytest.mark.parametrize("causal", [True, False])
def test_the_plain_attention_by_direct_sums(causal):
    """The model that the kernels' attention is compared with: sequences of other
    lengths, query heads that share a kv head, padded rows, rows that see nothing, a
    marked token that some rows see, and one that is all that a row sees."""
    rng = np.random.default_rng(5)
    batch, heads, kv, dim, vdim, n = 4, 4, 2, 5, 3, 6
    lengths, counts, scale = [70, 3, 66, 2], [6, 6, 2, 2], 0.7
    model = Model(batch, kv, dim, vdim)
    key = rng.standard_normal((batch, kv, 70, dim)).astype(np.float16)
    value = rng.standard_normal((batch, kv, 70, vdim)).astype(np.float16)
    key[0, 1, 67, 2] = np.inf
    value[3, 0, 0, 1] = np.nan
    model.append(key, value, lengths)
    q = rng.standard_normal((batch, heads, n, dim)).astype(np.float32)
    out, tol, weights, _ = model.attention(q, scale, causal, counts)
    want = np.zeros(weights.shape)
    kinds = set()
    for b in range(batch):
        assert np.isnan(out[b, :, counts[b]:]).all()
        for j in range(heads):
            h = j // (heads // kv)
            k = [None if model.marked[b][h][t] else row for t, row in enumerate(model.k[b][h].held())]
            v = model.v[b][h].held()
            for i in range(counts[b]):
                seen = lengths[b] if not causal else max(0, lengths[b] - counts[b] + i + 1)
                o, p = direct(q[b, j, i], k, v, scale, seen)
                kinds.add("nan" if o is None else "sums" if p else "nothing seen" if seen == 0 else "marked alone")
                if o is None:
                    assert np.isnan(out[b, j, i]).all()
                    continue
                # 70 products and sums in f64, the numbers no larger than 10
                assert np.abs(out[b, j, i] - o).max() < 1e-13
                assert (tol[b, j, i] > 0).all() == bool(p)
                for t, x in p.items():
                    want[b, h, t] += x
    assert kinds == ({"nan", "sums", "nothing seen", "marked alone"} if causal else {"nan", "sums"})
    assert np.abs(weights - want).max() < 1e-12


def test_the_plain_cache_by_direct_rounding():
    """Held values are the nearest of 255 steps of the block's largest, and the open
    block's are f16."""
    rng = np.random.default_rng(6)
    model = Model(1, 1, 4, 4)
    k, v = rng.standard_normal((2, 1, 1, 130, 4)).astype(np.float16)
    model.append(k[:, :, :70], v[:, :, :70])
    model.append(k[:, :, 70:], v[:, :, 70:])
    held = model.k[0][0].held()
    for block in (0, 64):
        x = k[0, 0, block:block + 64].astype(np.float64)
        a = np.abs(x).max()
        step = float(np.float32(a / 127))
        for i, j in np.ndindex(x.shape):
            codes = np.arange(-127, 128)
            best = codes[np.argmin(np.abs(codes * (a / 127) - x[i, j]))]
            assert held[block + i, j] == best * step
    assert np.array_equal(held[128:], k[0, 0, 128:])
