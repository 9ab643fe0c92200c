"""Shared attention of 2^26 query rows, as many as a call takes, with wide values: the
parts' join needs more threads than one launch holds."""
import ctypes

import numpy as np
import pytest

from tests.kv_model import u32s

pytestmark = pytest.mark.gpu

ROWS, DIM, VDIM = 2 ** 26, 1, 253
NEEDED = 175 << 30          # the output's 34 GB, the parts' 137, and some


def test_most_rows(sdk):
    free, total = ctypes.c_size_t(), ctypes.c_size_t()
    assert sdk.lib.hipMemGetInfo(ctypes.byref(free), ctypes.byref(total)) == 0
    if free.value < NEEDED:
        pytest.skip("too little device memory is free")
    rng = np.random.default_rng(1)
    caches, keys, values = [], [], []
    for n in (2, 3):
        k, v = (rng.standard_normal((1, 1, n, d)).astype(np.float16) for d in (DIM, VDIM))
        caches.append(sdk.kv_cache(1, 1, 64, DIM, VDIM))
        sdk.call("tensor_kv_cache_append_f16", caches[-1], sdk.from_numpy(k), sdk.from_numpy(v), None)
        keys.append(k[0, 0].astype(np.float64))
        values.append(v[0, 0].astype(np.float64))
    k, v = np.concatenate(keys), np.concatenate(values)
    q = rng.standard_normal((1, 1, ROWS, DIM), np.float32).astype(np.float16)
    out = sdk.tensor("f16", (1, 1, ROWS, VDIM))
    at = sdk.lib.tensor_buffer_device_handle_internal(out.handle)
    marks = np.full((8, VDIM), 99, np.float16)
    assert sdk.lib.hipMemcpy(ctypes.c_void_p(at + (ROWS - 8) * VDIM * 2), marks.ctypes.data_as(ctypes.c_void_p),
                             ctypes.c_size_t(marks.nbytes), 1) == 0
    there = ROWS - 5
    sdk.call("tensor_kv_cache_attention_shared_f16", *caches, sdk.from_numpy(q), None, u32s([there]), 0.7, 0, out)
    sdk.synchronize()
    for first in (0, 12345, ROWS // 2 - 500, 3 * (ROWS // 4), ROWS - 1000):
        got = np.empty((1000, VDIM), np.float16)
        assert sdk.lib.hipMemcpy(got.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(at + first * VDIM * 2),
                                 ctypes.c_size_t(got.nbytes), 2) == 0
        s = 0.7 * q[0, 0, first:first + 1000].astype(np.float64) @ k.T
        w = np.exp(s - s.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        want = w @ v
        # the weights' rounding to f16, relative to their rounded sum, the output's, and
        # that of the scores and sums in f32
        bound = 2.0 ** -11 * (2 * np.abs(want) + w @ np.abs(v)) + 2.0 ** -20 * np.abs(v).max()
        rows = min(1000, there - first)
        assert (np.abs(got.astype(np.float64) - want) <= bound)[:rows].all(), first
        assert (got[rows:] == 99).all()
