"""The 8-bit key/value cache without a GPU: what creation refuses, and that a
missing cache is refused, before any device work."""
import ctypes

import pytest

from tests.kv_model import u32s


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
