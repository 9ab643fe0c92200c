"""Lengths of a key/value cache whose launches fail, against a stand-in for the
runtime and the kernels, without a GPU: a call over more sequences than one launch
takes has done those before the launch that failed, and says so by their lengths."""
import os
import subprocess

import pytest

from tests.conftest import REPO

CSRC = os.path.join(REPO, "inference_c_amd", "csrc")
HIP_INCLUDE = "/opt/rocm/include"
COMPILER = "/opt/rocm/bin/amdclang++"

PROGRAM = r"""
#include "kv.hpp"
#include "sdk.hpp"
#include "tensor_kv_cache.h"
#include <cstdarg>
#include <cstdio>
#include <cstdlib>

static int good = 0;   // launches that succeed before one fails
static hipError_t launch() { return good-- > 0 ? hipSuccess : hipErrorInvalidConfiguration; }

extern "C" {
hipError_t hipMalloc(void **p, size_t n) { *p = std::malloc(n); return hipSuccess; }
hipError_t hipFree(void *p) { std::free(p); return hipSuccess; }
hipError_t hipMemsetAsync(void *, int, size_t, hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }

struct TensorBuffer { TensorDType dtype; size_t rank; uint64_t shape[4]; };
TensorDType tensor_buffer_dtype(const TensorBuffer *t) { return t->dtype; }
size_t tensor_buffer_rank(const TensorBuffer *t) { return t->rank; }
const uint64_t *tensor_buffer_shape(const TensorBuffer *t) { return t->shape; }
TensorBufferStorage tensor_buffer_storage(const TensorBuffer *) { return TENSOR_BUFFER_STORAGE_DEVICE; }
void *tensor_buffer_device_handle_internal(const TensorBuffer *) { return nullptr; }
}
namespace icsdk {
void set_error(char *error, size_t capacity, const char *format, ...) {
    va_list args;
    va_start(args, format);
    std::vsnprintf(error, capacity, format, args);
    va_end(args);
}
bool sdk_ready(char *, size_t) { return true; }
hipStream_t sdk_stream() { return nullptr; }
void bind_device() {}
bool hip_ok(hipError_t s, const char *what, char *error, size_t capacity) {
    if (s != hipSuccess) set_error(error, capacity, "%s", what);
    return s == hipSuccess;
}
Recording sdk_recording() { return Recording::kNo; }
void *scratch_acquire(size_t n) { return std::malloc(n); }
void scratch_release(void *p, size_t) { std::free(p); }
void *graph_scratch_acquire(size_t) { return nullptr; }
namespace kv {
hipError_t append(bool, const View &, uint32_t, uint32_t, const void *, const void *, uint32_t, const Counts &,
                  const Counts &, hipStream_t) { return launch(); }
hipError_t truncate(const View &, uint32_t, uint32_t, const Counts &, const Counts &, hipStream_t) { return launch(); }
hipError_t read(bool, const View &, uint32_t, void *, void *, uint32_t, uint32_t, hipStream_t) { return launch(); }
hipError_t evict(const View &, const View &, uint32_t, const EvictArgs &, hipStream_t) { return launch(); }
size_t attention_workspace(bool, const View &, const AttentionShape &) { return 0; }
hipError_t attention(bool, const View &, const AttentionShape &, const void *, void *, void *, hipStream_t) {
    return launch();
}
}
}

#define CHECK(x) do { if (!(x)) { std::printf("%d: %s (%s)\n", __LINE__, #x, text); return 1; } } while (0)
// the first `done` sequences hold a tokens, the others b
static bool holds(const TensorKvCache *c, size_t done, size_t a, size_t b) {
    for (size_t i = 0; i < 600; ++i)
        if (tensor_kv_cache_length(c, i) != (i < done ? a : b)) return false;
    return true;
}
int main() {
    char text[256] = "";
    TensorKvCache *c = nullptr, *other = nullptr;
    CHECK(tensor_kv_cache_create(600, 1, 100, 16, 16, &c, text, sizeof text));
    CHECK(tensor_kv_cache_create(600, 1, 100, 16, 16, &other, text, sizeof text));
    const TensorBuffer rows{TENSOR_DTYPE_F16, 4, {600, 1, 30, 16}};
    // 600 sequences go in three launches
    good = 0;
    CHECK(!tensor_kv_cache_append_f16(c, &rows, &rows, nullptr, text, sizeof text) && holds(c, 0, 0, 0));
    good = 2;
    CHECK(!tensor_kv_cache_append_f16(c, &rows, &rows, nullptr, text, sizeof text) && holds(c, 512, 30, 0));
    // the rest, as the lengths tell
    uint32_t counts[600], lengths[600];
    for (size_t i = 0; i < 600; ++i) counts[i] = 30 - (uint32_t)tensor_kv_cache_length(c, i), lengths[i] = 7;
    good = 3;
    CHECK(tensor_kv_cache_append_f16(c, &rows, &rows, counts, text, sizeof text) && holds(c, 600, 30, 30));
    good = 1;
    CHECK(!tensor_kv_cache_truncate(c, lengths, text, sizeof text) && holds(c, 256, 7, 30));
    good = 3;
    CHECK(tensor_kv_cache_truncate(c, lengths, text, sizeof text) && holds(c, 600, 7, 7));
    good = 0;
    CHECK(!tensor_kv_cache_evict(c, nullptr, 0, 0, 5, other, nullptr, nullptr, text, sizeof text));
    CHECK(holds(c, 600, 7, 7) && holds(other, 600, 0, 0));
    good = 1;
    CHECK(tensor_kv_cache_evict(c, nullptr, 0, 0, 5, other, nullptr, nullptr, text, sizeof text));
    CHECK(holds(c, 600, 7, 7) && holds(other, 600, 5, 5));
    // refusals come before any launch and change nothing
    good = 9;
    counts[599] = 31;
    CHECK(!tensor_kv_cache_append_f16(c, &rows, &rows, counts, text, sizeof text) && holds(c, 600, 7, 7) && good == 9);
    lengths[599] = 8;
    CHECK(!tensor_kv_cache_truncate(c, lengths, text, sizeof text) && holds(c, 600, 7, 7) && good == 9);
    CHECK(!tensor_kv_cache_evict(c, nullptr, 0, 0, 101, other, nullptr, nullptr, text, sizeof text) && good == 9);
    tensor_kv_cache_free(c);
    tensor_kv_cache_free(other);
    return 0;
}
"""


def test_lengths_after_failed_launches(tmp_path):
    if not os.path.isfile(COMPILER):
        pytest.skip("ROCm compiler absent")
    source, exe = tmp_path / "program.cpp", tmp_path / "program"
    source.write_text(PROGRAM)
    subprocess.run([COMPILER, "-std=c++17", "-x", "c++", "-D__HIP_PLATFORM_AMD__", "-isystem", HIP_INCLUDE, "-I", CSRC,
                    "-I", os.path.join(REPO, "include"), "-o", str(exe), str(source), os.path.join(CSRC, "kv_cache.cpp"),
                    "-pthread"], check=True)
    result = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert result.returncode == 0, result.stdout
