"""Copies and reorders of a key/value cache's sequences, and shared attention, without
a GPU: what is refused, before any launch, and the lengths after launches that fail,
against a stand-in for the runtime and the kernels."""
import os
import subprocess

import numpy as np
import pytest

from tests import beam_model
from tests.conftest import REPO
from tests.kv_model import Model
from tests.test_kv_cache_host import direct
from tests.test_kv_cache_launches import COMPILER, CSRC, HIP_INCLUDE, PROGRAM as CACHE_PROGRAM

STAND_IN = CACHE_PROGRAM[:CACHE_PROGRAM.index("#define CHECK")].replace(
    "Recording sdk_recording() { return Recording::kNo; }",
    "static bool recorded = false;\nRecording sdk_recording() { return recorded ? Recording::kYes : Recording::kNo; }")

PROGRAM = STAND_IN + r"""
static icsdk::kv::Counts told;       // the last copy's sources
static uint32_t told_batch, told_longest, told_most;
namespace icsdk {
namespace kv {
hipError_t copy(const View &, const View &, uint32_t, uint32_t batch, const Counts &source, uint32_t longest, size_t,
                hipStream_t) {
    told = source, told_batch = batch, told_longest = longest;
    return launch();
}
hipError_t reorder(const View &, uint32_t, uint32_t, const uint32_t *, uint32_t longest, hipStream_t) {
    told_longest = longest;
    return launch();
}
size_t attention_shared_workspace(bool, const View &, const PrefixShape &, const View &, const AttentionShape &) { return 64; }
hipError_t attention_shared(bool, const View &, const PrefixShape &p, const View &, const AttentionShape &a, const void *,
                            void *, void *, hipStream_t) {
    told_most = p.most, told_longest = p.longest, told_batch = a.batch;
    uint32_t sum = 0;
    for (uint32_t i = 0; i < p.batch; ++i) sum += p.members[i];
    return sum == a.batch ? launch() : hipErrorUnknown;
}
}
}
#define CHECK(x) do { if (!(x)) { std::printf("%d: %s (%s)\n", __LINE__, #x, text); return 1; } } while (0)
#include <cstring>
static char text[256];
static bool said(const char *what) { return std::strncmp(text, what, std::strlen(what)) == 0; }
static bool copy(const TensorKvCache *c, const uint32_t *s, TensorKvCache *t) {
    return tensor_kv_cache_copy(c, s, t, text, sizeof text) != 0;
}
int main() {
    const uint32_t keep = TENSOR_KV_CACHE_KEEP;
    TensorKvCache *c = nullptr, *small = nullptr, *large = nullptr, *wide = nullptr;
    CHECK(tensor_kv_cache_create(3, 2, 100, 16, 16, &c, text, sizeof text));
    CHECK(tensor_kv_cache_create(4, 2, 50, 16, 16, &small, text, sizeof text));
    CHECK(tensor_kv_cache_create(600, 2, 100, 16, 16, &large, text, sizeof text));
    CHECK(tensor_kv_cache_create(3, 2, 100, 16, 17, &wide, text, sizeof text));
    const TensorBuffer rows{TENSOR_DTYPE_F16, 4, {3, 2, 90, 16}};
    const uint32_t counts[] = {90, 20, 50};
    good = 1;
    CHECK(tensor_kv_cache_append_f16(c, &rows, &rows, counts, text, sizeof text));
    auto length = [](const TensorKvCache *x, size_t b) { return tensor_kv_cache_length(x, b); };

    // copies: refusals launch nothing and change nothing
    good = 9;
    const uint32_t past[] = {1, 3, 1, 1}, full[] = {1, 1, 0, 1}, chain[] = {1, 2, keep}, swap[] = {1, 0, keep};
    CHECK(!copy(nullptr, past, small) && said("cache copy requires a cache"));
    CHECK(!copy(c, nullptr, small) && !copy(c, past, nullptr));
    CHECK(!copy(c, chain, wide) && said("cache copy: the target's heads and dimensions"));
    CHECK(!copy(c, past, small) && said("cache copy: sequence 3 of 3"));
    CHECK(!copy(c, full, small) && said("cache copy: sequence 0 holds 90 tokens, the target has room for 50"));
    CHECK(!copy(c, chain, c) && said("cache copy: sequence 1 is copied from and to within one cache"));
    CHECK(!copy(c, swap, c) && length(small, 0) == 0 && length(c, 0) == 90 && good == 9);
    const uint32_t none[] = {keep, keep, keep, keep}, itself[] = {0, 1, 2};
    CHECK(copy(c, none, small) && copy(c, itself, c) && good == 9);
    icsdk::recorded = true;
    const uint32_t fits[] = {1, keep, 2, 1};
    CHECK(!copy(c, fits, small) && said("cache copy changes the cache's lengths") && good == 9);
    icsdk::recorded = false;
    CHECK(copy(c, fits, small) && good == 8 && told_longest == 50 && told_batch == 4 && told.n[1] == icsdk::kv::kKeep);
    CHECK(length(small, 0) == 20 && length(small, 1) == 0 && length(small, 2) == 50 && length(small, 3) == 20);
    const uint32_t within[] = {keep, 0, 2};
    CHECK(copy(c, within, c) && length(c, 1) == 90 && told.n[2] == icsdk::kv::kKeep && good == 7);
    // three launches, of which the middle one has nothing to do; those before one that fails are done
    uint32_t many[600];
    for (int b = 0; b < 600; ++b) many[b] = b < 256 || b >= 512 ? 2 : keep;
    good = 1;
    CHECK(!copy(c, many, large) && length(large, 0) == 50 && length(large, 255) == 50 && length(large, 256) == 0);
    CHECK(length(large, 512) == 0);
    good = 2;
    CHECK(copy(c, many, large) && good == 0 && length(large, 599) == 50 && length(large, 300) == 0);

    // reorders
    good = 9;
    auto reorder = [](TensorKvCache *x, TensorDType t, size_t rank, uint64_t g, uint64_t b) {
        const TensorBuffer parents{t, rank, {g, b}};
        return tensor_kv_cache_reorder(x, &parents, text, sizeof text) != 0;
    };
    CHECK(!tensor_kv_cache_reorder(small, nullptr, text, sizeof text) && said("cache reorder requires rank-2 U32"));
    CHECK(!reorder(nullptr, TENSOR_DTYPE_U32, 2, 1, 4) && said("cache reorder requires a cache"));
    CHECK(!reorder(small, TENSOR_DTYPE_I32, 2, 1, 4) && !reorder(small, TENSOR_DTYPE_U32, 1, 4, 1));
    const uint64_t shapes[][2] = {{1, 3}, {2, 4}, {0, 4}, {4, 0}, {1, 65}, {uint64_t{1} << 62, 8}, {3, 1}};
    for (auto &s : shapes) CHECK(!reorder(small, TENSOR_DTYPE_U32, 2, s[0], s[1]) && said("cache reorder: parents must be"));
    CHECK(!reorder(small, TENSOR_DTYPE_U32, 2, 1, 4) && said("cache reorder: the sequences of group 0 are not of one length"));
    CHECK(good == 9 && reorder(small, TENSOR_DTYPE_U32, 2, 4, 1) && good == 9);
    const uint32_t cut[] = {20, 0, 20, 20};
    CHECK(tensor_kv_cache_truncate(small, cut, text, sizeof text) && good == 8);
    CHECK(!reorder(small, TENSOR_DTYPE_U32, 2, 2, 2) && said("cache reorder: the sequences of group 0"));
    const uint32_t one[] = {1, 1, 1, 1};
    CHECK(copy(small, one, small) && length(small, 3) == 0 && good == 7);   // (sequence 1 stays as it is)
    const uint32_t zeros[] = {0, 0, 0, 0};
    CHECK(tensor_kv_cache_truncate(small, zeros, text, sizeof text) && reorder(small, TENSOR_DTYPE_U32, 2, 1, 4));
    icsdk::recorded = true;
    CHECK(reorder(small, TENSOR_DTYPE_U32, 2, 1, 4) && told_longest == 50);
    icsdk::recorded = false;

    // shared attention
    good = 9;
    const TensorBuffer q{TENSOR_DTYPE_F16, 4, {4, 4, 2, 16}}, out{TENSOR_DTYPE_F16, 4, {4, 4, 2, 16}};
    auto shared = [&](const TensorKvCache *p, const uint32_t *members, const uint32_t *n) {
        return tensor_kv_cache_attention_shared_f16(p, small, &q, members, n, 1.0f, 1, const_cast<TensorBuffer *>(&out),
                                                    text, sizeof text) != 0;
    };
    CHECK(!shared(small, nullptr, nullptr) && said("shared attention requires a prefix and another cache"));
    CHECK(!shared(nullptr, nullptr, nullptr) && said("shared attention requires a prefix"));
    CHECK(!shared(wide, nullptr, nullptr) && said("shared attention: the prefix's heads and dimensions"));
    CHECK(!shared(c, nullptr, nullptr) && said("shared attention: 3 sequences in equal groups, the cache has 4"));
    const uint32_t few[] = {1, 1, 1}, over[] = {4, 0xffffffffu, 1}, right[] = {0, 3, 1}, rows3[] = {2, 2, 3, 0};
    CHECK(!shared(c, few, nullptr) && said("shared attention: 3 sequences on the prefixes, the cache has 4"));
    CHECK(!shared(c, over, nullptr) && said("shared attention: 4294967300 sequences"));
    CHECK(!shared(c, right, rows3) && said("shared attention: a count exceeds the query rows") && good == 9);
    CHECK(shared(c, right, nullptr) && good == 8 && told_most == 3 && told_longest == 90 && told_batch == 4);
    const TensorBuffer huge{TENSOR_DTYPE_F16, 4, {4, 4, uint64_t{1} << 23, 16}};
    CHECK(!tensor_kv_cache_attention_shared_f16(c, small, &huge, right, nullptr, 1.0f, 1, const_cast<TensorBuffer *>(&out),
                                                text, sizeof text) && said("shared attention: query and output"));
    const TensorBuffer huge_out = huge;
    CHECK(!tensor_kv_cache_attention_shared_f16(c, small, &huge, right, nullptr, 1.0f, 1,
                                                const_cast<TensorBuffer *>(&huge_out), text, sizeof text) &&
          said("shared attention: too many query rows") && good == 8);
    icsdk::recorded = true;
    CHECK(!shared(c, right, nullptr) && said("shared attention: out of device memory"));   // (the stand-in has none)
    icsdk::recorded = false;
    tensor_kv_cache_free(c);
    tensor_kv_cache_free(small);
    tensor_kv_cache_free(large);
    tensor_kv_cache_free(wide);
    return 0;
}
"""


def test_lengths_and_refusals(tmp_path):
    if not os.path.isfile(COMPILER):
        pytest.skip("ROCm compiler absent")
    source, exe = tmp_path / "program.cpp", tmp_path / "program"
    source.write_text(PROGRAM)
    subprocess.run([COMPILER, "-std=c++17", "-x", "c++", "-D__HIP_PLATFORM_AMD__", "-isystem", HIP_INCLUDE, "-I", CSRC,
                    "-I", os.path.join(REPO, "include"), "-o", str(exe), str(source), os.path.join(CSRC, "kv_cache.cpp"),
                    os.path.join(CSRC, "kv_sequences.cpp"), "-pthread"], check=True)
    result = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert result.returncode == 0, result.stdout


@pytest.mark.parametrize("causal", [True, False])
def test_the_plain_shared_attention_by_direct_sums(causal):
    """Rows over a prefix's tokens and then own ones, one by one."""
    rng = np.random.default_rng(2)
    prefix, own = Model(2, 2, 5, 3), Model(3, 2, 5, 3)
    rows = [rng.standard_normal((b, 2, n, d)).astype(np.float16) for b, n in ((2, 70), (3, 9)) for d in (5, 3)]
    rows[0][1, 0, 66, 1] = np.nan
    prefix.append(*rows[:2], [70, 67])
    own.append(*rows[2:], [9, 2, 5])
    counts, members = [4, 2, 3], [1, 2]
    q = rng.standard_normal((3, 4, 4, 5)).astype(np.float32)
    out = beam_model.joined(prefix, own, members).attention(q, 0.6, causal, counts)[0]
    for b, p in enumerate((0, 1, 1)):
        for j in range(4):
            h = j // 2
            k = [None if m else row for x, i in ((prefix, p), (own, b)) for m, row in zip(x.marked[i][h], x.k[i][h].held())]
            v = [row for x, i in ((prefix, p), (own, b)) for row in x.v[i][h].held()]
            for i in range(counts[b]):
                seen = len(k) if not causal else prefix.length(p) + own.length(b) - counts[b] + i + 1
                want, _ = direct(q[b, j, i], k, v, 0.6, seen)
                assert np.isnan(out[b, j, i]).all() if want is None else np.abs(out[b, j, i] - want).max() < 1e-13
