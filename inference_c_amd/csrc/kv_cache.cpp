// The 8-bit key/value cache's entry points (include/tensor_kv_cache.h): handles,
// argument checks, and the launches of k_kv_cache.hip and k_kv_attention.hip.
//
// Every length is held twice: on the host, for the checks and the launch plans,
// and on the device, where the kernels that change a cache set it and the
// others read it (so that a recorded read or attention works on what the cache
// holds when it is replayed).
#include "kv.hpp"
#include "sdk.hpp"

#include "tensor_kv_cache.h"

#include <climits>
#include <cmath>
#include <cstdlib>
#include <mutex>
#include <new>

using namespace icsdk;

struct TensorKvCache {
    std::mutex mutex;
    size_t batch, capacity, bytes;
    kv::View view;
    void *memory;
    uint32_t *length;   // [batch]
};

namespace {

using Buf = const TensorBuffer *;

// A launch has fewer than 2^32 threads in a dimension: one for each token (of all
// sequences and heads: the fold's), or 32 for each of a head's (the weights': 16
// parts of its blocks in fours, 256 threads each).
constexpr size_t kMaxCapacity = size_t{1} << 27, kMaxTokens = size_t{1} << 31;
constexpr size_t kMaxBatch = 65535, kMaxHeads = 4096;

int fail(char *error, size_t capacity, const char *message) {
    set_error(error, capacity, "%s", message);
    return 0;
}

size_t round_up(size_t n, size_t to) { return (n + to - 1) / to * to; }

// Sizes of the cache's arrays one after another, or false where there are too many
// tokens.
struct Layout {
    size_t k, v, meta, kt, vt, length, total;
};
bool layout_of(size_t batch, size_t heads, size_t blocks, size_t kp, size_t vp, Layout *l) {
    const size_t pairs = batch * heads;   // below 2^28
    const size_t tokens = pairs * blocks * kv::kTokens;
    if (tokens > kMaxTokens) return false;
    l->k = 0;
    l->v = l->k + round_up(tokens * kp, 256);
    l->meta = l->v + round_up(tokens * vp, 256);
    l->kt = l->meta + round_up(pairs * blocks * sizeof(kv::Meta), 256);
    l->vt = l->kt + round_up(pairs * kv::kTokens * kp * 2, 256);
    l->length = l->vt + round_up(pairs * kv::kTokens * vp * 2, 256);
    l->total = l->length + round_up(batch * 4, 256);
    return true;
}

bool device_tensor(Buf t, TensorDType dtype, size_t rank) {
    return t != nullptr && tensor_buffer_dtype(t) == dtype && tensor_buffer_rank(t) == rank &&
           tensor_buffer_storage(t) == TENSOR_BUFFER_STORAGE_DEVICE;
}

bool shaped(Buf t, size_t a, size_t b, size_t c) {
    const uint64_t *s = tensor_buffer_shape(t);
    return s[0] == a && s[1] == b && s[2] == c;
}

bool shaped(Buf t, size_t a, size_t b, size_t c, size_t d) {
    return shaped(t, a, b, c) && tensor_buffer_shape(t)[3] == d;
}

void *dev(Buf t) { return t ? tensor_buffer_device_handle_internal(t) : nullptr; }

// A call that changes lengths cannot be replayed: the host's lengths would not
// follow.
bool not_recording(const char *what, char *error, size_t capacity) {
    if (sdk_recording() == Recording::kNo) return true;
    set_error(error, capacity, "%s changes the cache's lengths and cannot be recorded into a graph", what);
    return false;
}

uint32_t longest_of(const TensorKvCache *c) {
    uint32_t n = 0;
    for (size_t b = 0; b < c->batch; ++b) n = c->length[b] > n ? c->length[b] : n;
    return n;
}

// counts[b] <= n for every sequence
bool counts_fit(const TensorKvCache *c, const uint32_t *counts, size_t n) {
    for (size_t b = 0; counts != nullptr && b < c->batch; ++b)
        if (counts[b] > n) return false;
    return true;
}

int append(TensorDType dtype, TensorKvCache *c, Buf key, Buf value, const uint32_t *counts, char *error,
           size_t capacity) {
    if (c == nullptr) return fail(error, capacity, "cache append requires a cache");
    if (!device_tensor(key, dtype, 4) || !device_tensor(value, dtype, 4)) {
        set_error(error, capacity, "cache append requires rank-4 %s device tensors",
                  dtype == TENSOR_DTYPE_F32 ? "F32" : "F16");
        return 0;
    }
    const size_t n = tensor_buffer_shape(key)[2];
    if (!shaped(key, c->batch, c->view.heads, n, c->view.dim) ||
        !shaped(value, c->batch, c->view.heads, n, c->view.vdim))
        return fail(error, capacity, "cache append: key and value must be [batch, kv_heads, tokens, dim] of the cache");
    if (!counts_fit(c, counts, n)) return fail(error, capacity, "cache append: a count exceeds the tokens given");
    std::lock_guard<std::mutex> lock(c->mutex);
    for (size_t b = 0; b < c->batch; ++b) {
        const size_t add = counts ? counts[b] : n;
        if (add > c->capacity - c->length[b]) {
            set_error(error, capacity, "cache append: sequence %zu holds %u of %zu tokens, no room for %zu", b,
                      c->length[b], c->capacity, add);
            return 0;
        }
    }
    if (n > INT_MAX) return fail(error, capacity, "cache append: too many tokens");
    if (n == 0) return 1;
    if (!sdk_ready(error, capacity) || !not_recording("cache append", error, capacity)) return 0;
    for (size_t first = 0; first < c->batch; first += kv::kBatchPerLaunch) {
        const uint32_t batch = (uint32_t)(c->batch - first < kv::kBatchPerLaunch ? c->batch - first : kv::kBatchPerLaunch);
        kv::Counts start, count;
        for (uint32_t b = 0; b < batch; ++b) {
            start.n[b] = c->length[first + b];
            count.n[b] = counts ? counts[first + b] : (uint32_t)n;
        }
        if (!hip_ok(kv::append(dtype == TENSOR_DTYPE_F32, c->view, (uint32_t)first, batch, dev(key), dev(value),
                               (uint32_t)n, start, count, sdk_stream()),
                    "cache append: kernel launch", error, capacity))
            return 0;
        for (uint32_t b = 0; b < batch; ++b) c->length[first + b] += count.n[b];
    }
    return 1;
}

int read(TensorDType dtype, const TensorKvCache *c, TensorBuffer *key, TensorBuffer *value, char *error,
         size_t capacity) {
    if (c == nullptr) return fail(error, capacity, "cache read requires a cache");
    if ((key == nullptr && value == nullptr) || (key != nullptr && !device_tensor(key, dtype, 4)) ||
        (value != nullptr && !device_tensor(value, dtype, 4)) || key == value) {
        set_error(error, capacity, "cache read requires rank-4 %s device tensors, one for each output",
                  dtype == TENSOR_DTYPE_F32 ? "F32" : "F16");
        return 0;
    }
    const size_t rows = tensor_buffer_shape(key ? key : value)[2];
    if ((key != nullptr && !shaped(key, c->batch, c->view.heads, rows, c->view.dim)) ||
        (value != nullptr && !shaped(value, c->batch, c->view.heads, rows, c->view.vdim)))
        return fail(error, capacity, "cache read: key and value must be [batch, kv_heads, rows, dim] of the cache");
    TensorKvCache *const held = const_cast<TensorKvCache *>(c);
    std::lock_guard<std::mutex> lock(held->mutex);
    if (rows < longest_of(c)) return fail(error, capacity, "cache read: fewer rows than the longest sequence has tokens");
    if (rows > INT_MAX) return fail(error, capacity, "cache read: too many rows");
    if (rows == 0) return 1;
    if (!sdk_ready(error, capacity)) return 0;
    // a recorded call is replayed on later lengths: those the outputs have room for
    const size_t most = sdk_recording() == Recording::kNo ? longest_of(c) : c->capacity;
    const uint32_t fits = (uint32_t)(rows < c->capacity ? rows : c->capacity);
    return hip_ok(kv::read(dtype == TENSOR_DTYPE_F32, c->view, (uint32_t)c->batch, dev(key), dev(value), (uint32_t)rows,
                           most < fits ? (uint32_t)most : fits, sdk_stream()),
                  "cache read: kernel launch", error, capacity) ? 1 : 0;
}

int attention(TensorDType dtype, const TensorKvCache *c, Buf query, const uint32_t *counts, float scale, int causal,
              TensorBuffer *weights, TensorBuffer *output, char *error, size_t capacity) {
    if (c == nullptr) return fail(error, capacity, "cache attention requires a cache");
    if (!device_tensor(query, dtype, 4) || !device_tensor(output, dtype, 4) ||
        (weights != nullptr && !device_tensor(weights, TENSOR_DTYPE_F32, 3)) || !std::isfinite(scale) ||
        (causal != 0 && causal != 1) || output == query) {
        set_error(error, capacity, "cache attention requires rank-4 %s device tensors, an output of its own, finite "
                  "scale, causal 0 or 1, and optional rank-3 F32 device weights",
                  dtype == TENSOR_DTYPE_F32 ? "F32" : "F16");
        return 0;
    }
    const uint64_t *qs = tensor_buffer_shape(query);
    const size_t heads = qs[1], n = qs[2];
    if (heads == 0 || heads % c->view.heads != 0 || !shaped(query, c->batch, heads, n, c->view.dim) ||
        !shaped(output, c->batch, heads, n, c->view.vdim))
        return fail(error, capacity, "cache attention: query and output must be [batch, query_heads, rows, dim] of the "
                    "cache, query_heads a multiple of its kv_heads");
    if (n != 0 && heads > (size_t)INT_MAX / n) return fail(error, capacity, "cache attention: too many query rows");
    if (!counts_fit(c, counts, n)) return fail(error, capacity, "cache attention: a count exceeds the query rows");
    TensorKvCache *const held = const_cast<TensorKvCache *>(c);
    std::lock_guard<std::mutex> lock(held->mutex);
    size_t tokens = 0;
    if (weights != nullptr) {
        tokens = tensor_buffer_shape(weights)[2];
        if (!shaped(weights, c->batch, c->view.heads, tokens) || tokens < longest_of(c))
            return fail(error, capacity, "cache attention: weights must be [batch, kv_heads, tokens] with room for the "
                        "longest sequence");
    }
    if (n == 0) return 1;
    if (!sdk_ready(error, capacity)) return 0;
    const bool recording = sdk_recording() != Recording::kNo;
    const kv::AttentionShape shape{(uint32_t)c->batch, (uint32_t)heads, (uint32_t)n,
                                   recording ? (uint32_t)c->capacity : longest_of(c), scale, causal != 0, counts,
                                   static_cast<float *>(dev(weights)),
                                   (uint32_t)(tokens < c->capacity ? tokens : c->capacity), tokens};
    const size_t bytes = kv::attention_workspace(dtype == TENSOR_DTYPE_F32, c->view, shape);
    ScratchBlock workspace(bytes);
    if (bytes != 0 && workspace.get() == nullptr)
        return fail(error, capacity, "cache attention: out of device memory for its workspace");
    return hip_ok(kv::attention(dtype == TENSOR_DTYPE_F32, c->view, shape, dev(query), dev(output), workspace.get(),
                                sdk_stream()),
                  "cache attention: kernel launch", error, capacity) ? 1 : 0;
}

}  // namespace

extern "C" {

int tensor_kv_cache_create(size_t batch, size_t kv_heads, size_t capacity, size_t head_dim, size_t value_dim,
                           TensorKvCache **result, char *error, size_t error_capacity) {
    if (result != nullptr) *result = nullptr;
    if (result == nullptr || batch == 0 || batch > kMaxBatch || kv_heads == 0 || kv_heads > kMaxHeads || capacity == 0 ||
        capacity > kMaxCapacity || head_dim == 0 || head_dim > kv::kMaxDim || value_dim == 0 || value_dim > kv::kMaxDim)
        return fail(error, error_capacity, "cache requires a result pointer, 1 to 65535 sequences, 1 to 4096 heads, 1 to "
                    "2^27 tokens, and head and value dimensions of 1 to 256");
    const size_t blocks = (capacity + kv::kTokens - 1) / kv::kTokens;
    const size_t kp = round_up(head_dim, 16), vp = round_up(value_dim, 16);
    Layout l;
    if (!layout_of(batch, kv_heads, blocks, kp, vp, &l))
        return fail(error, error_capacity, "cache requires at most 2^31 tokens (in whole blocks) of all sequences and heads together");
    if (!sdk_ready(error, error_capacity)) return 0;
    if (sdk_recording() != Recording::kNo)
        return fail(error, error_capacity, "a cache cannot be created while a graph is recorded");
    auto *c = new (std::nothrow) TensorKvCache;
    uint32_t *length = static_cast<uint32_t *>(std::calloc(batch, sizeof(uint32_t)));
    if (c == nullptr || length == nullptr) {
        delete c;
        std::free(length);
        return fail(error, error_capacity, "out of memory creating cache");
    }
    char *memory = nullptr;
    if (!hip_ok(hipMalloc(reinterpret_cast<void **>(&memory), l.total), "cache: hipMalloc", error, error_capacity)) {
        delete c;
        std::free(length);
        return 0;
    }
    // columns past the dims are codes of 0 and zeros: they count in no block's largest
    // value, and meet a zero of q as what they are
    if (!hip_ok(hipMemsetAsync(memory, 128, l.meta, sdk_stream()), "cache: hipMemsetAsync", error, error_capacity) ||
        !hip_ok(hipMemsetAsync(memory + l.meta, 0, l.total - l.meta, sdk_stream()), "cache: hipMemsetAsync", error,
                error_capacity)) {
        (void)hipFree(memory);
        delete c;
        std::free(length);
        return 0;
    }
    c->batch = batch;
    c->capacity = capacity;
    c->bytes = l.total;
    c->memory = memory;
    c->length = length;
    c->view = kv::View{reinterpret_cast<uint8_t *>(memory + l.k), reinterpret_cast<uint8_t *>(memory + l.v),
                       reinterpret_cast<kv::Meta *>(memory + l.meta), reinterpret_cast<_Float16 *>(memory + l.kt),
                       reinterpret_cast<_Float16 *>(memory + l.vt), reinterpret_cast<uint32_t *>(memory + l.length),
                       (uint32_t)kv_heads, (uint32_t)blocks, (uint32_t)head_dim, (uint32_t)value_dim, (uint32_t)kp,
                       (uint32_t)vp};
    *result = c;
    return 1;
}

void tensor_kv_cache_free(TensorKvCache *cache) {
    if (cache == nullptr) return;
    bind_device();
    (void)hipStreamSynchronize(sdk_stream());   // queued kernels may still use it
    (void)hipFree(cache->memory);
    std::free(cache->length);
    delete cache;
}

size_t tensor_kv_cache_length(const TensorKvCache *cache, size_t sequence) {
    if (cache == nullptr || sequence >= cache->batch) return 0;
    std::lock_guard<std::mutex> lock(const_cast<TensorKvCache *>(cache)->mutex);
    return cache->length[sequence];
}

size_t tensor_kv_cache_capacity(const TensorKvCache *cache) { return cache ? cache->capacity : 0; }

size_t tensor_kv_cache_byte_length(const TensorKvCache *cache) { return cache ? cache->bytes : 0; }

int tensor_kv_cache_append_f32(TensorKvCache *cache, const TensorBuffer *key, const TensorBuffer *value,
                               const uint32_t *counts, char *error, size_t error_capacity) {
    return append(TENSOR_DTYPE_F32, cache, key, value, counts, error, error_capacity);
}

int tensor_kv_cache_append_f16(TensorKvCache *cache, const TensorBuffer *key, const TensorBuffer *value,
                               const uint32_t *counts, char *error, size_t error_capacity) {
    return append(TENSOR_DTYPE_F16, cache, key, value, counts, error, error_capacity);
}

int tensor_kv_cache_truncate(TensorKvCache *cache, const uint32_t *lengths, char *error, size_t error_capacity) {
    if (cache == nullptr) return fail(error, error_capacity, "cache truncate requires a cache");
    std::lock_guard<std::mutex> lock(cache->mutex);
    for (size_t b = 0; lengths != nullptr && b < cache->batch; ++b)
        if (lengths[b] > cache->length[b]) {
            set_error(error, error_capacity, "cache truncate: sequence %zu holds %u tokens, not %u", b, cache->length[b],
                      lengths[b]);
            return 0;
        }
    if (!sdk_ready(error, error_capacity) || !not_recording("cache truncate", error, error_capacity)) return 0;
    for (size_t first = 0; first < cache->batch; first += kv::kBatchPerLaunch) {
        const uint32_t batch =
            (uint32_t)(cache->batch - first < kv::kBatchPerLaunch ? cache->batch - first : kv::kBatchPerLaunch);
        kv::Counts from, to;
        for (uint32_t b = 0; b < batch; ++b) {
            from.n[b] = cache->length[first + b];
            to.n[b] = lengths ? lengths[first + b] : 0;
        }
        if (!hip_ok(kv::truncate(cache->view, (uint32_t)first, batch, from, to, sdk_stream()),
                    "cache truncate: kernel launch", error, error_capacity))
            return 0;
        for (uint32_t b = 0; b < batch; ++b) cache->length[first + b] = to.n[b];
    }
    return 1;
}

int tensor_kv_cache_read_f32(const TensorKvCache *cache, TensorBuffer *key, TensorBuffer *value, char *error,
                             size_t error_capacity) {
    return read(TENSOR_DTYPE_F32, cache, key, value, error, error_capacity);
}

int tensor_kv_cache_read_f16(const TensorKvCache *cache, TensorBuffer *key, TensorBuffer *value, char *error,
                             size_t error_capacity) {
    return read(TENSOR_DTYPE_F16, cache, key, value, error, error_capacity);
}

int tensor_kv_cache_attention_f32(const TensorKvCache *cache, const TensorBuffer *query, const uint32_t *counts,
                                  float scale, int causal, TensorBuffer *weights, TensorBuffer *output, char *error,
                                  size_t error_capacity) {
    return attention(TENSOR_DTYPE_F32, cache, query, counts, scale, causal, weights, output, error, error_capacity);
}

int tensor_kv_cache_attention_f16(const TensorKvCache *cache, const TensorBuffer *query, const uint32_t *counts,
                                  float scale, int causal, TensorBuffer *weights, TensorBuffer *output, char *error,
                                  size_t error_capacity) {
    return attention(TENSOR_DTYPE_F16, cache, query, counts, scale, causal, weights, output, error, error_capacity);
}

int tensor_kv_cache_evict(const TensorKvCache *cache, const TensorBuffer *weights, size_t first, size_t recent,
                          size_t keep, TensorKvCache *target, TensorBuffer *target_weights, TensorBuffer *kept,
                          char *error, size_t error_capacity) {
    if (cache == nullptr || target == nullptr || cache == target)
        return fail(error, error_capacity, "cache evict requires a cache and another one as its target");
    TensorKvCache *const source = const_cast<TensorKvCache *>(cache);
    if (target->batch != source->batch || target->view.heads != source->view.heads ||
        target->view.dim != source->view.dim || target->view.vdim != source->view.vdim)
        return fail(error, error_capacity, "cache evict: the target's batch, heads and dimensions must be the cache's");
    if (keep == 0 || keep > target->capacity || first > keep || recent > keep - first)
        return fail(error, error_capacity, "cache evict: keep must be positive, within the target's capacity and no less "
                    "than first + recent");
    if ((weights != nullptr && !device_tensor(weights, TENSOR_DTYPE_F32, 3)) ||
        (target_weights != nullptr && (!device_tensor(target_weights, TENSOR_DTYPE_F32, 3) || weights == nullptr ||
                                       target_weights == weights)) ||
        (kept != nullptr && !device_tensor(kept, TENSOR_DTYPE_U32, 3)))
        return fail(error, error_capacity, "cache evict: weights and target weights must be distinct rank-3 F32, kept "
                    "indices rank-3 U32 device tensors, and target weights need weights");
    std::scoped_lock lock(source->mutex, target->mutex);
    const size_t longest = longest_of(source), most = keep < longest ? keep : longest;
    const size_t heads = source->view.heads;
    size_t tokens = 0, slots = 0;
    if (weights != nullptr) {
        tokens = tensor_buffer_shape(weights)[2];
        if (!shaped(weights, source->batch, heads, tokens) || tokens < longest)
            return fail(error, error_capacity, "cache evict: weights must be [batch, kv_heads, tokens] with a weight for "
                        "every token");
    }
    for (Buf t : {(Buf)target_weights, (Buf)kept}) {
        if (t == nullptr) continue;
        const size_t n = tensor_buffer_shape(t)[2];
        if (!shaped(t, source->batch, heads, n) || n < most || (slots != 0 && n != slots))
            return fail(error, error_capacity, "cache evict: target weights and kept indices must be [batch, kv_heads, "
                        "slots] with a slot for every kept token");
        slots = n;
    }
    if (!sdk_ready(error, error_capacity) || !not_recording("cache evict", error, error_capacity)) return 0;
    if (slots > UINT32_MAX || tokens > UINT32_MAX)
        return fail(error, error_capacity, "cache evict: too many tokens or slots");
    const size_t bytes = source->batch * heads * most * sizeof(uint32_t);
    ScratchBlock workspace(bytes);
    if (bytes != 0 && workspace.get() == nullptr)
        return fail(error, error_capacity, "cache evict: out of device memory for its workspace");
    const kv::EvictArgs a{static_cast<const float *>(dev(weights)), (uint32_t)tokens, (uint32_t)first, (uint32_t)recent,
                          (uint32_t)keep, static_cast<float *>(dev(target_weights)), static_cast<uint32_t *>(dev(kept)),
                          (uint32_t)slots, static_cast<uint32_t *>(workspace.get()), (uint32_t)most,
                          (uint32_t)longest};
    if (!hip_ok(kv::evict(source->view, target->view, (uint32_t)source->batch, a, sdk_stream()),
                "cache evict: kernel launch", error, error_capacity))
        return 0;
    for (size_t b = 0; b < source->batch; ++b)
        target->length[b] = source->length[b] < keep ? source->length[b] : (uint32_t)keep;
    return 1;
}

}  // extern "C"
