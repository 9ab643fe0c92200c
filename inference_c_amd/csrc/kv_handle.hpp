// The key/value cache's handle, and the checks that its entry points share
// (kv_cache.cpp, kv_sequences.cpp).
#pragma once

#include "kv.hpp"
#include "sdk.hpp"

#include "tensor_kv_cache.h"

#include <mutex>

struct TensorKvCache {
    std::mutex mutex;
    size_t batch, capacity, bytes;
    icsdk::kv::View view;
    void *memory;
    uint32_t *length;   // [batch]
};

namespace icsdk {

using Buf = const TensorBuffer *;

inline int fail(char *error, size_t capacity, const char *message) {
    set_error(error, capacity, "%s", message);
    return 0;
}

inline bool device_tensor(Buf t, TensorDType dtype, size_t rank) {
    return t != nullptr && tensor_buffer_dtype(t) == dtype && tensor_buffer_rank(t) == rank &&
           tensor_buffer_storage(t) == TENSOR_BUFFER_STORAGE_DEVICE;
}

inline bool shaped(Buf t, size_t a, size_t b, size_t c) {
    const uint64_t *s = tensor_buffer_shape(t);
    return s[0] == a && s[1] == b && s[2] == c;
}

inline bool shaped(Buf t, size_t a, size_t b, size_t c, size_t d) {
    return shaped(t, a, b, c) && tensor_buffer_shape(t)[3] == d;
}

inline void *dev(Buf t) { return t ? tensor_buffer_device_handle_internal(t) : nullptr; }

// A call that changes lengths cannot be replayed: the host's lengths would not
// follow.
inline bool not_recording(const char *what, char *error, size_t capacity) {
    if (sdk_recording() == Recording::kNo) return true;
    set_error(error, capacity, "%s changes the cache's lengths and cannot be recorded into a graph", what);
    return false;
}

inline uint32_t longest_of(const TensorKvCache *c) {
    uint32_t n = 0;
    for (size_t b = 0; b < c->batch; ++b) n = c->length[b] > n ? c->length[b] : n;
    return n;
}

// counts[b] <= n for every sequence
inline bool counts_fit(const TensorKvCache *c, const uint32_t *counts, size_t n) {
    for (size_t b = 0; counts != nullptr && b < c->batch; ++b)
        if (counts[b] > n) return false;
    return true;
}

}  // namespace icsdk
