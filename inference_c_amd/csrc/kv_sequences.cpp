// The key/value cache's entry points for several continuations of one prompt
// (include/tensor_kv_cache.h): sequences copied and reordered as they are held
// (k_kv_copy.hip), and attention over a prefix that sequences share
// (k_kv_shared.hip).
#include "kv_handle.hpp"

#include <cmath>
#include <memory>
#include <new>

using namespace icsdk;

namespace {

bool same_rows(const TensorKvCache *a, const TensorKvCache *b) {
    return a->view.heads == b->view.heads && a->view.dim == b->view.dim && a->view.vdim == b->view.vdim;
}

// Locks two caches, or the one that both are.
class Locked {
public:
    Locked(const TensorKvCache *a, const TensorKvCache *b)
        : a_(const_cast<TensorKvCache *>(a)), b_(a == b ? nullptr : const_cast<TensorKvCache *>(b)) {
        if (b_ != nullptr) std::lock(a_->mutex, b_->mutex);
        else a_->mutex.lock();
    }
    Locked(const Locked &) = delete;
    Locked &operator=(const Locked &) = delete;
    ~Locked() {
        a_->mutex.unlock();
        if (b_ != nullptr) b_->mutex.unlock();
    }

private:
    TensorKvCache *a_, *b_;
};

int copy(const TensorKvCache *from, const uint32_t *source, TensorKvCache *to, char *error, size_t capacity) {
    if (from == nullptr || to == nullptr || source == nullptr)
        return fail(error, capacity, "cache copy requires a cache, source sequences and a target");
    if (!same_rows(from, to))
        return fail(error, capacity, "cache copy: the target's heads and dimensions must be the cache's");
    const Locked lock(from, to);
    uint32_t longest = 0;
    size_t tokens = 0;
    bool any = false;
    // within one cache, a copy of itself is what a sequence is already
    auto keeps = [&](size_t b) { return source[b] == TENSOR_KV_CACHE_KEEP || (from == to && source[b] == b); };
    for (size_t b = 0; b < to->batch; ++b) {
        if (keeps(b)) continue;
        if (source[b] >= from->batch) {
            set_error(error, capacity, "cache copy: sequence %u of %zu", source[b], from->batch);
            return 0;
        }
        if (from == to && !keeps(source[b])) {
            set_error(error, capacity, "cache copy: sequence %u is copied from and to within one cache", source[b]);
            return 0;
        }
        const uint32_t n = from->length[source[b]];
        if (n > to->capacity) {
            set_error(error, capacity, "cache copy: sequence %u holds %u tokens, the target has room for %zu", source[b], n,
                      to->capacity);
            return 0;
        }
        longest = n > longest ? n : longest;
        tokens += n;
        any = true;
    }
    if (!any) return 1;
    if (!sdk_ready(error, capacity) || !not_recording("cache copy", error, capacity)) return 0;
    for (size_t first = 0; first < to->batch; first += kv::kBatchPerLaunch) {
        const uint32_t batch =
            (uint32_t)(to->batch - first < kv::kBatchPerLaunch ? to->batch - first : kv::kBatchPerLaunch);
        kv::Counts sources;
        bool here = false;
        for (uint32_t b = 0; b < batch; ++b) {
            sources.n[b] = keeps(first + b) ? kv::kKeep : source[first + b];
            here = here || sources.n[b] != kv::kKeep;
        }
        if (!here) continue;
        if (!hip_ok(kv::copy(from->view, to->view, (uint32_t)first, batch, sources, longest, tokens, sdk_stream()),
                    "cache copy: kernel launch", error, capacity))
            return 0;
        for (uint32_t b = 0; b < batch; ++b)
            if (sources.n[b] != kv::kKeep) to->length[first + b] = from->length[sources.n[b]];
    }
    return 1;
}

int reorder(TensorKvCache *c, Buf parents, char *error, size_t capacity) {
    if (c == nullptr) return fail(error, capacity, "cache reorder requires a cache");
    if (!device_tensor(parents, TENSOR_DTYPE_U32, 2))
        return fail(error, capacity, "cache reorder requires rank-2 U32 device parents");
    const uint64_t *shape = tensor_buffer_shape(parents);
    const size_t groups = shape[0], beams = shape[1];
    if (beams == 0 || beams > kv::kMaxBeams || groups != c->batch / beams || c->batch % beams != 0)
        return fail(error, capacity, "cache reorder: parents must be [groups, beams] with 1 to 64 beams, groups * beams the "
                    "cache's batch");
    std::lock_guard<std::mutex> lock(c->mutex);
    for (size_t b = 0; b < c->batch; ++b)
        if (c->length[b] != c->length[b / beams * beams]) {
            set_error(error, capacity, "cache reorder: the sequences of group %zu are not of one length", b / beams);
            return 0;
        }
    if (!sdk_ready(error, capacity)) return 0;
    // a recorded call is replayed on later lengths
    const uint32_t longest = sdk_recording() == Recording::kNo ? longest_of(c) : (uint32_t)c->capacity;
    if (longest == 0 || beams == 1) return 1;
    return hip_ok(kv::reorder(c->view, (uint32_t)groups, (uint32_t)beams, static_cast<const uint32_t *>(dev(parents)),
                              longest, sdk_stream()),
                  "cache reorder: kernel launch", error, capacity) ? 1 : 0;
}

// Query rows of a call, at most: a pass's launch holds fewer than 2^32 threads.
constexpr size_t kMaxSharedRows = size_t{1} << 26;

int attention_shared(TensorDType dtype, const TensorKvCache *prefix, const TensorKvCache *c, Buf query,
                     const uint32_t *members, const uint32_t *counts, float scale, int causal, TensorBuffer *output,
                     char *error, size_t capacity) {
    if (prefix == nullptr || c == nullptr || prefix == c)
        return fail(error, capacity, "shared attention requires a prefix and another cache of the sequences' own tokens");
    if (!device_tensor(query, dtype, 4) || !device_tensor(output, dtype, 4) || !std::isfinite(scale) ||
        (causal != 0 && causal != 1) || output == query) {
        set_error(error, capacity, "shared attention requires rank-4 %s device tensors, an output of its own, finite "
                  "scale, and causal 0 or 1", dtype == TENSOR_DTYPE_F32 ? "F32" : "F16");
        return 0;
    }
    if (!same_rows(prefix, c))
        return fail(error, capacity, "shared attention: the prefix's heads and dimensions must be the cache's");
    const uint64_t *qs = tensor_buffer_shape(query);
    const size_t heads = qs[1], n = qs[2];
    if (heads == 0 || heads % c->view.heads != 0 || !shaped(query, c->batch, heads, n, c->view.dim) ||
        !shaped(output, c->batch, heads, n, c->view.vdim))
        return fail(error, capacity, "shared attention: query and output must be [batch, query_heads, rows, dim] of the "
                    "cache, query_heads a multiple of its kv_heads");
    if (n != 0 && (heads > kMaxSharedRows / n || c->batch > kMaxSharedRows / (heads * n)))
        return fail(error, capacity, "shared attention: too many query rows");
    if (!counts_fit(c, counts, n)) return fail(error, capacity, "shared attention: a count exceeds the query rows");
    size_t sum = 0, most = 0;
    for (size_t p = 0; p < prefix->batch; ++p) {
        const size_t m = members ? members[p] : c->batch / prefix->batch;
        sum += m;
        most = m > most ? m : most;
    }
    if (sum != c->batch) {
        set_error(error, capacity, members ? "shared attention: %zu sequences on the prefixes, the cache has %zu"
                                           : "shared attention: %zu sequences in equal groups, the cache has %zu",
                  sum, c->batch);
        return 0;
    }
    if (n == 0) return 1;
    const Locked lock(prefix, c);
    if (!sdk_ready(error, capacity)) return 0;
    std::unique_ptr<uint32_t[]> equal;
    if (members == nullptr) {
        equal.reset(new (std::nothrow) uint32_t[prefix->batch]);
        if (!equal) return fail(error, capacity, "shared attention: out of memory");
        for (size_t p = 0; p < prefix->batch; ++p) equal[p] = (uint32_t)most;
        members = equal.get();
    }
    // a recorded call is replayed on later lengths
    const bool recording = sdk_recording() != Recording::kNo;
    const kv::PrefixShape over{(uint32_t)prefix->batch, (uint32_t)most,
                               recording ? (uint32_t)prefix->capacity : longest_of(prefix), members};
    const kv::AttentionShape shape{(uint32_t)c->batch, (uint32_t)heads, (uint32_t)n,
                                   recording ? (uint32_t)c->capacity : longest_of(c), scale, causal != 0, counts,
                                   nullptr, 0, 0};
    const bool f32 = dtype == TENSOR_DTYPE_F32;
    const size_t bytes = kv::attention_shared_workspace(f32, prefix->view, over, c->view, shape);
    ScratchBlock workspace(bytes);
    if (bytes != 0 && workspace.get() == nullptr)
        return fail(error, capacity, "shared attention: out of device memory for its workspace");
    return hip_ok(kv::attention_shared(f32, prefix->view, over, c->view, shape, dev(query), dev(output), workspace.get(),
                                       sdk_stream()),
                  "shared attention: kernel launch", error, capacity) ? 1 : 0;
}

}  // namespace

extern "C" {

int tensor_kv_cache_copy(const TensorKvCache *cache, const uint32_t *source, TensorKvCache *target, char *error,
                         size_t error_capacity) {
    return copy(cache, source, target, error, error_capacity);
}

int tensor_kv_cache_reorder(TensorKvCache *cache, const TensorBuffer *parents, char *error, size_t error_capacity) {
    return reorder(cache, parents, error, error_capacity);
}

int tensor_kv_cache_attention_shared_f32(const TensorKvCache *prefix, const TensorKvCache *cache,
                                         const TensorBuffer *query, const uint32_t *members, const uint32_t *counts,
                                         float scale, int causal, TensorBuffer *output, char *error,
                                         size_t error_capacity) {
    return attention_shared(TENSOR_DTYPE_F32, prefix, cache, query, members, counts, scale, causal, output, error,
                            error_capacity);
}

int tensor_kv_cache_attention_shared_f16(const TensorKvCache *prefix, const TensorKvCache *cache,
                                         const TensorBuffer *query, const uint32_t *members, const uint32_t *counts,
                                         float scale, int causal, TensorBuffer *output, char *error,
                                         size_t error_capacity) {
    return attention_shared(TENSOR_DTYPE_F16, prefix, cache, query, members, counts, scale, causal, output, error,
                            error_capacity);
}

}  // extern "C"
