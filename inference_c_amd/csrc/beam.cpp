// Beam search's choice over beams and vocabulary (include/tensor_ops_ext.h,
// tensor_beam_select_*): argument checks, staging of host operands, and the launches
// of k_beam.hip.
#include "kernels.hpp"
#include "sdk.hpp"
#include "staging.hpp"

#include "tensor_buffer.h"
#include "tensor_ops_ext.h"

using namespace icsdk;

namespace {

using Buf = const TensorBuffer *;

constexpr size_t kMaxVocab = size_t{1} << 26, kMaxRows = size_t{1} << 24;

bool is(Buf t, TensorDType dtype, size_t rank) {
    return t != nullptr && tensor_buffer_dtype(t) == dtype && tensor_buffer_rank(t) == rank;
}
bool shaped(Buf t, uint64_t a, uint64_t b) { return tensor_buffer_shape(t)[0] == a && tensor_buffer_shape(t)[1] == b; }

const void *in(Staging &st, Buf t) {
    if (t == nullptr) return nullptr;
    return st.host() ? st.in(tensor_buffer_data(t), tensor_buffer_byte_length(t)) : tensor_buffer_device_handle_internal(t);
}
void *out(Staging &st, TensorBuffer *t) {
    if (t == nullptr) return nullptr;
    return st.host() ? st.out(tensor_buffer_data_mut(t), tensor_buffer_byte_length(t))
                     : tensor_buffer_device_handle_internal(t);
}

int select(TensorDType dtype, Buf logits, Buf scores, Buf ended, uint32_t end_token, TensorBuffer *parents,
           TensorBuffer *tokens, TensorBuffer *new_scores, TensorBuffer *new_ended, char *error, size_t capacity) {
    if (!is(logits, dtype, 3) || !is(scores, TENSOR_DTYPE_F32, 2) ||
        (ended != nullptr && !is(ended, TENSOR_DTYPE_U32, 2)) || !is(parents, TENSOR_DTYPE_U32, 2) ||
        !is(tokens, TENSOR_DTYPE_U32, 2) || !is(new_scores, TENSOR_DTYPE_F32, 2) ||
        (new_ended != nullptr && !is(new_ended, TENSOR_DTYPE_U32, 2))) {
        set_error(error, capacity, "beam select requires rank-3 %s logits, rank-2 F32 scores, optional rank-2 U32 ended "
                  "flags, and rank-2 outputs: U32 parents and tokens, F32 scores, optional U32 ended flags",
                  dtype == TENSOR_DTYPE_F32 ? "F32" : "F16");
        return 0;
    }
    const uint64_t *shape = tensor_buffer_shape(logits);
    const size_t groups = shape[0], beams = shape[1], vocab = shape[2], keep = tensor_buffer_shape(parents)[1];
    if (beams == 0 || beams > k::kBeamMax || keep == 0 || keep > k::kBeamMaxKeep || vocab == 0 || vocab > kMaxVocab ||
        groups > kMaxRows / beams || end_token >= vocab) {
        set_error(error, capacity, "beam select requires 1 to 64 beams, 1 to 64 kept candidates, 1 to 2^26 tokens with the "
                  "end token among them, and at most 2^24 beams of all groups");
        return 0;
    }
    if (!shaped(scores, groups, beams) || (ended != nullptr && !shaped(ended, groups, beams)) ||
        !shaped(parents, groups, keep) || !shaped(tokens, groups, keep) || !shaped(new_scores, groups, keep) ||
        (new_ended != nullptr && !shaped(new_ended, groups, keep))) {
        set_error(error, capacity, "beam select: scores and ended flags must be [groups, beams] of the logits, and every "
                  "output [groups, keep]");
        return 0;
    }
    // (of one type and shape only scores and ended flags can be an output too)
    const bool apart = parents != tokens && parents != new_ended && tokens != new_ended &&
                       (ended == nullptr || ((Buf)parents != ended && (Buf)tokens != ended));
    if (!apart) {
        set_error(error, capacity, "beam select: outputs must be tensors of their own (new scores may be the scores, and "
                  "new ended flags the ended flags)");
        return 0;
    }
    const bool host = tensor_buffer_storage(logits) == TENSOR_BUFFER_STORAGE_HOST;
    for (Buf t : {logits, scores, ended, (Buf)parents, (Buf)tokens, (Buf)new_scores, (Buf)new_ended})
        if (t != nullptr && (tensor_buffer_storage(t) == TENSOR_BUFFER_STORAGE_HOST) != host) {
            set_error(error, capacity, "beam select operands must use the same storage type");
            return 0;
        }
    if (groups == 0) return 1;
    Staging st("beam select", host, error, capacity);
    if (!st.begin()) return 0;
    const void *px = in(st, logits), *ps = in(st, scores), *pe = in(st, ended);
    void *pp = out(st, parents), *pt = out(st, tokens), *pn = out(st, new_scores), *pd = out(st, new_ended);
    if (st.failed()) return 0;
    const k::BeamShape b{groups, beams, vocab, keep};
    const bool f32 = dtype == TENSOR_DTYPE_F32;
    ScratchBlock workspace(k::beam_select_workspace(b, f32));
    if (workspace.get() == nullptr) {
        set_error(error, capacity, "beam select: out of device memory for its workspace");
        return 0;
    }
    return st.finish(k::beam_select(f32, b, px, static_cast<const float *>(ps), static_cast<const uint32_t *>(pe), end_token,
                                    static_cast<uint32_t *>(pp), static_cast<uint32_t *>(pt), static_cast<float *>(pn),
                                    static_cast<uint32_t *>(pd), workspace.get(), st.stream())) ? 1 : 0;
}

}  // namespace

extern "C" {

int tensor_beam_select_f32(Buf logits, Buf scores, Buf ended, uint32_t end_token, TensorBuffer *parents,
                           TensorBuffer *tokens, TensorBuffer *new_scores, TensorBuffer *new_ended, char *error,
                           size_t capacity) {
    return select(TENSOR_DTYPE_F32, logits, scores, ended, end_token, parents, tokens, new_scores, new_ended, error, capacity);
}
int tensor_beam_select_f16(Buf logits, Buf scores, Buf ended, uint32_t end_token, TensorBuffer *parents,
                           TensorBuffer *tokens, TensorBuffer *new_scores, TensorBuffer *new_ended, char *error,
                           size_t capacity) {
    return select(TENSOR_DTYPE_F16, logits, scores, ended, end_token, parents, tokens, new_scores, new_ended, error, capacity);
}

}  // extern "C"
