// The 8-bit key/value cache in device memory, and the launchers of its kernels
// (k_kv_cache.hip: append, read, truncate, evict; k_kv_copy.hip: copy, reorder;
// k_kv_attention.hip: attention; k_kv_shared.hip: attention over a shared prefix).
//
// Of each (sequence, kv head), in blocks of 64 tokens:
//   k     [block][token][kp]   codes + 128 as bytes, kp = head dim in whole 16s
//   v     [block][dim][64]     likewise, the tokens of a dim side by side, vp =
//                              value dim in whole 16s
//   meta  [block]              scales and the mark bits of the block's tokens
//   kt    [token][kp], vt [dim][64]   the open block in f16
// Keys lie by token and values by dim because that is how the two matrix
// products of attention read them: a lane's 16 bytes of k are 16 dims of one
// key, its 16 bytes of v 16 keys of one dim, and both go into MFMA operands as
// they come. Codes and f16 are zeros at creation, columns past the dims stay that,
// and every f16 in kt and vt is finite, so rows and columns past the data may be
// read: their products are dropped or meet zeros.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace icsdk {
namespace kv {

constexpr uint32_t kTokens = 64;       // tokens per block
constexpr uint32_t kMaxDim = 256;
constexpr uint32_t kBatchPerLaunch = 256;

struct Meta {
    float k_scale, v_scale;
    uint64_t marked;   // bit t: token t is marked (its score is NaN)
};

struct View {
    uint8_t *k, *v;
    Meta *meta;
    _Float16 *kt, *vt;
    uint32_t *length;              // [batch]
    uint32_t heads, blocks;        // blocks per (sequence, head)
    uint32_t dim, vdim, kp, vp;
};

// Per-sequence numbers of one launch, passed by value.
struct Counts {
    uint32_t n[kBatchPerLaunch];
};

// Sequences first .. first + batch - 1: from start[b] on, count[b] tokens of
// key / value rows [b][head][row of n]. length[b] becomes start + count.
hipError_t append(bool f32, const View &c, uint32_t first, uint32_t batch, const void *key, const void *value,
                  uint32_t n, const Counts &start, const Counts &count, hipStream_t s);
// Lengths from `from` to `to` (not above); cut blocks are opened.
hipError_t truncate(const View &c, uint32_t first, uint32_t batch, const Counts &from, const Counts &to,
                    hipStream_t s);
// Rows of the outputs (either may be null); `longest` bounds the lengths.
hipError_t read(bool f32, const View &c, uint32_t batch, void *key, void *value, uint32_t rows, uint32_t longest,
                hipStream_t s);

struct EvictArgs {
    const float *weights;   // [batch, heads, tokens] or null
    uint32_t tokens, first, recent, keep;
    float *target_weights;  // [batch, heads, slots] or null
    uint32_t *kept;         // likewise
    uint32_t slots;
    uint32_t *index;        // workspace [batch, heads, keep_most]
    uint32_t keep_most;     // min(keep, longest length)
    uint32_t longest;
};
hipError_t evict(const View &from, const View &to, uint32_t batch, const EvictArgs &a, hipStream_t s);

// Sequences first .. first + batch - 1 of `to` become copies of sequences source[b] of
// `from` (kKeep: stay as they are); `longest` bounds the sources' lengths, `tokens` are
// all that the call copies. `to` may be `from` where no sequence is both read and written.
constexpr uint32_t kKeep = 0xffffffffu;
hipError_t copy(const View &from, const View &to, uint32_t first, uint32_t batch, const Counts &source, uint32_t longest,
                size_t tokens, hipStream_t s);
// In each group of `beams` sequences (of one length, at most `longest`), sequence i
// becomes what sequence parents[i] was.
constexpr uint32_t kMaxBeams = 64;
hipError_t reorder(const View &c, uint32_t groups, uint32_t beams, const uint32_t *parents, uint32_t longest,
                   hipStream_t s);

struct AttentionShape {
    uint32_t batch, q_heads, n;   // n query rows per head
    uint32_t longest;             // bound of the lengths, for the plan
    float scale;
    bool causal;
    const uint32_t *counts;       // host [batch] or null
    float *weights;               // [batch, heads, weight_stride] or null
    uint32_t weight_tokens;       // of each row, those that a token may have
    size_t weight_stride;
};
// Bytes of workspace of a call (0: none).
size_t attention_workspace(bool f32, const View &c, const AttentionShape &a);
hipError_t attention(bool f32, const View &c, const AttentionShape &a, const void *query, void *output,
                     void *workspace, hipStream_t s);

// The same with the tokens of `prefix` before each sequence's own: sequences of `c`
// lie in groups, one per sequence of the prefix, of members[p] each (host; `most`: the
// largest). No weights.
struct PrefixShape {
    uint32_t batch, most, longest;
    const uint32_t *members;
};
// Rows that a launch of its parts' join takes, a thread for each four of their elements:
// fewer than 2^32 threads.
constexpr uint32_t join_rows(uint32_t vdim) { return (1u << 31) / ((vdim + 3) / 4); }
size_t attention_shared_workspace(bool f32, const View &prefix, const PrefixShape &p, const View &c,
                                  const AttentionShape &a);
hipError_t attention_shared(bool f32, const View &prefix, const PrefixShape &p, const View &c, const AttentionShape &a,
                            const void *query, void *output, void *workspace, hipStream_t s);

}  // namespace kv
}  // namespace icsdk
