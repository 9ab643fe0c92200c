// What the kernels of attention over the 8-bit cache share: arguments, the codes
// as f16, the rules of rows, outputs and weights (kv_rows.hpp describes them;
// kv_tiles.hpp has the kernel for many rows), and the plan.
#pragma once

#include "kern_common.hpp"
#include "kv.hpp"

namespace icsdk {
namespace kv {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWaves = 4;
constexpr uint32_t kRows = 16;         // packed rows of a wave
constexpr double kLog2e = 1.4426950408889634;
constexpr float kTiny = 1.1754944e-38f, kHuge = 3.0e38f;   // what a factor of raw products is kept between
constexpr float kUnitRange = 8.0f;     // a value scale further from the unit moves it
// f16: P of a row whose maximum is M is 2^(s - M + kHeadroom): as far up as the unit's
// range and the lazy rescale of the maximum (by more than 2^kLazy) leave room for, 2^15
// in all, so that small weights keep their bits: absolute errors of P, relative to the
// row's largest, are below 2^-26 (P is rounded to 2^-11 anyway). f32, whose maximum
// is never left behind: the weight 2^(s - M), with its exponent near 0 for the largest
// ones, times kPairScale; errors below 2^-34.
template <typename S> constexpr float kLazy = sizeof(S) == 4 ? 0.0f : 8.0f;
template <typename S> constexpr float kHeadroom = sizeof(S) == 4 ? 0.0f : 4.0f;
template <typename S> constexpr float kPairScale = sizeof(S) == 4 ? 4096.0f : 1.0f;

// Arguments of a launch over sequences first .. (pairs / heads of them).
template <typename S> struct Args {
    View c;
    const S *q;
    S *out;
    float *part_o;       // [part][row][vdim], rows of all sequences
    f32x2 *part_ml;      // [part][row] running maximum (log2 units) and sum
    float *part_exact;   // [part][row] sum of the weights before P's rounding, or null
    f32x2 *row_ml;       // [row] maximum and 1 / sum (0: the row adds no weight), or null
    float *weights;
    float *scores;       // [row][score_stride] scores in log2 units, or null
    size_t rows;         // of all sequences
    size_t score_stride;
    size_t weight_stride;
    uint32_t weight_tokens;
    uint32_t first, pairs, group, n, parts, row_group0, row_groups, longest;
    double scale2;       // scale * log2 e
    int causal;
    Counts count;
};

// Of a pass of attention over a prefix and own tokens (k_kv_shared.hip), whose rows'
// parts meet another pass's. Over a prefix, a packed row of (sequence first + b, head) of
// the pass's cache is row r % own_rows of that head of sequence count.n[b] + r / own_rows
// of q and the parts: `count` has where the groups start. Over own tokens, own_rows is 0
// and all is as in Args. Outputs are parts, however few.
template <typename S> struct SharedArgs : Args<S> {
    uint32_t own_rows;   // packed rows of a sequence and head
    uint32_t last;       // where the last group of the launch ends
    uint32_t columns;    // of a head, workgroups of the rows kernel
    // Over a prefix, where some of the query heads' n rows are padding: n (else 0), and
    // every sequence's count (null: the other pass's `count`, which follows, has them).
    uint32_t padded;
    const uint32_t *counts;
};
// Arguments where a kernel finds them: memory that nothing writes.
template <typename A> using Constant = const __attribute__((address_space(4))) A;
template <typename A> __device__ inline Constant<A> &kernel_arguments(uint32_t offset) {
    return *(Constant<A> *)((const __attribute__((address_space(4))) char *)__builtin_amdgcn_kernarg_segment_ptr() + offset);
}
template <typename A> constexpr bool kIsShared = false;
template <typename S> constexpr bool kIsShared<Constant<SharedArgs<S>>> = true;

// How many of a query head's rows are there.
template <typename S> __device__ inline uint32_t rows_there(Constant<Args<S>> &a, uint32_t b) { return a.count.n[b]; }
template <typename S> __device__ inline uint32_t rows_there(Constant<SharedArgs<S>> &a, uint32_t b) {
    if (a.own_rows == 0) return a.count.n[b];
    // (over a prefix `count` has where the groups start)
    const uint32_t end = (b + 1) * a.c.heads < a.pairs ? a.count.n[b + 1] : a.last;
    return (end - a.count.n[b]) * a.own_rows;
}
// The packed row that a lane of row r (i of its query head) loads: of padding, and of rows
// past the head, the last one of a query head that is there (count > 0), which is then in
// the wave twice and changes nothing: what the padding holds is not looked at.
__device__ inline uint32_t loaded_row(uint32_t r, uint32_t i, uint32_t in_head, uint32_t n, uint32_t count) {
    return r < in_head ? r - i + min(i, count - 1) : in_head - n + count - 1;
}
// The row of q, the parts and the output that packed row r is.
template <typename S>
__device__ inline size_t shared_row(Constant<SharedArgs<S>> &a, uint32_t r, uint32_t b, uint32_t h, uint32_t in_head) {
    if (a.own_rows == 0) return ((size_t)(a.first + b) * a.c.heads + h) * in_head + r;
    const uint32_t m = r / a.own_rows, sequence = a.count.n[b] + m;
    return ((size_t)sequence * a.c.heads + h) * a.own_rows + (r - m * a.own_rows);
}

// Whether packed row r over a prefix is no padding.
template <typename S> __device__ inline bool no_padding(Constant<SharedArgs<S>> &a, uint32_t r, uint32_t b) {
    const uint32_t m = r / a.own_rows, sequence = a.count.n[b] + m, i = (r - m * a.own_rows) % a.padded;
    return i < (a.counts != nullptr ? a.counts[sequence] : (&a)[1].count.n[sequence]);
}
// The row of one of the lanes in `some`.
__device__ inline size_t row_among(size_t row, uint64_t some) {
    const int lane = __builtin_ctzll(some);
    return (size_t)(uint32_t)__builtin_amdgcn_readlane((int)(row >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)row, lane);
}

// A block's Meta through the scalar cache (no kernel writes it while one that
// reads it runs): a vector load would wait in line with the codes asked for ahead.
__device__ inline Meta scalar_meta(const Meta *at) {
    typedef const __attribute__((address_space(4))) u32x4 Constant;
    return __builtin_bit_cast(Meta, *(Constant *)(uintptr_t)at);
}

// Eight codes (as bytes + 128) as f16, exact.
__device__ inline half8 codes(uint32_t a, uint32_t b) {
    const uint32_t one = 0x64646464u;
    const half2_t bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    u32x4 r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(one, a, 0x04010400u)) - bias);
    r[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(one, a, 0x04030402u)) - bias);
    r[2] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(one, b, 0x04010400u)) - bias);
    r[3] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(one, b, 0x04030402u)) - bias);
    return __builtin_bit_cast(half8, r);
}

// Element e of a query row as f16 operands: an f16 one as it is. An f32 one (|x| <
// 2^14) as three that add up to it to 2^-21 and 2^-33 of it or better, the last a multiple
// of 8. An MFMA cuts its products off at 2^-24 or so of the largest one, and with a
// pair (x rounded to f16, and the rest) f32 attention was off by 2e-6, twice as far as its
// plain f32 form. Multiples of one power of two, 11 bits of them, times codes add up
// exactly, and what is cut off the small parts' products does not count: 5e-7. The
// small parts' products come first.
template <typename S> constexpr uint32_t kPieces = sizeof(S) == 4 ? 3 : 1;
__device__ inline void pieces_of(float x, half8 &p0, half8 &p1, half8 &p2, uint32_t e) {
    constexpr float kEights = 1.5f * 0x1p26f;   // its f32 neighbours are 8 apart
    const float most = (x + kEights) - kEights, rest = x - most;
    p2[e] = (_Float16)most;
    p1[e] = (_Float16)rest;
    p0[e] = (_Float16)(rest - (float)p1[e]);
}

// Elements d .. d + 7 of an f32 row, zeros past its end (rows of whole fours are
// asked for without a test).
__device__ inline void load8(const float *row, uint32_t dim, uint32_t d, float (&x)[8]) {
    if (dim % 4 == 0) {
#pragma unroll
        for (uint32_t i = 0; i < 8; i += 4) {
            f32x4 v = *reinterpret_cast<const f32x4 *>(row + (d + i < dim ? d + i : 0));
            if (d + i >= dim) v = f32x4{0, 0, 0, 0};
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) x[i + e] = v[e];
        }
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) x[e] = d + e < dim ? row[d + e] : 0.0f;
    }
}

// How many keys packed row r sees (0 or fewer: none); those that are loaded in the
// place of padding and past the head see all, as the row that they repeat does.
__device__ inline int seen_by(uint32_t i, bool live, uint32_t length, uint32_t count, int causal) {
    return causal && live ? (int)length - (int)count + (int)i + 1 : (int)length;
}

template <typename S>
__device__ inline void store_out(S *row, uint32_t vdim, uint32_t d, f32x4 v) {
    if (vdim % 4 == 0) {
        if (d < vdim) {
            if constexpr (sizeof(S) == 4) *reinterpret_cast<f32x4 *>(row + d) = v;
            else *reinterpret_cast<half4 *>(row + d) = half4{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
        }
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            if (d + e < vdim) row[d + e] = (S)v[e];
    }
}

// Outputs of a row from its maximum, its sum and its sum of weighted values.
__device__ inline f32x4 finish(f32x4 o, float big, float total) {
    if (!__builtin_isfinite(big)) return f32x4{0, 0, 0, 0};
    const float inverse = 1.0f / total;
    return f32x4{o.x * inverse, o.y * inverse, o.z * inverse, o.w * inverse};
}
__device__ inline f32x2 weight_terms(float big, float total) {
    const bool counts = __builtin_isfinite(big) && __builtin_isfinite(total);
    return f32x2{counts ? big : 0.0f, counts ? 1.0f / total : 0.0f};
}

// Many packed rows per head (k_kv_tiles.hip): kTileRows of a workgroup. `widest`:
// the wider of the padded dims. False where no such kernel is built.
constexpr uint32_t kTileRows = 128;
bool tiles_fit(bool f32, uint32_t widest);
// Whether a CU holds two of its workgroups (their registers decide).
constexpr bool tiles_twice(bool f32, uint32_t widest) { return !f32 && widest <= 128; }
template <typename S>
hipError_t launch_tiles(const Args<S> &a, uint32_t widest, uint32_t groups, hipStream_t s);
// Weights from the rows' maxima and sums; row_parts > 1: `partial` holds row_parts
// sums for each token of every (sequence, head).
template <typename S>
hipError_t launch_weights(const Args<S> &a, uint32_t widest, uint32_t batch, uint32_t blocks, uint32_t row_parts,
                          float *partial, hipStream_t s);

// Joins `parts` parts of the rows of a launch's sequences, by wide workgroups or not;
// its workgroups after those take token weights from the stored scores, if there are any.
template <typename S>
hipError_t launch_fold(const Args<S> &a, uint32_t parts, bool scores, uint32_t longest, bool wide, hipStream_t s);

struct Plan {
    bool many;     // rows enough for a tile to take less time than workgroups of 16 rows
    bool tiles;    // and products enough: k_kv_tiles.hip
    bool scores;   // the weights come from scores that the rows kernel stores (never with tiles)
    uint32_t row_groups, parts, row_parts;
    size_t rows, score_stride;
    size_t o_bytes, ml_bytes, exact_bytes, row_bytes, score_bytes, partial_bytes;
    size_t bytes() const { return o_bytes + ml_bytes + exact_bytes + row_bytes + score_bytes + partial_bytes; }
};

inline size_t whole256(size_t bytes) { return (bytes + 255) / 256 * 256; }
inline uint32_t widest_of(const View &c) { return c.kp > c.vp ? c.kp : c.vp; }
constexpr uint32_t kWorkgroups = 512;   // two for every CU
// Whether a CU holds two workgroups of the rows kernel (their registers decide).
constexpr bool rows_twice(bool f32, uint32_t widest) { return widest <= (f32 ? 128u : 192u); }
Plan plan_of(bool f32, const View &c, const AttentionShape &a);

// Codes past what the 256 MB cache behind the L2s holds to the next call are read
// as a stream. One sequence of 131000 tokens (268 MB): 62.5 -> 56.6 us; 8 x 4096
// (67 MB, found there by calls in a row): 19.5, as a stream 20.6.
constexpr size_t kStreamBytes = size_t{192} << 20;

}  // namespace kv
}  // namespace icsdk
