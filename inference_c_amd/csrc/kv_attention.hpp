// What the kernels of attention over the 8-bit cache share: arguments, the codes
// as f16, and the rules of rows, outputs and weights (k_kv_attention.hip describes
// them; k_kv_tiles.hip has the kernels for many rows).
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

// How many keys packed row r sees (0 or fewer: none); padded rows and rows past
// the head see all.
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

}  // namespace kv
}  // namespace icsdk
