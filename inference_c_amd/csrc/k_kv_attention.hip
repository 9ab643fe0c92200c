// Attention over the 8-bit key/value cache (kv.hpp), f16 and f32.
//
// The query heads of a kv head and their n rows are consecutive in q and out,
// so packed row r of a kv head is row r of a [group * n, dim] matrix; its
// position in the sequence goes by i = r % n.
//
// v_mfma_f32_16x16x32_f16: A[m][k] in lane l at m = l % 16, k = 8 g + e, g = l / 16;
// B[k][n] at n = l % 16 likewise; D[m][n] at n = l % 16, m = 4 g + e. Per block of
// 64 keys a wave of 16 rows computes
//   S^T = K Q^T in four sub-tiles u: A row m is key 16 (m / 4) + 4 u + m % 4 of
//     the block, so lane l gets of row l % 16 the keys 16 g + 4 u + e: all four
//     sub-tiles together 16 consecutive ones;
//   out^T = V^T P^T: step s contracts over keys 16 g + 8 s + e, of which the lane
//     has P in registers, and of the block's v rows (a dim's 64 keys side by
//     side) the same keys are half s of the 16 bytes at 16 g.
// The codes go from memory to registers and, turned to f16, into the MFMA; no
// LDS. A code byte u = code + 128 is put behind a byte 0x64, which is the f16
// 1024 + u, and 1152 is subtracted, exactly: one v_perm_b32 and one v_pk_add_f16
// per two codes.
//
// Scales: a block's key scale multiplies its scores. Its value scale v multiplies
// P, relative to a running unit of the output: P v / unit, with the unit moved to
// v (the output rescaled) when the ratio leaves 2^-3 .. 2^3, so P keeps f16's
// range whatever the blocks' scales are.
//
// f32: q and P each are a pair of f16 (q scaled by a power of two to a largest
// element of 2^13 .. 2^14), 22 significant bits, and codes are exact: two MFMAs
// in place of one.
#include "kern_common.hpp"
#include "kv.hpp"

namespace icsdk {
namespace kv {
namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWaves = 4;
constexpr uint32_t kRows = 16;         // packed rows of a wave
constexpr double kLog2e = 1.4426950408889634;
constexpr float kUnitRange = 8.0f;     // a value scale further from the unit moves it
// P of a row whose maximum is M is 2^(s - M + kHeadroom): as far up in f16 as the
// unit's range and the lazy rescale of the maximum (by more than 2^kLazy) leave
// room for, 2^15 in all, so that small weights keep their bits: absolute
// errors of P, relative to the row's largest, are below 2^-26 (f16; P is rounded
// to 2^-11 anyway) and 2^-34 (f32, whose maximum is never left behind).
template <typename S> constexpr float kLazy = sizeof(S) == 4 ? 0.0f : 8.0f;
template <typename S> constexpr float kHeadroom = sizeof(S) == 4 ? 12.0f : 4.0f;
// Arguments of a launch over sequences first .. (pairs / heads of them).
template <typename S> struct Args {
    View c;
    const S *q;
    S *out;
    float *part_o;       // [part][row][vdim], rows of all sequences
    f32x2 *part_ml;      // [part][row] running maximum (log2 units) and sum
    f32x2 *row_ml;       // [row] maximum and 1 / sum (0: the row adds no weight), or null
    float *weights;
    float *scores;       // [row][score_stride] scores in log2 units, or null
    size_t rows;         // of all sequences
    size_t score_stride;
    size_t weight_stride;
    uint32_t weight_tokens;
    uint32_t first, pairs, group, n, parts, row_group0;
    double scale2;       // scale * log2 e
    int causal;
    Counts count;
};

// Largest and sum over the four lanes that hold one row.
__device__ inline float groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ inline float groups_sum(float v) {
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
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

// The dims that a lane's operand of k step s has: 64-dim chunks of 16 per lane
// group in two steps, then (P an odd multiple of 32) one of 8 per lane group.
template <uint32_t P> __device__ inline uint32_t step_dim(uint32_t s, uint32_t g) {
    return s / 2 < P / 64 ? s / 2 * 64 + g * 16 + s % 2 * 8 : P / 64 * 64 + g * 8;
}

// A wave's 16 query rows as B operands, one per k step (f32: and their rest).
template <typename S, uint32_t P> struct Query {
    static constexpr uint32_t kSteps = P / 32;
    static constexpr bool kPair = sizeof(S) == 4;
    half8 hi[kSteps], lo[kPair ? kSteps : 1];
    float factor;   // the power of two that a f32 row was divided by

    __device__ inline void load(const S *row, uint32_t dim, uint32_t g) {
        factor = 1.0f;
        if constexpr (!kPair) {
#pragma unroll
            for (uint32_t s = 0; s < kSteps; ++s) {
                const uint32_t d = step_dim<P>(s, g);
                if (dim % 8 == 0) {
                    hi[s] = *reinterpret_cast<const half8 *>(row + (d < dim ? d : 0));
                    if (d >= dim) hi[s] = half8{};
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) hi[s][e] = d + e < dim ? row[d + e] : (_Float16)0.0f;
                }
            }
        } else {
            float x[kSteps][8], big = 0.0f;
            bool finite = true;
#pragma unroll
            for (uint32_t s = 0; s < kSteps; ++s) {
                const uint32_t d = step_dim<P>(s, g);
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) {
                    x[s][e] = d + e < dim ? row[d + e] : 0.0f;
                    big = fmaxf(big, fabsf(x[s][e]));
                    finite = finite && __builtin_isfinite(x[s][e]);
                }
            }
            big = groups_max(finite ? big : __builtin_inff());
            // a row with an element that is not finite has no finite score: NaN ones
            // leave its maximum at -inf, and it is zeros
            const bool usable = big > 0.0f && __builtin_isfinite(big);
            const int exponent = usable ? __builtin_amdgcn_frexp_expf(big) : 14;   // big in [2^(e-1), 2^e)
            factor = __builtin_isfinite(big) ? __builtin_ldexpf(1.0f, exponent - 14) : __builtin_nanf("");
#pragma unroll
            for (uint32_t s = 0; s < kSteps; ++s)
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) {
                    const float y = usable ? __builtin_ldexpf(x[s][e], 14 - exponent) : 0.0f;
                    hi[s][e] = (_Float16)y;
                    lo[s][e] = (_Float16)(y - (float)hi[s][e]);
                }
        }
    }
};

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

// One workgroup: 16 packed rows of one (sequence, kv head) and one part of its
// blocks; wave w takes blocks w, w + 4, ... of the part and the waves' results
// meet in LDS.
template <typename S, uint32_t P>
__global__ __launch_bounds__(kThreads) void kv_rows_kernel(Args<S> a) {
    constexpr bool kPair = sizeof(S) == 4;
    constexpr uint32_t NC = P / 64, NV = P / 16;
    constexpr bool kOdd = P % 64 != 0;
    __shared__ f32x4 lds_o[kWaves][NV][kWave];
    __shared__ f32x2 lds_ml[kWaves][kRows];
    const View &c = a.c;
    const uint32_t lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t part = blockIdx.x % a.parts, pr = blockIdx.x / a.parts;
    const uint32_t pair = pr % a.pairs, row0 = (a.row_group0 + pr / a.pairs) * kRows;
    const uint32_t b = pair / c.heads, h = pair % c.heads, seq = a.first + b;
    const size_t head = (size_t)seq * c.heads + h;
    const uint32_t length = c.length[seq], count = a.count.n[b];
    const uint32_t in_head = a.group * a.n;
    const uint32_t r = row0 + m, i = r % a.n;
    const bool live = r < in_head && i < count;
    if (!wave_any(live)) return;
    const size_t row = head * in_head + (r < in_head ? r : in_head - 1);   // (rows past the head repeat its last)
    const int seen = seen_by(i, live, length, count, a.causal);
    int most = live ? seen : 0, least = live ? seen : (int)length;
#pragma unroll
    for (int d = 1; d < 16; d *= 2) {
        most = max(most, __shfl_xor(most, d, kWave));
        least = min(least, __shfl_xor(least, d, kWave));
    }
    most = __builtin_amdgcn_readfirstlane(most);
    least = __builtin_amdgcn_readfirstlane(least);
    const uint32_t blocks = ((uint32_t)max(most, 0) + kTokens - 1) / kTokens;
    const uint32_t whole = length / kTokens;   // blocks held as codes
    const uint32_t share = ((blocks + a.parts - 1) / a.parts + kWaves - 1) / kWaves * kWaves;
    const uint32_t begin = min(part * share, blocks), end = min(begin + share, blocks);

    Query<S, P> q;
    q.load(a.q + row * c.dim, c.dim, g);

    const float neg_inf = -__builtin_inff();
    f32x4 o[NV];
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) o[j] = f32x4{0, 0, 0, 0};
    float big = neg_inf, sum = 0.0f, unit = 1.0f;

    // one block: kf(u, s) and vf(j, s) give the A operands
    auto step = [&](uint32_t t, Meta meta, auto kf, auto vf, auto keys_done) {
        const double factor2 = (double)meta.k_scale * a.scale2;
        const float factor = (float)factor2 * q.factor;
        // f32: what rounding takes off the factor and the scores is added back in
        // the exponent (scores of 10 would be off by 1e-6 of their weight)
        const float factor_rest = (float)(factor2 - (double)(float)factor2) * q.factor;
        float p[16], rest[kPair ? 16 : 1];
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
            f32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t s = 0; s < Query<S, P>::kSteps; ++s) {
                const half8 k = kf(u, s);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q.hi[s], acc, 0, 0, 0);
                if constexpr (kPair) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q.lo[s], acc, 0, 0, 0);
            }
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                p[4 * u + e] = acc[e] * factor;
                if constexpr (kPair) {
                    const float off = __builtin_fmaf(acc[e], factor, -p[4 * u + e]) + acc[e] * factor_rest;
                    rest[4 * u + e] = fabsf(p[4 * u + e]) < 1e30f ? off : 0.0f;
                }
            }
        }
        keys_done();
        if ((int)(t * kTokens + kTokens) > least || meta.marked != 0) {
            const uint32_t mine = (uint32_t)(meta.marked >> (16 * g));
#pragma unroll
            for (uint32_t e = 0; e < 16; ++e) {
                if (mine >> e & 1) p[e] = __builtin_nanf("");
                if ((int)(t * kTokens + 16 * g + e) >= seen) p[e] = neg_inf;
            }
        }
        if (a.scores != nullptr && live) {
            float *const out = a.scores + row * a.score_stride + t * kTokens + 16 * g;
#pragma unroll
            for (uint32_t e = 0; e < 16; e += 4)
                *reinterpret_cast<f32x4 *>(out + e) = f32x4{p[e], p[e + 1], p[e + 2], p[e + 3]};
        }
        float top = neg_inf;
#pragma unroll
        for (uint32_t e = 0; e < 16; ++e) top = fmaxf(top, p[e]);
        if (__builtin_amdgcn_ballot_w64(top > big + kLazy<S>) != 0) {
            const float now = groups_max(fmaxf(top, big));
            const float alpha = now == neg_inf ? 1.0f : __builtin_amdgcn_exp2f(big - now);
            sum *= alpha;
#pragma unroll
            for (uint32_t j = 0; j < NV; ++j) o[j] *= alpha;
            big = now;
        }
        // nothing seen yet: every score is -inf (p = 0) or NaN
        const float base = big == neg_inf ? 0.0f : big - kHeadroom<S>;
        float ratio = meta.v_scale / unit;
        if (meta.v_scale == 0.0f) {
            ratio = 1.0f;   // its codes are zeros
        } else if (ratio > kUnitRange || ratio < 1.0f / kUnitRange) {
#pragma unroll
            for (uint32_t j = 0; j < NV; ++j) o[j] *= unit / meta.v_scale;
            unit = meta.v_scale;
            ratio = 1.0f;
        }
        half8 ph[2], pl[kPair ? 2 : 1];
        float add = 0.0f;
#pragma unroll
        for (uint32_t e = 0; e < 16; ++e) {
            float x = p[e] - base;
            if constexpr (kPair) x += rest[e];
            x = __builtin_amdgcn_exp2f(x);
            const float y = x * ratio;
            ph[e / 8][e % 8] = (_Float16)y;
            if constexpr (kPair) {
                pl[e / 8][e % 8] = (_Float16)(y - (float)ph[e / 8][e % 8]);
                add += x;
            } else {
                add += (float)ph[e / 8][e % 8];   // the sum of P as the product has it
            }
        }
        sum += kPair ? add : add * (1.0f / ratio);
#pragma unroll
        for (uint32_t j = 0; j < NV; ++j) {
            if (j * 16 >= c.vp) continue;
#pragma unroll
            for (uint32_t s = 0; s < 2; ++s) {
                const half8 v = vf(j, s);
                o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[s], o[j], 0, 0, 0);
                if constexpr (kPair) o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl[s], o[j], 0, 0, 0);
            }
        }
    };

    const Meta *const meta = c.meta + head * c.blocks;
    const uint32_t key_of = (m / 4) * 16 + m % 4;   // + 4 u: the lane's key row
    u32x4 kr[4][NC > 0 ? NC : 1], vr[NV];
    u32x2 ko[4];
    auto load_k = [&](uint32_t t) {
        const uint8_t *base = c.k + ((head * c.blocks + t) * kTokens + key_of) * c.kp;
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
#pragma unroll
            for (uint32_t ch = 0; ch < NC; ++ch) {
                const uint32_t d = ch * 64 + g * 16;   // past the row: its start, against zeros of q
                kr[u][ch] = *reinterpret_cast<const u32x4 *>(base + 4 * u * c.kp + (d < c.kp ? d : 0));
            }
            if constexpr (kOdd) {
                const uint32_t d = NC * 64 + g * 8;
                ko[u] = *reinterpret_cast<const u32x2 *>(base + 4 * u * c.kp + (d < c.kp ? d : 0));
            }
        }
    };
    auto load_v = [&](uint32_t t) {
        const uint8_t *base = c.v + ((head * c.blocks + t) * c.vp + m) * kTokens + g * 16;
#pragma unroll
        for (uint32_t j = 0; j < NV; ++j)
            if (j * 16 < c.vp) vr[j] = *reinterpret_cast<const u32x4 *>(base + j * 16 * kTokens);
    };
    const uint32_t end_whole = min(end, whole);
    uint32_t t = begin + wave;
    if (t < end_whole) {
        load_k(t);
        load_v(t);
    }
    for (; t < end_whole; t += kWaves) {
        const uint32_t next = t + kWaves;
        step(
            t, meta[t],
            [&](uint32_t u, uint32_t s) {
                if (s / 2 < NC) return codes(kr[u][s / 2][s % 2 * 2], kr[u][s / 2][s % 2 * 2 + 1]);
                return codes(ko[u].x, ko[u].y);
            },
            [&](uint32_t j, uint32_t s) { return codes(vr[j][2 * s], vr[j][2 * s + 1]); },
            [&] {
                if (next < end_whole) load_k(next);
            });
        if (next < end_whole) load_v(next);
    }
    if (t == whole && t < end) {   // the open block, in f16
        const _Float16 *kt = c.kt + (head * kTokens + key_of) * c.kp;
        const _Float16 *vt = c.vt + (head * c.vp + m) * kTokens + g * 16;
        step(
            t, Meta{1.0f, 1.0f, meta[t].marked},
            [&](uint32_t u, uint32_t s) {
                const uint32_t d = step_dim<P>(s, g);
                return *reinterpret_cast<const half8 *>(kt + 4 * u * c.kp + (d < c.kp ? d : 0));
            },
            [&](uint32_t j, uint32_t s) { return *reinterpret_cast<const half8 *>(vt + j * 16 * kTokens + s * 8); }, [] {});
    }

    // the waves meet
    sum = groups_sum(sum);
    big -= kHeadroom<S>;   // what P's exponents are relative to
    if (g == 0) lds_ml[wave][m] = f32x2{big, sum};
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) lds_o[wave][j][lane] = o[j] * unit;
    __syncthreads();
    float top = neg_inf, total = 0.0f, w[kWaves];
#pragma unroll
    for (uint32_t k = 0; k < kWaves; ++k) top = fmaxf(top, lds_ml[k][m].x);
#pragma unroll
    for (uint32_t k = 0; k < kWaves; ++k) {
        // (a wave that saw nothing has weight 0, and a NaN in it stays)
        w[k] = top == neg_inf ? 1.0f : __builtin_amdgcn_exp2f(lds_ml[k][m].x - top);
        total += w[k] * lds_ml[k][m].y;
    }
    const bool writes = live && r < in_head;
    if (a.parts == 1) {
        S *const out = a.out + row * c.vdim;
#pragma unroll
        for (uint32_t j = wave; j < NV; j += kWaves) {
            f32x4 v = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t k = 0; k < kWaves; ++k) v += lds_o[k][j][lane] * w[k];
            if (writes) store_out(out, c.vdim, 16 * j + 4 * g, finish(v, top, total));
        }
        if (writes && g == 0 && wave == 0) {
            if (a.row_ml != nullptr) a.row_ml[row] = weight_terms(top, total);
            if (a.scores != nullptr) a.part_ml[row] = f32x2{top, total};
        }
    } else {
        float *const out = a.part_o + ((size_t)part * a.rows + row) * c.vdim;
#pragma unroll
        for (uint32_t j = wave; j < NV; j += kWaves) {
            f32x4 v = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t k = 0; k < kWaves; ++k) v += lds_o[k][j][lane] * w[k];
            if (writes) store_out(out, c.vdim, 16 * j + 4 * g, v);
        }
        if (writes && g == 0 && wave == 0) a.part_ml[(size_t)part * a.rows + row] = f32x2{top, total};
    }
}

// Maximum and sum of a row from its parts', by one wave.
__device__ inline f32x2 fold_ml(const f32x2 *ml, uint32_t parts, size_t rows, uint32_t lane) {
    float top = -__builtin_inff(), total = 0.0f;
    for (uint32_t s = lane; s < parts; s += kWave) top = fmaxf(top, ml[s * rows].x);
    top = wave_max(top);
    for (uint32_t s = lane; s < parts; s += kWave) {
        const f32x2 v = ml[s * rows];
        total += (top == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(v.x - top)) * v.y;
    }
    return f32x2{top, wave_sum(total)};
}

// Merges the parts of a row, one workgroup per row: its waves take every fourth
// part, a lane four output elements. The workgroups after `folds` do 256 tokens
// of one (sequence, head) each: their weights from the stored scores.
template <typename S>
__global__ __launch_bounds__(kThreads) void kv_fold_kernel(Args<S> a, uint32_t folds, uint32_t token_groups) {
    __shared__ f32x4 lds_o[kWaves][kWave];
    __shared__ f32x2 lds_ml[kRows];
    const View &c = a.c;
    const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t in_head = a.group * a.n;
    if (blockIdx.x >= folds) {
        const uint32_t tg = (blockIdx.x - folds) % token_groups, pair = (blockIdx.x - folds) / token_groups;
        const uint32_t b = pair / c.heads, seq = a.first + b, length = min(c.length[seq], a.weight_tokens);
        const size_t head = (size_t)seq * c.heads + pair % c.heads;
        if (tg * kThreads >= length) return;
        for (uint32_t r = wave; r < in_head; r += kWaves) {
            const size_t row = head * in_head + r;
            const f32x2 ml = r % a.n < a.count.n[b] ? fold_ml(a.part_ml + row, a.parts, a.rows, lane)
                                                    : f32x2{-__builtin_inff(), 0.0f};
            if (lane == 0) lds_ml[r] = weight_terms(ml.x, ml.y);
        }
        __syncthreads();
        const uint32_t t = tg * kThreads + threadIdx.x;
        if (t >= length) return;
        float total = 0.0f;
        for (uint32_t r = 0; r < in_head; ++r) {
            const f32x2 ml = lds_ml[r];
            if (ml.y != 0.0f)
                total += __builtin_amdgcn_exp2f(a.scores[(head * in_head + r) * a.score_stride + t] - ml.x) * ml.y;
        }
        a.weights[head * a.weight_stride + t] += total;
        return;
    }
    const uint32_t b = blockIdx.x / (in_head * c.heads);
    if (blockIdx.x % a.n >= a.count.n[b]) return;
    const size_t row = (size_t)a.first * c.heads * in_head + blockIdx.x;
    const f32x2 all = fold_ml(a.part_ml + row, a.parts, a.rows, lane);
    f32x4 v = {0, 0, 0, 0};
    const uint32_t d = 4 * lane;
    const bool fours = c.vdim % 4 == 0;
#pragma unroll 4
    for (uint32_t s = wave; s < a.parts; s += kWaves) {
        const float m = a.part_ml[(size_t)s * a.rows + row].x;
        const float w = all.x == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - all.x);
        const float *src = a.part_o + ((size_t)s * a.rows + row) * c.vdim;
        if (fours) {
            v += *reinterpret_cast<const f32x4 *>(src + (d < c.vdim ? d : 0)) * w;
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                if (d + e < c.vdim) v[e] += src[d + e] * w;
        }
    }
    lds_o[wave][lane] = v;
    __syncthreads();
    if (wave != 0) return;
    for (uint32_t k = 1; k < kWaves; ++k) v += lds_o[k][lane];
    store_out(a.out + row * c.vdim, c.vdim, d, finish(v, all.x, all.y));
    if (a.row_ml != nullptr && lane == 0) a.row_ml[row] = weight_terms(all.x, all.y);
}

// Softmax weights of one block's tokens, summed over the rows that see them: the
// scores again, now with the rows' maxima and sums known. The block's keys stay
// in registers and each wave walks every fourth group of 16 rows.
template <typename S, uint32_t P>
__global__ __launch_bounds__(kThreads) void kv_weights_kernel(Args<S> a) {
    constexpr bool kPair = sizeof(S) == 4;
    constexpr uint32_t KS = P / 32;
    __shared__ float lds_w[kWaves][kTokens];
    const View &c = a.c;
    const uint32_t lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t t = blockIdx.x, h = blockIdx.y, b = blockIdx.z, seq = a.first + b;
    const size_t head = (size_t)seq * c.heads + h;
    const uint32_t length = c.length[seq], count = a.count.n[b];
    if (t * kTokens >= length || count == 0) return;
    const uint32_t in_head = a.group * a.n;
    const bool open = t == length / kTokens;
    const Meta meta = c.meta[head * c.blocks + t];
    const float k_scale = open ? 1.0f : meta.k_scale;
    const uint32_t key_of = (m / 4) * 16 + m % 4;
    half8 k[4][KS];
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u)
#pragma unroll
        for (uint32_t s = 0; s < KS; ++s) {
            const uint32_t d = step_dim<P>(s, g), at = d < c.kp ? d : 0;
            if (open) {
                k[u][s] = *reinterpret_cast<const half8 *>(c.kt + (head * kTokens + key_of + 4 * u) * c.kp + at);
            } else {
                const u32x2 w = *reinterpret_cast<const u32x2 *>(
                    c.k + ((head * c.blocks + t) * kTokens + key_of + 4 * u) * c.kp + at);
                k[u][s] = codes(w.x, w.y);
            }
        }
    float acc[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
    const uint32_t marked = (uint32_t)(meta.marked >> (16 * g));
    for (uint32_t row0 = wave * kRows; row0 < in_head; row0 += kWaves * kRows) {
        const uint32_t r = row0 + m, i = r % a.n;
        const bool live = r < in_head && i < count;
        const int seen = seen_by(i, live, length, count, a.causal);
        if (!wave_any(live && seen > (int)(t * kTokens))) continue;
        const size_t row = head * in_head + min(r, in_head - 1);
        Query<S, P> q;
        q.load(a.q + row * c.dim, c.dim, g);
        const f32x2 ml = live ? a.row_ml[row] : f32x2{0.0f, 0.0f};
        const float factor = (float)((double)k_scale * a.scale2) * q.factor;
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
            f32x4 s4 = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t s = 0; s < KS; ++s) {
                s4 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[u][s], q.hi[s], s4, 0, 0, 0);
                if constexpr (kPair) s4 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[u][s], q.lo[s], s4, 0, 0, 0);
            }
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                const uint32_t at = 4 * u + e;
                const bool counts = ml.y != 0.0f && (int)(t * kTokens + 16 * g + at) < seen && !(marked >> at & 1);
                acc[at] += counts ? __builtin_amdgcn_exp2f(s4[e] * factor - ml.x) * ml.y : 0.0f;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
#pragma unroll
        for (int d = 1; d < 16; d *= 2) acc[e] += __shfl_xor(acc[e], d, kWave);
        if (m == 0) lds_w[wave][16 * g + e] = acc[e];
    }
    __syncthreads();
    const uint32_t token = t * kTokens + lane;
    if (wave == 0 && token < min(length, a.weight_tokens)) {
        float total = 0.0f;
        for (uint32_t w = 0; w < kWaves; ++w) total += lds_w[w][lane];
        a.weights[head * a.weight_stride + token] += total;
    }
}

// ---- plan and launch ---------------------------------------------------------------

struct Plan {
    uint32_t row_groups, parts;
    bool scores;   // the weights come from scores that the rows kernel stores
    size_t rows, score_stride;
    size_t o_bytes, ml_bytes, row_bytes, score_bytes;
};

size_t whole256(size_t bytes) { return (bytes + 255) / 256 * 256; }

Plan plan_of(const View &c, const AttentionShape &a) {
    Plan p;
    const uint32_t in_head = a.q_heads / c.heads * a.n;
    p.row_groups = (in_head + kRows - 1) / kRows;
    const uint32_t blocks = (a.longest + kTokens - 1) / kTokens;
    // parts: workgroups for every CU twice over, a block for each wave at least
    const uint64_t base = (uint64_t)a.batch * c.heads * p.row_groups;
    uint64_t parts = base >= 512 ? 1 : 512 / base;
    const uint32_t most = (blocks + kWaves - 1) / kWaves;
    parts = parts < most ? parts : most;
    p.parts = parts < 1 ? 1 : (uint32_t)parts;
    p.rows = (size_t)a.batch * a.q_heads * a.n;
    p.o_bytes = p.parts > 1 ? whole256(p.parts * p.rows * c.vdim * 4) : 0;
    // a token's scores, 4 bytes per row written and read again, against its key
    // again: for up to a tile of rows the scores
    p.scores = a.weights != nullptr && in_head <= kRows;
    p.score_stride = (size_t)blocks * kTokens;
    p.ml_bytes = p.parts > 1 || p.scores ? whole256(p.parts * p.rows * sizeof(f32x2)) : 0;
    p.row_bytes = a.weights != nullptr && !p.scores ? whole256(p.rows * sizeof(f32x2)) : 0;
    p.score_bytes = p.scores ? whole256(p.rows * p.score_stride * 4) : 0;
    return p;
}

template <typename S, uint32_t P>
hipError_t launch(Args<S> a, const Plan &p, uint32_t batch, uint32_t longest, hipStream_t s) {
    const uint32_t blocks = (longest + kTokens - 1) / kTokens;
    // (a launch holds fewer than 2^32 threads)
    const uint32_t most = (1u << 23) / (a.pairs * p.parts) < 1 ? 1 : (1u << 23) / (a.pairs * p.parts);
    for (uint32_t g0 = 0; g0 < p.row_groups; g0 += most) {
        a.row_group0 = g0;
        const uint32_t groups = p.row_groups - g0 < most ? p.row_groups - g0 : most;
        kv_rows_kernel<S, P><<<groups * a.pairs * p.parts, kThreads, 0, s>>>(a);
        const hipError_t status = hipGetLastError();
        if (status != hipSuccess) return status;
    }
    if (p.parts > 1 || p.scores) {
        // (at most 512 row groups where there are parts)
        const uint32_t folds = p.parts > 1 ? a.pairs * a.group * a.n : 0;
        const uint32_t token_groups = p.scores ? (blocks * kTokens + kThreads - 1) / kThreads : 0;
        if (folds + a.pairs * token_groups == 0) return hipSuccess;
        kv_fold_kernel<S><<<folds + a.pairs * token_groups, kThreads, 0, s>>>(a, folds, token_groups);
        const hipError_t status = hipGetLastError();
        if (status != hipSuccess) return status;
    }
    if (a.row_ml != nullptr && blocks > 0) {
        kv_weights_kernel<S, P><<<dim3(blocks, a.c.heads, batch), kThreads, 0, s>>>(a);
        return hipGetLastError();
    }
    return hipSuccess;
}

template <typename S>
hipError_t run(const View &c, const AttentionShape &sh, const void *query, void *output, void *workspace,
               hipStream_t s) {
    const Plan p = plan_of(c, sh);
    Args<S> a;
    a.c = c;
    a.q = static_cast<const S *>(query);
    a.out = static_cast<S *>(output);
    char *ws = static_cast<char *>(workspace);
    a.part_o = reinterpret_cast<float *>(ws);
    a.part_ml = reinterpret_cast<f32x2 *>(ws + p.o_bytes);
    a.row_ml = p.row_bytes ? reinterpret_cast<f32x2 *>(ws + p.o_bytes + p.ml_bytes) : nullptr;
    a.scores = p.scores ? reinterpret_cast<float *>(ws + p.o_bytes + p.ml_bytes + p.row_bytes) : nullptr;
    a.score_stride = p.score_stride;
    a.weights = sh.weights;
    a.weight_tokens = sh.weight_tokens;
    a.weight_stride = sh.weight_stride;
    a.rows = p.rows;
    a.group = sh.q_heads / c.heads;
    a.n = sh.n;
    a.parts = p.parts;
    a.scale2 = (double)sh.scale * kLog2e;
    a.causal = sh.causal;
    const uint32_t widest = c.kp > c.vp ? c.kp : c.vp;
    for (uint32_t first = 0; first < sh.batch; first += kBatchPerLaunch) {
        const uint32_t batch = sh.batch - first < kBatchPerLaunch ? sh.batch - first : kBatchPerLaunch;
        for (uint32_t b = 0; b < batch; ++b) a.count.n[b] = sh.counts ? sh.counts[first + b] : sh.n;
        a.first = first;
        a.pairs = batch * c.heads;
        hipError_t status;
        if (widest <= 32) status = launch<S, 32>(a, p, batch, sh.longest, s);
        else if (widest <= 64) status = launch<S, 64>(a, p, batch, sh.longest, s);
        else if (widest <= 96) status = launch<S, 96>(a, p, batch, sh.longest, s);
        else if (widest <= 128) status = launch<S, 128>(a, p, batch, sh.longest, s);
        else if (widest <= 192) status = launch<S, 192>(a, p, batch, sh.longest, s);
        else status = launch<S, 256>(a, p, batch, sh.longest, s);
        if (status != hipSuccess) return status;
    }
    return hipSuccess;
}

}  // namespace

size_t attention_workspace(const View &c, const AttentionShape &a) {
    const Plan p = plan_of(c, a);
    return p.o_bytes + p.ml_bytes + p.row_bytes + p.score_bytes;
}

hipError_t attention(bool f32, const View &c, const AttentionShape &a, const void *query, void *output,
                     void *workspace, hipStream_t s) {
    return f32 ? run<float>(c, a, query, output, workspace, s) : run<_Float16>(c, a, query, output, workspace, s);
}

}  // namespace kv
}  // namespace icsdk
