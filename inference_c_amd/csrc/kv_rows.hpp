// The kernel of attention over the 8-bit cache for few query rows, as a function of
// its workgroup (k_kv_attention.hip and k_kv_shared.hip make kernels of it).
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
// f32: q is three f16 operands (scaled by a power of two to a largest element of 2^13 ..
// 2^14), P a pair, 22 significant bits, and codes are exact. A block's output is added
// to the running one in f32, rounded to nearest, as the MFMA does not.
//
// f16: the output is divided by the sum of P as rounded to f16, so that a row with one
// large weight has its value exactly; accumulated token weights, which are f32, go by the
// sum before that rounding. Token weights of either type go by scores in one f32, off by
// 2^-24 of the score: sums of many rows' weights, for which 32 bits are enough.
#pragma once

#include "kv_attention.hpp"

namespace icsdk {
namespace kv {

// Largest and sum over the four lanes that hold one row.
__device__ inline float groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ inline float groups_sum(float v) {
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
}

// The dims that a lane's operand of k step s has: 64-dim chunks of 16 per lane
// group in two steps, then (P an odd multiple of 32) one of 8 per lane group.
template <uint32_t P> __device__ inline uint32_t step_dim(uint32_t s, uint32_t g) {
    return s / 2 < P / 64 ? s / 2 * 64 + g * 16 + s % 2 * 8 : P / 64 * 64 + g * 8;
}

// A wave's 16 query rows as B operands, one per k step and piece.
template <typename S, uint32_t P> struct Query {
    static constexpr uint32_t kSteps = P / 32;
    static constexpr bool kPair = sizeof(S) == 4;
    half8 piece[kPieces<S>][kSteps];
    int shift = 0;   // an f32 row was divided by 2^shift

    __device__ inline void load(const S *row, uint32_t dim, uint32_t g) {
        if constexpr (!kPair) {
#pragma unroll
            for (uint32_t s = 0; s < kSteps; ++s) {
                const uint32_t d = step_dim<P>(s, g);
                if (dim % 8 == 0) {
                    piece[0][s] = *reinterpret_cast<const half8 *>(row + (d < dim ? d : 0));
                    if (d >= dim) piece[0][s] = half8{};
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) piece[0][s][e] = d + e < dim ? row[d + e] : (_Float16)0.0f;
                }
            }
        } else {
            float x[kSteps][8], big = 0.0f;
            bool finite = true;
#pragma unroll
            for (uint32_t s = 0; s < kSteps; ++s) {
                const uint32_t d = step_dim<P>(s, g);
                load8(row, dim, d, x[s]);
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) {
                    big = fmaxf(big, fabsf(x[s][e]));
                    finite = finite && __builtin_isfinite(x[s][e]);
                }
            }
            big = groups_max(finite ? big : __builtin_inff());
            // a row with an element that is not finite has no finite score: NaN ones
            // leave its maximum at -inf, and it is zeros
            const bool usable = big > 0.0f && __builtin_isfinite(big);
            const int exponent = usable ? __builtin_amdgcn_frexp_expf(big) : 14;   // big in [2^(e-1), 2^e)
            shift = exponent - 14;
            const float none = big > 0.0f ? __builtin_nanf("") : 0.0f;
#pragma unroll
            for (uint32_t s = 0; s < kSteps; ++s)
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) {
                    const float y = usable ? __builtin_ldexpf(x[s][e], -shift) : none;
                    pieces_of(y, piece[0][s], piece[1][s], piece[2][s], e);
                }
        }
    }
};

template <bool kStream, typename V> __device__ inline V load_codes(const V *p) {
    return kStream ? __builtin_nontemporal_load(p) : *p;
}

// One workgroup: 16 packed rows of one (sequence, kv head) and one part of its
// blocks; wave w takes blocks w, w + 4, ... of the part and the waves' results
// meet in LDS. Bound by the codes' way from memory: 8 x 8 heads x 4096 tokens of D 128
// (67 MB) 14 us, 4.7 TB/s, and the fold 3; one sequence of 131000 tokens (268 MB) 47 us,
// 5.7 TB/s (a copy of 1 GiB: 5.1). Two workgroups for every CU: three or four make more
// parts to fold (8 x 4096 18 -> 22 us).
// What the first loads wait for comes as leading arguments, which are in scalar
// registers when a wave starts: the struct behind them takes a microsecond to
// arrive. (8 x 4096 tokens, from the wave's start to its first loads' issue: 2 us
// out of 12 with the struct alone.)
// A is Args, or SharedArgs for a pass of attention over a prefix and own tokens. kSolo
// (of such a pass): a wave has 16 rows and a part by itself, and its own x, h and b.
// kMeet of 8: four waves have the prefix, where b is the sequence's one, and four its own
// tokens; rows are those of `own`, and all eight meet.
template <uint32_t P, uint32_t kMeet = kWaves> using RowsOut = f32x4[kMeet][P / 16][kWave];
template <uint32_t kMeet = kWaves> using RowsMl = f32x4[kMeet][kRows];   // maximum, sums of P rounded and not
struct OwnRows {
    uint32_t sequence, count;
};
template <typename S, uint32_t P, bool kStream, bool kSolo, uint32_t kMeet = kWaves, typename A>
__device__ __forceinline__ void rows_of(RowsOut<P, kMeet> &lds_o, RowsMl<kMeet> &lds_ml, const uint8_t *keys, const uint8_t *values,
                                        const uint32_t *lengths, const Meta *metas, const S *queries, uint32_t all_blocks,
                                        uint32_t heads, uint32_t parts_first, uint32_t pitches, uint32_t n,
                                        uint32_t group, A &a, uint32_t x, uint32_t h, uint32_t b,
                                        OwnRows own = {}) {
    constexpr bool kPair = sizeof(S) == 4, kShared = kIsShared<A>, kBoth = kMeet != kWaves;
    constexpr uint32_t NC = P / 64, NV = P / 16;
    constexpr bool kOdd = P % 64 != 0;
    auto &c = a.c;
    const uint32_t lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const uint32_t place = (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / kWave), wave = kBoth ? place % kWaves : place;
    const uint32_t parts = parts_first & 0xffffu, kp = pitches & 0xffffu, vp = pitches >> 16;
    const uint32_t seq = (parts_first >> 16) + b;
    const uint32_t length = lengths[seq];
    const uint32_t part = x % parts;
    const size_t head = (size_t)seq * heads + h;
    // the part's blocks, the open one (the last, in f16) among them
    const uint32_t whole = length / kTokens, held = (length + kTokens - 1) / kTokens;
    constexpr uint32_t kEvery = kSolo ? 1 : kWaves;
    const uint32_t share = ((held + parts - 1) / parts + kEvery - 1) / kEvery * kEvery;
    const uint32_t begin = min(part * share, held);
    uint32_t t = begin + (kSolo ? 0 : wave);

    const Meta *const meta = metas + head * all_blocks;
    const uint32_t key_of = (m / 4) * 16 + m % 4;   // + 4 u: the lane's key row
    u32x4 kr[4][NC > 0 ? NC : 1], vr[NV];
    u32x2 ko[4];
    auto load_k = [&](uint32_t t) {
        const uint8_t *base = keys + ((head * all_blocks + t) * kTokens + key_of) * kp;
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
#pragma unroll
            for (uint32_t ch = 0; ch < NC; ++ch) {
                const uint32_t d = ch * 64 + g * 16;   // past the row: its start, against zeros of q
                kr[u][ch] = load_codes<kStream>(reinterpret_cast<const u32x4 *>(base + 4 * u * kp + (d < kp ? d : 0)));
            }
            if constexpr (kOdd) {
                const uint32_t d = NC * 64 + g * 8;
                ko[u] = load_codes<kStream>(reinterpret_cast<const u32x2 *>(base + 4 * u * kp + (d < kp ? d : 0)));
            }
        }
    };
    auto load_v = [&](uint32_t t) {
        const uint8_t *base = values + ((head * all_blocks + t) * vp + m) * kTokens + g * 16;
#pragma unroll
        for (uint32_t j = 0; j < NV; ++j)
            if (j * 16 < vp) vr[j] = load_codes<kStream>(reinterpret_cast<const u32x4 *>(base + j * 16 * kTokens));
    };
    Meta now_meta = scalar_meta(meta + min(t, all_blocks - 1));
    // (a part of rows that see less than it holds asks for a block it does not use)
    if (t < min(begin + share, whole)) {
        load_k(t);
        load_v(t);
    }
    const uint32_t in_head = group * n, count = kBoth ? own.count : rows_there(a, b);
    // (the last rows, which see most keys, first)
    const uint32_t row0 = (a.row_groups - 1 - a.row_group0 - x / parts) * kRows;
    // what the rows see, from the first one's place among its query head's n
    const uint32_t i0 = n == 1 ? 0 : row0 % n;
    const bool another = row0 + (n - i0) < in_head && i0 + kRows > n;   // rows of a next query head too
    if (count == 0 || (i0 >= count && !another)) return;
    const uint32_t last = i0 + kRows >= n ? n - 1 : i0 + kRows - 1;
    const int before = (int)length - (int)count;
    const int most = a.causal ? before + (int)min(last, count - 1) + 1 : (int)length;
    const int least = a.causal ? before + (int)(another ? 0 : i0) + 1 : (int)length;
    const uint32_t blocks = ((uint32_t)max(most, 0) + kTokens - 1) / kTokens;
    const uint32_t end = min(begin + share, blocks), end_whole = min(end, whole);
    const uint32_t r = row0 + m, i = n == 1 ? 0 : r % n;
    bool live = r < in_head && i < count;
    const uint32_t loaded = loaded_row(r, i, in_head, n, count);
    size_t row = head * in_head + loaded;
    if constexpr (kBoth) row = ((size_t)own.sequence * heads + h) * in_head + loaded;
    else if constexpr (kShared) {
        row = shared_row(a, loaded, b, h, in_head);
        if (a.padded != 0) {   // (all of the workgroup's waves have the same rows)
            live = live && no_padding(a, loaded, b);
            const uint64_t some = __builtin_amdgcn_ballot_w64(live);
            if (some == 0) return;
            row = live ? row : row_among(row, some);
        }
    }
    const int seen = seen_by(i, live, length, count, a.causal);
    Query<S, P> q;
    q.load(queries + row * c.dim, c.dim, g);

    const float neg_inf = -__builtin_inff();
    f32x4 o[NV];
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) o[j] = f32x4{0, 0, 0, 0};
    float big = neg_inf, sum = 0.0f, exact = 0.0f, unit = 1.0f, inverse_unit = 1.0f;

    // one block: kf(u, s) and vf(j, s) give the A operands
    auto step = [&](uint32_t t, Meta meta, auto kf, auto vf, auto keys_done) {
        // The factor of raw products, for f32 times the row's 2^shift, is kept finite:
        // a product of 0 is a score of 0 at any scale. f32: what rounding takes off the
        // factor and the scores is added back in the exponent (scores of 10 would be
        // off by 1e-6 of their weight)
        double whole_factor = (double)meta.k_scale * a.scale2;
        if constexpr (kPair) whole_factor = __builtin_ldexp(whole_factor, q.shift);
        const float factor = fminf(fmaxf((float)whole_factor, -kHuge), kHuge);
        float factor_rest = 0.0f;
        if constexpr (kPair) factor_rest = fabsf(factor) < kHuge ? (float)(whole_factor - (double)factor) : 0.0f;
        float p[16], rest[kPair ? 16 : 1];
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
            f32x4 acc = {0, 0, 0, 0};
            half8 k[Query<S, P>::kSteps];
#pragma unroll
            for (uint32_t s = 0; s < Query<S, P>::kSteps; ++s) k[s] = kf(u, s);
#pragma unroll
            for (uint32_t i = 0; i < kPieces<S>; ++i)
#pragma unroll
                for (uint32_t s = 0; s < Query<S, P>::kSteps; ++s)
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[s], q.piece[i][s], acc, 0, 0, 0);
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
                p[e] = mine >> e & 1 ? __builtin_nanf("") : p[e];
                p[e] = (int)(t * kTokens + 16 * g + e) >= seen ? neg_inf : p[e];
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
            exact *= alpha;
#pragma unroll
            for (uint32_t j = 0; j < NV; ++j) o[j] *= alpha;
            big = now;
        }
        // nothing seen yet: every score is -inf (p = 0) or NaN
        const float base = big == neg_inf ? 0.0f : big - kHeadroom<S>;
        float ratio = meta.v_scale * inverse_unit;
        if (meta.v_scale == 0.0f) {
            ratio = 1.0f;   // its codes are zeros
        } else if (ratio > kUnitRange || ratio < 1.0f / kUnitRange) {
#pragma unroll
            for (uint32_t j = 0; j < NV; ++j) o[j] *= unit / meta.v_scale;
            unit = meta.v_scale;
            inverse_unit = 1.0f / unit;
            ratio = 1.0f;
        }
        half8 ph[2], pl[kPair ? 2 : 1];
        float add = 0.0f;
#pragma unroll
        for (uint32_t e = 0; e < 16; ++e) {
            float x = p[e] - base;
            if constexpr (kPair) x += rest[e];
            x = p[e] = __builtin_amdgcn_exp2f(x);
            float y = x * (ratio * kPairScale<S>);
            // (an f32 here: the compiler may take one f16 from the product's f32 and
            // another, elsewhere, from the product itself, and the rest of the wrong one)
            if constexpr (kPair) asm("" : "+v"(y));
            ph[e / 8][e % 8] = (_Float16)y;
            if constexpr (kPair) {
                pl[e / 8][e % 8] = (_Float16)(y - (float)ph[e / 8][e % 8]);
                add += x;
            } else {
                add += (float)ph[e / 8][e % 8];   // the sum of P as the product has it
            }
        }
        sum += kPair ? add : add * fast_rcp(ratio);
        if (!kPair && a.part_exact != nullptr) {
            add = 0.0f;
#pragma unroll
            for (uint32_t e = 0; e < 16; ++e) add += p[e];
            exact += add;
        }
#pragma unroll
        for (uint32_t j = 0; j < NV; ++j) {
            if (j * 16 >= vp) continue;
            if constexpr (kPair) {
                const half8 v[2] = {vf(j, 0), vf(j, 1)};
                f32x4 x = {0, 0, 0, 0};
#pragma unroll
                for (uint32_t s = 0; s < 2; ++s) x = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[s], pl[s], x, 0, 0, 0);
#pragma unroll
                for (uint32_t s = 0; s < 2; ++s) x = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[s], ph[s], x, 0, 0, 0);
                o[j] += x;
            } else {
#pragma unroll
                for (uint32_t s = 0; s < 2; ++s) o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf(j, s), ph[s], o[j], 0, 0, 0);
            }
        }
    };

    for (; t < end_whole; t += kEvery) {
        const uint32_t next = t + kEvery;
        Meta next_meta;
        step(
            t, now_meta,
            [&](uint32_t u, uint32_t s) {
                if (s / 2 < NC) return codes(kr[u][s / 2][s % 2 * 2], kr[u][s / 2][s % 2 * 2 + 1]);
                return codes(ko[u].x, ko[u].y);
            },
            [&](uint32_t j, uint32_t s) { return codes(vr[j][2 * s], vr[j][2 * s + 1]); },
            [&] {
                // (asked for a block ahead as the codes are, but where this block's is in:
                // a wait for one scalar load waits for all)
                next_meta = scalar_meta(meta + min(next, all_blocks - 1));
                if (next < end_whole) load_k(next);
            });
        if (next < end_whole) load_v(next);
        now_meta = next_meta;
    }
    if (t == whole && t < end) {   // the open block, in f16
        const _Float16 *kt = c.kt + (head * kTokens + key_of) * c.kp;
        const _Float16 *vt = c.vt + (head * c.vp + m) * kTokens + g * 16;
        step(
            t, Meta{1.0f, 1.0f, now_meta.marked},
            [&](uint32_t u, uint32_t s) {
                const uint32_t d = step_dim<P>(s, g);
                return *reinterpret_cast<const half8 *>(kt + 4 * u * c.kp + (d < c.kp ? d : 0));
            },
            [&](uint32_t j, uint32_t s) { return *reinterpret_cast<const half8 *>(vt + j * 16 * kTokens + s * 8); }, [] {});
    }

    // the waves meet
    sum = groups_sum(sum);
    exact = kPair ? sum : groups_sum(exact);
    big -= kHeadroom<S>;   // what P's exponents are relative to
    if constexpr (kSolo) {
        static_assert(kShared);
        if (!live || r >= in_head) return;
        float *const out = a.part_o + ((size_t)part * a.rows + row) * c.vdim;
#pragma unroll
        for (uint32_t j = 0; j < NV; ++j) store_out(out, c.vdim, 16 * j + 4 * g, o[j] * (unit / kPairScale<S>));
        if (g == 0) a.part_ml[(size_t)part * a.rows + row] = f32x2{big, sum};
        return;
    }
    if (g == 0) lds_ml[place][m] = f32x4{big, sum, exact, 0.0f};
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) lds_o[place][j][lane] = o[j] * (unit / kPairScale<S>);
    __syncthreads();
    float top = neg_inf, total = 0.0f, total_exact = 0.0f, w[kMeet];
#pragma unroll
    for (uint32_t k = 0; k < kMeet; ++k) top = fmaxf(top, lds_ml[k][m].x);
#pragma unroll
    for (uint32_t k = 0; k < kMeet; ++k) {
        // (a wave that saw nothing has weight 0, and a NaN in it stays)
        w[k] = top == neg_inf ? 1.0f : __builtin_amdgcn_exp2f(lds_ml[k][m].x - top);
        total += w[k] * lds_ml[k][m].y;
        total_exact += w[k] * lds_ml[k][m].z;
    }
    const bool writes = live && r < in_head;
    if (kBoth || (!kShared && parts == 1)) {
        S *const out = a.out + row * c.vdim;
#pragma unroll
        for (uint32_t j = place; j < NV; j += kMeet) {
            f32x4 v = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t k = 0; k < kMeet; ++k) v += lds_o[k][j][lane] * w[k];
            if (writes) store_out(out, c.vdim, 16 * j + 4 * g, finish(v, top, total));
        }
        if (writes && g == 0 && place == 0) {
            if (a.row_ml != nullptr) a.row_ml[row] = weight_terms(top, total_exact);
            if (a.scores != nullptr) {
                a.part_ml[row] = f32x2{top, total};
                a.part_exact[row] = total_exact;
            }
        }
    } else {
        float *const out = a.part_o + ((size_t)part * a.rows + row) * c.vdim;
#pragma unroll
        for (uint32_t j = place; j < NV; j += kMeet) {
            f32x4 v = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t k = 0; k < kMeet; ++k) v += lds_o[k][j][lane] * w[k];
            if (writes) store_out(out, c.vdim, 16 * j + 4 * g, v);
        }
        if (writes && g == 0 && place == 0) {
            a.part_ml[(size_t)part * a.rows + row] = f32x2{top, total};
            if (a.part_exact != nullptr) a.part_exact[(size_t)part * a.rows + row] = total_exact;
        }
    }
}

}  // namespace kv
}  // namespace icsdk
