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
// f32: q is three f16 operands (scaled by a power of two to a largest element of 2^13 ..
// 2^14), P a pair, 22 significant bits, and codes are exact. A block's output is added
// to the running one in f32, rounded to nearest, as the MFMA does not.
//
// f16: the output is divided by the sum of P as rounded to f16, so that a row with one
// large weight has its value exactly; accumulated token weights, which are f32, go by the
// sum before that rounding. Token weights of either type go by scores in one f32, off by
// 2^-24 of the score: sums of many rows' weights, for which 32 bits are enough.
#include "kv_attention.hpp"

namespace icsdk {
namespace kv {
namespace {

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
// kShared: a pass of attention over a prefix and own tokens.
template <typename S, uint32_t P, bool kStream, bool kShared>
__global__ __launch_bounds__(kThreads) void kv_rows_kernel(const uint8_t *keys, const uint8_t *values,
                                                           const uint32_t *lengths, const Meta *metas, const S *queries,
                                                           uint32_t all_blocks, uint32_t heads, uint32_t parts_first,
                                                           uint32_t pitches, uint32_t n, uint32_t group,
                                                           typename ArgsOf<S, kShared>::type a) {
    constexpr bool kPair = sizeof(S) == 4;
    constexpr uint32_t NC = P / 64, NV = P / 16;
    constexpr bool kOdd = P % 64 != 0;
    __shared__ f32x4 lds_o[kWaves][NV][kWave];
    __shared__ f32x4 lds_ml[kWaves][kRows];   // maximum, sums of P rounded and not
    const View &c = a.c;
    const uint32_t lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t parts = parts_first & 0xffffu, kp = pitches & 0xffffu, vp = pitches >> 16;
    const uint32_t h = blockIdx.y, b = blockIdx.z, seq = (parts_first >> 16) + b;
    const uint32_t length = lengths[seq];
    const uint32_t part = blockIdx.x % parts;
    const size_t head = (size_t)seq * heads + h;
    // the part's blocks, the open one (the last, in f16) among them
    const uint32_t whole = length / kTokens, held = (length + kTokens - 1) / kTokens;
    const uint32_t share = ((held + parts - 1) / parts + kWaves - 1) / kWaves * kWaves;
    const uint32_t begin = min(part * share, held);
    uint32_t t = begin + wave;

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
    const uint32_t in_head = group * n, count = a.count.n[b];
    // (the last rows, which see most keys, first)
    const uint32_t row0 = (a.row_groups - 1 - a.row_group0 - blockIdx.x / parts) * kRows;
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
    const bool live = r < in_head && i < count;
    size_t row = head * in_head + (r < in_head ? r : in_head - 1);   // (rows past the head repeat its last)
    if constexpr (kShared) row = shared_row(a, r, b, h, in_head, count);
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

    for (; t < end_whole; t += kWaves) {
        const uint32_t next = t + kWaves;
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
    if (g == 0) lds_ml[wave][m] = f32x4{big, sum, exact, 0.0f};
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) lds_o[wave][j][lane] = o[j] * (unit / kPairScale<S>);
    __syncthreads();
    float top = neg_inf, total = 0.0f, total_exact = 0.0f, w[kWaves];
#pragma unroll
    for (uint32_t k = 0; k < kWaves; ++k) top = fmaxf(top, lds_ml[k][m].x);
#pragma unroll
    for (uint32_t k = 0; k < kWaves; ++k) {
        // (a wave that saw nothing has weight 0, and a NaN in it stays)
        w[k] = top == neg_inf ? 1.0f : __builtin_amdgcn_exp2f(lds_ml[k][m].x - top);
        total += w[k] * lds_ml[k][m].y;
        total_exact += w[k] * lds_ml[k][m].z;
    }
    const bool writes = live && r < in_head;
    if (!kShared && parts == 1) {
        S *const out = a.out + row * c.vdim;
#pragma unroll
        for (uint32_t j = wave; j < NV; j += kWaves) {
            f32x4 v = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t k = 0; k < kWaves; ++k) v += lds_o[k][j][lane] * w[k];
            if (writes) store_out(out, c.vdim, 16 * j + 4 * g, finish(v, top, total));
        }
        if (writes && g == 0 && wave == 0) {
            if (a.row_ml != nullptr) a.row_ml[row] = weight_terms(top, total_exact);
            if (a.scores != nullptr) {
                a.part_ml[row] = f32x2{top, total};
                a.part_exact[row] = total_exact;
            }
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
        if (writes && g == 0 && wave == 0) {
            a.part_ml[(size_t)part * a.rows + row] = f32x2{top, total};
            if (a.part_exact != nullptr) a.part_exact[(size_t)part * a.rows + row] = total_exact;
        }
    }
}

// Maximum and sum (`exact`: the one before P's rounding) of a row from its parts',
// by one wave.
__device__ inline f32x2 fold_ml(const f32x2 *ml, const float *exact, uint32_t parts, size_t rows, uint32_t lane) {
    float top = -__builtin_inff(), total = 0.0f;
    for (uint32_t s = lane; s < parts; s += kWave) top = fmaxf(top, ml[s * rows].x);
    top = wave_max(top);
    for (uint32_t s = lane; s < parts; s += kWave) {
        const f32x2 v = ml[s * rows];
        total += (top == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(v.x - top)) *
                 (exact != nullptr ? exact[s * rows] : v.y);
    }
    return f32x2{top, wave_sum(total)};
}

// Merges the parts of rows, kRowWaves waves for each: the waves take the parts in
// turn, a lane four output elements. The workgroups after `folds` do a token per
// thread of one (sequence, head): their weights from the stored scores. Bound by
// its chain of memory latencies: up to 4 parts one wave per row, up to 16 four. 3 to 6
// us. (The last workgroup of a row folding in the rows kernel instead: 60 us more, for
// the fences that order its parts.)
template <typename S, uint32_t kFoldWaves, uint32_t kRowWaves>
__global__ __launch_bounds__(kFoldWaves *kWave) void kv_fold_kernel(const float *part_o, const f32x2 *part_ml, size_t rows,
                                                                  uint32_t parts, uint32_t n, uint32_t in_head,
                                                                  uint32_t vdim, uint32_t folds, uint32_t first_row,
                                                                  uint32_t token_groups, uint32_t all_rows, Args<S> a) {
    constexpr uint32_t kFoldThreads = kFoldWaves * kWave, kHeld = 4;
    __shared__ f32x4 lds_o[kFoldWaves][kWave];
    __shared__ f32x2 lds_ml[kRows];
    const View &c = a.c;
    const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (blockIdx.x >= folds) {
        const uint32_t tg = (blockIdx.x - folds) % token_groups, pair = (blockIdx.x - folds) / token_groups;
        const uint32_t b = pair / c.heads, seq = a.first + b, length = min(c.length[seq], a.weight_tokens);
        const size_t head = (size_t)seq * c.heads + pair % c.heads;
        if (tg * kFoldThreads >= length) return;
        for (uint32_t r = wave; r < in_head; r += kFoldWaves) {
            const size_t row = head * in_head + r;
            const f32x2 ml = r % a.n < a.count.n[b] ? fold_ml(a.part_ml + row, a.part_exact + row, a.parts, a.rows, lane)
                                                    : f32x2{-__builtin_inff(), 0.0f};
            if (lane == 0) lds_ml[r] = weight_terms(ml.x, ml.y);
        }
        __syncthreads();
        const uint32_t t = tg * kFoldThreads + threadIdx.x;
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
    const uint32_t of_pairs = blockIdx.x * (kFoldWaves / kRowWaves) + wave / kRowWaves, first = wave % kRowWaves;
    if (of_pairs >= all_rows) return;   // (with one row per workgroup, none)
    const size_t row = (size_t)first_row + of_pairs;
    // four of the wave's parts are asked for along with all parts' maxima (a part
    // past the last one again, left out of the sums)
    f32x4 v = {0, 0, 0, 0}, held[kHeld];
    float held_m[kHeld];
    const uint32_t d = 4 * lane, last = parts - 1;
    auto load = [&](uint32_t s) {
        const float *src = part_o + ((size_t)min(s, last) * rows + row) * vdim;
        f32x4 x;
        if (vdim % 4 == 0) {
            x = *reinterpret_cast<const f32x4 *>(src + (d < vdim ? d : 0));
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) x[e] = src[d + e < vdim ? d + e : 0];
        }
        return x;
    };
#pragma unroll
    for (uint32_t k = 0; k < kHeld; ++k) {
        held[k] = load(first + k * kRowWaves);
        held_m[k] = part_ml[(size_t)min(first + k * kRowWaves, last) * rows + row].x;
    }
    // a row of padding has no parts: what is there is read, and not used
    const uint32_t b = of_pairs / (in_head * c.heads);
    const bool there = of_pairs % n < a.count.n[b];
    const f32x2 all = fold_ml(part_ml + row, nullptr, parts, rows, lane);
    auto weight = [&](float m) { return all.x == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - all.x); };
#pragma unroll
    for (uint32_t k = 0; k < kHeld; ++k)
        if (first + k * kRowWaves < parts) v += held[k] * weight(held_m[k]);
#pragma unroll 4
    for (uint32_t s = first + kHeld * kRowWaves; s < parts; s += kRowWaves)
        v += load(s) * weight(part_ml[(size_t)s * rows + row].x);
    if constexpr (kRowWaves > 1) {
        lds_o[wave][lane] = v;
        __syncthreads();
        if (first != 0) return;
        for (uint32_t k = 1; k < kRowWaves; ++k) v += lds_o[k][lane];
    }
    if (!there) return;
    store_out(a.out + row * vdim, vdim, d, finish(v, all.x, all.y));
    if (a.row_ml != nullptr) {
        const f32x2 whole = fold_ml(part_ml + row, a.part_exact + row, parts, rows, lane);
        if (lane == 0) a.row_ml[row] = weight_terms(whole.x, whole.y);
    }
}

// ---- plan and launch ---------------------------------------------------------------

struct Plan {
    bool tiles;    // many rows: k_kv_tiles.hip
    bool scores;   // the weights come from scores that the rows kernel stores (never with tiles)
    uint32_t row_groups, parts, row_parts;
    size_t rows, score_stride;
    size_t o_bytes, ml_bytes, exact_bytes, row_bytes, score_bytes, partial_bytes;
    size_t bytes() const { return o_bytes + ml_bytes + exact_bytes + row_bytes + score_bytes + partial_bytes; }
};

size_t whole256(size_t bytes) { return (bytes + 255) / 256 * 256; }
uint32_t widest_of(const View &c) { return c.kp > c.vp ? c.kp : c.vp; }

// Products of a call from which the kernel of 128-row tiles is used: it reads each
// operand for twice the rows and takes each code to f16 once for 128, but a
// workgroup's turn lasts long. Measured (us, rows kernel and tiles, causal): f16 D 128,
// 8 heads x 512 rows x 2000 keys (1.0e9) 22 and 30, 8 x 384 x 8000 (3.1e9) 54 and 48,
// 32 x 512 x 8000 175 and 90; D 64, 32 x 384 x 2000 (1.6e9) 23 and 38, 32 x 256 x 8000
// (4.2e9) 53 and 43; D 256, 8 x 512 x 2000 (1.8e9) 50 and 42; f32 D 80, 32 x 512 x 2000
// (2.3e9) 58 and 63, 32 x 1024 x 2000 (3.9e9) 102 and 87; D 128, 32 x 256 x 2000
// (2.0e9) 44 and 52, 8 x 512 x 8000 (4.1e9) 72 and 74, 32 x 512 x 8000 226 and 201.
constexpr double kTileProducts = 2.6e9, kTileProductsF32 = 3.5e9;
// ... where it takes less than the rows kernel's workgroups of 16 rows do: it multiplies
// 128 rows whatever is there, in the time of two of those at f16, of four at dims up to 32
// and of five at f32. Measured at 64 heads x 8000 keys, from 2.6e9 products on (us, rows
// kernel and tiles): f16 D 128, 32 rows 48 and 47, 48 rows 69 and 50, 96 rows 125 and 57; D
// 256, 32 rows 94 and 103, 48 rows 149 and 109; 64 x 32000, D 128, 16 rows 93 and 168; D 64,
// 32 rows 90 and 99, 48 rows 137 and 107; D 32, 64 rows 84 and 88, 96 rows 144 and 91; f32
// D 128, 64 rows 349 and 378, 96 rows 589 and 399; D 64, 64 rows 211 and 255, 96 rows 339
// and 254; 64 x 8000, 160 rows 112 and 129, 256 rows 148 and 134.
constexpr uint32_t rows_for_tile(bool f32, uint32_t widest) { return kRows * (f32 ? 5 : widest <= 32 ? 4 : 2); }
constexpr uint32_t kWorkgroups = 512;   // two for every CU
// Whether a CU holds two workgroups of the rows kernel (their registers decide).
constexpr bool rows_twice(bool f32, uint32_t widest) { return widest <= (f32 ? 128u : 192u); }

Plan plan_of(bool f32, const View &c, const AttentionShape &a) {
    Plan p{};
    const uint32_t in_head = a.q_heads / c.heads * a.n;
    const uint32_t blocks = (a.longest + kTokens - 1) / kTokens;
    const uint64_t pairs = (uint64_t)a.batch * c.heads;
    // keys that a row sees on average
    const double keys = a.longest - (a.causal ? 0.5 * (a.n < a.longest ? a.n : a.longest) : 0.0);
    const double products = (double)pairs * in_head * keys * widest_of(c);
    const uint32_t whole_rows = (in_head + kRows - 1) / kRows * kRows;
    const uint32_t row_tiles = (in_head + kTileRows - 1) / kTileRows;
    p.tiles = whole_rows > (uint64_t)row_tiles * rows_for_tile(f32, widest_of(c)) &&
              products >= (f32 ? kTileProductsF32 : kTileProducts) && tiles_fit(f32, widest_of(c));
    const uint32_t rows_each = p.tiles ? kTileRows : kRows;
    p.row_groups = (in_head + rows_each - 1) / rows_each;
    // parts: workgroups for every CU twice over (once for those of which a CU holds one:
    // tiles, f32 D 128, 8 heads x 512 rows x 8000 keys 74 us, twice over 87; rows, f16 D
    // 256, 8 x 8 heads x 4096 keys 30 us, twice over 35), with a block for each wave
    // (tiles: four blocks) at least
    const uint64_t base = pairs * p.row_groups;
    const bool twice = p.tiles ? tiles_twice(f32, widest_of(c)) : rows_twice(f32, widest_of(c));
    const uint32_t fill = twice ? kWorkgroups : kWorkgroups / 2;
    uint64_t parts = base >= fill ? 1 : fill / base;
    const uint32_t most = (blocks + kWaves - 1) / kWaves;
    parts = parts < most ? parts : most;
    p.parts = parts < 1 ? 1 : (uint32_t)parts;
    p.rows = (size_t)a.batch * a.q_heads * a.n;
    p.o_bytes = p.parts > 1 ? whole256(p.parts * p.rows * c.vdim * 4) : 0;
    // a token's scores, 4 bytes per row written and read again, against its key and
    // the rows again: for up to 16 rows the scores (which the rows kernel, that these
    // always take, stores). Measured (us, scores and a second pass): f16 D 128, 8 heads
    // x 1000 tokens, 4 rows 14 and 22, 16 rows 17 and 22; 256 heads x 8000, 4 rows 143
    // and 238, 16 rows 207 and 240; f32 16 rows 196 and 264; f16 D 64, 8 rows 107 and 128.
    // Of 16 rows at D 64 and less it holds for small caches alone: 8 heads x 1000 15 and
    // 19, 64 x 4000 29 and 31, 256 x 8000 148 and 129 (D 32: 132 and 94)
    p.scores = a.weights != nullptr && in_head <= kRows;
    p.score_stride = (size_t)blocks * kTokens;
    p.ml_bytes = p.parts > 1 || p.scores ? whole256(p.parts * p.rows * sizeof(f32x2)) : 0;
    p.exact_bytes = a.weights != nullptr ? whole256(p.parts * p.rows * sizeof(float)) : 0;
    p.row_bytes = a.weights != nullptr && !p.scores ? whole256(p.rows * sizeof(f32x2)) : 0;
    p.score_bytes = p.scores ? whole256(p.rows * p.score_stride * 4) : 0;
    p.row_parts = 1;
    if (p.row_bytes != 0 && blocks != 0) {
        // weights: workgroups (of four blocks) for every CU twice over, with four
        // steps of 32 rows at least; and, since of causal rows the first blocks are
        // seen by more than the last, at most 24 steps for what of it is uneven (f16
        // D 64, 2 x 15 heads x 4000 rows, of 12000 per kv head: 4 parts 272 us, 13 parts
        // 229; 1500 rows: 9 parts 69 us, 18 parts 72)
        const uint64_t groups = pairs * ((blocks + kWaves - 1) / kWaves), fit = (in_head + kTileRows - 1) / kTileRows;
        uint64_t want = (kWorkgroups + groups - 1) / groups;
        if (a.causal) {
            const uint64_t uneven = (uint64_t)in_head * (a.n < a.longest ? a.n : a.longest) / a.longest;
            const uint64_t more = uneven / (24 * 32) < 16 ? uneven / (24 * 32) : 16;   // (partial sums are memory)
            want = want < more ? more : want;
        }
        p.row_parts = (uint32_t)(want < fit ? want : fit);
        if (p.row_parts > 1) p.partial_bytes = whole256(p.row_parts * pairs * p.score_stride * 4);
    }
    return p;
}

// Codes past what the 256 MB cache behind the L2s holds to the next call are read
// as a stream. One sequence of 131000 tokens (268 MB): 62.5 -> 56.6 us; 8 x 4096
// (67 MB, found there by calls in a row): 19.5, as a stream 20.6.
constexpr size_t kStreamBytes = size_t{192} << 20;

template <typename S, uint32_t P, bool kShared>
hipError_t launch_rows(const typename ArgsOf<S, kShared>::type &a, uint32_t groups, hipStream_t s) {
    const dim3 grid(groups * a.parts, a.c.heads, a.pairs / a.c.heads);
    const size_t bytes = (size_t)a.pairs * a.longest * (a.c.kp + a.c.vp);
    const auto kernel = bytes > kStreamBytes ? kv_rows_kernel<S, P, true, kShared> : kv_rows_kernel<S, P, false, kShared>;
    kernel<<<grid, kThreads, 0, s>>>(a.c.k, a.c.v, a.c.length, a.c.meta, a.q, a.c.blocks, a.c.heads,
                                     a.parts | a.first << 16, a.c.kp | a.c.vp << 16, a.n, a.group, a);
    return hipGetLastError();
}
template <typename S, bool kShared>
hipError_t launch_rows(const typename ArgsOf<S, kShared>::type &a, uint32_t widest, uint32_t groups, hipStream_t s) {
    if (widest <= 32) return launch_rows<S, 32, kShared>(a, groups, s);
    if (widest <= 64) return launch_rows<S, 64, kShared>(a, groups, s);
    if (widest <= 96) return launch_rows<S, 96, kShared>(a, groups, s);
    if (widest <= 128) return launch_rows<S, 128, kShared>(a, groups, s);
    if (widest <= 192) return launch_rows<S, 192, kShared>(a, groups, s);
    return launch_rows<S, 256, kShared>(a, groups, s);
}

// The rows' (or tiles') launches of a plan.
template <typename S, bool kShared>
hipError_t launch_pass(typename ArgsOf<S, kShared>::type a, const Plan &p, hipStream_t s) {
    const uint32_t widest = widest_of(a.c);
    // (a launch holds fewer than 2^32 threads)
    const uint32_t most = (1u << 23) / (a.pairs * p.parts) < 1 ? 1 : (1u << 23) / (a.pairs * p.parts);
    for (uint32_t g0 = 0; g0 < p.row_groups; g0 += most) {
        a.row_group0 = g0;
        const uint32_t groups = p.row_groups - g0 < most ? p.row_groups - g0 : most;
        const hipError_t status = p.tiles ? launch_tiles<S, kShared>(a, widest, groups, s)
                                          : launch_rows<S, kShared>(a, widest, groups, s);
        if (status != hipSuccess) return status;
    }
    return hipSuccess;
}

// Joins `parts` parts of the rows of a launch's sequences; its workgroups after those
// take weights from the stored scores, if there are any.
template <typename S>
hipError_t launch_fold(const Args<S> &a, uint32_t parts, bool scores, uint32_t longest, hipStream_t s) {
    const uint32_t blocks = (longest + kTokens - 1) / kTokens;
    // (at most 512 row groups where there are parts)
    const uint32_t folds = parts > 1 ? a.pairs * a.group * a.n : 0;
    const uint32_t threads = parts > 16 ? 16 * kWave : kThreads;
    const uint32_t token_groups = scores ? (blocks * kTokens + threads - 1) / threads : 0;
    const uint32_t workgroups = parts <= kWaves ? (folds + kWaves - 1) / kWaves : folds;
    const uint32_t grid = workgroups + a.pairs * token_groups;
    if (grid == 0) return hipSuccess;
    auto fold = [&](auto kernel) {
        kernel<<<grid, threads, 0, s>>>(a.part_o, a.part_ml, a.rows, parts, a.n, a.group * a.n, a.c.vdim, workgroups,
                                        a.first * a.c.heads * a.group * a.n, token_groups, folds, a);
    };
    if (parts <= kWaves) fold(kv_fold_kernel<S, kWaves, 1>);
    else if (threads == kThreads) fold(kv_fold_kernel<S, kWaves, kWaves>);
    else fold(kv_fold_kernel<S, 16, 16>);
    return hipGetLastError();
}

template <typename S>
hipError_t launch(const Args<S> &a, const Plan &p, uint32_t batch, uint32_t longest, float *partial, hipStream_t s) {
    const uint32_t blocks = (longest + kTokens - 1) / kTokens;
    hipError_t status = launch_pass<S, false>(a, p, s);
    if (status == hipSuccess && (p.parts > 1 || p.scores)) status = launch_fold(a, p.parts, p.scores, longest, s);
    if (status != hipSuccess) return status;
    if (a.row_ml != nullptr && blocks > 0) return launch_weights(a, widest_of(a.c), batch, blocks, p.row_parts, partial, s);
    return hipSuccess;
}

template <typename S>
hipError_t run(const View &c, const AttentionShape &sh, const void *query, void *output, void *workspace,
               hipStream_t s) {
    const Plan p = plan_of(sizeof(S) == 4, c, sh);
    Args<S> a;
    a.c = c;
    a.q = static_cast<const S *>(query);
    a.out = static_cast<S *>(output);
    char *ws = static_cast<char *>(workspace);
    auto take = [&](size_t bytes) {
        char *const at = bytes ? ws : nullptr;
        ws += bytes;
        return at;
    };
    a.part_o = reinterpret_cast<float *>(take(p.o_bytes));
    a.part_ml = reinterpret_cast<f32x2 *>(take(p.ml_bytes));
    a.part_exact = reinterpret_cast<float *>(take(p.exact_bytes));
    a.row_ml = reinterpret_cast<f32x2 *>(take(p.row_bytes));
    a.scores = reinterpret_cast<float *>(take(p.score_bytes));
    float *const partial = reinterpret_cast<float *>(take(p.partial_bytes));
    a.score_stride = p.score_stride;
    a.weights = sh.weights;
    a.weight_tokens = sh.weight_tokens;
    a.weight_stride = sh.weight_stride;
    a.rows = p.rows;
    a.group = sh.q_heads / c.heads;
    a.n = sh.n;
    a.parts = p.parts;
    a.longest = sh.longest;
    a.row_groups = p.row_groups;
    a.scale2 = (double)sh.scale * kLog2e;
    a.causal = sh.causal;
    for (uint32_t first = 0; first < sh.batch; first += kBatchPerLaunch) {
        const uint32_t batch = sh.batch - first < kBatchPerLaunch ? sh.batch - first : kBatchPerLaunch;
        for (uint32_t b = 0; b < batch; ++b) a.count.n[b] = sh.counts ? sh.counts[first + b] : sh.n;
        a.first = first;
        a.pairs = batch * c.heads;
        const hipError_t status = launch(a, p, batch, sh.longest, partial, s);
        if (status != hipSuccess) return status;
    }
    return hipSuccess;
}

// ---- a prefix and own tokens ---------------------------------------------------------

// Attention of sequences whose tokens follow a prefix that several of them share, in
// two passes into the same rows' parts: over the prefix the rows of a group's sequences
// are packed as one head's rows, so that its codes are read once for all of them, then
// over each sequence's own tokens. A softmax over both is their parts' join.
struct SharedPlan {
    AttentionShape over;   // of the pass over the prefix
    Plan prefix, own;
    size_t rows, o_bytes, ml_bytes;
};

SharedPlan plan_of(bool f32, const View &prefix, const PrefixShape &ps, const View &c, const AttentionShape &a) {
    SharedPlan p;
    p.over = AttentionShape{ps.batch, prefix.heads, ps.most * (a.q_heads / c.heads) * a.n, ps.longest, a.scale, false,
                            nullptr, nullptr, 0, 0};
    p.prefix = plan_of(f32, prefix, p.over);
    p.own = plan_of(f32, c, a);
    p.rows = p.own.rows;
    const size_t parts = p.prefix.parts + p.own.parts;
    p.o_bytes = whole256(parts * p.rows * c.vdim * 4);
    p.ml_bytes = whole256(parts * p.rows * sizeof(f32x2));
    return p;
}

template <typename S>
hipError_t run_shared(const View &prefix, const PrefixShape &ps, const View &c, const AttentionShape &sh,
                      const void *query, void *output, void *workspace, hipStream_t s) {
    const SharedPlan p = plan_of(sizeof(S) == 4, prefix, ps, c, sh);
    const uint32_t group = sh.q_heads / c.heads;
    SharedArgs<S> a{};
    a.q = static_cast<const S *>(query);
    a.out = static_cast<S *>(output);
    a.part_o = static_cast<float *>(workspace);
    a.part_ml = reinterpret_cast<f32x2 *>(static_cast<char *>(workspace) + p.o_bytes);
    a.rows = p.rows;
    a.scale2 = (double)sh.scale * kLog2e;
    a.own_rows = group * sh.n;
    // a group's rows are one head's rows here, all of them there
    a.c = prefix;
    a.group = 1;
    a.n = p.over.n;
    a.parts = p.prefix.parts;
    a.longest = ps.longest;
    a.row_groups = p.prefix.row_groups;
    uint32_t sequence = 0;
    for (uint32_t first = 0; first < ps.batch; first += kBatchPerLaunch) {
        const uint32_t batch = ps.batch - first < kBatchPerLaunch ? ps.batch - first : kBatchPerLaunch;
        for (uint32_t b = 0; b < batch; ++b) {
            a.member.n[b] = ps.members[first + b] != 0 ? sequence : 0;   // (of none, a row that is there)
            a.count.n[b] = ps.members[first + b] * a.own_rows;
            sequence += ps.members[first + b];
        }
        a.first = first;
        a.pairs = batch * c.heads;
        const hipError_t status = launch_pass<S, true>(a, p.prefix, s);
        if (status != hipSuccess) return status;
    }
    a.c = c;
    a.group = group;
    a.n = sh.n;
    a.parts = p.own.parts;
    a.longest = sh.longest;
    a.row_groups = p.own.row_groups;
    a.causal = sh.causal;
    float *const part_o = a.part_o;
    f32x2 *const part_ml = a.part_ml;
    for (uint32_t first = 0; first < sh.batch; first += kBatchPerLaunch) {
        const uint32_t batch = sh.batch - first < kBatchPerLaunch ? sh.batch - first : kBatchPerLaunch;
        for (uint32_t b = 0; b < batch; ++b) {
            a.member.n[b] = first + b;
            a.count.n[b] = sh.counts ? sh.counts[first + b] : sh.n;
        }
        a.first = first;
        a.pairs = batch * c.heads;
        a.part_o = part_o + (size_t)p.prefix.parts * p.rows * c.vdim;
        a.part_ml = part_ml + (size_t)p.prefix.parts * p.rows;
        hipError_t status = launch_pass<S, true>(a, p.own, s);
        a.part_o = part_o;
        a.part_ml = part_ml;
        if (status == hipSuccess) status = launch_fold<S>(a, p.prefix.parts + p.own.parts, false, 0, s);
        if (status != hipSuccess) return status;
    }
    return hipSuccess;
}

}  // namespace

size_t attention_workspace(bool f32, const View &c, const AttentionShape &a) { return plan_of(f32, c, a).bytes(); }

hipError_t attention(bool f32, const View &c, const AttentionShape &a, const void *query, void *output,
                     void *workspace, hipStream_t s) {
    return f32 ? run<float>(c, a, query, output, workspace, s) : run<_Float16>(c, a, query, output, workspace, s);
}

size_t attention_shared_workspace(bool f32, const View &prefix, const PrefixShape &p, const View &c,
                                  const AttentionShape &a) {
    const SharedPlan plan = plan_of(f32, prefix, p, c, a);
    return plan.o_bytes + plan.ml_bytes;
}

hipError_t attention_shared(bool f32, const View &prefix, const PrefixShape &p, const View &c, const AttentionShape &a,
                            const void *query, void *output, void *workspace, hipStream_t s) {
    return f32 ? run_shared<float>(prefix, p, c, a, query, output, workspace, s)
               : run_shared<_Float16>(prefix, p, c, a, query, output, workspace, s);
}

}  // namespace kv
}  // namespace icsdk
