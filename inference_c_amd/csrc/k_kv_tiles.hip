// Attention over the 8-bit cache for many query rows: tiles of 128 packed rows
// and 64 keys (kv_attention.hpp, kv.hpp).
//
// v_mfma_f32_32x32x16_f16: A[m][k] in lane l at m = l % 32, k = 8 (l / 32) + e;
// B[k][n] at n = l % 32 likewise; D[m][n] at n = l % 32, m = 8 (r / 4) + 4 (l / 32) +
// r % 4. A wave of 32 rows computes, per block of 64 keys,
//   S^T = K Q^T in two halves of 32 keys. A row m is key m with its bits 2 and 3
//     exchanged, so that accumulator registers 8 c .. 8 c + 7 of a lane are the
//     keys 16 c + 8 (l / 32) + 0 .. 7: consecutive, and
//   out^T = V^T P^T takes them as B operands in their order, with the dim's same
//     keys side by side in memory: one 16-byte LDS read per A operand.
// Each block's codes are turned to f16 once, on their way into LDS (key rows 8
// halves longer than the data, dim rows of 72: no bank conflicts).
// Scores stay raw products; the block's factor k_scale * scale * log2 e enters with
// the maximum in one fma, the ratio of its value scale to the unit as an addend of
// the exponent (k_kv_attention.hip has the rules).
#include "flash.hpp"
#include "kv_attention.hpp"

namespace icsdk {
namespace kv {
namespace {

typedef float float16v __attribute__((ext_vector_type(16)));

// 32 query rows as B operands, one per 16 dims and piece, times `sign`
// (the scale's; 0 where the scale is).
template <typename S, uint32_t P> struct TileQuery {
    static constexpr uint32_t kSteps = P / 16;
    static constexpr bool kPair = sizeof(S) == 4;
    half8 piece[kPieces<S>][kSteps];
    int shift = 0;   // an f32 row was divided by 2^shift

    __device__ inline void load(const S *row, uint32_t dim, uint32_t half, float sign) {
        if constexpr (!kPair) {
            const _Float16 s = (_Float16)sign;
            if (dim % 8 == 0) {
#pragma unroll
                for (uint32_t c = 0; c < kSteps; ++c) {
                    const uint32_t d = 16 * c + 8 * half;
                    piece[0][c] = *reinterpret_cast<const half8 *>(row + (d < dim ? d : 0));
                }
#pragma unroll
                for (uint32_t c = 0; c < kSteps; ++c) {
                    piece[0][c] *= s;
                    if (16 * c + 8 * half >= dim) piece[0][c] = half8{};
                }
            } else {
#pragma unroll
                for (uint32_t c = 0; c < kSteps; ++c)
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) {
                        const uint32_t d = 16 * c + 8 * half + e;
                        piece[0][c][e] = d < dim ? row[d] * s : (_Float16)0.0f;
                    }
            }
        } else {
            float x[kSteps][8], big = 0.0f;
            bool finite = true;
#pragma unroll
            for (uint32_t c = 0; c < kSteps; ++c) load8(row, dim, 16 * c + 8 * half, x[c]);
#pragma unroll
            for (uint32_t c = 0; c < kSteps; ++c)
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) {
                    x[c][e] *= sign;
                    big = fmaxf(big, fabsf(x[c][e]));
                    finite = finite && __builtin_isfinite(x[c][e]);
                }
            big = flash::pair_max(finite ? big : __builtin_inff());
            const bool usable = big > 0.0f && __builtin_isfinite(big);
            const int exponent = usable ? __builtin_amdgcn_frexp_expf(big) : 14;
            shift = exponent - 14;
            const float none = big > 0.0f ? __builtin_nanf("") : 0.0f;   // (not finite: no score is)
#pragma unroll
            for (uint32_t c = 0; c < kSteps; ++c)
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) {
                    const float y = usable ? __builtin_ldexpf(x[c][e], -shift) : none;
                    pieces_of(y, piece[0][c], piece[1][c], piece[2][c], e);
                }
        }
    }
};

// A block's factor of raw products, for f32 times the query row's 2^shift, and what
// rounding took off it. Positive (queries carry the scale's sign) and finite: masked
// products are -inf before it. Below kTiny products come to nothing either way. A block
// of zero keys has raw products 0: any factor.
template <typename S, bool kExact> __device__ inline f32x2 block_factor(float k_scale, double scale2, int shift) {
    const float k = k_scale == 0.0f ? 1.0f : k_scale;
    const double scale = scale2 == 0.0 ? 1.0 : fabs(scale2);
    if constexpr (sizeof(S) == 2 && !kExact) {
        return f32x2{fminf(fmaxf(k * (float)scale, kTiny), kHuge), 0.0f};
    } else {
        const double f = sizeof(S) == 4 ? __builtin_ldexp((double)k * scale, shift) : (double)k * scale;
        const float hi = fminf(fmaxf((float)f, kTiny), kHuge);
        return f32x2{hi, (float)(f - (double)hi)};
    }
}

// Key row of the block that A row m of a half reads.
__device__ inline uint32_t swap23(uint32_t m) { return (m & 0x13u) | (m & 4u) << 1 | (m & 8u) >> 1; }

// The mark bits of a lane's 32 keys, in its order of them (16 i + 8 half + 0 .. 7).
__device__ inline uint32_t marks_of(uint64_t marked, uint32_t half) {
    const uint64_t m = marked >> (8 * half);
    return (uint32_t)(m & 255u) | (uint32_t)(m >> 8 & 0xff00u) | (uint32_t)(m >> 16 & 0xff0000u) |
           (uint32_t)(m >> 24 & 0xff000000u);
}

// N matrix steps with other work in between: operand(i) reads step i's A operand
// (four steps ahead), product(i, operand) issues its MFMA, work(i) is step i's share
// of the rest, and nothing moves from one step to another. An MFMA takes 8 cycles to
// issue and 32 to complete, and the SIMD issues 6 vector instructions (3
// transcendental ones) meanwhile at no cost, but only if they come in between: of
// two waves on a SIMD, one in a stretch of MFMAs and one in a stretch of vector
// instructions, neither gained, and the compiler by itself makes such stretches.
template <uint32_t N, typename R, typename M, typename W>
__device__ inline void steps(R operand, M product, W work) {
    constexpr uint32_t kAhead = 4;
    half8 a[N];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (uint32_t i = 0; i < kAhead && i < N; ++i) a[i] = operand(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
        product(i, a[i]);
        if (i + kAhead < N) a[i + kAhead] = operand(i + kAhead);
        work(i);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// A workgroup: 128 packed rows, 32 per wave, of one (sequence, kv head), and one
// part of its blocks; the open block first. The loop is skewed: turn s multiplies
// P of tile s - 1 with its values while it takes the maxima of tile s and turns
// codes to f16, then multiplies the keys of tile s + 1 while it takes the
// exponentials of tile s.
// 32 heads x 2048 rows over 8192 keys, D 128, f16: 268 us, 900 TFLOP/s, where a library
// product of 8192^3 reaches 1340. MFMAs take half of the cycles; a turn has 1024 of
// them, 1260 of vector instructions, of which those between MFMAs hide, and LDS reads
// for 70% of its time. Measured and left: 256 rows on eight waves (250 us here, but
// 4 x 8 heads x 2000 rows over themselves 57 -> 65 us, being one round of uneven
// workgroups), two groups of four waves a phase apart (332 us), first operands of a
// phase asked for in the one before (1%).
// kExact: with the sum of P before its rounding to f16 too, for the weights.
template <typename S, uint32_t P, bool kExact>
__global__ __launch_bounds__(kThreads, tiles_twice(sizeof(S) == 4, P) ? 2 : 1) void kv_tiles_kernel(Args<S> a) {
    constexpr bool kPair = sizeof(S) == 4;
    static_assert(!kPair || !kExact);   // (its sum is exact by itself)
    constexpr uint32_t KC = P / 16, VT = (P + 31) / 32;
    constexpr uint32_t KROW = P + 8, VROW = kTokens + 8;   // LDS rows, halves
    constexpr uint32_t KTILE = kTokens * KROW, VTILE = VT * 32 * VROW;
    constexpr uint32_t KPER = (kTokens * P / 16 + kThreads - 1) / kThreads;   // 16-byte pieces of codes per thread
    // Of a row's groups of 8 the even ones lie in its first half and the odd ones
    // in its second, so that a wave's lanes write 16 bytes side by side.
    constexpr uint32_t KHALF = P / 2, VHALF = kTokens / 2;
    // (each tile with a spare place, for pieces past the end)
    __shared__ __attribute__((aligned(16))) _Float16 ks[2][KTILE + KHALF + 8], vs[2][VTILE + VHALF + 8];
    __shared__ int wave_most[kWaves];
    const View &c = a.c;
    const uint32_t tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane(tid / kWave);
    // workgroup -> (rows, part, (sequence, head)): the last rows, which see most
    // keys, first; one head's workgroups on one XCD where the heads are whole eights
    const uint32_t in_head = a.group * a.n, row_blocks = (in_head + kTileRows - 1) / kTileRows;
    const uint32_t pair = blockIdx.x % a.pairs, rest = blockIdx.x / a.pairs + a.row_group0 * a.parts;
    const uint32_t part = rest % a.parts, row_block = row_blocks - 1 - rest / a.parts;
    const uint32_t b = pair / c.heads, h = pair % c.heads, seq = a.first + b;
    const size_t head = (size_t)seq * c.heads + h;
    const uint32_t length = c.length[seq], count = a.count.n[b];
    const uint32_t r = row_block * kTileRows + wave * 32 + col, i = r % a.n;
    const bool live = r < in_head && i < count;
    const size_t row = head * in_head + min(r, in_head - 1);
    const int seen = seen_by(i, live, length, count, a.causal);
    // keys that some row of the workgroup, and that every row of the wave, sees
    int most = live ? seen : 0, least = live ? seen : (int)length;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        most = max(most, __shfl_xor(most, d, kWave));
        least = min(least, __shfl_xor(least, d, kWave));
    }
    least = __builtin_amdgcn_readfirstlane(least);
    if (lane == 0) wave_most[wave] = most;
    __syncthreads();
    most = wave_most[0];
#pragma unroll
    for (uint32_t w = 1; w < kWaves; ++w) most = max(most, wave_most[w]);
    most = __builtin_amdgcn_readfirstlane(most);
    const uint32_t blocks = ((uint32_t)max(most, 0) + kTokens - 1) / kTokens, whole = length / kTokens;
    const uint32_t share = (blocks + a.parts - 1) / a.parts;
    const uint32_t begin = min(part * share, blocks), end = min(begin + share, blocks), tiles = end - begin;
    // tile s is block begin + s, or with the open block among them that one first
    const uint32_t open_first = end > whole ? 1 : 0;
    auto block_of = [&](uint32_t s) { return open_first && s == 0 ? whole : min(begin + s - open_first, c.blocks - 1); };

    TileQuery<S, P> q;
    q.load(a.q + row * c.dim, c.dim, half, a.scale2 > 0.0 ? 1.0f : a.scale2 < 0.0 ? -1.0f : 0.0f);
    const Meta *const meta = c.meta + head * c.blocks;
    const uint8_t *const kcodes = c.k + head * c.blocks * kTokens * c.kp;
    const uint8_t *const vcodes = c.v + head * c.blocks * kTokens * c.vp;
    // A tile's Meta comes by a vector load ahead of the codes of the turn before,
    // and is there when they are: a scalar load, which may return before or after any
    // LDS read, would have to be waited for by the next of those.
    uint32_t zero = 0;
    asm volatile("" : "+v"(zero));   // (a lane's address: no scalar load)
    u32x4 meta_ahead;
    auto fetch_meta = [&](uint32_t s) {
        meta_ahead = *reinterpret_cast<const u32x4 *>(reinterpret_cast<const char *>(meta + block_of(s)) + zero);
    };
    auto take_meta = [&](uint32_t s) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (uint32_t)__builtin_amdgcn_readfirstlane((int)meta_ahead[i]);
        Meta m = __builtin_bit_cast(Meta, w);
        if (open_first && s == 0) m.k_scale = m.v_scale = 1.0f;
        return m;
    };

    // the thread's 16-byte pieces of a block's codes (pieces past the end repeat the
    // last one and go to the spare place: no branch lies between the MFMAs)
    const uint32_t kpieces = kTokens * c.kp / 16, vpieces = c.vp * 4;
    uint32_t kto[KPER], vto[KPER];
#pragma unroll
    for (uint32_t u = 0; u < KPER; ++u) {
        const uint32_t p = tid + u * kThreads;
        kto[u] = p < kpieces ? p * 16 / c.kp * KROW + p * 16 % c.kp / 2 : KTILE;
        vto[u] = p < vpieces ? p / 4 * VROW + p % 4 * 8 : VTILE;
    }
    u32x4 kreg[KPER], vreg[KPER];
    // (asked for without a test, past the end some block again: the count of loads
    // in flight is then known wherever one is waited for)
    auto fetch_k = [&](uint32_t s) {
        const u32x4 *from = reinterpret_cast<const u32x4 *>(kcodes + (size_t)block_of(s) * kTokens * c.kp);
#pragma unroll
        for (uint32_t u = 0; u < KPER; ++u) kreg[u] = from[min(tid + u * kThreads, kpieces - 1)];
    };
    auto fetch_v = [&](uint32_t s) {
        const u32x4 *from = reinterpret_cast<const u32x4 *>(vcodes + (size_t)block_of(s) * kTokens * c.vp);
#pragma unroll
        for (uint32_t u = 0; u < KPER; ++u) vreg[u] = from[min(tid + u * kThreads, vpieces - 1)];
    };
    auto put = [&](_Float16 *to, uint32_t far, half8 lo, half8 hi) {
        *reinterpret_cast<half8 *>(to) = lo;
        *reinterpret_cast<half8 *>(to + far) = hi;
    };
    auto stash_k = [&](uint32_t buf) {
#pragma unroll
        for (uint32_t u = 0; u < KPER; ++u)
            put(&ks[buf][kto[u]], KHALF, codes(kreg[u].x, kreg[u].y), codes(kreg[u].z, kreg[u].w));
    };

    const float neg_inf = -__builtin_inff();
    float16v o[VT], st[2];
    half8 ph[4], pl[kPair ? 4 : 1];
#pragma unroll
    for (uint32_t t = 0; t < VT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[t][e] = 0.0f;
#pragma unroll
    for (uint32_t ch = 0; ch < 4; ++ch) {
        ph[ch] = half8{};
        if constexpr (kPair) pl[ch] = half8{};
    }
    float big = neg_inf, sum = 0.0f, exact = 0.0f, unit = 1.0f;   // (sums of the lane's keys)
    // matrix steps of a tile's scores (piece by piece) and outputs (f32: P's rests first)
    constexpr uint32_t NS1 = 2 * KC, NO1 = 4 * VT, NS = kPieces<S> * NS1, NO = kPair ? 2 * NO1 : NO1;
    float16v fresh[kPair ? VT : 1];   // f32: a tile's outputs
    auto key_operand = [&](uint32_t buf, uint32_t i) {
        i %= NS1;
        return *reinterpret_cast<const half8 *>(&ks[buf][(32 * (i % 2) + swap23(col)) * KROW + 8 * (i / 2) + KHALF * half]);
    };
    auto value_operand = [&](uint32_t buf, uint32_t i) {
        i %= NO1;
        return *reinterpret_cast<const half8 *>(&vs[buf][(32 * (i % VT) + col) * VROW + 8 * (i / VT) + VHALF * half]);
    };
    auto score = [&](float16v (&to)[2], uint32_t i, half8 k) {
        to[i % 2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q.piece[i / NS1][i % NS1 / 2], to[i % 2], 0, 0, 0);
    };
    auto output = [&](uint32_t i, half8 v) {
        const bool rest = kPair && i < NO1;
        const half8 x = rest ? pl[kPair ? i % NO1 / VT : 0] : ph[i % NO1 / VT];
        float16v &to = kPair ? fresh[kPair ? i % VT : 0] : o[i % VT];
        to = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, x, to, 0, 0, 0);
    };
    // f16: the sum of P as the product has it, beside that product
    float add[4], inverse_ratio = 1.0f;
    auto clear_add = [&] { add[0] = add[1] = add[2] = add[3] = 0.0f; };
    auto add_p = [&](uint32_t i) {
        if constexpr (!kPair)
#pragma unroll
            for (uint32_t e = i * 16 / NO; e < (i + 1) * 16 / NO; ++e) {
                const half2_t two = {ph[e / 4][e % 4 * 2], ph[e / 4][e % 4 * 2 + 1]};
                add[e % 4] = __builtin_amdgcn_fdot2(two, half2_t{(_Float16)1.0f, (_Float16)1.0f}, add[e % 4], false);
            }
    };
    auto clear_fresh = [&] {
        if constexpr (kPair)
#pragma unroll
            for (uint32_t t = 0; t < VT; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) fresh[t][e] = 0.0f;
    };
    auto add_fresh = [&] {
        if constexpr (kPair)
#pragma unroll
            for (uint32_t t = 0; t < VT; ++t) o[t] += fresh[t];
    };
    auto clear = [](float16v (&to)[2]) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int e = 0; e < 16; ++e) to[s][e] = 0.0f;
    };
    // unit u of a turn's codes: 8 of the thread's, to f16 and into LDS
    auto unit_of_codes = [&](uint32_t u, uint32_t buf) {
        const bool keys = u >= 2 * KPER;
        const uint32_t piece = u / 2 % KPER, second = u % 2;
        const u32x4 w = keys ? kreg[piece] : vreg[piece];
        const half8 x = second ? codes(w.z, w.w) : codes(w.x, w.y);
        _Float16 *const to = keys ? &ks[buf][kto[piece]] : &vs[buf][vto[piece]];
        *reinterpret_cast<half8 *>(to + (keys ? KHALF : VHALF) * second) = x;
    };

    // columns past the padded dim meet zeros of q, and the first turn's P of no
    // tile meets these values: neither may be NaN
    for (uint32_t p = tid; p < kTokens * (P - c.kp) / 8; p += kThreads) {
        const uint32_t per = (P - c.kp) / 8, t = p / per, group = c.kp / 8 + p % per, d = group % 2 * KHALF + group / 2 * 8;
        *reinterpret_cast<half8 *>(&ks[0][t * KROW + d]) = half8{};
        *reinterpret_cast<half8 *>(&ks[1][t * KROW + d]) = half8{};
    }
    for (uint32_t p = tid; p < VTILE / 8; p += kThreads) reinterpret_cast<half8 *>(vs[1])[p] = half8{};
    fetch_meta(0);
    fetch_k(0);
    fetch_v(0);
    if (tiles != 0) {
        if (open_first) {   // it lies in f16
            const half8 *kt = reinterpret_cast<const half8 *>(c.kt + head * kTokens * c.kp);
#pragma unroll
            for (uint32_t u = 0; u < KPER; ++u) {
                const uint32_t p = min(tid + u * kThreads, kpieces - 1);
                put(&ks[0][kto[u]], KHALF, kt[2 * p], kt[2 * p + 1]);
            }
        } else {
            stash_k(0);
        }
    }
    fetch_k(1);
    stash_k(1);
    Meta next_meta = take_meta(0);
    fetch_meta(1);
    fetch_k(2);
    float inverse_unit = 1.0f;
    __syncthreads();
    clear(st);
    steps<NS>([&](uint32_t i) { return key_operand(0, i); }, [&](uint32_t i, half8 k) { score(st, i, k); }, [](uint32_t) {});
    auto turn = [&](uint32_t s, float16v (&now)[2], float16v (&ahead)[2]) {
        const Meta m = next_meta;
        const uint32_t t = block_of(s);
        __syncthreads();
        if ((int)(t * kTokens + kTokens) > least || m.marked != 0) {
            const int last = seen - (int)(t * kTokens);
            const uint32_t mine = marks_of(m.marked, half);
#pragma unroll
            for (uint32_t e = 0; e < 32; ++e) {
                const uint32_t key = e / 8 * 16 + 8 * half + e % 8;
                const float x = mine >> e & 1 ? __builtin_nanf("") : now[e / 16][e % 16];
                now[e / 16][e % 16] = (int)key >= last ? neg_inf : x;
            }
        }
        const f32x2 f2 = block_factor<S, kExact>(m.k_scale, a.scale2, q.shift);
        const float factor = f2.x;
        float part_max[4] = {neg_inf, neg_inf, neg_inf, neg_inf};
        clear_fresh();
        clear_add();
        steps<NO>([&](uint32_t i) { return value_operand((s + 1) & 1, i); }, [&](uint32_t i, half8 v) { output(i, v); },
                  [&](uint32_t i) {
#pragma unroll
                      for (uint32_t u = i * 4 * KPER / NO; u < (i + 1) * 4 * KPER / NO; ++u) unit_of_codes(u, s & 1);
#pragma unroll
                      for (uint32_t e = i * 32 / NO; e < (i + 1) * 32 / NO; ++e)
                          part_max[e % 4] = fmaxf(part_max[e % 4], now[e / 16][e % 16]);
                      add_p(i);
                  });
        add_fresh();
        if constexpr (!kPair) sum += ((add[0] + add[1]) + (add[2] + add[3])) * inverse_ratio;
        const float raw = fmaxf(fmaxf(part_max[0], part_max[1]), fmaxf(part_max[2], part_max[3]));
        next_meta = take_meta(s + 1);
        fetch_meta(s + 2);
        fetch_v(s + 1);
        fetch_k(s + 3);
        const float top = raw * factor;
        if (__builtin_amdgcn_ballot_w64(top > big + kLazy<S>) != 0) {
            const float up = flash::pair_max(fmaxf(top, big));
            const float alpha = up == neg_inf ? 1.0f : __builtin_amdgcn_exp2f(big - up);
            sum *= alpha;
            exact *= alpha;
#pragma unroll
            for (uint32_t v = 0; v < VT; ++v) o[v] *= alpha;
            big = up;
        }
        float ratio = m.v_scale * inverse_unit;
        if (m.v_scale == 0.0f) {
            ratio = 1.0f;
        } else if (ratio > kUnitRange || ratio < 1.0f / kUnitRange) {
#pragma unroll
            for (uint32_t v = 0; v < VT; ++v) o[v] *= unit / m.v_scale;
            unit = m.v_scale;
            inverse_unit = 1.0f / unit;
            ratio = 1.0f;
        }
        // exponents are relative to this; with nothing seen every score is -inf or NaN.
        // The ratio is an addend of the exponent where f16's P is all that comes of it.
        constexpr bool kInExponent = !kPair && !kExact;
        const float base = (big == neg_inf ? 0.0f : big - kHeadroom<S>) -
                           (kInExponent ? __builtin_amdgcn_logf(ratio) : 0.0f);
        const float to_p = ratio * kPairScale<S>;
        float add_exact = 0.0f;
        clear_add();
        clear(ahead);
        // (after the last tile: the scores of an old one, not used)
        steps<NS>([&](uint32_t i) { return key_operand((s + 1) & 1, i); }, [&](uint32_t i, half8 k) { score(ahead, i, k); },
                  [&](uint32_t i) {
#pragma unroll
                      for (uint32_t e = i * 32 / NS; e < (i + 1) * 32 / NS; ++e) {
                          const float raw_score = now[e / 16][e % 16];
                          float x = __builtin_fmaf(raw_score, factor, -base);
                          if constexpr (kPair) {
                              const float off = raw_score * f2.y;
                              x += fabsf(off) < 1.0f ? off : 0.0f;   // (not for -inf)
                          }
                          x = __builtin_amdgcn_exp2f(x);
                          if constexpr (kExact) add_exact += x;
                          if constexpr (kPair) add[e % 4] += x;
                          float y = kInExponent ? x : x * to_p;
                          if constexpr (kPair) asm volatile("" : "+v"(y));   // (one f32 for both its f16s)
                          ph[e / 8][e % 8] = (_Float16)y;
                          if constexpr (kPair) pl[e / 8][e % 8] = (_Float16)(y - (float)ph[e / 8][e % 8]);
                          // (taken here, not moved to where it is used)
                          if (e % 8 == 7) {
                              asm volatile("" : "+v"(ph[e / 8]));
                              if constexpr (kPair) asm volatile("" : "+v"(pl[e / 8]));
                              if constexpr (kExact) asm volatile("" : "+v"(add_exact));
                          }
                      }
                  });
        if constexpr (kPair) sum += (add[0] + add[1]) + (add[2] + add[3]);
        else inverse_ratio = fast_rcp(ratio);
        if constexpr (kExact) exact += add_exact;
    };
    float16v other[2];
    for (uint32_t s = 0; s < tiles; s += 2) {   // (two score tiles in turn: no copies)
        turn(s, st, other);
        if (open_first && s == 0) {   // its values, over what turn 0 wrote in their place
            const half8 *vt = reinterpret_cast<const half8 *>(c.vt + head * kTokens * c.vp);
#pragma unroll
            for (uint32_t u = 0; u < KPER; ++u) {
                const uint32_t p = min(tid + u * kThreads, vpieces - 1);
                put(&vs[0][vto[u]], VHALF, vt[2 * p], vt[2 * p + 1]);
            }
        }
        if (s + 1 < tiles) turn(s + 1, other, st);
    }
    __syncthreads();
    clear_fresh();
    clear_add();
    steps<NO>([&](uint32_t i) { return value_operand((tiles + 1) & 1, i); }, [&](uint32_t i, half8 v) { output(i, v); },
              add_p);
    add_fresh();
    if constexpr (!kPair) sum += ((add[0] + add[1]) + (add[2] + add[3])) * inverse_ratio;
    sum = flash::pair_sum(sum);
    exact = kExact ? flash::pair_sum(exact) : sum;
    big -= kHeadroom<S>;
    if (!live) return;
    const bool direct = a.parts == 1;
#pragma unroll
    for (uint32_t v = 0; v < VT; ++v)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            const f32x4 x = f32x4{o[v][4 * e], o[v][4 * e + 1], o[v][4 * e + 2], o[v][4 * e + 3]} * (unit / kPairScale<S>);
            const uint32_t d = 32 * v + 8 * e + 4 * half;
            if (direct) store_out(a.out + row * c.vdim, c.vdim, d, finish(x, big, sum));
            else store_out(a.part_o + ((size_t)part * a.rows + row) * c.vdim, c.vdim, d, x);
        }
    if (half != 0) return;
    if (!direct) {
        a.part_ml[(size_t)part * a.rows + row] = f32x2{big, sum};
        if (a.part_exact != nullptr) a.part_exact[(size_t)part * a.rows + row] = exact;
    } else if (a.row_ml != nullptr) {
        a.row_ml[row] = weight_terms(big, exact);
    }
}

// Softmax weights of four blocks' tokens, a wave each, summed over the rows that
// see them: the scores again, now with the rows' maxima and sums known. A block's
// keys stay in its wave's registers as A operands; the rows pass through LDS, 32
// at a time, the next ones' loads ahead. Where there are too few blocks for the
// chip, `row_parts` workgroups share four blocks' rows, and
// kv_weights_add_kernel adds their sums in order. Bound by its chain of steps (rows
// from memory to LDS, products, exponentials, a barrier): 2 x 15 heads x 1500 rows, D 64,
// f16 26 us and the addition 5.
template <typename S, uint32_t P>
__global__ __launch_bounds__(kThreads, P <= 64 ? 3 : P <= 128 ? 2 : 1) void kv_weights_kernel(Args<S> a, uint32_t row_parts,
                                                                               float *partial) {
    constexpr bool kPair = sizeof(S) == 4;
    constexpr uint32_t KC = P / 16, QROW = P + 8, kStep = 32;
    constexpr uint32_t G = (P / 8 + 7) / 8;   // groups of 8 dims of a thread: 8 threads stage a row
    __shared__ __attribute__((aligned(16))) _Float16 qs[2][kPieces<S>][kStep * QROW];
    __shared__ f32x4 terms[2][kStep];         // of a row: maximum, 1 / sum (0: adds nothing), shift
    const View &c = a.c;
    const uint32_t tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane(tid / kWave);
    const uint32_t t0 = blockIdx.x / row_parts * kWaves, row_part = blockIdx.x % row_parts;
    const uint32_t h = blockIdx.y, b = blockIdx.z, seq = a.first + b;
    const size_t head = (size_t)seq * c.heads + h;
    const uint32_t length = c.length[seq], count = a.count.n[b];
    if (t0 * kTokens >= length || count == 0) return;
    const uint32_t blocks = (length + kTokens - 1) / kTokens;
    const uint32_t t = min(t0 + wave, blocks - 1);   // (waves past the end repeat the last block)
    const uint32_t in_head = a.group * a.n;
    const bool open = t == length / kTokens;
    const Meta meta = c.meta[head * c.blocks + t];
    half8 k[2][KC];
#pragma unroll
    for (uint32_t s = 0; s < 2; ++s)
#pragma unroll
        for (uint32_t ch = 0; ch < KC; ++ch) {
            const uint32_t d = 16 * ch + 8 * half, at = d < c.kp ? d : 0, key = 32 * s + swap23(col);
            if (open) {
                k[s][ch] = *reinterpret_cast<const half8 *>(c.kt + (head * kTokens + key) * c.kp + at);
            } else {
                const u32x2 w = *reinterpret_cast<const u32x2 *>(c.k + ((head * c.blocks + t) * kTokens + key) * c.kp + at);
                k[s][ch] = codes(w.x, w.y);
            }
        }
    const float sign = a.scale2 > 0.0 ? 1.0f : a.scale2 < 0.0 ? -1.0f : 0.0f;
    const float k_scale = open ? 1.0f : meta.k_scale;
    float acc[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) acc[e] = 0.0f;

    const uint32_t steps = (in_head + kStep - 1) / kStep;
    // the workgroup's steps: every row_parts-th, but those whose rows end before its blocks
    auto skip = [&](uint32_t step) {
        if (!a.causal) return false;
        const uint32_t i = step * kStep % a.n, last = i + kStep - 1 < a.n ? i + kStep - 1 : a.n - 1;
        return (int)length - (int)count + (int)min(last, count - 1) + 1 <= (int)(t0 * kTokens);
    };
    auto from = [&](uint32_t step) {
        while (step < steps && skip(step)) step += row_parts;
        return step;
    };
    // staging: row tid / 8 of the step, groups tid % 8, + 8, ... of its dims
    const uint32_t srow = tid / 8, sub = tid % 8;
    typedef S vec8 __attribute__((ext_vector_type(8)));
    struct Staged {
        vec8 x[G];
        f32x2 ml;
    };
    auto fetch = [&](uint32_t step, Staged &to) {
        vec8 (&x)[G] = to.x;
        f32x2 &ml = to.ml;
        const uint32_t r = min(step, steps - 1) * kStep + srow;
        const size_t row = head * in_head + min(r, in_head - 1);
        const S *src = a.q + row * c.dim;
        ml = a.row_ml[row];
        if (r >= in_head || r % a.n >= count) ml = f32x2{0.0f, 0.0f};
#pragma unroll
        for (uint32_t g = 0; g < G; ++g) {
            const uint32_t d = (sub + 8 * g) * 8;
            if (c.dim % 8 == 0) {
                x[g] = *reinterpret_cast<const vec8 *>(src + (d < c.dim ? d : 0));
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) x[g][e] = src[d + e < c.dim ? d + e : 0];
            }
        }
    };
    auto stash = [&](uint32_t buf, Staged &from) {
        vec8 (&x)[G] = from.x;
        const f32x2 ml = from.ml;
        // a row that adds nothing: zeros, so that its raw products are finite
#pragma unroll
        for (uint32_t g = 0; g < G; ++g) {
            const uint32_t d = (sub + 8 * g) * 8;
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) x[g][e] = ml.y != 0.0f && d + e < c.dim ? x[g][e] * (S)sign : (S)0.0f;
        }
        int shift = 0;
        if constexpr (kPair) {
            float big = 0.0f;
#pragma unroll
            for (uint32_t g = 0; g < G; ++g)
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[g][e]));
#pragma unroll
            for (int d = 1; d < 8; d *= 2) big = fmaxf(big, __shfl_xor(big, d, kWave));
            shift = big > 0.0f ? __builtin_amdgcn_frexp_expf(big) - 14 : 0;
#pragma unroll
            for (uint32_t g = 0; g < G; ++g) {
                half8 piece[3];
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e)
                    pieces_of(__builtin_ldexpf(x[g][e], -shift), piece[0], piece[1], piece[2], e);
                const uint32_t d = (sub + 8 * g) * 8;
                if (d < P)
#pragma unroll
                    for (uint32_t i = 0; i < 3; ++i) *reinterpret_cast<half8 *>(&qs[buf][i][srow * QROW + d]) = piece[i];
            }
        } else {
#pragma unroll
            for (uint32_t g = 0; g < G; ++g) {
                const uint32_t d = (sub + 8 * g) * 8;
                if (d < P) *reinterpret_cast<half8 *>(&qs[buf][0][srow * QROW + d]) = x[g];
            }
        }
        if (sub == 0) terms[buf][srow] = f32x4{ml.x, ml.y, (float)shift, 0.0f};
    };
    // two steps' rows are on their way while a step is computed
    Staged even, odd;
    const uint32_t first = from(row_part);
    uint32_t second = from(first + row_parts);
    fetch(first, even);
    stash(0, even);
    fetch(second, odd);
    __syncthreads();
    // one step, from LDS buffer buf; `next` is staged, the one after it asked for
    auto turn = [&](uint32_t step, uint32_t next, uint32_t buf, Staged &staged, Staged &ahead) {
        const uint32_t after = from(next + row_parts);
        fetch(after, ahead);
        const uint32_t r = step * kStep + col, i = r % a.n;
        const bool live = r < in_head && i < count;
        const int seen = seen_by(i, live, length, count, a.causal);
        if (wave_any(live && seen > (int)(t * kTokens))) {
            const f32x4 term = terms[buf][col];
            const float factor = block_factor<S, true>(k_scale, a.scale2, (int)term.z).x;
            float16v st[2];
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int e = 0; e < 16; ++e) st[s][e] = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < kPieces<S>; ++i)
#pragma unroll
                for (uint32_t ch = 0; ch < KC; ++ch) {
                    const half8 x = *reinterpret_cast<const half8 *>(&qs[buf][i][col * QROW + 16 * ch + 8 * half]);
#pragma unroll
                    for (uint32_t s = 0; s < 2; ++s)
                        st[s] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[s][ch], x, st[s], 0, 0, 0);
                }
            if (wave_any(live && seen < (int)(t * kTokens + kTokens)) || meta.marked != 0) {
                const int last = seen - (int)(t * kTokens);
                const uint32_t mine = marks_of(meta.marked, half);
#pragma unroll
                for (uint32_t e = 0; e < 32; ++e) {
                    const uint32_t key = e / 8 * 16 + 8 * half + e % 8;
                    st[e / 16][e % 16] = (mine >> e & 1) != 0 || (int)key >= last ? -__builtin_inff() : st[e / 16][e % 16];
                }
            }
#pragma unroll
            for (int e = 0; e < 32; ++e)
                acc[e] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(st[e / 16][e % 16], factor, -term.x)), term.y,
                                        acc[e]);
        }
        stash(buf ^ 1, staged);
        __syncthreads();
        return after;
    };
    for (uint32_t step = first; step < steps;) {
        const uint32_t third = turn(step, second, 0, odd, even);
        step = second;
        if (step >= steps) break;
        second = turn(step, third, 1, even, odd);
        step = third;
    }
    // sums over the 32 rows of a half wave: each exchange halves the values, and
    // lane col ends with value col
#pragma unroll
    for (uint32_t n = 16; n >= 1; n /= 2)
#pragma unroll
        for (uint32_t j = 0; j < n; ++j) {
            const bool upper = col & n;
            const float mine = upper ? acc[j + n] : acc[j], other = upper ? acc[j] : acc[j + n];
            acc[j] = mine + __shfl_xor(other, n, kWave);
        }
    const uint32_t token = t * kTokens + col / 8 * 16 + 8 * half + col % 8;
    if (t0 + wave >= blocks || token >= min(length, a.weight_tokens)) return;
    if (row_parts == 1)
        a.weights[head * a.weight_stride + token] += acc[0];
    else
        partial[((size_t)row_part * a.pairs + (size_t)b * c.heads + h) * a.score_stride + token] = acc[0];
}

template <typename S>
__global__ __launch_bounds__(kThreads) void kv_weights_add_kernel(Args<S> a, uint32_t row_parts,
                                                                  const float *partial) {
    const View &c = a.c;
    const uint32_t t = blockIdx.x * kThreads + threadIdx.x, h = blockIdx.y, b = blockIdx.z, seq = a.first + b;
    if (a.count.n[b] == 0 || t >= min(c.length[seq], a.weight_tokens)) return;
    float total = 0.0f;
    for (uint32_t p = 0; p < row_parts; ++p)
        total += partial[((size_t)p * a.pairs + (size_t)b * c.heads + h) * a.score_stride + t];
    a.weights[((size_t)seq * c.heads + h) * a.weight_stride + t] += total;
}

template <typename S, uint32_t P>
hipError_t tiles(const Args<S> &a, uint32_t groups, hipStream_t s) {
    const dim3 grid(groups * a.pairs * a.parts);
    if constexpr (sizeof(S) == 2) {
        if (a.weights != nullptr) {
            kv_tiles_kernel<S, P, true><<<grid, kThreads, 0, s>>>(a);
            return hipGetLastError();
        }
    }
    kv_tiles_kernel<S, P, false><<<grid, kThreads, 0, s>>>(a);
    return hipGetLastError();
}

template <typename S, uint32_t P>
hipError_t weights(const Args<S> &a, uint32_t batch, uint32_t blocks, uint32_t row_parts, float *partial, hipStream_t s) {
    const uint32_t fours = (blocks + kWaves - 1) / kWaves;
    kv_weights_kernel<S, P><<<dim3(fours * row_parts, a.c.heads, batch), kThreads, 0, s>>>(a, row_parts, partial);
    const hipError_t status = hipGetLastError();
    if (status != hipSuccess || row_parts == 1) return status;
    kv_weights_add_kernel<S><<<dim3((blocks * kTokens + kThreads - 1) / kThreads, a.c.heads, batch), kThreads, 0, s>>>(
        a, row_parts, partial);
    return hipGetLastError();
}

}  // namespace

bool tiles_fit(bool f32, uint32_t widest) { return !f32 || widest <= 128; }

template <typename S>
hipError_t launch_tiles(const Args<S> &a, uint32_t widest, uint32_t groups, hipStream_t s) {
    if (widest <= 32) return tiles<S, 32>(a, groups, s);
    if (widest <= 64) return tiles<S, 64>(a, groups, s);
    if (widest <= 96) return tiles<S, 96>(a, groups, s);
    if (widest <= 128) return tiles<S, 128>(a, groups, s);
    if constexpr (sizeof(S) == 2) {
        if (widest <= 192) return tiles<S, 192>(a, groups, s);
        return tiles<S, 256>(a, groups, s);
    }
    return hipErrorInvalidValue;
}

template <typename S>
hipError_t launch_weights(const Args<S> &a, uint32_t widest, uint32_t batch, uint32_t blocks, uint32_t row_parts,
                          float *partial, hipStream_t s) {
    if (widest <= 32) return weights<S, 32>(a, batch, blocks, row_parts, partial, s);
    if (widest <= 64) return weights<S, 64>(a, batch, blocks, row_parts, partial, s);
    if (widest <= 96) return weights<S, 96>(a, batch, blocks, row_parts, partial, s);
    if (widest <= 128) return weights<S, 128>(a, batch, blocks, row_parts, partial, s);
    if (widest <= 192) return weights<S, 192>(a, batch, blocks, row_parts, partial, s);
    return weights<S, 256>(a, batch, blocks, row_parts, partial, s);
}

template hipError_t launch_tiles<float>(const Args<float> &, uint32_t, uint32_t, hipStream_t);
template hipError_t launch_tiles<_Float16>(const Args<_Float16> &, uint32_t, uint32_t, hipStream_t);
template hipError_t launch_weights<float>(const Args<float> &, uint32_t, uint32_t, uint32_t, uint32_t, float *, hipStream_t);
template hipError_t launch_weights<_Float16>(const Args<_Float16> &, uint32_t, uint32_t, uint32_t, uint32_t, float *,
                                             hipStream_t);

}  // namespace kv
}  // namespace icsdk
