// Attention over the 8-bit cache for many query rows (kv_tiles.hpp), and the softmax
// weights of its tokens.
#include "kv_tiles.hpp"

namespace icsdk {
namespace kv {
namespace {

template <typename S, uint32_t P, bool kExact>
__global__ __launch_bounds__(kThreads, tiles_twice(sizeof(S) == 4, P) ? 2 : 1) void kv_tiles_kernel(Args<S> a) {
    __shared__ __attribute__((aligned(16))) typename TilesLds<P>::Keys ks;
    __shared__ __attribute__((aligned(16))) typename TilesLds<P>::Values vs;
    __shared__ typename TilesLds<P>::Most wave_most;
    tiles_of<S, P, kExact>(ks, vs, wave_most, kernel_arguments<Args<S>>(0), blockIdx.x);
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
        const size_t row = head * in_head + (count == a.n ? min(r, in_head - 1) : loaded_row(r, r % a.n, in_head, a.n, count));
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
