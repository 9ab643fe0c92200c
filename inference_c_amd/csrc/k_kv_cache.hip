// Filling, reading, cutting and thinning of the 8-bit key/value cache
// (kv.hpp has its layout). One workgroup does one block of 64 tokens of one
// (sequence, head), keys and values both: a token is marked by either, and the
// block's rows pass through LDS once, where the values are turned from token
// rows into dim rows.
//
// Codes. With a the largest |x| of the block (f16), code = rne(127 x / a). The
// kernels compute q = x * fl(127 / a), whose relative error is below 2^-23, and
// round that. A quotient that is no tie lies at least 2^(k - 20) from one where
// |code| < 2^(k + 1) (127 x and (2 c + 1) a / 2 are whole multiples of a
// common unit, x and a having 11 significant bits), four times q's error, so
// only exact ties need a second look: r = 127 x - c a is exact in f32 (18-bit
// products), a tie is |2 r| = a, and the odd one of its two codes gives way.
#include "kern_common.hpp"
#include "kv.hpp"

namespace icsdk {
namespace kv {
namespace {

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWaves = kThreads / kWave;

__device__ inline bool finite16(uint16_t bits) { return (bits & 0x7c00u) != 0x7c00u; }
__device__ inline uint16_t bits16(_Float16 v) { return __builtin_bit_cast(uint16_t, v); }
__device__ inline _Float16 half_of(uint16_t v) { return __builtin_bit_cast(_Float16, v); }

// Code of x (f16 as f32) in a block of largest |x| a > 0; inverse = 127 / a.
__device__ inline int code_of(float x, float a, float inverse) {
    const float c = rintf(x * inverse);
    const float r = __builtin_fmaf(-c, a, 127.0f * x);
    int code = (int)c;
    if (fabsf(r) * 2.0f == a && (code & 1)) code += r > 0.0f ? 1 : -1;
    return code;
}

// Largest of the workgroup's values (all >= 0), for every thread.
__device__ inline float block_max(float v, float *slots) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) slots[threadIdx.x / kWave] = v;
    __syncthreads();
    float m = slots[0];
#pragma unroll
    for (uint32_t i = 1; i < kWaves; ++i) m = fmaxf(m, slots[i]);
    return m;
}

// ---- append --------------------------------------------------------------------

template <typename S> struct AppendArgs {
    View c;
    const S *key, *value;
    uint32_t n, first;
    Counts start, count;
};

// Rows [lo, hi) of a block from memory into LDS rows of `pitch` halves (the
// columns from dim to its whole 16s as zeros), marking those with an element
// that f16 does not hold.
template <typename S>
__device__ inline void load_rows(const S *src, uint32_t lo, uint32_t hi, uint32_t dim, uint16_t *rows,
                                 uint32_t pitch, uint32_t *marks) {
    const uint32_t padded = (dim + 15) / 16 * 16, tid = threadIdx.x;
    constexpr uint32_t E = Vec16<S>::N;
    if (dim % E == 0) {   // rows of whole, aligned vectors
        const uint32_t per = dim / E;
        for (uint32_t i = tid; i < (hi - lo) * per; i += kThreads) {
            const uint32_t t = lo + i / per, d = i % per * E;
            const Vec16<S> v = load16_stream(src + (size_t)i * E);
            bool good = true;
#pragma unroll
            for (uint32_t e = 0; e < E; e += 2) {
                const uint16_t x = bits16((_Float16)v.v[e]), y = bits16((_Float16)v.v[e + 1]);
                good = good && finite16(x) && finite16(y);
                *reinterpret_cast<uint32_t *>(&rows[t * pitch + d + e]) = x | (uint32_t)y << 16;
            }
            if (!good) atomicOr(&marks[t / 32], 1u << (t % 32));
        }
    } else {
        for (uint32_t i = tid; i < (hi - lo) * dim; i += kThreads) {
            const uint32_t t = lo + i / dim;
            const uint16_t x = bits16((_Float16)src[i]);
            rows[t * pitch + i % dim] = x;
            if (!finite16(x)) atomicOr(&marks[t / 32], 1u << (t % 32));
        }
    }
    for (uint32_t i = tid; i < (hi - lo) * (padded - dim); i += kThreads)
        rows[(lo + i / (padded - dim)) * pitch + dim + i % (padded - dim)] = 0;
}

// Bound by its bytes (rows in, codes out). The 16-byte pieces of a v row are
// written by four neighbouring lanes; v's LDS rows are two halves longer than
// the data, so that those lanes' columns lie in different banks.
template <typename S, uint32_t P>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(AppendArgs<S> a) {
    __shared__ __attribute__((aligned(16))) uint16_t rk[kTokens * P], rv[kTokens * (P + 2)];
    __shared__ uint32_t marks[2];
    __shared__ float slots[kWaves];
    const View &c = a.c;
    const uint32_t tid = threadIdx.x, h = blockIdx.y, b = blockIdx.z, seq = a.first + b;
    const uint32_t start = a.start.n[b], count = a.count.n[b];
    if (count == 0) return;
    const uint32_t end = start + count, first_block = start / kTokens, open_block = end / kTokens;
    if (blockIdx.x > 0 && first_block + blockIdx.x >= open_block) return;
    const size_t head = (size_t)seq * c.heads + h;
    if (blockIdx.x == 0 && h == 0 && tid == 0) c.length[seq] = end;
    const uint32_t kp = c.kp, vp = c.vp, vpitch = vp + 2;
    _Float16 *const kt = c.kt + head * kTokens * kp, *const vt = c.vt + head * kTokens * vp;

    // The open block's rows in f16 are one place for all blocks: the workgroup
    // that takes the first block, which may need the rows held there, writes the
    // last block's rows after it.
    uint32_t j = first_block + blockIdx.x;
    for (;;) {
        const uint32_t from = j == first_block ? start % kTokens : 0;   // rows the block has
        const uint32_t to = j == open_block ? end % kTokens : kTokens;
        const bool closed = to == kTokens;
        if (tid < 2) marks[tid] = 0;
        __syncthreads();
        const size_t row = head * a.n + (size_t)j * kTokens + from - start;
        load_rows(a.key + row * c.dim, from, to, c.dim, rk, kp, marks);
        load_rows(a.value + row * c.vdim, from, to, c.vdim, rv, vpitch, marks);
        if (closed) {
            for (uint32_t i = tid; i < from * kp / 8; i += kThreads)
                reinterpret_cast<u32x4 *>(rk)[i] = reinterpret_cast<const u32x4 *>(kt)[i];
            for (uint32_t i = tid; i < from * vp; i += kThreads)
                rv[i % from * vpitch + i / from] = bits16(vt[i / from * kTokens + i % from]);
        }
        __syncthreads();
        Meta *const meta = c.meta + head * c.blocks + j;
        const uint64_t fresh = marks[0] | (uint64_t)marks[1] << 32;
        if (fresh != 0) {   // marked rows are held as zeros
            for (uint32_t t = from; t < to; ++t) {
                if (!(fresh >> t & 1)) continue;
                for (uint32_t d = tid; d < kp; d += kThreads) rk[t * kp + d] = 0;
                for (uint32_t d = tid; d < vp; d += kThreads) rv[t * vpitch + d] = 0;
            }
            __syncthreads();
        }
        float k_scale = 1.0f, v_scale = 1.0f;
        if (closed) {
            float kmax = 0.0f, vmax = 0.0f;
            for (uint32_t i = tid; i < kTokens * kp / 8; i += kThreads) {
                const half8 x = reinterpret_cast<const half8 *>(rk)[i];
#pragma unroll
                for (int e = 0; e < 8; ++e) kmax = fmaxf(kmax, fabsf((float)x[e]));
            }
            for (uint32_t i = tid; i < kTokens * vp / 2; i += kThreads) {
                const uint32_t t = i / (vp / 2), d = i % (vp / 2) * 2;
                const uint32_t x = *reinterpret_cast<const uint32_t *>(&rv[t * vpitch + d]);
                vmax = fmaxf(vmax, fmaxf(fabsf((float)half_of((uint16_t)x)), fabsf((float)half_of((uint16_t)(x >> 16)))));
            }
            kmax = block_max(kmax, slots);
            vmax = block_max(vmax, slots);
            k_scale = kmax / 127.0f;
            v_scale = vmax / 127.0f;
            // (an all-zero block: inverse 0 makes every code 0)
            const float kinv = kmax > 0.0f ? 127.0f / kmax : 0.0f, vinv = vmax > 0.0f ? 127.0f / vmax : 0.0f;
            const size_t block = head * c.blocks + j;
            u32x4 *const ko = reinterpret_cast<u32x4 *>(c.k + block * kTokens * kp);
            u32x4 *const vo = reinterpret_cast<u32x4 *>(c.v + block * kTokens * vp);
            for (uint32_t i = tid; i < kTokens * kp / 16; i += kThreads) {
                u32x4 out;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t word = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        word |= (uint32_t)(code_of((float)half_of(rk[i * 16 + w * 4 + e]), kmax, kinv) + 128) << (8 * e);
                    out[w] = word;
                }
                ko[i] = out;
            }
            for (uint32_t i = tid; i < vp * 4; i += kThreads) {
                const uint32_t d = i / 4, t0 = i % 4 * 16;
                u32x4 out;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t word = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        word |= (uint32_t)(code_of((float)half_of(rv[(t0 + w * 4 + e) * vpitch + d]), vmax, vinv) + 128)
                                << (8 * e);
                    out[w] = word;
                }
                vo[i] = out;
            }
        } else {
            for (uint32_t i = tid; i < (to - from) * kp; i += kThreads) kt[from * kp + i] = half_of(rk[from * kp + i]);
            for (uint32_t i = tid; i < (to - from) * vp; i += kThreads) {
                const uint32_t t = from + i % (to - from), d = i / (to - from);
                vt[d * kTokens + t] = half_of(rv[t * vpitch + d]);
            }
        }
        if (tid == 0) {
            const uint64_t held = from == 0 ? 0 : meta->marked & ((uint64_t{1} << from) - 1);
            *meta = Meta{k_scale, v_scale, fresh | held};
        }
        if (blockIdx.x != 0 || j == open_block || end % kTokens == 0) return;
        j = open_block;
        __syncthreads();
    }
}

// ---- read ------------------------------------------------------------------------

template <typename S> struct ReadArgs {
    View c;
    S *key, *value;
    uint32_t rows;
};

// Values of one block, written as rows. Keys go straight from 16-byte pieces to
// rows, values through LDS. Bound by its bytes.
template <typename S, uint32_t P>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(ReadArgs<S> a) {
    __shared__ __attribute__((aligned(16))) _Float16 rows[kTokens * (P + 2)];
    const View &c = a.c;
    const uint32_t tid = threadIdx.x, j = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const uint32_t length = min(c.length[b], a.rows);
    const uint32_t t0 = j * kTokens;
    if (t0 >= length) return;
    const uint32_t live = min(length - t0, kTokens);
    const size_t head = (size_t)b * c.heads + h, block = head * c.blocks + j;
    const Meta meta = c.meta[block];
    const bool open = c.length[b] / kTokens == j;
    const float nan = __builtin_nanf("");
    auto write = [&](S *out, uint32_t dim, uint32_t pitch, float scale) {
        for (uint32_t i = tid; i < live * dim; i += kThreads) {
            const uint32_t t = i / dim, d = i % dim;
            const float x = (float)rows[t * pitch + d];
            out[i] = meta.marked >> t & 1 ? (S)nan : (S)(x * scale);
        }
    };
    if (a.key != nullptr) {
        const uint8_t *src = c.k + block * kTokens * c.kp;
        const _Float16 *half = c.kt + head * kTokens * c.kp;
        for (uint32_t i = tid; i < live * c.kp; i += kThreads)
            rows[i / c.kp * (c.kp + 2) + i % c.kp] = open ? half[i] : (_Float16)(int)(src[i] - 128);
        __syncthreads();
        write(a.key + (head * a.rows + t0) * c.dim, c.dim, c.kp + 2, open ? 1.0f : meta.k_scale);
        __syncthreads();
    }
    if (a.value != nullptr) {
        const uint8_t *src = c.v + block * kTokens * c.vp;
        const _Float16 *half = c.vt + head * kTokens * c.vp;
        for (uint32_t i = tid; i < kTokens * c.vp; i += kThreads)
            rows[i % kTokens * (c.vp + 2) + i / kTokens] = open ? half[i] : (_Float16)(int)(src[i] - 128);
        __syncthreads();
        write(a.value + (head * a.rows + t0) * c.vdim, c.vdim, c.vp + 2, open ? 1.0f : meta.v_scale);
    }
}

// ---- truncate --------------------------------------------------------------------

struct TruncateArgs {
    View c;
    uint32_t first;
    Counts from, to;
};

__global__ __launch_bounds__(kThreads) void kv_truncate_kernel(TruncateArgs a) {
    const View &c = a.c;
    const uint32_t h = blockIdx.x, b = blockIdx.y, seq = a.first + b;
    const uint32_t from = a.from.n[b], to = a.to.n[b], j = to / kTokens;
    if (h == 0 && threadIdx.x == 0) c.length[seq] = to;
    if (from / kTokens == j || to % kTokens == 0) return;
    // a full block is cut: what it held goes on in f16 (marked tokens: zeros)
    const size_t head = (size_t)seq * c.heads + h, block = head * c.blocks + j;
    const Meta meta = c.meta[block];
    for (uint32_t i = threadIdx.x; i < kTokens * c.kp; i += kThreads)
        c.kt[head * kTokens * c.kp + i] = (_Float16)((float)((int)c.k[block * kTokens * c.kp + i] - 128) * meta.k_scale);
    for (uint32_t i = threadIdx.x; i < kTokens * c.vp; i += kThreads)
        c.vt[head * kTokens * c.vp + i] = (_Float16)((float)((int)c.v[block * kTokens * c.vp + i] - 128) * meta.v_scale);
    __syncthreads();
    if (threadIdx.x == 0) c.meta[block] = Meta{1.0f, 1.0f, meta.marked};
}

// ---- evict -----------------------------------------------------------------------

constexpr uint32_t kSelectThreads = 1024;
constexpr uint32_t kSelectWaves = kSelectThreads / kWave;

// Unsigned image of a weight in its order: NaN lowest, the two zeros equal.
__device__ inline uint32_t order_of(float w) {
    if (w != w) return 0;
    const uint32_t u = __builtin_bit_cast(uint32_t, w == 0.0f ? 0.0f : w);
    return u >> 31 ? ~u : u | 0x80000000u;
}

// Which tokens a head keeps: one workgroup per (sequence, head). The n-th
// largest weight is found by its bytes, from the top (a histogram of the next
// byte among the weights that share the bytes so far); then every wave counts
// the tokens above and at it in its part of the sequence and, from the counts
// of the parts before, writes the kept ones in order, the earliest of those
// that equal it.
__global__ __launch_bounds__(kSelectThreads) void kv_select_kernel(View from, EvictArgs a) {
    __shared__ uint32_t bins[256], chosen[2];
    __shared__ uint32_t above[kSelectWaves], equal[kSelectWaves];
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const uint32_t h = blockIdx.x, b = blockIdx.y;
    const size_t head = (size_t)b * from.heads + h;
    const uint32_t length = from.length[b];
    const float *w = a.weights ? a.weights + head * a.tokens : nullptr;
    uint32_t *index = a.index + head * a.keep_most;
    auto put = [&](uint32_t slot, uint32_t t) {
        index[slot] = t;
        if (a.kept) a.kept[head * a.slots + slot] = t;
        if (a.target_weights) a.target_weights[head * a.slots + slot] = w[t];
    };
    if (length <= a.keep) {
        for (uint32_t t = tid; t < length; t += kSelectThreads) put(t, t);
        return;
    }
    // first + recent <= keep < length: the two do not meet
    const uint32_t lo = a.first, hi = length - a.recent, want = a.keep - a.first - a.recent;
    if (w == nullptr) {
        for (uint32_t i = tid; i < a.keep; i += kSelectThreads) put(i, i < lo ? i : length - a.keep + i);
        return;
    }
    uint32_t prefix = 0, left = want;   // the bytes found; how many are wanted among those that share them
    for (int shift = 24; shift >= 0 && want != 0; shift -= 8) {
        if (tid < 256) bins[tid] = 0;
        __syncthreads();
        for (uint32_t t = lo + tid; t < hi; t += kSelectThreads) {
            const uint32_t u = order_of(w[t]);
            if (shift == 24 || u >> (shift + 8) == prefix) atomicAdd(&bins[u >> shift & 255u], 1u);
        }
        __syncthreads();
        if (wave == 0) {
            // lane l has bins 4 l .. 4 l + 3; how many lie in higher lanes
            uint32_t n[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += n[i] = bins[4 * lane + i];
            uint32_t higher = sum;
#pragma unroll
            for (int d = 1; d < kWave; d *= 2) {
                const uint32_t other = __shfl_down(higher, d, kWave);
                if (lane + d < kWave) higher += other;
            }
            higher -= sum;
#pragma unroll
            for (int i = 3; i >= 0; --i) {
                if (higher < left && higher + n[i] >= left) {
                    chosen[0] = 4 * lane + i;
                    chosen[1] = left - higher;
                }
                higher += n[i];
            }
        }
        __syncthreads();
        prefix = prefix << 8 | chosen[0];
        left = chosen[1];
        __syncthreads();
    }
    const uint32_t per = (length + kSelectThreads - 1) / kSelectThreads * kWave;   // a wave's tokens
    const uint32_t begin = min(wave * per, length), end = min(begin + per, length);
    auto ranks = [&](uint32_t t, bool &over, bool &same) {
        over = same = false;
        if (t >= end) return;
        if (t < lo || t >= hi) {
            over = true;
        } else if (want != 0) {
            const uint32_t u = order_of(w[t]);
            over = u > prefix;
            same = u == prefix;
        }
    };
    uint32_t n_above = 0, n_equal = 0;
    for (uint32_t t = begin; t < end; t += kWave) {
        bool over, same;
        ranks(t + lane, over, same);
        n_above += __popcll(__builtin_amdgcn_ballot_w64(over));
        n_equal += __popcll(__builtin_amdgcn_ballot_w64(same));
    }
    if (lane == 0) {
        above[wave] = n_above;
        equal[wave] = n_equal;
    }
    __syncthreads();
    n_above = n_equal = 0;
    for (uint32_t i = 0; i < wave; ++i) {
        n_above += above[i];
        n_equal += equal[i];
    }
    const uint64_t below = (uint64_t{1} << lane) - 1;
    for (uint32_t t = begin; t < end; t += kWave) {
        bool over, same;
        ranks(t + lane, over, same);
        const uint64_t overs = __builtin_amdgcn_ballot_w64(over), sames = __builtin_amdgcn_ballot_w64(same);
        const uint32_t e = n_equal + __popcll(sames & below);
        if (over || (same && e < left)) put(n_above + __popcll(overs & below) + min(e, left), t + lane);
        n_above += __popcll(overs);
        n_equal += __popcll(sames);
    }
}

struct MoveArgs {
    View from, to;
    const uint32_t *index;
    uint32_t keep, keep_most;
};

// One block of the target from the tokens kept. The values code * scale are
// held anew: their largest, a, is taken in f64 (exact products), and a code is
// rne(127 value / a). It is computed as code * fl(127 scale / a) in f32, off by
// at most 2^-16 (|result| <= 127.5, three roundings of 2^-24), and only within
// 2^-12 of a tie decided by the f64 quotient. A block whose tokens
// all come from one block keeps its codes and its scale: its largest code is
// 127, so a / 127 is that scale.
template <uint32_t P>
__global__ __launch_bounds__(kThreads) void kv_move_kernel(MoveArgs a) {
    __shared__ __attribute__((aligned(16))) uint16_t rows[kTokens * (P + 2)];
    __shared__ uint32_t token[kTokens];
    __shared__ float scale_of[2][kTokens];
    __shared__ double largest;
    __shared__ uint32_t opened[2], marks[2];
    const View &f = a.from, &c = a.to;
    const uint32_t tid = threadIdx.x, j = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const size_t head = (size_t)b * c.heads + h;
    const uint32_t length = f.length[b], kept = min(length, a.keep);
    if (j == 0 && h == 0 && tid == 0) c.length[b] = kept;
    if (j * kTokens >= kept) return;
    const uint32_t live = min(kept - j * kTokens, kTokens);
    const bool closed = live == kTokens;
    if (tid < 2) opened[tid] = marks[tid] = 0;
    __syncthreads();
    if (tid < kTokens) {
        // rows past the last token repeat it; they are not kept
        const uint32_t t = a.index[head * a.keep_most + j * kTokens + min(tid, live - 1)];
        const bool open = t / kTokens == length / kTokens;
        const Meta meta = f.meta[head * f.blocks + t / kTokens];
        token[tid] = t;
        scale_of[0][tid] = open ? 1.0f : meta.k_scale;
        scale_of[1][tid] = open ? 1.0f : meta.v_scale;
        if (open) atomicOr(&opened[tid / 32], 1u << (tid % 32));
        if ((meta.marked >> (t % kTokens) & 1) && tid < live) atomicOr(&marks[tid / 32], 1u << (tid % 32));
    }
    __syncthreads();
    const uint64_t open_bits = opened[0] | (uint64_t)opened[1] << 32;
    float scales[2];
    for (int which = 0; which < 2; ++which) {
        const uint32_t width = which ? c.vp : c.kp, pitch = width + 2;
        const float *const scale = scale_of[which];
        // rows[token][dim]: a code, or the f16 of the open block
        if (which == 0) {
            for (uint32_t i = tid; i < kTokens * width / 4; i += kThreads) {
                const uint32_t r = i / (width / 4), d = i % (width / 4) * 4, t = token[r];
                if (open_bits >> r & 1) {
                    const _Float16 *src = f.kt + (head * kTokens + t % kTokens) * width + d;
#pragma unroll
                    for (int e = 0; e < 4; ++e) rows[r * pitch + d + e] = bits16(src[e]);
                } else {
                    const uint32_t word = *reinterpret_cast<const uint32_t *>(f.k + ((head * f.blocks) * kTokens + t) * width + d);
#pragma unroll
                    for (int e = 0; e < 4; ++e) rows[r * pitch + d + e] = (uint16_t)((word >> (8 * e) & 255u) - 128u);
                }
            }
        } else {
            for (uint32_t i = tid; i < kTokens * width; i += kThreads) {
                const uint32_t r = i % kTokens, d = i / kTokens, t = token[r];
                rows[r * pitch + d] =
                    open_bits >> r & 1
                        ? bits16(f.vt[(head * width + d) * kTokens + t % kTokens])
                        : (uint16_t)((uint32_t)f.v[((head * f.blocks + t / kTokens) * width + d) * kTokens + t % kTokens] - 128u);
            }
        }
        __syncthreads();
        auto value = [&](uint32_t r, uint32_t d) -> double {
            const uint16_t x = rows[r * pitch + d];
            return open_bits >> r & 1 ? (double)(float)half_of(x) : (double)(int16_t)x * (double)scale[r];
        };
        if (closed) {
            // the largest |value|: four threads per token, then the tokens' in one wave
            {
                const uint32_t r = tid / 4;
                const bool open = open_bits >> r & 1;
                float m = 0.0f;
                for (uint32_t d = tid % 4; d < width; d += 4) {
                    const uint16_t x = rows[r * pitch + d];
                    m = fmaxf(m, fabsf(open ? (float)half_of(x) : (float)(int16_t)x));
                }
                m = fmaxf(m, __shfl_xor(m, 1, kWave));
                m = fmaxf(m, __shfl_xor(m, 2, kWave));
                double big = (double)m * (double)scale[r];
                for (int d = 4; d < kWave; d *= 2) big = fmax(big, __shfl_xor(big, d, kWave));
                __shared__ double wave_big[kWaves];
                if ((tid & (kWave - 1)) == 0) wave_big[tid / kWave] = big;
                __syncthreads();
                if (tid == 0) {
                    for (uint32_t i = 1; i < kWaves; ++i) big = fmax(big, wave_big[i]);
                    largest = big;
                }
                __syncthreads();
            }
            const double big = largest;
            scales[which] = (float)(big / 127.0);
            auto code = [&](uint32_t r, uint32_t d) -> uint32_t {
                if (big == 0.0) return 128u;
                const uint16_t x = rows[r * pitch + d];
                const float ratio = (float)(127.0 * (double)scale[r] / big);
                const float q = (open_bits >> r & 1 ? (float)half_of(x) : (float)(int16_t)x) * ratio;
                float n = rintf(q);
                if (fabsf(fabsf(q - n) - 0.5f) < 0x1p-12f) n = (float)rint(127.0 * value(r, d) / big);
                return (uint32_t)((int)n + 128);
            };
            const size_t block = (head * c.blocks + j) * kTokens * width;
            if (which == 0) {
                for (uint32_t i = tid; i < kTokens * width / 4; i += kThreads) {
                    const uint32_t r = i / (width / 4), d = i % (width / 4) * 4;
                    uint32_t word = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) word |= code(r, d + e) << (8 * e);
                    reinterpret_cast<uint32_t *>(c.k + block)[i] = word;
                }
            } else {
                for (uint32_t i = tid; i < kTokens * width / 4; i += kThreads) {
                    const uint32_t d = i / (kTokens / 4), r = i % (kTokens / 4) * 4;
                    uint32_t word = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) word |= code(r + e, d) << (8 * e);
                    reinterpret_cast<uint32_t *>(c.v + block)[i] = word;
                }
            }
        } else {
            scales[which] = 1.0f;
            for (uint32_t i = tid; i < live * width; i += kThreads) {
                if (which == 0) {
                    const uint32_t r = i / width, d = i % width;
                    c.kt[(head * kTokens + r) * width + d] = (_Float16)(float)value(r, d);
                } else {
                    const uint32_t r = i % live, d = i / live;
                    c.vt[(head * width + d) * kTokens + r] = (_Float16)(float)value(r, d);
                }
            }
        }
        __syncthreads();
    }
    if (tid == 0) c.meta[head * c.blocks + j] = Meta{scales[0], scales[1], marks[0] | (uint64_t)marks[1] << 32};
}

uint32_t class_of(const View &c) {
    const uint32_t widest = c.kp > c.vp ? c.kp : c.vp;
    return widest <= 64 ? 64 : widest <= 128 ? 128 : 256;
}

template <typename S>
void launch_append(const AppendArgs<S> &a, dim3 grid, hipStream_t s) {
    switch (class_of(a.c)) {
        case 64: kv_append_kernel<S, 64><<<grid, kThreads, 0, s>>>(a); break;
        case 128: kv_append_kernel<S, 128><<<grid, kThreads, 0, s>>>(a); break;
        default: kv_append_kernel<S, 256><<<grid, kThreads, 0, s>>>(a); break;
    }
}

template <typename S>
void launch_read(const ReadArgs<S> &a, dim3 grid, hipStream_t s) {
    switch (class_of(a.c)) {
        case 64: kv_read_kernel<S, 64><<<grid, kThreads, 0, s>>>(a); break;
        case 128: kv_read_kernel<S, 128><<<grid, kThreads, 0, s>>>(a); break;
        default: kv_read_kernel<S, 256><<<grid, kThreads, 0, s>>>(a); break;
    }
}

}  // namespace

hipError_t append(bool f32, const View &c, uint32_t first, uint32_t batch, const void *key, const void *value,
                  uint32_t n, const Counts &start, const Counts &count, hipStream_t s) {
    uint32_t most = 0;   // blocks that the longest sequence's tokens close, at least one
    for (uint32_t b = 0; b < batch; ++b) {
        const uint32_t blocks = (start.n[b] + count.n[b]) / kTokens - start.n[b] / kTokens;
        if (count.n[b] != 0) most = blocks > most ? blocks : most == 0 ? 1 : most;
    }
    if (most == 0) return hipSuccess;
    const dim3 grid(most, c.heads, batch);
    if (f32)
        launch_append(AppendArgs<float>{c, static_cast<const float *>(key), static_cast<const float *>(value), n, first,
                                        start, count}, grid, s);
    else
        launch_append(AppendArgs<_Float16>{c, static_cast<const _Float16 *>(key), static_cast<const _Float16 *>(value),
                                           n, first, start, count}, grid, s);
    return hipGetLastError();
}

hipError_t truncate(const View &c, uint32_t first, uint32_t batch, const Counts &from, const Counts &to,
                    hipStream_t s) {
    kv_truncate_kernel<<<dim3(c.heads, batch), kThreads, 0, s>>>(TruncateArgs{c, first, from, to});
    return hipGetLastError();
}

hipError_t read(bool f32, const View &c, uint32_t batch, void *key, void *value, uint32_t rows, uint32_t longest,
                hipStream_t s) {
    const uint32_t most = longest < rows ? longest : rows, blocks = (most + kTokens - 1) / kTokens;
    if (blocks == 0) return hipSuccess;
    const dim3 grid(blocks, c.heads, batch);
    if (f32)
        launch_read(ReadArgs<float>{c, static_cast<float *>(key), static_cast<float *>(value), rows}, grid, s);
    else
        launch_read(ReadArgs<_Float16>{c, static_cast<_Float16 *>(key), static_cast<_Float16 *>(value), rows}, grid, s);
    return hipGetLastError();
}

hipError_t evict(const View &from, const View &to, uint32_t batch, const EvictArgs &a, hipStream_t s) {
    kv_select_kernel<<<dim3(from.heads, batch), kSelectThreads, 0, s>>>(from, a);
    const hipError_t status = hipGetLastError();
    if (status != hipSuccess) return status;
    const MoveArgs m{from, to, a.index, a.keep, a.keep_most};
    const uint32_t blocks = (a.keep_most + kTokens - 1) / kTokens;
    const dim3 grid(blocks == 0 ? 1 : blocks, from.heads, batch);   // (one block sets the lengths)
    switch (class_of(from)) {
        case 64: kv_move_kernel<64><<<grid, kThreads, 0, s>>>(m); break;
        case 128: kv_move_kernel<128><<<grid, kThreads, 0, s>>>(m); break;
        default: kv_move_kernel<256><<<grid, kThreads, 0, s>>>(m); break;
    }
    return hipGetLastError();
}

}  // namespace kv
}  // namespace icsdk
