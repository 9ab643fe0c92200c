// Filling, reading, cutting and thinning of the 8-bit key/value cache
// (kv.hpp has its layout). One workgroup does one block of 64 tokens of one
// (sequence, head), keys and values both: a token is marked by either, and the
// block's rows pass through LDS once, where the values are turned from token
// rows into dim rows.
//
// Codes. With a the largest |x| of the block (f16), code = rne(127 x / a). The
// kernels compute the quotient as a division does: q = 127 x * fl(1 / a), its exact
// remainder by one fma, and q + remainder * fl(1 / a), which is the correctly
// rounded quotient; then its rounding to a whole number by adding 1.5 * 2^23. Ties
// (x = a / 2 is one) come out exactly, being representable, and a quotient that is
// none lies at least 2^(k - 20) from one where |code| < 2^(k + 1) (127 x and
// (2 c + 1) a / 2 are whole multiples of a common unit, x and a having 11
// significant bits), eight times the f32 step there.
#include "kern_common.hpp"
#include "kv.hpp"

namespace icsdk {
namespace kv {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWaves = kThreads / kWave;

__device__ inline bool finite16(uint16_t bits) { return (bits & 0x7c00u) != 0x7c00u; }
__device__ inline uint16_t bits16(_Float16 v) { return __builtin_bit_cast(uint16_t, v); }
__device__ inline _Float16 half_of(uint16_t v) { return __builtin_bit_cast(_Float16, v); }

// code * scale as f32, the value that a code stands for: f16 outputs round it a
// second time. (Left to itself the compiler may round the exact product to f16
// in one instruction, in some places and not in others.)
__device__ inline float value_of(float code, float scale) {
    float v = code * scale;
    asm("" : "+v"(v));
    return v;
}

// What makes codes of a block's elements; an all-zero block's are all 0.
struct Coder {
    float a, inverse;
    __device__ explicit Coder(float largest) : a(largest), inverse(largest > 0.0f ? 1.0f / largest : 0.0f) {}
    // code + 128 in the low byte
    __device__ inline uint32_t byte(float x) const {
        const float x127 = 127.0f * x, q = x127 * inverse;
        const float quotient = __builtin_fmaf(__builtin_fmaf(-q, a, x127), inverse, q);
        return __builtin_bit_cast(uint32_t, quotient + (12582912.0f + 128.0f));
    }
    __device__ inline uint32_t four(float x0, float x1, float x2, float x3) const {
        const uint32_t lo = __builtin_amdgcn_perm(byte(x1), byte(x0), 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(byte(x3), byte(x2), 0x04000c0cu);
        return lo | hi;
    }
};

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
    FastDiv k_groups, v_groups;   // groups of 8 elements per row
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

// For rows that are not whole groups of 8 (kv_append_groups_kernel has the others).
// Bound by its passes over LDS, element by element: 8 heads x 16400 tokens of 100 +
// 100 from f16 70 us. The 16-byte pieces of a v row are written by four neighbouring lanes; v's LDS rows are two halves longer than
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
            const Coder kcoder(kmax), vcoder(vmax);
            const size_t block = head * c.blocks + j;
            u32x4 *const ko = reinterpret_cast<u32x4 *>(c.k + block * kTokens * kp);
            u32x4 *const vo = reinterpret_cast<u32x4 *>(c.v + block * kTokens * vp);
            for (uint32_t i = tid; i < kTokens * kp / 16; i += kThreads) {
                u32x4 out;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint16_t *x = &rk[i * 16 + w * 4];
                    out[w] = kcoder.four((float)half_of(x[0]), (float)half_of(x[1]), (float)half_of(x[2]), (float)half_of(x[3]));
                }
                ko[i] = out;
            }
            for (uint32_t i = tid; i < vp * 4; i += kThreads) {
                const uint32_t d = i / 4, t0 = i % 4 * 16;
                u32x4 out;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint16_t *x = &rv[(t0 + w * 4) * vpitch + d];
                    out[w] = vcoder.four((float)half_of(x[0]), (float)half_of(x[vpitch]), (float)half_of(x[2 * vpitch]),
                                         (float)half_of(x[3 * vpitch]));
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

// As kv_append_kernel, for rows of whole groups of 8 elements: a block stays in
// registers. Four waves have 8-element groups of the key rows, whose codes go
// out as they lie, four have of the value rows the same group of four
// neighbouring tokens, whose codes they turn into four tokens' bytes per dim;
// those pass through LDS to become whole 64-byte rows.
// Bound by its bytes: 8 heads x 16400 tokens of 128 + 128 from f16 (101 MB) 25 us,
// 4.0 TB/s. 16 waves a CU: registers for 24 spill, and the call that appends and reads
// back takes 57 us where it takes 50.
template <typename S> __device__ inline half8 load8(const S *p) {
    if constexpr (sizeof(S) == 2) {
        return __builtin_bit_cast(half8, __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p)));
    } else {
        const Vec16<float> a = load16_stream(p), b = load16_stream(p + 4);
        half8 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            r[e] = (_Float16)a.v[e];
            r[4 + e] = (_Float16)b.v[e];
        }
        return r;
    }
}
// Bits of the largest |element|; 0x7c00 and more: one is not finite.
__device__ inline uint32_t largest8(half8 v) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    const u32x4 w = __builtin_bit_cast(u32x4, v);
    u16x2 m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu);
    const u16x2 x = __builtin_elementwise_max(__builtin_elementwise_max(m[0], m[1]), __builtin_elementwise_max(m[2], m[3]));
    return x.x > x.y ? x.x : x.y;
}
__device__ inline uint32_t pack4(half8 v, int first, const Coder &coder) {
    return coder.four((float)v[first], (float)v[first + 1], (float)v[first + 2], (float)v[first + 3]);
}
// Rows w[0..3] of four bytes each become columns.
__device__ inline void transpose4(uint32_t (&w)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

template <typename S, uint32_t P>
__global__ __launch_bounds__(2 * kThreads, P <= 128 ? 4 : 2) void kv_append_groups_kernel(AppendArgs<S> a) {
    constexpr uint32_t N = P <= 128 ? 4 : 8;   // groups of a thread: 64 P / 8 / 256, whole fours
    constexpr uint32_t kPitch = kTokens + 4;
    __shared__ __attribute__((aligned(16))) uint8_t turned[P * kPitch];
    __shared__ uint32_t marks[2];
    __shared__ float slots[2 * kWaves];
    const View &c = a.c;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const bool values = wave >= kWaves;   // what the wave does
    const uint32_t tid = threadIdx.x % kThreads, h = blockIdx.y, b = blockIdx.z, seq = a.first + b;
    const uint32_t start = a.start.n[b], count = a.count.n[b];
    if (count == 0) return;
    const uint32_t end = start + count, first_block = start / kTokens, open_block = end / kTokens;
    if (blockIdx.x > 0 && first_block + blockIdx.x >= open_block) return;
    const size_t head = (size_t)seq * c.heads + h;
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) c.length[seq] = end;
    const uint32_t kp = c.kp, vp = c.vp;
    _Float16 *const kt = c.kt + head * kTokens * kp, *const vt = c.vt + head * kTokens * vp;
    // the thread's groups: token and dim of each. Keys: groups tid, tid + 256, ...
    // of the block's rows; values: of rows 4 q .. 4 q + 3 the same group.
    const FastDiv &per = values ? a.v_groups : a.k_groups;
    uint32_t token[N], dim[N];
#pragma unroll
    for (uint32_t u = 0; u < N; ++u) {
        const uint32_t i = values ? tid + u / 4 * kThreads : tid + u * kThreads, row = fast_div(i, per);
        token[u] = values ? 4 * row + u % 4 : row;
        dim[u] = (i - row * per.divisor) * 8;
    }
    const S *const memory = values ? a.value : a.key;
    const uint32_t width = values ? c.vdim : c.dim;

    uint32_t j = first_block + blockIdx.x;
    for (;;) {   // (the open block's f16 rows: as in kv_append_kernel)
        const uint32_t from = j == first_block ? start % kTokens : 0;
        const uint32_t to = j == open_block ? end % kTokens : kTokens;
        const bool closed = to == kTokens;
        if (threadIdx.x < 2) marks[threadIdx.x] = 0;
        // row t of the block is row t of the memory from here; rows that are not
        // new read one that is, so that no load waits for a test
        const S *const rows = memory + ((ptrdiff_t)(head * a.n) + (ptrdiff_t)j * kTokens - start) * (ptrdiff_t)width;
        half8 x[N];
        uint32_t largest[N];
#pragma unroll
        for (uint32_t u = 0; u < N; ++u)
            if (values || u < P / 32) x[u] = load8(rows + (size_t)min(max(token[u], from), to - 1) * width + dim[u]);
        __syncthreads();
#pragma unroll
        for (uint32_t u = 0; u < N; ++u) {
            const uint32_t t = token[u];
            if (t < from || t >= to) x[u] = half8{};   // (and those past the block)
            largest[u] = largest8(x[u]);
            if (largest[u] >= 0x7c00u) atomicOr(&marks[t / 32], 1u << (t % 32));
        }
        if (closed && from != 0) {   // the rows the open block had
#pragma unroll
            for (uint32_t u = 0; u < N; ++u) {
                if (token[u] >= from) continue;
                if (!values) {
                    x[u] = *reinterpret_cast<const half8 *>(kt + token[u] * kp + dim[u]);
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) x[u][e] = vt[(dim[u] + e) * kTokens + token[u]];
                }
                largest[u] = largest8(x[u]);
            }
        }
        __syncthreads();
        Meta *const meta = c.meta + head * c.blocks + j;
        const uint64_t fresh = marks[0] | (uint64_t)marks[1] << 32;
        if (fresh != 0) {   // marked rows are held as zeros
#pragma unroll
            for (uint32_t u = 0; u < N; ++u)
                if (fresh >> (token[u] & 63) & 1) {
                    x[u] = half8{};
                    largest[u] = 0;
                }
        }
        float scale = 1.0f;
        if (closed) {
            uint32_t most = 0;
#pragma unroll
            for (uint32_t u = 0; u < N; ++u) most = max(most, largest[u]);
            float big = wave_max((float)half_of((uint16_t)most));
            if ((threadIdx.x & (kWave - 1)) == 0) slots[wave] = big;
            __syncthreads();
            big = slots[values * kWaves];
#pragma unroll
            for (uint32_t i = 1; i < kWaves; ++i) big = fmaxf(big, slots[values * kWaves + i]);
            scale = big / 127.0f;
            const Coder coder(big);
            if (!values) {
                uint8_t *const out = c.k + (head * c.blocks + j) * kTokens * kp;
#pragma unroll
                for (uint32_t u = 0; u < N; ++u)
                    if (token[u] < kTokens)
                        *reinterpret_cast<uint2 *>(out + token[u] * kp + dim[u]) =
                            uint2{pack4(x[u], 0, coder), pack4(x[u], 4, coder)};
            } else {
#pragma unroll
                for (uint32_t u = 0; u < N; u += 4) {
                    if (token[u] >= kTokens) continue;
#pragma unroll
                    for (uint32_t half = 0; half < 2; ++half) {
                        uint32_t w[4];
#pragma unroll
                        for (uint32_t r = 0; r < 4; ++r) w[r] = pack4(x[u + r], 4 * half, coder);
                        transpose4(w);
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e)
                            *reinterpret_cast<uint32_t *>(&turned[(dim[u] + 4 * half + e) * kPitch + token[u]]) = w[e];
                    }
                }
            }
            __syncthreads();
            uint8_t *const out = c.v + (head * c.blocks + j) * kTokens * vp;
            for (uint32_t i = threadIdx.x; i < c.vdim * 4; i += 2 * kThreads) {
                const uint32_t *src = reinterpret_cast<const uint32_t *>(&turned[i / 4 * kPitch + i % 4 * 16]);
                reinterpret_cast<u32x4 *>(out)[i] = u32x4{src[0], src[1], src[2], src[3]};
            }
        } else {
#pragma unroll
            for (uint32_t u = 0; u < N; ++u) {
                if (token[u] < from || token[u] >= to) continue;
                if (!values) {
                    *reinterpret_cast<half8 *>(kt + token[u] * kp + dim[u]) = x[u];
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) vt[(dim[u] + e) * kTokens + token[u]] = x[u][e];
                }
            }
        }
        if (tid == 0) {
            if (values) {
                meta->v_scale = scale;
            } else {
                const uint64_t held = from == 0 ? 0 : meta->marked & ((uint64_t{1} << from) - 1);
                meta->k_scale = scale;
                meta->marked = fresh | held;
            }
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
    FastDiv k_quads, v_quads;   // groups of 4 elements per row
};

template <typename S> __device__ inline void store4(S *p, uint32_t word, float scale, bool marked) {
    const float nan = __builtin_nanf("");
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = marked ? nan : value_of((float)((int)(word >> (8 * e) & 255u) - 128), scale);
    if constexpr (sizeof(S) == 4) {
        *reinterpret_cast<f32x4 *>(p) = f32x4{x[0], x[1], x[2], x[3]};
    } else {
        typedef _Float16 half4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<half4 *>(p) = half4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
    }
}

// Values of one block, written as rows. kQuads (dims of whole fours): a thread
// turns 4 codes of a key row, or 16 tokens of 4 dims of the values, whose bytes
// it transposes in registers. Other dims go element by element through LDS.
// Bound by its bytes: 64 heads x 4096 tokens of 128 + 128 to f16 (201 MB) 36 us, 5.6
// TB/s; 8 heads x 16400 (101 MB) 23 us.
template <typename S, uint32_t P, bool kQuads>
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
    if (kQuads && open) {
        auto write = [&](S *out, const _Float16 *src, uint32_t dim, const FastDiv &quads, uint32_t by_token, uint32_t by_dim) {
            const _Float16 nan = (_Float16)__builtin_nanf("");
            for (uint32_t i = tid; i < live * (dim / 4); i += kThreads) {
                const uint32_t t = fast_div(i, quads), d = (i - t * (dim / 4)) * 4;
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    out[(size_t)i * 4 + e] = (S)(meta.marked >> t & 1 ? nan : src[t * by_token + (d + e) * by_dim]);
            }
        };
        if (a.key != nullptr)
            write(a.key + (head * a.rows + t0) * c.dim, c.kt + head * kTokens * c.kp, c.dim, a.k_quads, c.kp, 1);
        if (a.value != nullptr)
            write(a.value + (head * a.rows + t0) * c.vdim, c.vt + head * kTokens * c.vp, c.vdim, a.v_quads, 1, kTokens);
        return;
    }
    if (kQuads) {
        if (a.key != nullptr) {
            const uint8_t *src = c.k + block * kTokens * c.kp;
            S *out = a.key + (head * a.rows + t0) * c.dim;
            for (uint32_t i = tid; i < live * (c.dim / 4); i += kThreads) {
                const uint32_t t = fast_div(i, a.k_quads), q = i - t * (c.dim / 4);
                store4(out + (size_t)i * 4, *reinterpret_cast<const uint32_t *>(src + t * c.kp + q * 4), meta.k_scale,
                       meta.marked >> t & 1);
            }
        }
        if (a.value != nullptr) {
            const uint8_t *src = c.v + block * kTokens * c.vp;
            S *out = a.value + (head * a.rows + t0) * c.vdim;
            for (uint32_t i = tid; i < c.vdim; i += kThreads) {
                const uint32_t d = i / 4 * 4, first = i % 4 * 16;
                u32x4 w[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) w[r] = *reinterpret_cast<const u32x4 *>(src + (d + r) * kTokens + first);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t x[4] = {w[0][q], w[1][q], w[2][q], w[3][q]};
                    transpose4(x);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const uint32_t t = first + 4 * q + r;
                        if (t < live) store4(out + (size_t)t * c.vdim + d, x[r], meta.v_scale, meta.marked >> t & 1);
                    }
                }
            }
        }
        return;
    }
    const float nan = __builtin_nanf("");
    auto write = [&](S *out, uint32_t dim, uint32_t pitch, float scale) {
        for (uint32_t i = tid; i < live * dim; i += kThreads) {
            const uint32_t t = i / dim, d = i % dim;
            const float x = (float)rows[t * pitch + d];
            out[i] = meta.marked >> t & 1 ? (S)nan : (S)value_of(x, scale);
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

// One workgroup per (sequence, head): 1.5 us.
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
        c.kt[head * kTokens * c.kp + i] =
            (_Float16)value_of((float)((int)c.k[block * kTokens * c.kp + i] - 128), meta.k_scale);
    for (uint32_t i = threadIdx.x; i < kTokens * c.vp; i += kThreads)
        c.vt[head * kTokens * c.vp + i] =
            (_Float16)value_of((float)((int)c.v[block * kTokens * c.vp + i] - 128), meta.v_scale);
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

// Which tokens a head keeps: one workgroup per (sequence, head), a wave per
// sixteenth of the sequence. The want-th largest weight is found by its bits,
// 11, 11 and 10 from the top (a histogram of the next ones among the weights that
// share those so far); then every wave counts the tokens above and at it in its
// part and, from the counts of the parts before, writes the kept ones in order,
// the earliest of those that equal it.
// kHeld: up to 32768 tokens, whose images stay in registers; longer sequences
// are read anew each time.
// Bound by its chain of steps, each a memory or LDS latency and a barrier: 3 heads x
// 1100 tokens 9 us, 64 x 8200 17 us.
constexpr uint32_t kHeldKeys = 32;   // of a thread
constexpr uint32_t kBins = 2048;
template <bool kHeld>
__global__ __launch_bounds__(kSelectThreads) void kv_select_kernel(View from, EvictArgs a) {
    __shared__ uint32_t bins[kBins], chosen[2];
    __shared__ uint32_t above[kSelectWaves], equal[kSelectWaves];
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1);
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane(tid / kWave);
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
    // the wave's tokens: begin + 64 i + lane, i < steps
    const uint32_t steps = (length + kSelectThreads - 1) / kSelectThreads, begin = wave * steps * kWave;
    uint32_t held[kHeld ? kHeldKeys : 1];
    if constexpr (kHeld) {
#pragma unroll
        for (uint32_t i = 0; i < kHeldKeys; ++i) {
            if (i % 8 == 0 && i >= steps) break;
            held[i] = order_of(w[min(begin + i * kWave + lane, length - 1)]);
        }
    }
    auto each = [&](auto &&f) {   // f(token, image)
        if constexpr (kHeld) {
#pragma unroll
            for (uint32_t i = 0; i < kHeldKeys; ++i) {
                if (i >= steps) break;
                f(begin + i * kWave + lane, held[i]);
            }
        } else {
#pragma unroll 8
            for (uint32_t i = 0; i < steps; ++i) {
                const uint32_t t = begin + i * kWave + lane;
                f(t, order_of(w[min(t, length - 1)]));
            }
        }
    };
    uint32_t prefix = 0, left = want;   // the bits found; how many are wanted among those that share them
    for (uint32_t pass = 0; pass < 3 && want != 0; ++pass) {
        const uint32_t shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, mask = pass == 2 ? 1023 : 2047;
        const uint32_t above_shift = pass == 1 ? 21 : 10;
        bins[tid] = bins[tid + kSelectThreads] = 0;
        __syncthreads();
        each([&](uint32_t t, uint32_t u) {
            if (t >= lo && t < hi && (pass == 0 || u >> above_shift == prefix)) atomicAdd(&bins[u >> shift & mask], 1u);
        });
        __syncthreads();
        // thread i has bins 2047 - 2 i and 2046 - 2 i: a running sum from the top
        const uint32_t n0 = bins[kBins - 1 - 2 * tid], n1 = bins[kBins - 2 - 2 * tid];
        uint32_t upto = n0 + n1;
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) {
            const uint32_t other = __shfl_up(upto, d, kWave);
            if (lane >= (uint32_t)d) upto += other;
        }
        if (lane == kWave - 1) above[wave] = upto;
        __syncthreads();
        uint32_t higher = upto - n0 - n1;
#pragma unroll
        for (uint32_t i = 0; i < kSelectWaves; ++i) higher += i < wave ? above[i] : 0;
        if (higher < left && higher + n0 >= left) {
            chosen[0] = kBins - 1 - 2 * tid;
            chosen[1] = left - higher;
        } else if (higher + n0 < left && higher + n0 + n1 >= left) {
            chosen[0] = kBins - 2 - 2 * tid;
            chosen[1] = left - higher - n0;
        }
        __syncthreads();
        prefix = prefix << (pass == 2 ? 10 : 11) | chosen[0];
        left = chosen[1];
    }
    auto ranks = [&](uint32_t t, uint32_t u, bool &over, bool &same) {
        const bool middle = t >= lo && t < hi;
        over = t < length && (!middle || (want != 0 && u > prefix));
        same = middle && want != 0 && u == prefix;
    };
    uint32_t n_above = 0, n_equal = 0;
    each([&](uint32_t t, uint32_t u) {
        bool over, same;
        ranks(t, u, over, same);
        n_above += __popcll(__builtin_amdgcn_ballot_w64(over));
        n_equal += __popcll(__builtin_amdgcn_ballot_w64(same));
    });
    __syncthreads();   // (above[] has been read)
    if (lane == 0) {
        above[wave] = n_above;
        equal[wave] = n_equal;
    }
    __syncthreads();
    n_above = n_equal = 0;
#pragma unroll
    for (uint32_t i = 0; i < kSelectWaves; ++i) {
        n_above += i < wave ? above[i] : 0;
        n_equal += i < wave ? equal[i] : 0;
    }
    const uint64_t below = (uint64_t{1} << lane) - 1;
    each([&](uint32_t t, uint32_t u) {
        bool over, same;
        ranks(t, u, over, same);
        const uint64_t overs = __builtin_amdgcn_ballot_w64(over), sames = __builtin_amdgcn_ballot_w64(same);
        const uint32_t e = n_equal + __popcll(sames & below);
        if (over || (same && e < left)) put(n_above + __popcll(overs & below) + min(e, left), t);
        n_above += __popcll(overs);
        n_equal += __popcll(sames);
    });
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
//
// A thread has 16-byte pieces of one kept key row (four threads per row), and of
// the values one kept token (a lane each) in four neighbouring dims of every
// sixteen, byte by byte: the lanes' tokens lie in a few 64-byte rows of the
// source. Four lanes turn their new codes of four dims into four tokens of one
// dim each, and store words. 64 heads x 4096 of 8200 tokens of 128 + 128 (134 MB out of
// the kept ones and in) 48 us, 2.8 TB/s: the value rows are read whole for half of
// their bytes, by the workgroups of two blocks, and index, codes and maxima are had
// one after another. (Half the arithmetic gave nothing; the source's blocks brought
// to LDS whole, and the bytes read there, 56 us.)
__device__ inline uint32_t value_dim(uint32_t u, uint32_t wave) { return u / 4 * 16 + wave * 4 + u % 4; }
// Bytes (dims 0 .. 3 of one lane's token) to bytes (tokens of four lanes) of the
// dim lane % 4: exchanges with lane ^ 1, then lane ^ 2.
__device__ inline uint32_t quad_transpose(uint32_t own, uint32_t lane) {
    const uint32_t p = (uint32_t)dpp_i32<kQuadSwap1>(0, (int)own);
    const uint32_t y = __builtin_amdgcn_perm(p, own, lane & 1 ? 0x03070105u : 0x06020400u);
    const uint32_t z = (uint32_t)dpp_i32<kQuadSwap2>(0, (int)y);
    return __builtin_amdgcn_perm(z, y, lane & 2 ? 0x03020706u : 0x05040100u);
}
__device__ inline double wave_max_f64(double v) {
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) v = fmax(v, __shfl_xor(v, d, kWave));
    return v;
}

// Values anew: x is a code with its block's scale, or (scale 1) an f16.
struct Recoder {
    float scale, ratio;   // ratio = 127 scale / largest; an all-zero block's is 0
    double big;
    // Codes + 128 of four elements as bytes.
    __device__ inline uint32_t four(const _Float16 *x) const {
        constexpr float kWhole = 12582912.0f + 128.0f;   // 1.5 * 2^23: rounds to whole numbers
        uint32_t b[4];
        bool near = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float q = (float)x[e] * ratio, n = q + kWhole;
            near = near || fabsf(q - (n - kWhole)) > 0.5f - 0x1p-12f;
            b[e] = __builtin_bit_cast(uint32_t, n);
        }
        if (near) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                b[e] = big > 0.0 ? (uint32_t)(int)rint(127.0 * ((double)(float)x[e] * (double)scale) / big) + 128u : 128u;
        }
        return __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u) | __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
    }
};

template <uint32_t P>
__global__ __launch_bounds__(kThreads) void kv_move_kernel(MoveArgs a) {
    __shared__ double biggest[2][kWaves];
    __shared__ uint32_t marks[2];
    const View &f = a.from, &c = a.to;
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1);
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane(tid / kWave);
    const uint32_t j = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const size_t head = (size_t)b * c.heads + h;
    const uint32_t length = f.length[b], kept = min(length, a.keep);
    if (j == 0 && h == 0 && tid == 0) c.length[b] = kept;
    if (j * kTokens >= kept) return;
    const uint32_t live = min(kept - j * kTokens, kTokens), kp = f.kp, vp = f.vp;
    const bool closed = live == kTokens;
    const uint32_t *const index = a.index + head * a.keep_most + j * kTokens;
    const uint32_t open_block = length / kTokens;
    if (tid < 2) marks[tid] = 0;

    // keys: row tid / 4, pieces tid % 4, + 4, ... (rows past the last kept token
    // repeat it; they are not written)
    const uint32_t row = tid / 4, kt = index[min(row, live - 1)];
    const bool k_open = kt / kTokens == open_block;
    const Meta km = f.meta[head * f.blocks + kt / kTokens];
    const float k_old = k_open ? 1.0f : km.k_scale;
    // values: token `lane`, dims 16 i + 4 wave .. + 3
    const uint32_t vtoken = index[min(lane, live - 1)];
    const bool v_open = vtoken / kTokens == open_block;
    const Meta vm = f.meta[head * f.blocks + vtoken / kTokens];
    const float v_old = v_open ? 1.0f : vm.v_scale;
    // (columns past the width read the last ones again and are not written: no
    // load waits behind a test)
    u32x4 kw[P / 64];
    uint8_t vw[P / 4];
    const uint8_t *const ksrc = f.k + (head * f.blocks * kTokens + kt) * kp;
    const uint8_t *const vsrc = f.v + (head * f.blocks + vtoken / kTokens) * vp * kTokens + vtoken % kTokens;
#pragma unroll
    for (uint32_t u = 0; u < P / 64; ++u)
        kw[u] = *reinterpret_cast<const u32x4 *>(ksrc + min((tid % 4 + 4 * u) * 16, kp - 16));
#pragma unroll
    for (uint32_t u = 0; u < P / 4; ++u) vw[u] = vsrc[min(value_dim(u, wave), vp - 1) * kTokens];
    _Float16 kx[P / 64][16], vx[P / 4];
    float kmax = 0.0f, vmax = 0.0f;
#pragma unroll
    for (uint32_t u = 0; u < P / 64; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) kx[u][e] = (_Float16)(int)((kw[u][e / 4] >> (8 * (e % 4)) & 255u) - 128u);
#pragma unroll
    for (uint32_t u = 0; u < P / 4; ++u) vx[u] = (_Float16)((int)vw[u] - 128);
    if (wave_any(k_open)) {
        const _Float16 *const src = f.kt + (head * kTokens + kt % kTokens) * kp;
        if (k_open)
#pragma unroll
            for (uint32_t u = 0; u < P / 64; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) kx[u][e] = src[min((tid % 4 + 4 * u) * 16, kp - 16) + e];
    }
    if (wave_any(v_open)) {
        const _Float16 *const src = f.vt + head * vp * kTokens + vtoken % kTokens;
        if (v_open)
#pragma unroll
            for (uint32_t u = 0; u < P / 4; ++u) vx[u] = src[min(value_dim(u, wave), vp - 1) * kTokens];
    }
#pragma unroll
    for (uint32_t u = 0; u < P / 64; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) kmax = fmaxf(kmax, fabsf((float)kx[u][e]));
#pragma unroll
    for (uint32_t u = 0; u < P / 4; ++u) vmax = fmaxf(vmax, fabsf((float)vx[u]));
    const double kwide = wave_max_f64((double)kmax * (double)k_old), vwide = wave_max_f64((double)vmax * (double)v_old);
    __syncthreads();   // (marks are cleared)
    if (lane == 0) {
        biggest[0][wave] = kwide;
        biggest[1][wave] = vwide;
    }
    if (wave == 0 && lane < live && (vm.marked >> (vtoken % kTokens) & 1)) atomicOr(&marks[lane / 32], 1u << (lane % 32));
    __syncthreads();
    if (!closed) {
        _Float16 *const ko = c.kt + head * kTokens * kp, *const vo = c.vt + head * vp * kTokens;
#pragma unroll
        for (uint32_t u = 0; u < P / 64; ++u) {
            const uint32_t d = (tid % 4 + 4 * u) * 16;
            if (d >= kp || row >= live) continue;
#pragma unroll
            for (int e = 0; e < 16; ++e) ko[row * kp + d + e] = (_Float16)value_of((float)kx[u][e], k_old);
        }
#pragma unroll
        for (uint32_t u = 0; u < P / 4; ++u)
            if (value_dim(u, wave) < vp && lane < live)
                vo[value_dim(u, wave) * kTokens + lane] = (_Float16)value_of((float)vx[u], v_old);
        if (tid == 0) c.meta[head * c.blocks + j] = Meta{1.0f, 1.0f, marks[0] | (uint64_t)marks[1] << 32};
        return;
    }
    double big[2] = {0.0, 0.0};
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w)
#pragma unroll
        for (int i = 0; i < 2; ++i) big[i] = fmax(big[i], biggest[i][w]);
    const Recoder keys{k_old, big[0] > 0.0 ? (float)(127.0 * (double)k_old / big[0]) : 0.0f, big[0]};
    const Recoder values{v_old, big[1] > 0.0 ? (float)(127.0 * (double)v_old / big[1]) : 0.0f, big[1]};
    const size_t block = head * c.blocks + j;
#pragma unroll
    for (uint32_t u = 0; u < P / 64; ++u) {
        const uint32_t d = (tid % 4 + 4 * u) * 16;
        if (d >= kp) continue;
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = keys.four(&kx[u][4 * e]);
        *reinterpret_cast<u32x4 *>(c.k + (block * kTokens + row) * kp + d) = w;
    }
#pragma unroll
    for (uint32_t u = 0; u < P / 4; u += 4) {
        const uint32_t d = value_dim(u, wave);
        if (d >= vp) continue;
        *reinterpret_cast<uint32_t *>(c.v + (block * vp + d + lane % 4) * kTokens + lane / 4 * 4) =
            quad_transpose(values.four(&vx[u]), lane);
    }
    if (tid == 0)
        c.meta[block] = Meta{(float)(big[0] / 127.0), (float)(big[1] / 127.0), marks[0] | (uint64_t)marks[1] << 32};
}

uint32_t class_of(const View &c) {
    const uint32_t widest = c.kp > c.vp ? c.kp : c.vp;
    return widest <= 64 ? 64 : widest <= 128 ? 128 : 256;
}

template <typename S>
void launch_append(AppendArgs<S> a, dim3 grid, hipStream_t s) {
    if (a.c.dim % 8 == 0 && a.c.vdim % 8 == 0) {
        a.k_groups = make_fast_div(a.c.dim / 8);
        a.v_groups = make_fast_div(a.c.vdim / 8);
        switch (class_of(a.c)) {
            case 64: kv_append_groups_kernel<S, 64><<<grid, 2 * kThreads, 0, s>>>(a); break;
            case 128: kv_append_groups_kernel<S, 128><<<grid, 2 * kThreads, 0, s>>>(a); break;
            default: kv_append_groups_kernel<S, 256><<<grid, 2 * kThreads, 0, s>>>(a); break;
        }
        return;
    }
    switch (class_of(a.c)) {
        case 64: kv_append_kernel<S, 64><<<grid, kThreads, 0, s>>>(a); break;
        case 128: kv_append_kernel<S, 128><<<grid, kThreads, 0, s>>>(a); break;
        default: kv_append_kernel<S, 256><<<grid, kThreads, 0, s>>>(a); break;
    }
}

template <typename S, bool kQuads>
void launch_read(const ReadArgs<S> &a, dim3 grid, hipStream_t s) {
    switch (class_of(a.c)) {
        case 64: kv_read_kernel<S, 64, kQuads><<<grid, kThreads, 0, s>>>(a); break;
        case 128: kv_read_kernel<S, 128, kQuads><<<grid, kThreads, 0, s>>>(a); break;
        default: kv_read_kernel<S, 256, kQuads><<<grid, kThreads, 0, s>>>(a); break;
    }
}
template <typename S>
void launch_read(ReadArgs<S> a, dim3 grid, hipStream_t s) {
    if (a.c.dim % 4 == 0 && a.c.vdim % 4 == 0) {
        a.k_quads = make_fast_div(a.c.dim / 4);
        a.v_quads = make_fast_div(a.c.vdim / 4);
        launch_read<S, true>(a, grid, s);
    } else {
        launch_read<S, false>(a, grid, s);
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
                                        {}, {}, start, count}, grid, s);
    else
        launch_append(AppendArgs<_Float16>{c, static_cast<const _Float16 *>(key), static_cast<const _Float16 *>(value),
                                           n, first, {}, {}, start, count}, grid, s);
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
        launch_read(ReadArgs<float>{c, static_cast<float *>(key), static_cast<float *>(value), rows, {}, {}}, grid, s);
    else
        launch_read(ReadArgs<_Float16>{c, static_cast<_Float16 *>(key), static_cast<_Float16 *>(value), rows, {}, {}}, grid, s);
    return hipGetLastError();
}

hipError_t evict(const View &from, const View &to, uint32_t batch, const EvictArgs &a, hipStream_t s) {
    if (a.longest <= kHeldKeys * kSelectThreads)
        kv_select_kernel<true><<<dim3(from.heads, batch), kSelectThreads, 0, s>>>(from, a);
    else
        kv_select_kernel<false><<<dim3(from.heads, batch), kSelectThreads, 0, s>>>(from, a);
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
