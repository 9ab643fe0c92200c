// Attention over the 8-bit key/value cache (kv.hpp), f16 and f32.
//
// kv_rows.hpp has the kernel for few rows and the arithmetic, k_kv_tiles.hip the one
// for many; here are their launches, the join of their parts, and the plan.
#include "kv_rows.hpp"

namespace icsdk {
namespace kv {
namespace {

constexpr uint32_t kRowsArguments = 64;   // where the struct behind the leading ones lies

template <typename S, uint32_t P, bool kStream>
__global__ __launch_bounds__(kThreads) void kv_rows_kernel(const uint8_t *keys, const uint8_t *values,
                                                           const uint32_t *lengths, const Meta *metas, const S *queries,
                                                           uint32_t all_blocks, uint32_t heads, uint32_t parts_first,
                                                           uint32_t pitches, uint32_t n, uint32_t group, Args<S> a) {
    __shared__ RowsOut<P> lds_o;
    __shared__ RowsMl<> lds_ml;
    rows_of<S, P, kStream, false>(lds_o, lds_ml, keys, values, lengths, metas, queries, all_blocks, heads, parts_first, pitches, n, group,
                           kernel_arguments<Args<S>>(kRowsArguments), blockIdx.x, blockIdx.y, blockIdx.z);
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

}  // namespace

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
    p.many = whole_rows > (uint64_t)row_tiles * rows_for_tile(f32, widest_of(c)) && tiles_fit(f32, widest_of(c));
    p.tiles = p.many && products >= (f32 ? kTileProductsF32 : kTileProducts);
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

namespace {

template <typename S, uint32_t P>
hipError_t launch_rows(const Args<S> &a, uint32_t groups, hipStream_t s) {
    const dim3 grid(groups * a.parts, a.c.heads, a.pairs / a.c.heads);
    const size_t bytes = (size_t)a.pairs * a.longest * (a.c.kp + a.c.vp);
    const auto kernel = bytes > kStreamBytes ? kv_rows_kernel<S, P, true> : kv_rows_kernel<S, P, false>;
    kernel<<<grid, kThreads, 0, s>>>(a.c.k, a.c.v, a.c.length, a.c.meta, a.q, a.c.blocks, a.c.heads,
                                     a.parts | a.first << 16, a.c.kp | a.c.vp << 16, a.n, a.group, a);
    return hipGetLastError();
}
template <typename S>
hipError_t launch_rows(const Args<S> &a, uint32_t widest, uint32_t groups, hipStream_t s) {
    if (widest <= 32) return launch_rows<S, 32>(a, groups, s);
    if (widest <= 64) return launch_rows<S, 64>(a, groups, s);
    if (widest <= 96) return launch_rows<S, 96>(a, groups, s);
    if (widest <= 128) return launch_rows<S, 128>(a, groups, s);
    if (widest <= 192) return launch_rows<S, 192>(a, groups, s);
    return launch_rows<S, 256>(a, groups, s);
}

}  // namespace

template <typename S>
hipError_t launch_fold(const Args<S> &a, uint32_t parts, bool scores, uint32_t longest, bool wide, hipStream_t s) {
    const uint32_t blocks = (longest + kTokens - 1) / kTokens;
    // (at most 512 row groups where there are more parts than a workgroup has waves)
    const uint32_t folds = parts > 1 ? a.pairs * a.group * a.n : 0;
    const uint32_t threads = wide ? 16 * kWave : kThreads;
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
template hipError_t launch_fold<float>(const Args<float> &, uint32_t, bool, uint32_t, bool, hipStream_t);
template hipError_t launch_fold<_Float16>(const Args<_Float16> &, uint32_t, bool, uint32_t, bool, hipStream_t);

namespace {

template <typename S>
hipError_t launch(Args<S> a, const Plan &p, uint32_t batch, uint32_t longest, float *partial, hipStream_t s) {
    const uint32_t blocks = (longest + kTokens - 1) / kTokens, widest = widest_of(a.c);
    // (a launch holds fewer than 2^32 threads)
    const uint32_t most = (1u << 23) / (a.pairs * p.parts) < 1 ? 1 : (1u << 23) / (a.pairs * p.parts);
    for (uint32_t g0 = 0; g0 < p.row_groups; g0 += most) {
        a.row_group0 = g0;
        const uint32_t groups = p.row_groups - g0 < most ? p.row_groups - g0 : most;
        const hipError_t status = p.tiles ? launch_tiles(a, widest, groups, s) : launch_rows(a, widest, groups, s);
        if (status != hipSuccess) return status;
    }
    if (p.parts > 1 || p.scores) {
        const hipError_t status = launch_fold<S>(a, p.parts, p.scores, longest, p.parts > 16, s);
        if (status != hipSuccess) return status;
    }
    if (a.row_ml != nullptr && blocks > 0) return launch_weights(a, widest, batch, blocks, p.row_parts, partial, s);
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

}  // namespace

size_t attention_workspace(bool f32, const View &c, const AttentionShape &a) { return plan_of(f32, c, a).bytes(); }

hipError_t attention(bool f32, const View &c, const AttentionShape &a, const void *query, void *output,
                     void *workspace, hipStream_t s) {
    return f32 ? run<float>(c, a, query, output, workspace, s) : run<_Float16>(c, a, query, output, workspace, s);
}

}  // namespace kv
}  // namespace icsdk
