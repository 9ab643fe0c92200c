// Attention over the 8-bit cache of sequences whose tokens follow a prefix that
// several of them share.
//
// Of few tokens a workgroup has both, a wave some blocks of either (kv_shared_close_kernel).
// Else two passes into the same rows' parts: over the prefix the rows of a group's sequences
// are packed as one head's rows, so that its codes are read once for 16 or 128 of them,
// and over each sequence's own tokens as in attention without a prefix. A softmax over
// both is their parts' join (kv_join_kernel; kv_fold_kernel for many parts of few rows). The passes are one launch: neither waits
// for the other, and where the prefix is bound by its products (tiles) and the own
// tokens by memory (rows), a CU has one of each. Padded rows lie among a group's packed
// ones; they are not loaded, and a workgroup that has no others ends at once (4 x 512
// rows on 8000 tokens 300 us, of which 512, 400, 300 and 1 are there 247, one each of three
// 221).
#include "kv_rows.hpp"
#include "kv_tiles.hpp"

namespace icsdk {
namespace kv {
namespace {

template <typename S> struct Both {
    SharedArgs<S> pass[2];   // the prefix, own tokens
    uint32_t first;          // workgroups of the first pass; those behind are the second's
};

// Workgroup i of a pass by the rows kernel; kSolo: each wave does what a workgroup
// would, the waves of four of them.
template <typename S, uint32_t P, bool kStream, bool kSolo>
__device__ __forceinline__ void rows_of(RowsOut<P> &lds_o, RowsMl<> &lds_ml, Constant<SharedArgs<S>> &a, uint32_t i) {
    if constexpr (kSolo) {
        i = i * kWaves + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
        if (i >= a.columns * a.pairs) return;
    }
    const uint32_t pair = i % a.pairs, x = i / a.pairs, h = pair % a.c.heads, b = pair / a.c.heads;
    rows_of<S, P, kStream, kSolo>(lds_o, lds_ml, a.c.k, a.c.v, a.c.length, a.c.meta, a.q, a.c.blocks, a.c.heads,
                                  a.parts | a.first << 16, a.c.kp | a.c.vp << 16, a.n, a.group, a, x, h, b);
}

// Both by the rows kernel. 14 f32 sequences of 130 tokens with 4 rows of 16 heads on three
// prefixes of 1500, D 80: 11 us, and the join 4, for 4 MB of codes: bound by a workgroup's
// chain (arguments, lengths, queries, two or three blocks for each wave, the waves' meeting).
template <typename S, uint32_t P, bool kStream>
__global__ __launch_bounds__(kThreads) void kv_shared_rows_kernel(Both<S>) {
    __shared__ RowsOut<P> lds_o;
    __shared__ RowsMl<> lds_ml;
    auto &both = kernel_arguments<Both<S>>(0);
    const uint32_t second = blockIdx.x >= both.first ? 1 : 0;
    rows_of<S, P, kStream, false>(lds_o, lds_ml, both.pass[second], blockIdx.x - (second ? both.first : 0));
}

// Own tokens by waves alone. 8 x 8 sequences of 100 tokens on 2000, 32/8 heads of 128: 18 us
// for 47 MB (2.6 TB/s), bound by latency: three blocks for each wave of the prefix, one
// after another, and registers for two workgroups in a CU. A fourth part of the prefix is a
// second round of workgroups (the call 28 us for 21); three in a CU spill registers (27).
template <typename S, uint32_t P>
__global__ __launch_bounds__(kThreads) void kv_shared_solo_kernel(Both<S>) {
    __shared__ RowsOut<P> lds_o;
    __shared__ RowsMl<> lds_ml;
    auto &both = kernel_arguments<Both<S>>(0);
    if (blockIdx.x < both.first) rows_of<S, P, false, false>(lds_o, lds_ml, both.pass[0], blockIdx.x);
    else rows_of<S, P, false, true>(lds_o, lds_ml, both.pass[1], blockIdx.x - both.first);
}

// Both by tiles. Four sequences' 512 rows behind 8000 tokens, 32/8 heads of 128, f16: 285 us
// (975 TFLOP/s; 330 in the first calls, before the clock settles), bound as kv_tiles_kernel
// is. A pass over own tokens that goes on over the prefix, without parts, took 344 us against
// 322 and the join's 16: its workgroups end all at once.
template <typename S, uint32_t P>
__global__ __launch_bounds__(kThreads, tiles_twice(sizeof(S) == 4, P) ? 2 : 1) void kv_shared_tiles_kernel(Both<S>) {
    __shared__ __attribute__((aligned(16))) typename TilesLds<P>::Keys ks;
    __shared__ __attribute__((aligned(16))) typename TilesLds<P>::Values vs;
    __shared__ typename TilesLds<P>::Most wave_most;
    auto &both = kernel_arguments<Both<S>>(0);
    const uint32_t second = blockIdx.x >= both.first ? 1 : 0;
    tiles_of<S, P, false>(ks, vs, wave_most, both.pass[second], blockIdx.x - (second ? both.first : 0));
}

// Tiles over the prefix, rows over own tokens. 64 sequences of up to 500 tokens on 16000,
// 32/8 heads of 128, f16: 40 us, where the tiles alone take 35 and the rows alone 18. Bound
// by a tile's turn (1.8 us with one workgroup of tiles in a CU, 16 turns each). More parts
// (24: 56 us for 48, the call), or own workgroups before some of the prefix's (58 to 75 us),
// make the passes follow each other.
template <typename S, uint32_t P>
__global__ __launch_bounds__(kThreads, 2) void kv_shared_mixed_kernel(Both<S>) {
    static_assert(tiles_twice(sizeof(S) == 4, P) && sizeof(RowsOut<P>) + sizeof(RowsMl<>) <= sizeof(typename TilesLds<P>::Keys));
    __shared__ __attribute__((aligned(16))) typename TilesLds<P>::Keys ks;
    __shared__ __attribute__((aligned(16))) typename TilesLds<P>::Values vs;
    __shared__ typename TilesLds<P>::Most wave_most;
    auto &both = kernel_arguments<Both<S>>(0);
    if (blockIdx.x < both.first) {
        tiles_of<S, P, false>(ks, vs, wave_most, both.pass[0], blockIdx.x);
    } else {
        char *const lds = reinterpret_cast<char *>(ks);
        rows_of<S, P, false, false>(*reinterpret_cast<RowsOut<P> *>(lds),
                                    *reinterpret_cast<RowsMl<> *>(lds + sizeof(RowsOut<P>)), both.pass[1],
                                    blockIdx.x - both.first);
    }
}

// Both by one workgroup, and no parts: of its eight waves four have the prefix and four
// own tokens, of one sequence's rows. Four sequences of 20 tokens on 200, 9/3 heads of 64:
// 6.4 us (6.1 and the join's 1.8 by parts), a chain of latencies.
template <typename S, uint32_t P>
__global__ __launch_bounds__(2 * kThreads) void kv_shared_close_kernel(Both<S>) {
    constexpr uint32_t kMeet = 2 * kWaves;
    __shared__ RowsOut<P, kMeet> lds_o;
    __shared__ RowsMl<kMeet> lds_ml;
    auto &both = kernel_arguments<Both<S>>(0);
    const uint32_t second = (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
    auto &a = both.pass[second];
    const uint32_t pair = blockIdx.x % a.pairs, x = blockIdx.x / a.pairs, h = pair % a.c.heads, b = pair / a.c.heads;
    const uint32_t sequence = both.pass[1].first + b, of = second ? sequence : both.pass[0].count.n[b];
    rows_of<S, P, false, false, kMeet>(lds_o, lds_ml, a.c.k, a.c.v, a.c.length, a.c.meta, a.q, a.c.blocks, a.c.heads, 1,
                                       a.c.kp | a.c.vp << 16, a.n, a.group, a, x, h, of,
                                       OwnRows{sequence, both.pass[1].count.n[b]});
}

// Counts of sequences where the kernels of a call of more than a launch's find them.
__global__ __launch_bounds__(kBatchPerLaunch) void kv_counts_kernel(uint32_t *counts, uint32_t batch, Counts of) {
    if (threadIdx.x < batch) counts[threadIdx.x] = of.n[threadIdx.x];
}

// ---- the parts' join ------------------------------------------------------------------------

struct JoinArgs {
    const float *part_o;
    const f32x2 *part_ml;
    size_t rows, first_row;    // of all sequences; of the first of `count`
    uint32_t parts, vdim, from, all;   // the launch's rows: from first_row + from on, `all` of them
    FastDiv per_row;             // threads of a row, four elements each
    bool padded;                 // some rows are padding, by `count`
    FastDiv n, per_sequence;     // rows of a query head, and of a sequence
    Counts count;
};

// A thread has four elements of a row; kHeld parts are asked for at once. 4 x 32 heads x 512
// rows of two parts (67 MB read, 17 written) 16 us, 5.2 TB/s; by four waves for each row 32.
// Few rows of a few parts: 3.8 us, two latencies and the launch. (Past the
// last part that one again, and not used.)
template <typename S, uint32_t kHeld> __global__ __launch_bounds__(kThreads) void kv_join_kernel(S *out, JoinArgs a) {
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x, r = fast_div(i, a.per_row), d = 4 * (i - r * a.per_row.divisor);
    if (r >= a.all) return;
    const uint32_t at = a.from + r;
    const size_t row = a.first_row + at;
    if (a.padded && at - fast_div(at, a.n) * a.n.divisor >= a.count.n[fast_div(at, a.per_sequence)]) return;
    const uint32_t last = a.parts - 1;
    auto load = [&](uint32_t s) {
        const float *const src = a.part_o + ((size_t)s * a.rows + row) * a.vdim + d;
        f32x4 x;
        if (a.vdim % 4 == 0) {
            x = *reinterpret_cast<const f32x4 *>(src);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) x[e] = d + e < a.vdim ? src[e] : 0.0f;
        }
        return x;
    };
    f32x4 v = {0, 0, 0, 0}, held[kHeld];
    f32x2 ml[kHeld];
#pragma unroll
    for (uint32_t k = 0; k < kHeld; ++k) {
        const uint32_t s = min(k, last);
        held[k] = load(s);
        ml[k] = a.part_ml[(size_t)s * a.rows + row];
    }
    float top = ml[0].x, total = 0.0f;
#pragma unroll
    for (uint32_t k = 1; k < kHeld; ++k) top = fmaxf(top, ml[k].x);
#pragma unroll 8
    for (uint32_t s = kHeld; s < a.parts; ++s) top = fmaxf(top, a.part_ml[(size_t)s * a.rows + row].x);
    // (a part that saw nothing has weight 0, and a NaN in it stays)
    auto weight = [&](float m) { return top == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - top); };
#pragma unroll
    for (uint32_t k = 0; k < kHeld; ++k)
        if (k < a.parts) {
            const float w = weight(ml[k].x);
            v += held[k] * w;
            total += ml[k].y * w;
        }
#pragma unroll 8
    for (uint32_t s = kHeld; s < a.parts; ++s) {
        const f32x2 x = a.part_ml[(size_t)s * a.rows + row];
        const float w = weight(x.x);
        v += load(s) * w;
        total += x.y * w;
    }
    store_out(out + row * a.vdim, a.vdim, d, finish(v, top, total));
}

// Few rows of many parts are joined by 16 waves each (kv_fold_kernel).
constexpr size_t kWideRows = 512;

// ---- plan --------------------------------------------------------------------------------

// Measured (us, the call, four waves and solo; f16, one query row): 8 prefixes of 2000 x 8
// sequences, 8 heads of 128, own tokens of 2 blocks 24.5 and 20.9, of 8 37.9 and 34.9, of 12
// 45.7 and 43.1, of 16 50.3 and 51.3; 5 heads of 64, 8 x 8 sequences of 15 blocks 17.8 and
// 25.6. With f32 queries (28 for 22) or beside tiles (49 for 46) it loses.
constexpr uint32_t kSoloBlocks = 8;

// A pass: its kernel and its workgroups.
struct Pass {
    bool tiles, solo;   // (solo: rows, by waves alone)
    uint32_t batch, row_groups, parts;
};
struct SharedPlan {
    Pass prefix, own;
    bool close;      // both by one workgroup
    bool together;   // in one launch
    uint32_t n;      // rows of a prefix's head
    size_t rows, o_bytes, ml_bytes, counts_bytes;
};

Pass pass_of(const View &c, bool tiles, uint32_t batch, uint32_t in_head, uint32_t longest, uint64_t workgroups) {
    Pass p{tiles, false, batch, 0, 1};
    const uint32_t rows = tiles ? kTileRows : kRows, blocks = (longest + kTokens - 1) / kTokens;
    p.row_groups = (in_head + rows - 1) / rows;
    const uint64_t base = (uint64_t)batch * c.heads * p.row_groups, most = (blocks + kWaves - 1) / kWaves;
    uint64_t parts = base == 0 ? 1 : workgroups / base;
    parts = parts < most ? parts : most;
    p.parts = parts < 1 ? 1 : (uint32_t)parts;
    return p;
}

uint64_t workgroups_of(const View &c, const Pass &p) {
    const uint64_t n = (uint64_t)p.batch * c.heads * p.row_groups * p.parts;
    return p.solo ? (n + kWaves - 1) / kWaves : n;
}

// Few blocks are done by one workgroup of a sequence's rows (kv_shared_close_kernel): no
// parts and no join, but a prefix is read for each sequence. Measured (us, the call, a
// workgroup for both and parts; 2 prefixes, own tokens of 200, 8 heads, workgroups x tokens
// of a prefix): f16 D 64, 64 x 250 7.7 and 11.3, 64 x 1000 9.1 and 11.1, 64 x 2000 (own 50)
// 11.9 and 9.4, 512 x 500 11.9 and 14.7, 1024 x 500 19 and 17; D 128, 64 x 500 10.5 and 12.4,
// 64 x 1000 14.4 and 13.1, 256 x 500 12.7 and 18.9, 512 x 250 20 and 19; D 192, 64 x 500 15.1
// and 15.1, 256 x 500 17 and 23; f32 D 32, 64 x 1000 9.1 and 11.0, 512 x 500 10.5 and 12.1; D
// 64, 64 x 500 8.8 and 11.2, 64 x 1000 11.7 and 11.5, 512 x 250 15.3 and 15.0; D 128, 64 x
// 250 11.0 and 13.0, 64 x 500 14.0 and 13.8, 256 x 500 15.6 and 17.4; D 80, 64 x (500, own
// 300) 11.8 and 10.2.
constexpr uint32_t kCloseBlocks = 12, kCloseBlocksMore = 20, kCloseWorkgroups = 256;
// (wider ones do not find registers for eight waves)
constexpr bool close_built(bool f32, uint32_t widest) { return widest <= (f32 ? 128u : 192u); }
bool close_fits(bool f32, const PrefixShape &ps, const View &c, const AttentionShape &a) {
    const uint32_t widest = widest_of(c), in_head = a.q_heads / c.heads * a.n;
    const uint32_t row_groups = (in_head + kRows - 1) / kRows;
    const uint64_t blocks = ((uint64_t)ps.longest + kTokens - 1) / kTokens + ((uint64_t)a.longest + kTokens - 1) / kTokens;
    const bool twice = widest <= (f32 ? 32u : 64u);   // two workgroups in a CU
    return close_built(f32, widest) && blocks <= (widest <= (f32 ? 32u : 96u) ? kCloseBlocksMore : kCloseBlocks) &&
           (uint64_t)a.batch * c.heads * row_groups <= (twice ? 2 : 1) * kCloseWorkgroups;
}

bool padded(const AttentionShape &a) {
    for (uint32_t b = 0; a.counts != nullptr && b < a.batch; ++b)
        if (a.counts[b] < a.n) return true;
    return false;
}

SharedPlan plan_of(bool f32, const View &prefix, const PrefixShape &ps, const View &c, const AttentionShape &a) {
    SharedPlan p{};
    const uint32_t widest = widest_of(c), own_rows = a.q_heads / c.heads * a.n;
    p.n = ps.most * own_rows;
    const Plan over = icsdk::kv::plan_of(f32, prefix, AttentionShape{ps.batch, prefix.heads, p.n, ps.longest, a.scale, false,
                                                                     nullptr, nullptr, 0, 0});
    const Plan own = icsdk::kv::plan_of(f32, c, a);
    p.close = close_fits(f32, ps, c, a);
    if (p.close) {
        p.own = pass_of(c, false, a.batch, own_rows, a.longest, 1);
        return p;
    }
    // beside a pass by tiles another one by tiles needs no products enough to fill the chip
    const bool own_tiles = own.tiles || (over.tiles && own.many), prefix_tiles = over.tiles || (own_tiles && over.many);
    const bool mixed = prefix_tiles && !own_tiles;
    p.together = prefix_tiles == own_tiles || (mixed && tiles_twice(f32, widest));
    const bool twice = prefix_tiles || own_tiles ? tiles_twice(f32, widest) : rows_twice(f32, widest);
    const uint32_t fill = twice ? kWorkgroups : kWorkgroups / 2;
    p.own = pass_of(c, own_tiles, a.batch, own_rows, a.longest, fill);
    // own tokens of few blocks, of which four waves would have one or two each, where the
    // workgroups of their own would take the chip from the prefix
    p.own.solo = !f32 && !prefix_tiles && !own_tiles && a.longest <= kSoloBlocks * kTokens &&
                 workgroups_of(c, p.own) >= fill / 2;
    // the prefix has what the own tokens leave of the chip, half at least
    const uint64_t taken = p.together ? workgroups_of(c, p.own) : 0;
    p.prefix = pass_of(prefix, prefix_tiles, ps.batch, p.n, ps.longest, fill - (taken < fill / 2 ? taken : fill / 2));
    p.rows = (size_t)a.batch * a.q_heads * a.n;
    const size_t parts = p.prefix.parts + p.own.parts;
    p.o_bytes = whole256(parts * p.rows * c.vdim * 4);
    p.ml_bytes = whole256(parts * p.rows * sizeof(f32x2));
    p.counts_bytes = padded(a) && a.batch > kBatchPerLaunch ? whole256(a.batch * sizeof(uint32_t)) : 0;
    return p;
}

// ---- launch --------------------------------------------------------------------------------

// The launches that a pass is in: 256 sequences and 2^22 workgroups each.
template <typename S> struct Cursor {
    const View &c;
    const Pass &pass;
    uint32_t first = 0, group = 0;

    bool done() const { return first >= pass.batch; }
    // Sequences, row groups and workgroups of the next launch.
    uint32_t batch() const { return pass.batch - first < kBatchPerLaunch ? pass.batch - first : kBatchPerLaunch; }
    uint32_t next(SharedArgs<S> &a) {
        a.first = first;
        a.pairs = batch() * c.heads;
        a.row_group0 = group;
        const uint32_t fit = (1u << 22) / (a.pairs * pass.parts), most = fit < 1 ? 1 : fit;
        const uint32_t groups = pass.row_groups - group < most ? pass.row_groups - group : most;
        a.columns = groups * pass.parts;
        group += groups;
        if (group == pass.row_groups) {
            first += batch();
            group = 0;
        }
        const uint32_t n = a.columns * a.pairs;
        return pass.solo ? (n + kWaves - 1) / kWaves : n;
    }
};

// Which kernel a launch takes.
struct Kernels {
    bool tiles[2], solo, stream;
};
template <typename S, uint32_t P> hipError_t launch(const Both<S> &both, uint32_t grid, const Kernels &k, hipStream_t s) {
    auto go = [&](auto kernel) {
        kernel<<<grid, kThreads, 0, s>>>(both);
        return hipGetLastError();
    };
    if constexpr (tiles_twice(sizeof(S) == 4, P))
        if (k.tiles[0] && !k.tiles[1]) return go(kv_shared_mixed_kernel<S, P>);
    if constexpr (sizeof(S) == 2 || P <= 128)
        if (k.tiles[0] && k.tiles[1]) return go(kv_shared_tiles_kernel<S, P>);
    if (k.tiles[0] || k.tiles[1]) return hipErrorInvalidValue;   // (no plan has them)
    if constexpr (sizeof(S) == 2)
        if (k.solo) return go(kv_shared_solo_kernel<S, P>);
    return k.stream ? go(kv_shared_rows_kernel<S, P, true>) : go(kv_shared_rows_kernel<S, P, false>);
}
template <typename S> hipError_t launch_close(const Both<S> &both, uint32_t widest, uint32_t grid, hipStream_t s) {
    auto go = [&](auto kernel) {
        kernel<<<grid, 2 * kThreads, 0, s>>>(both);
        return hipGetLastError();
    };
    if (widest <= 32) return go(kv_shared_close_kernel<S, 32>);
    if (widest <= 64) return go(kv_shared_close_kernel<S, 64>);
    if (widest <= 96) return go(kv_shared_close_kernel<S, 96>);
    if (widest <= 128) return go(kv_shared_close_kernel<S, 128>);
    if constexpr (close_built(sizeof(S) == 4, 192))
        if (widest <= 192) return go(kv_shared_close_kernel<S, 192>);
    return hipErrorInvalidValue;   // (no plan has them)
}
template <typename S>
hipError_t launch(const Both<S> &both, uint32_t widest, uint32_t grid, const Kernels &k, hipStream_t s) {
    if (widest <= 32) return launch<S, 32>(both, grid, k, s);
    if (widest <= 64) return launch<S, 64>(both, grid, k, s);
    if (widest <= 96) return launch<S, 96>(both, grid, k, s);
    if (widest <= 128) return launch<S, 128>(both, grid, k, s);
    if (widest <= 192) return launch<S, 192>(both, grid, k, s);
    return launch<S, 256>(both, grid, k, s);
}

template <typename S>
hipError_t run(const View &prefix, const PrefixShape &ps, const View &c, const AttentionShape &sh, const void *query,
               void *output, void *workspace, hipStream_t s) {
    const SharedPlan p = plan_of(sizeof(S) == 4, prefix, ps, c, sh);
    const uint32_t group = sh.q_heads / c.heads;
    Both<S> both{};
    SharedArgs<S> &over = both.pass[0], &own = both.pass[1];
    own.q = static_cast<const S *>(query);
    own.out = static_cast<S *>(output);
    own.part_o = static_cast<float *>(workspace);
    own.part_ml = reinterpret_cast<f32x2 *>(static_cast<char *>(workspace) + p.o_bytes);
    own.rows = p.rows;
    own.scale2 = (double)sh.scale * kLog2e;
    if (p.close) {
        own.c = c;
        own.group = group;
        own.n = sh.n;
        own.parts = 1;
        own.row_groups = p.own.row_groups;
        over = own;
        over.c = prefix;
        own.causal = sh.causal;
        uint32_t on = 0, left = ps.members[0];
        for (own.first = 0; own.first < sh.batch; own.first += kBatchPerLaunch) {
            const uint32_t batch = sh.batch - own.first < kBatchPerLaunch ? sh.batch - own.first : kBatchPerLaunch;
            for (uint32_t b = 0; b < batch; ++b, --left) {
                while (left == 0) left = ps.members[++on];
                over.count.n[b] = on;
                own.count.n[b] = sh.counts ? sh.counts[own.first + b] : sh.n;
            }
            over.pairs = own.pairs = batch * c.heads;
            const hipError_t status = launch_close(both, widest_of(c), own.pairs * own.row_groups, s);
            if (status != hipSuccess) return status;
        }
        return hipSuccess;
    }
    over = own;
    over.c = prefix;
    over.group = 1;   // a group's rows are one head's rows there
    over.n = p.n;
    over.own_rows = group * sh.n;
    over.parts = p.prefix.parts;
    over.longest = ps.longest;
    over.row_groups = p.prefix.row_groups;
    own.c = c;
    own.group = group;
    own.n = sh.n;
    own.parts = p.own.parts;
    own.longest = sh.longest;
    own.row_groups = p.own.row_groups;
    own.causal = sh.causal;
    own.part_o += (size_t)p.prefix.parts * p.rows * c.vdim;
    own.part_ml += (size_t)p.prefix.parts * p.rows;
    const size_t held = (size_t)(ps.batch * (uint64_t)ps.longest + sh.batch * (uint64_t)sh.longest) * c.heads * (c.kp + c.vp);
    auto go = [&](uint32_t grid, bool tiles0, bool tiles1) {
        return launch(both, widest_of(c), grid, Kernels{{tiles0, tiles1}, p.own.solo, held > kStreamBytes}, s);
    };

    auto batch_from = [&](uint32_t first) { return sh.batch - first < kBatchPerLaunch ? sh.batch - first : kBatchPerLaunch; };
    auto take_counts = [&](uint32_t first) {
        for (uint32_t b = 0; b < batch_from(first); ++b) own.count.n[b] = sh.counts ? sh.counts[first + b] : sh.n;
    };
    take_counts(0);
    over.padded = padded(sh) ? sh.n : 0;
    if (p.counts_bytes != 0) {
        uint32_t *const counts = reinterpret_cast<uint32_t *>(static_cast<char *>(workspace) + p.o_bytes + p.ml_bytes);
        for (uint32_t first = 0; first < sh.batch; first += kBatchPerLaunch) {
            take_counts(first);
            kv_counts_kernel<<<1, kBatchPerLaunch, 0, s>>>(counts + first, batch_from(first), own.count);
            const hipError_t status = hipGetLastError();
            if (status != hipSuccess) return status;
        }
        over.counts = counts;
    }

    Cursor<S> of_prefix{prefix, p.prefix}, of_own{c, p.own};
    uint32_t sequence = 0;   // where the next group starts
    while (!of_prefix.done() || !of_own.done()) {
        both.first = 0;
        uint32_t grid = 0;
        if (!of_prefix.done()) {
            if (of_prefix.group == 0) {   // the next prefixes
                for (uint32_t b = 0; b < of_prefix.batch(); ++b) {
                    over.count.n[b] = sequence;
                    sequence += ps.members[of_prefix.first + b];
                }
                over.last = sequence;
            }
            both.first = grid = of_prefix.next(over);
        }
        if (grid != 0 && !p.together) {
            const hipError_t status = go(grid, p.prefix.tiles, p.prefix.tiles);
            if (status != hipSuccess) return status;
            both.first = grid = 0;
        }
        if (!of_own.done()) {
            take_counts(of_own.first);
            grid += of_own.next(own);
        }
        if (grid == 0) continue;
        const hipError_t status = go(grid, p.together ? p.prefix.tiles : p.own.tiles, p.own.tiles);
        if (status != hipSuccess) return status;
    }

    // the parts' join, for 256 sequences each
    const uint32_t parts = p.prefix.parts + p.own.parts;
    own.part_o = over.part_o;
    own.part_ml = over.part_ml;
    for (uint32_t first = 0; first < sh.batch; first += kBatchPerLaunch) {
        const uint32_t batch = batch_from(first);
        take_counts(first);
        const uint32_t per_sequence = sh.q_heads * sh.n;
        hipError_t status = hipSuccess;
        if (parts > 16 && p.rows <= kWideRows) {
            own.first = first;
            own.pairs = batch * c.heads;
            status = launch_fold<S>(own, parts, false, 0, true, s);
        } else {
            const uint32_t threads = (c.vdim + 3) / 4, most = join_rows(c.vdim), rows = batch * per_sequence;
            JoinArgs j{own.part_o, own.part_ml, p.rows, (size_t)first * per_sequence, parts, c.vdim, 0, 0,
                       make_fast_div(threads), sh.counts != nullptr, make_fast_div(sh.n), make_fast_div(per_sequence),
                       own.count};
            for (; j.from < rows && status == hipSuccess; j.from += j.all) {
                j.all = rows - j.from < most ? rows - j.from : most;
                auto join = [&](auto kernel) {
                    kernel<<<(j.all * threads + kThreads - 1) / kThreads, kThreads, 0, s>>>(static_cast<S *>(output), j);
                };
                if (parts <= 2) join(kv_join_kernel<S, 2>);
                else if (parts <= 4) join(kv_join_kernel<S, 4>);
                else join(kv_join_kernel<S, 8>);
                status = hipGetLastError();
            }
        }
        if (status != hipSuccess) return status;
    }
    return hipSuccess;
}

}  // namespace

size_t attention_shared_workspace(bool f32, const View &prefix, const PrefixShape &p, const View &c,
                                  const AttentionShape &a) {
    const SharedPlan plan = plan_of(f32, prefix, p, c, a);
    return plan.o_bytes + plan.ml_bytes + plan.counts_bytes;
}

hipError_t attention_shared(bool f32, const View &prefix, const PrefixShape &p, const View &c, const AttentionShape &a,
                            const void *query, void *output, void *workspace, hipStream_t s) {
    return f32 ? run<float>(prefix, p, c, a, query, output, workspace, s)
               : run<_Float16>(prefix, p, c, a, query, output, workspace, s);
}

}  // namespace kv
}  // namespace icsdk
