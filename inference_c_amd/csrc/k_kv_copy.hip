// Sequences of the 8-bit key/value cache (kv.hpp) moved as they are held: into
// another cache or another place of the same one, and in place among the beams of a
// group. Codes, scales and marks are copied, nothing is held anew.
//
// Of a (sequence, kv head) there are the codes of the whole blocks' keys and values,
// each one run of memory, the blocks' Meta, and with a partial block its f16 rows.
// What lies behind a sequence's tokens is not copied: it is codes or finite f16 of
// earlier tokens, which nothing uses.
#include "kern_common.hpp"
#include "kv.hpp"

namespace icsdk {
namespace kv {
namespace {

constexpr uint32_t kThreads = 256;

// What a (sequence, head) holds of each kind, in bytes (whole 16s).
struct Held {
    size_t k, v;           // codes of whole blocks
    uint32_t meta, kt, vt;
    __device__ Held(const View &c, uint32_t length) {
        const uint32_t whole = length / kTokens, open = length % kTokens;
        k = (size_t)whole * kTokens * c.kp;
        v = (size_t)whole * kTokens * c.vp;
        meta = (whole + (open ? 1 : 0)) * (uint32_t)sizeof(Meta);
        kt = open * c.kp * 2;   // rows by token
        vt = open ? kTokens * c.vp * 2 : 0;
    }
};

// ---- copies ----------------------------------------------------------------------

struct CopyArgs {
    View from, to;
    uint32_t first, k_pieces, v_pieces;
    Counts source;   // of the target's sequences first ..: the one copied (kKeep: none)
};

constexpr uint32_t kPer = 4, kPiece = kThreads * kPer * 16;   // bytes of a workgroup

__device__ inline void copy_run(const void *from, void *to, size_t bytes) {
    for (size_t at = threadIdx.x * 16; at < bytes; at += kThreads * 16)
        *reinterpret_cast<u32x4 *>(static_cast<char *>(to) + at) =
            *reinterpret_cast<const u32x4 *>(static_cast<const char *>(from) + at);
}

// A workgroup: 16 KB of one (sequence, head)'s codes; the last one of each the rest.
// Bound by memory: 4 sequences of 2000 tokens of 8 heads of 128 + 128 into 32 (131 MB
// written, the sources being found in the caches) 24 us, 5.4 TB/s. Codes past what the caches
// hold to the next call are written as a stream (kStream): that copy then takes 34 us, but
// its read 87 for 104, both 115 for 129; 64 MB 90, as a stream 92.
constexpr size_t kStreamBytes = size_t{96} << 20;

template <bool kStream>
__global__ __launch_bounds__(kThreads) void kv_copy_kernel(CopyArgs a) {
    const View &f = a.from, &c = a.to;
    const uint32_t piece = blockIdx.x, h = blockIdx.y, b = a.first + blockIdx.z, s = a.source.n[blockIdx.z];
    if (s == kKeep) return;
    const uint32_t length = f.length[s];
    const Held held(f, length);
    const size_t from = (size_t)s * f.heads + h, to = (size_t)b * c.heads + h;
    if (piece == a.k_pieces + a.v_pieces) {
        if (h == 0 && threadIdx.x == 0) c.length[b] = length;
        copy_run(f.meta + from * f.blocks, c.meta + to * c.blocks, held.meta);
        copy_run(f.kt + from * kTokens * f.kp, c.kt + to * kTokens * c.kp, held.kt);
        copy_run(f.vt + from * kTokens * f.vp, c.vt + to * kTokens * c.vp, held.vt);
        return;
    }
    const bool keys = piece < a.k_pieces;
    const uint32_t pitch = keys ? f.kp : f.vp;
    const size_t bytes = keys ? held.k : held.v, first = (size_t)(keys ? piece : piece - a.k_pieces) * kPiece;
    const uint8_t *const src = (keys ? f.k : f.v) + from * f.blocks * kTokens * pitch;
    uint8_t *const dst = (keys ? c.k : c.v) + to * c.blocks * kTokens * pitch;
    u32x4 x[kPer];
#pragma unroll
    for (uint32_t u = 0; u < kPer; ++u) {
        const size_t at = first + (u * kThreads + threadIdx.x) * 16;
        if (at < bytes) x[u] = *reinterpret_cast<const u32x4 *>(src + at);
    }
#pragma unroll
    for (uint32_t u = 0; u < kPer; ++u) {
        const size_t at = first + (u * kThreads + threadIdx.x) * 16;
        if (at >= bytes) continue;
        if constexpr (kStream) __builtin_nontemporal_store(x[u], reinterpret_cast<u32x4 *>(dst + at));
        else *reinterpret_cast<u32x4 *>(dst + at) = x[u];
    }
}

// ---- beams in place ----------------------------------------------------------------

struct ReorderArgs {
    View c;
    const uint32_t *parents;   // [groups][beams]
    uint32_t beams, k_pieces, v_pieces;
};

// Beams' cache memory in place: a thread has the same 16 bytes of every sequence of
// its group, reads those that replace others, and then writes them, so no copy needs a
// place in between. kBeams: at least the group's. Bound by memory, read and written in
// turn: 16 groups of 8 x 850 tokens on average, 8 heads of 128 + 128, of which half move
// (116 MB read, as often as it goes to several, and written) 50 us, 4.7 TB/s of that. A
// workgroup does kColumns of its 16 bytes' columns, kAhead of them at once. Measured (us,
// 16 x 8 x 850 and 4 groups of 16 x 1000): one column 57 and 56, two one after another 54
// and 59, four 53 and 49, four by twos 50 and 50, eight by twos 53 and 55; 32 groups of 4 x
// 100 tokens 10.5 one by one, 8.7 by twos. More than 16 beams run short of scalar registers
// for their parents, and 64 of vector registers too (a wave per SIMD, and spills): 128
// sequences of 1000 tokens, of which 114 to 125 move, in groups of 8 78 us, of 16 103, of 32
// 119 (4.3 TB/s), of 64 266 (1.9 TB/s).
constexpr uint32_t kColumns = 4, kColumn = kThreads * 16;
template <uint32_t kBeams>
__global__ __launch_bounds__(kThreads) void kv_reorder_kernel(ReorderArgs a) {
    const View &c = a.c;
    const uint32_t piece = blockIdx.x, h = blockIdx.y, first = blockIdx.z * a.beams;
    const Held held(c, c.length[first]);
    uint32_t parent[kBeams];
#pragma unroll
    for (uint32_t i = 0; i < kBeams; ++i) {
        const uint32_t p = i < a.beams ? a.parents[first + i] : i;
        parent[i] = p < a.beams ? p : i;   // (an index past the group: the sequence stays)
    }
    // the thread's next kAhead columns of one kind: `pitch` bytes from one sequence to the next
    constexpr uint32_t kAhead = kBeams <= 16 ? 2 : 1;
    auto column = [&](void *memory, size_t pitch, size_t at, size_t bytes) {
        char *const base = static_cast<char *>(memory) + ((size_t)first * c.heads + h) * pitch;
        const size_t next = c.heads * pitch;
        u32x4 x[kAhead][kBeams];
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u)
#pragma unroll
            for (uint32_t i = 0; i < kBeams; ++i)
                if (parent[i] != i && at + u * kColumn < bytes)
                    x[u][i] = *reinterpret_cast<const u32x4 *>(base + at + u * kColumn + parent[i] * next);
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u)
#pragma unroll
            for (uint32_t i = 0; i < kBeams; ++i)
                if (parent[i] != i && at + u * kColumn < bytes)
                    *reinterpret_cast<u32x4 *>(base + at + u * kColumn + i * next) = x[u][i];
    };
    const size_t lane = threadIdx.x * 16;
    if (piece < a.k_pieces) {
        for (size_t u = 0; u < kColumns; u += kAhead)
            column(c.k, (size_t)c.blocks * kTokens * c.kp, (piece * kColumns + u) * kColumn + lane, held.k);
    } else if (piece < a.k_pieces + a.v_pieces) {
        for (size_t u = 0; u < kColumns; u += kAhead)
            column(c.v, (size_t)c.blocks * kTokens * c.vp, ((piece - a.k_pieces) * kColumns + u) * kColumn + lane, held.v);
    } else {
        for (size_t at = lane; at < held.meta; at += kAhead * kColumn) column(c.meta, (size_t)c.blocks * sizeof(Meta), at, held.meta);
        for (size_t at = lane; at < held.kt; at += kAhead * kColumn) column(c.kt, (size_t)kTokens * c.kp * 2, at, held.kt);
        for (size_t at = lane; at < held.vt; at += kAhead * kColumn) column(c.vt, (size_t)kTokens * c.vp * 2, at, held.vt);
    }
}

uint32_t pieces_of(uint32_t longest, uint32_t pitch, uint32_t piece) {
    return (uint32_t)(((size_t)(longest / kTokens) * kTokens * pitch + piece - 1) / piece);
}

}  // namespace

hipError_t copy(const View &from, const View &to, uint32_t first, uint32_t batch, const Counts &source, uint32_t longest,
                size_t tokens, hipStream_t s) {
    const CopyArgs a{from, to, first, pieces_of(longest, from.kp, kPiece), pieces_of(longest, from.vp, kPiece), source};
    const dim3 grid(a.k_pieces + a.v_pieces + 1, from.heads, batch);
    if (tokens * from.heads * (from.kp + from.vp) > kStreamBytes) kv_copy_kernel<true><<<grid, kThreads, 0, s>>>(a);
    else kv_copy_kernel<false><<<grid, kThreads, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t reorder(const View &c, uint32_t groups, uint32_t beams, const uint32_t *parents, uint32_t longest,
                   hipStream_t s) {
    const ReorderArgs a{c, parents, beams, pieces_of(longest, c.kp, kColumns * kColumn),
                        pieces_of(longest, c.vp, kColumns * kColumn)};
    const dim3 grid(a.k_pieces + a.v_pieces + 1, c.heads, groups);
    if (beams <= 4) kv_reorder_kernel<4><<<grid, kThreads, 0, s>>>(a);
    else if (beams <= 8) kv_reorder_kernel<8><<<grid, kThreads, 0, s>>>(a);
    else if (beams <= 16) kv_reorder_kernel<16><<<grid, kThreads, 0, s>>>(a);
    else if (beams <= 32) kv_reorder_kernel<32><<<grid, kThreads, 0, s>>>(a);
    else kv_reorder_kernel<64><<<grid, kThreads, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace kv
}  // namespace icsdk
