// One step's choice of a beam search over beams and vocabulary: of every group the
// `keep` candidates (beam, token) of largest score[b] + x[b, v] - log sum exp x[b, :].
//
// Within a beam the order is that of the logits, so a beam's own `keep` largest
// logits are all that can be chosen of it. beam_scan_kernel reads each row once, a wave
// per part of it, and leaves of each part the running sum of exp(x - max) and its
// largest logits in order; beam_pick_kernel, a workgroup per group, joins the sums of a
// row and takes the best of all parts' candidates by their scores.
//
// Scores are f64 from exact logits; of the log sums only the exponentials, and the sums of
// 16 of them, are f32. An exponential of t = x - max is off by at most (2 |t| + 2) 2^-24 of
// itself (t and its exponent rounded, and the last place), a sum of 16 by four roundings
// more, so a log sum by (2 log vocab + 6) 2^-24 at the very most, where all terms round the
// same way; 4e-8 is the largest seen over plateaus, steps and rows far from 0. Two beams'
// candidates change places only where their scores are that close.
#include "kernels.hpp"
#include "kern_common.hpp"

namespace icsdk {
namespace k {
namespace {

constexpr uint32_t kMaxKeep = kBeamMaxKeep;   // a lane each at the end
static_assert(kMaxKeep == kWave);
constexpr uint32_t kTokenBits = 26;
// Kept candidates from which bounds are taken of more than a lane's one: of four sets of
// its logits here, of several pieces of a list there. Measured (us, with and without, the
// call): 64 x 16 beams x 8000 logits, 64 kept 42 and 52; 2 x 16 x 128256, 32 kept 19.6 and
// 20.2; 16 x 8 x 32003, 16 kept 17 and 14.
constexpr uint32_t kManyKept = 24;
constexpr uint32_t kMaxParts = 128;           // of a row

struct Entry {
    float logit;
    uint32_t token;
};
struct PartSum {
    double sum;   // of exp(x - max); NaN where a logit is
    float max;
    uint32_t pad;
};

// Keys in the order of the floats they stand for (+0 and -0 alike; no NaN).
__device__ inline uint32_t key_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ inline float from_key(uint32_t k) {
    return __builtin_bit_cast(float, k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ inline uint64_t key_of(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);
    return b ^ ((uint64_t)((int64_t)b >> 63) | uint64_t{1} << 63);
}
__device__ inline double from_key(uint64_t k) {
    return __builtin_bit_cast(double, k ^ (k >> 63 ? uint64_t{1} << 63 : ~uint64_t{0}));
}

// Orders a wave's own LDS accesses (which the hardware does by itself) for the compiler.
__device__ inline void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

__device__ inline uint32_t lanes(bool flag) { return (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(flag)); }
__device__ inline uint32_t lanes_below(bool flag, uint32_t lane) {
    return (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(flag) & ((uint64_t{1} << lane) - 1));
}

__device__ inline uint32_t wave_or(uint32_t v) {
    int x = (int)v;
    x |= dpp_i32<kQuadSwap1>(0, x);
    x |= dpp_i32<kQuadSwap2>(0, x);
    x |= dpp_i32<kRowHalfMirror>(0, x);
    x |= dpp_i32<kRowMirror>(0, x);
    x |= dpp_i32<kRowBcast15, 0xa>(0, x);
    x |= dpp_i32<kRowBcast31, 0xc>(0, x);
    return (uint32_t)__builtin_amdgcn_readlane(x, kWave - 1);
}
__device__ inline uint64_t wave_or(uint64_t v) {
    return (uint64_t)wave_or((uint32_t)(v >> 32)) << 32 | wave_or((uint32_t)v);
}
__device__ inline uint32_t of_lane(uint32_t v, uint32_t lane) {
    return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)lane);
}
__device__ inline uint64_t of_lane(uint64_t v, uint32_t lane) {
    return (uint64_t)of_lane((uint32_t)(v >> 32), lane) << 32 | of_lane((uint32_t)v, lane);
}

// The want-th largest of the wave's keys (kSlots per lane, the first `slots` looked at;
// a key of 0 is none, and there are `want` others), or a smaller number above which there
// are exactly `want`: after the bits that all keys have in common, from the highest on, a
// bit is set where at least `want` keys reach it.
template <typename K, uint32_t kSlots>
__device__ inline K largest(const K (&key)[kSlots], uint32_t slots, uint32_t want) {
    // some key, and the bits in which others differ from it
    K some = 0, differ = 0;
#pragma unroll
    for (uint32_t i = 0; i < kSlots; ++i) some = key[i] != 0 ? key[i] : some;
    some = of_lane(some, (uint32_t)__builtin_ctzll(__builtin_amdgcn_ballot_w64(some != 0)));
#pragma unroll
    for (uint32_t i = 0; i < kSlots; ++i) differ |= key[i] != 0 ? key[i] ^ some : 0;
    differ = wave_or(differ);
    if (differ == 0) return some;
    const uint32_t top = 63 - (uint32_t)__builtin_clzll((uint64_t)differ);
    K least = some >> top >> 1 << top << 1;
    for (K bit = K{1} << top; bit != 0; bit >>= 1) {
        const K at = least | bit;
        uint32_t n = 0;
#pragma unroll
        for (uint32_t i = 0; i < kSlots; ++i)
            if (i < slots) n += lanes(key[i] >= at);
        if (n >= want) least = at;
        if (n == want) break;
    }
    return least;
}

// ---- of each part of a row ---------------------------------------------------------

struct ScanArgs {
    Entry *entries;   // [rows][parts][pitch]
    PartSum *sums;    // [rows][parts]
    uint32_t pitch;
};

// exp(t) for t <= 0 (and NaN): log2 e in two pieces, so that the exponent is off by
// one rounding alone.
__device__ inline float exp_below(float t) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(t, 1.4426950216293335f, t * 1.925963033500001e-8f));
}
// Pairwise: no term is rounded more than log2 N times.
template <uint32_t N> __device__ inline float sum_of(const float *x) {
    if constexpr (N == 1) return x[0];
    else return sum_of<N / 2>(x) + sum_of<N / 2>(x + N / 2);
}

typedef uint32_t Vector __attribute__((ext_vector_type(4), aligned(2)));   // 16 bytes of logits from any on

constexpr uint32_t kLogits = 16, kTile = kLogits * kWave;   // of a lane and of a wave, at a time
constexpr uint32_t kTiles = 16;                             // between two looks for candidates
constexpr uint32_t kSets = 4;                               // of a lane's logits, each with its largest
constexpr uint32_t kFewLanes = 8;                           // of several hits each, which a cut or two takes
// Entries of a wave, and above how many they are cut to the best.
constexpr uint32_t kSpare = 2 * kMaxKeep, kHeld = kSpare + kWave, kSlots = kHeld / kWave;

// A wave has a part of a row. It sums up to 16 tiles, leaving of each every lane's
// largest logit in LDS; the largest ones so far of `keep` lanes, or of sets of a lane's
// logits, reach a bound, and only where a tile's lane reaches it are logits looked at
// again, one lane for each such place. 256 rows of 128256 f32 (131 MB) 27 us, 4.8 TB/s,
// where a copy of 1 GiB reaches 5.1; f16 19 us, bound by vector instructions (a quarter of
// them the exponentials, at a quarter of the rate). One tile each (16 x 8 x 32003 f16) 8.5
// us: the chain of load, sum, bound, sort and store, 4 us of them for a wave alone. Measured
// and left: candidates looked for in every tile (f32 31 us, f16 25), workgroups of four
// waves (the same). Logits that equal the bound are candidates too, the first `keep` of
// them: all but three of 128256 at the type's lowest number 35 us (f32) and 26 (f16), where
// each of them looked at took ten times as long.
template <typename T>
__global__ __launch_bounds__(kWave) void beam_scan_kernel(const T *x, const uint32_t *ended, uint32_t vocab, uint32_t per_part,
                                                          uint32_t keep, ScanArgs a) {
    constexpr uint32_t E = Vec16<T>::N, U = kLogits / E, kStep = U * kWave;   // kStep: a tile's vectors
    __shared__ uint64_t held[kHeld];   // a logit's key, then the earlier token as the larger one
    __shared__ float largests[kTiles * kWave];
    __shared__ uint16_t places[kTiles * kWave];
    const uint32_t lane = threadIdx.x, row = blockIdx.x, part = blockIdx.y;
    const float neg_inf = -__builtin_inff(), inf = __builtin_inff();
    // tokens lie in vectors from the row's first on, wherever in memory that is (a load
    // needs no alignment), so that rows alike have sums alike
    x += (uint64_t)row * vocab;
    const uint32_t vectors = (vocab + E - 1) / E;
    const uint32_t begin = min(part * per_part, vectors), end = min(begin + per_part, vectors);
    // a place: vectors at, at + 64, ..., 16 logits (of vectors that are not whole nothing)
    auto load = [&](Vector (&to)[U], uint32_t at) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t v = at + u * kWave;
            if (v < end && (v + 1) * E <= vocab) to[u] = __builtin_nontemporal_load(reinterpret_cast<const Vector *>(x + v * E));
        }
    };
    Vector ahead[U];
    load(ahead, begin + lane);
    if (ended != nullptr && ended[row] != 0) return;

    // m: the lane's largest logit; base: the wave's; s: the lane's sum of exp(x - base)
    float now[kLogits], m = neg_inf, base = neg_inf, of_set[kSets] = {neg_inf, neg_inf, neg_inf, neg_inf};
    double s = 0.0;
    float low = -3.4028234663852886e38f;   // entries are at least this (never -inf or NaN)
    uint32_t n = 0;
    // Places of earlier tiles with a logit of at least `counted`: once there are `keep`, one
    // that equals it is behind them all.
    uint32_t sure = 0;
    float counted = low;
    auto take = [&](const Vector (&from)[U], uint32_t at, bool whole) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            struct Elements {
                T v[E];
            };
            const Elements w = __builtin_bit_cast(Elements, from[u]);
#pragma unroll
            for (uint32_t e = 0; e < E; ++e) now[u * E + e] = (float)w.v[e];
        }
        if (whole) return;
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t v = at + u * kWave;
            if (v < end && (v + 1) * E <= vocab) continue;
#pragma unroll
            for (uint32_t e = 0; e < E; ++e)
                now[u * E + e] = v < end && v * E + e < vocab ? (float)x[v * E + e] : neg_inf;
        }
    };
    // Of the wave's hits that equal the bound, for each of a place's vectors, the first
    // `keep` (places are in the order of their tokens).
    auto first_equal = [&](uint32_t hits) {
        uint32_t equal = 0;
#pragma unroll
        for (uint32_t j = 0; j < kLogits; ++j) equal |= now[j] == low ? 1u << j : 0u;
        equal &= hits;
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t its = (uint32_t)__builtin_popcount(equal >> u * E & ((1u << E) - 1));
            uint32_t before = 0;
#pragma unroll
            for (uint32_t bit = 0; 1u << bit <= E; ++bit) before += lanes_below((its >> bit & 1) != 0, lane) << bit;
#pragma unroll
            for (uint32_t j = u * E; j < (u + 1) * E; ++j) {
                if (before >= keep) hits &= ~(equal & 1u << j);
                before += equal >> j & 1;
            }
        }
        return hits;
    };
    // cuts the entries to the `keep` best
    auto cut = [&] {
        wave_order();
        uint64_t key[kSlots];
#pragma unroll
        for (uint32_t i = 0; i < kSlots; ++i) key[i] = i * kWave + lane < n ? held[i * kWave + lane] : 0;
        const uint64_t bound = largest(key, kSlots, keep);
        wave_order();
        n = 0;
        uint32_t lowest = 0xffffffffu;
#pragma unroll
        for (uint32_t i = 0; i < kSlots; ++i) {
            const bool stays = key[i] >= bound;
            const uint32_t to = n + lanes_below(stays, lane);
            if (stays) {
                held[to] = key[i];
                lowest = min(lowest, (uint32_t)(key[i] >> 32));
            }
            n += lanes(stays);
        }
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) lowest = min(lowest, (uint32_t)__shfl_xor((int)lowest, d, kWave));
        low = fmaxf(low, from_key(lowest));
    };
    for (uint32_t from = begin; from < end; from += kTiles * kStep) {
        const uint32_t to = min(from + kTiles * kStep, end), tiles = (to - from + kStep - 1) / kStep;
        for (uint32_t t = 0; t < tiles; ++t) {
            const uint32_t at = from + t * kStep;
            take(ahead, at + lane, at + kStep <= end && (at + kStep) * E <= vocab);
            if (at + kStep < end) load(ahead, at + kStep + lane);
            float top = neg_inf;
#pragma unroll
            for (uint32_t k = 0; k < kSets; ++k) {
                float of = now[k];
#pragma unroll
                for (uint32_t j = k + kSets; j < kLogits; j += kSets) of = fmaxf(of, now[j]);
                of_set[k] = fmaxf(of_set[k], of);
                top = fmaxf(top, of);
            }
            m = fmaxf(m, top);
            if (wave_any(m > base)) {
                const float next = wave_max(m);
                if (base != neg_inf) s *= exp((double)base - (double)next);
                base = next;
            }
            // A tile's terms in f32, tiles in f64: in one f32 the terms of flat rows, which
            // all round the same way, left sums of 32003 off by 1e-5.
            float term[kLogits];
            if (base == inf) {
#pragma unroll
                for (uint32_t j = 0; j < kLogits; ++j) term[j] = now[j] == inf ? 1.0f : now[j] != now[j] ? now[j] : 0.0f;
            } else {
                const float from_base = base == neg_inf ? 0.0f : base;
#pragma unroll
                for (uint32_t j = 0; j < kLogits; ++j) term[j] = exp_below(now[j] - from_base);
            }
            s += (double)sum_of<kLogits>(term);
            largests[t * kWave + lane] = top;
        }
        // the bound, and the places that reach it
        if (keep < kManyKept) {
            const uint32_t ms[1] = {m == neg_inf ? 0 : key_of(m)};
            if (lanes(ms[0] != 0) >= keep) low = fmaxf(low, from_key(largest(ms, 1, keep)));
        } else {
            uint32_t ms[kSets], there = 0;
#pragma unroll
            for (uint32_t k = 0; k < kSets; ++k) {
                ms[k] = of_set[k] == neg_inf ? 0 : key_of(of_set[k]);
                there += lanes(ms[k] != 0);
            }
            if (there >= keep) low = fmaxf(low, from_key(largest(ms, kSets, keep)));
        }
        const bool one = tiles == 1;   // (its logits are still in their lanes)
        uint32_t all = one ? kWave : 0;
        if (!one) {
            if (counted != low) {
                counted = low;
                sure = 0;
            }
            const float above = from_key(key_of(low) + 1);
            wave_order();
            for (uint32_t t = 0; t < tiles; ++t) {
                const bool reaches = largests[t * kWave + lane] >= (sure < keep ? low : above);
                const uint32_t i = all + lanes_below(reaches, lane);
                if (reaches) places[i] = (uint16_t)(t * kWave + lane);
                all += lanes(reaches);
                sure += lanes(reaches);
            }
            wave_order();
        }
        for (uint32_t i = 0; i < all; i += kWave) {
            uint32_t at = from + lane;
            if (!one) {
                const uint32_t place = places[min(i + lane, all - 1)];
                at = from + place / kWave * kStep + place % kWave;
                Vector again[U];
                load(again, at);
                take(again, at, false);
            }
            uint32_t hits = 0;   // a lane's
#pragma unroll
            for (uint32_t j = 0; j < kLogits; ++j) hits |= now[j] >= low ? 1u << j : 0u;
            if (i + lane >= all) hits = 0;
            if (lanes(__builtin_popcount(hits) > 2) > kFewLanes) hits = first_equal(hits);
            while (wave_any(hits != 0)) {
                const uint32_t j = (uint32_t)__builtin_ctz(hits | 1u << (kLogits - 1));
                // now[j], by the bits of j (chosen as conditions, the compiler makes a chain of
                // 16 comparisons of each)
                uint32_t pick[kLogits];
#pragma unroll
                for (uint32_t k = 0; k < kLogits; ++k) pick[k] = __builtin_bit_cast(uint32_t, now[k]);
#pragma unroll
                for (uint32_t half = kLogits / 2; half > 0; half /= 2) {
                    const uint32_t upper = j & half ? 0xffffffffu : 0;
#pragma unroll
                    for (uint32_t k = 0; k < half; ++k) pick[k] = (pick[k + half] & upper) | (pick[k] & ~upper);
                }
                const float y = __builtin_bit_cast(float, pick[0]);
                const bool passes = hits != 0 && y >= low;
                const uint32_t slot = n + lanes_below(passes, lane);
                if (passes) held[slot] = (uint64_t)key_of(y) << 32 | ~((at + j / E * kWave) * E + j % E);
                n += lanes(passes);
                hits &= hits - 1;
                if (n > kSpare) cut();
            }
        }
    }
    if (n > kWave) cut();
    // in order, each entry behind those that are larger
    wave_order();
    const uint64_t mine = lane < n ? held[lane] : 0;
    uint32_t rank = 0;
    for (uint32_t i = 0; i < n; ++i) rank += of_lane(mine, i) > mine;
    const size_t list = (size_t)row * gridDim.y + part;
    if (lane >= n) rank = lane;
    if (rank < a.pitch)
        a.entries[list * a.pitch + rank] = lane < n ? Entry{from_key((uint32_t)(mine >> 32)), ~(uint32_t)mine} : Entry{neg_inf, 0};
    const double sum = wave_sum_f64(s);
    if (lane == 0) a.sums[list] = PartSum{sum, base, 0};
}

// ---- of a group ----------------------------------------------------------------------

struct PickArgs {
    uint32_t *parents, *tokens;
    float *new_scores;
    uint32_t *new_ended;
    uint32_t end_token;
};

constexpr uint32_t kPickWaves = 8;
constexpr uint32_t kAhead = 4;   // entries of a list asked for at once
// Entries of a wave, and above how many they are cut to the best.
constexpr uint32_t kPickSpare = 2 * kMaxKeep, kPickHeld = kPickSpare + kAhead * kWave, kPickSlots = kPickHeld / kWave;

// A candidate: its score, and what goes before where scores are equal (the lower
// beam, the larger logit, the lower token), both as keys.
struct Candidate {
    uint64_t score, rest;
};
__device__ inline Candidate candidate(double score, uint32_t beam, float logit, uint32_t token) {
    return Candidate{key_of(score), (uint64_t)(kBeamMax - 1 - beam) << 58 | (uint64_t)key_of(logit) << kTokenBits |
                                        ((1u << kTokenBits) - 1 - token)};
}

// Bound by its chain: 13000 cycles (4.5 to 6 us) for a group alone, of which 2500 are the
// first loads and the f64 exponentials and logarithms, 2800 scores and bound, 1500 the
// candidates, 2500 their order. (Ordered by one wave in LDS, and cut by each before, 5.9 to
// 11 us.)
__global__ __launch_bounds__(kPickWaves *kWave) void beam_pick_kernel(const Entry *entries, const PartSum *sums,
                                                                     const float *scores, const uint32_t *ended,
                                                                     uint32_t beams, uint32_t parts, uint32_t keep,
                                                                     uint32_t pitch, PickArgs a) {
    __shared__ Candidate held[kPickWaves][kPickHeld];
    __shared__ uint32_t count[kPickWaves];
    __shared__ uint64_t bound[2][kPickWaves];
    __shared__ uint32_t evenly[kPickWaves];
    __shared__ double log_sum[kBeamMax];   // of a beam; NaN: it has no candidates
    __shared__ float most[kBeamMax], score[kBeamMax];
    __shared__ uint32_t over[kBeamMax], ranks[kWave];
    const uint32_t lane = threadIdx.x % kWave, wave = (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t group = blockIdx.x, first = group * beams, lists = beams * parts;
    const float neg_inf = -__builtin_inff();
    // A lane has a piece of four of a list's entries, the first pieces of every list going
    // to the first lanes; those and the first beams' sums are asked for at once (of a beam
    // that has ended whatever is there, not used).
    const uint32_t pieces = pitch / kAhead, place = wave * kWave + lane;
    uint32_t span = 1, first_piece = 0, list = min(place, lists - 1);   // span: pieces of a list at a time
    if (keep >= kManyKept) {
        span = min(pieces, kPickWaves * kWave / lists);
        first_piece = place / lists;
        list = place - first_piece * lists;
    }
    const u32x4 *const mine_at = reinterpret_cast<const u32x4 *>(entries + ((size_t)first * parts + list) * pitch);
    u32x4 w[kAhead / 2];
    auto load = [&](uint32_t piece) {
#pragma unroll
        for (uint32_t i = 0; i < kAhead / 2; ++i) w[i] = mine_at[min(piece, pieces - 1) * (kAhead / 2) + i];
    };
    load(first_piece);
    const uint32_t beam = list / parts;
    for (uint32_t b = wave; b < beams; b += kPickWaves) {
        const PartSum *const of = sums + (size_t)(first + b) * parts;
        const PartSum one = of[min(lane, parts - 1)];
        const float sc = scores[first + b];
        const bool is_over = ended != nullptr && ended[first + b] != 0;
        float top = one.max;
        for (uint32_t p = lane + kWave; p < parts; p += kWave) top = fmaxf(top, of[p].max);
        top = wave_max(top);
        auto part = [&](const PartSum &x) { return x.sum * (x.max == top ? 1.0 : exp((double)x.max - (double)top)); };
        double sum = lane < parts ? part(one) : 0.0;
        for (uint32_t p = lane + kWave; p < parts; p += kWave) sum += part(of[p]);
        sum = log(wave_sum_f64(sum));
        if (lane == 0) {
            log_sum[b] = sum;
            most[b] = top;
            score[b] = sc;
            over[b] = is_over ? 1 : 0;
        }
    }
    __syncthreads();
    Candidate *const mine = held[wave];
    uint32_t n = 0;
    uint64_t least = 0;   // `keep` candidates reach it
    // cuts the wave's candidates to the `keep` best
    auto cut = [&] {
        wave_order();
        uint64_t sc[kPickSlots], rest[kPickSlots];
        const uint32_t slots = (n + kWave - 1) / kWave;
#pragma unroll
        for (uint32_t i = 0; i < kPickSlots; ++i) {
            const uint32_t at = i * kWave + lane;
            sc[i] = rest[i] = 0;
            if (at < n) {
                sc[i] = mine[at].score;
                rest[i] = mine[at].rest;
            }
        }
        const uint64_t to_reach = largest(sc, slots, keep);
        uint32_t above = 0, same = 0;
#pragma unroll
        for (uint32_t i = 0; i < kPickSlots; ++i) {
            above += lanes(sc[i] > to_reach);
            same += lanes(sc[i] == to_reach && sc[i] != 0);
        }
        uint64_t first_rest = 0;
        if (above + same > keep) {
            uint64_t of[kPickSlots];
#pragma unroll
            for (uint32_t i = 0; i < kPickSlots; ++i) of[i] = sc[i] == to_reach ? rest[i] : 0;
            first_rest = largest(of, slots, keep - above);
        }
        wave_order();
        uint32_t to = 0;
        uint64_t lowest = ~uint64_t{0};
#pragma unroll
        for (uint32_t i = 0; i < kPickSlots; ++i) {
            const bool stays = sc[i] != 0 && (sc[i] > to_reach || (sc[i] == to_reach && rest[i] >= first_rest));
            const uint32_t at = to + lanes_below(stays, lane);
            if (stays) {
                mine[at] = Candidate{sc[i], rest[i]};
                lowest = sc[i] < lowest ? sc[i] : lowest;
            }
            to += lanes(stays);
        }
        n = to;
        wave_order();
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) {
            const uint64_t other = (uint64_t)__shfl_xor((unsigned long long)lowest, d, kWave);
            lowest = other < lowest ? other : lowest;
        }
        least = lowest > least ? lowest : least;   // (there were more than `keep`)
    };
    auto add = [&](bool passes, const Candidate &c) {
        const uint32_t at = n + lanes_below(passes, lane);
        if (passes) mine[at] = c;
        n += lanes(passes);
    };

    // a list, which is in order of its logits, is done with its first candidate that is
    // not among the best so far
    const double sc = (double)score[beam], sum = log_sum[beam];
    const float top = most[beam];
    bool going = place < lists * span && over[beam] == 0;
    for (uint32_t piece = first_piece, past = 0; past < keep; piece += span, past += span * kAhead) {
        if (past != 0) {
            if (!wave_any(going)) break;
            load(piece);
        }
#pragma unroll
        for (uint32_t e = 0; e < kAhead; ++e) {
            const uint32_t bits = w[e / 2][e % 2 * 2], token = w[e / 2][e % 2 * 2 + 1];
            const float x = __builtin_bit_cast(float, bits);
            const double to_top = x == top ? 0.0 : (double)x - (double)top;
            const double s = sc + (to_top - sum);
            going = going && piece * kAhead + e < keep && x > neg_inf && s > -__builtin_inf();
            const Candidate c = candidate(s, beam, x, token);
            if (e == 0 && past == 0) {
                // What `keep` pieces' first candidates reach is a bound: the keep-th of a
                // wave's, the largest of all waves, or an even share of `keep` in every wave
                // that has any, the smallest of all. (By the keys' upper halves.)
                const uint32_t heads[1] = {going ? (uint32_t)(c.score >> 32) : 0}, there = lanes(going);
                const uint32_t waves = (lists * span + kWave - 1) / kWave, share = (keep + waves - 1) / waves;
                const uint32_t reach = there >= keep ? largest(heads, 1, keep) : 0;
                const uint32_t even = waves > 1 && there >= share ? largest(heads, 1, share) : 0;
                if (lane == 0) {
                    bound[0][wave] = (uint64_t)reach << 32;
                    evenly[wave] = even;
                }
                __syncthreads();
                uint32_t lowest = 0xffffffffu;
                for (uint32_t i = 0; i < waves; ++i) {
                    least = bound[0][i] > least ? bound[0][i] : least;
                    lowest = min(lowest, evenly[i]);
                }
                least = (uint64_t)lowest << 32 > least ? (uint64_t)lowest << 32 : least;
            }
            going = going && c.score >= least;
            add(going, c);
        }
        if (n > kPickSpare) cut();
    }
    if (wave == 0 && ended != nullptr) {   // the beams that have ended
        const uint32_t b = min(lane, beams - 1);
        add(lane < beams && over[b] != 0 && score[b] > neg_inf, candidate((double)score[b], b, 0.0f, a.end_token));
    }
    if (lane == 0) {
        count[wave] = n;
        bound[1][wave] = least;
    }
    if (wave == 0) ranks[lane] = 0;
    __syncthreads();
    const size_t out = (size_t)group * keep;
    uint32_t all = 0, before = 0, from = 0;   // lane i of every wave has the i-th of all candidates
#pragma unroll
    for (uint32_t i = 0; i < kPickWaves; ++i) {
        const uint32_t its = count[i];
        if (lane >= all) {
            from = i;
            before = all;
        }
        all += its;
    }
    Candidate c{};
    uint32_t rank;
    if (all <= kWave) {
        // each wave compares them with an eighth of them
        n = all;
        if (lane < n) c = held[from][lane - before];
        rank = 0;
        for (uint32_t i = wave; i < n; i += kPickWaves) {
            const uint64_t other = of_lane(c.score, i);
            rank += other > c.score || (other == c.score && of_lane(c.rest, i) > c.rest);
        }
        if (rank != 0) atomicAdd(&ranks[lane], rank);
        __syncthreads();
        if (wave != 0) return;
        rank = lane < n ? ranks[lane] : lane;
    } else {
        if (wave != 0) return;
        for (uint32_t i = 1; i < kPickWaves; ++i) least = bound[1][i] > least ? bound[1][i] : least;
        for (uint32_t i = 1; i < kPickWaves; ++i) {
            const uint32_t its = count[i];
            for (uint32_t at = lane; wave_any(at < its); at += kWave) {
                const Candidate x = held[i][min(at, kPickHeld - 1)];   // (of an entry that is not there, not used)
                add(at < its && x.score >= least, x);
            }
            if (n > kPickSpare || (i == kPickWaves - 1 && n > kWave)) cut();
        }
        wave_order();
        if (lane < n) c = mine[lane];
        rank = lane;
        if (lane < n) rank = 0;
        for (uint32_t i = 0; i < n; ++i) {
            const uint64_t other = of_lane(c.score, i);
            const bool ahead = other > c.score || (other == c.score && of_lane(c.rest, i) > c.rest);
            rank += ahead && lane < n;
        }
    }
    if (rank >= keep) return;
    const bool there = lane < n;
    const uint32_t token = there ? (1u << kTokenBits) - 1 - ((uint32_t)c.rest & ((1u << kTokenBits) - 1)) : a.end_token;
    a.parents[out + rank] = there ? kBeamMax - 1 - (uint32_t)(c.rest >> 58) : 0;
    a.tokens[out + rank] = token;
    a.new_scores[out + rank] = there ? (float)from_key(c.score) : neg_inf;
    if (a.new_ended != nullptr) a.new_ended[out + rank] = token == a.end_token ? 1 : 0;
}

// ---- plan and launch -------------------------------------------------------------------

// Waves of a call, 16 for every CU. Measured (us, 2048, 4096 and 8192 of them): 32 x 8 x
// 128256 f32 32.8, 33.0 and 34.1, f16 24.1, 22.9 and 24.4; 16 x 8 x 32003 f32 14.8, 13.5
// (a tile each) and 13.5.
constexpr uint32_t kWavesWanted = 4096;

struct Plan {
    uint32_t parts, per_part, pitch;
    size_t entry_bytes, sum_bytes;
};

Plan plan_of(size_t rows, size_t beams, size_t vocab, size_t keep, size_t elem) {
    Plan p;
    const size_t tile = kTile * elem / 16, tiles = (vocab + kTile - 1) / kTile;   // (of vectors)
    size_t parts = kWavesWanted / rows;
    parts = parts < 1 ? 1 : parts > kMaxParts ? kMaxParts : parts;
    parts = parts > tiles ? tiles : parts;
    // (a group's lists are its workgroup's lanes)
    const size_t lists = kPickWaves * kWave / beams;
    parts = parts > lists ? lists : parts;
    const size_t each = (tiles + parts - 1) / parts;
    p.per_part = (uint32_t)(each * tile);
    p.parts = (uint32_t)((tiles + each - 1) / each);
    p.pitch = (uint32_t)((keep + kAhead - 1) / kAhead * kAhead);
    p.entry_bytes = (rows * p.parts * p.pitch * sizeof(Entry) + 255) / 256 * 256;
    p.sum_bytes = rows * p.parts * sizeof(PartSum);
    return p;
}

}  // namespace

size_t beam_select_workspace(const BeamShape &b, bool f32) {
    const Plan p = plan_of(b.groups * b.beams, b.beams, b.vocab, b.keep, f32 ? 4 : 2);
    return p.entry_bytes + p.sum_bytes;
}

hipError_t beam_select(bool f32, const BeamShape &b, const void *logits, const float *scores, const uint32_t *ended,
                       uint32_t end_token, uint32_t *parents, uint32_t *tokens, float *new_scores, uint32_t *new_ended,
                       void *workspace, hipStream_t s) {
    const size_t rows = b.groups * b.beams;
    const Plan p = plan_of(rows, b.beams, b.vocab, b.keep, f32 ? 4 : 2);
    Entry *const entries = static_cast<Entry *>(workspace);
    PartSum *const sums = reinterpret_cast<PartSum *>(static_cast<char *>(workspace) + p.entry_bytes);
    auto scan = [&](auto kernel, auto *x) {
        kernel<<<dim3((uint32_t)rows, p.parts), kWave, 0, s>>>(x, ended, (uint32_t)b.vocab, p.per_part, (uint32_t)b.keep,
                                                             ScanArgs{entries, sums, p.pitch});
    };
    if (f32) scan(beam_scan_kernel<float>, static_cast<const float *>(logits));
    else scan(beam_scan_kernel<_Float16>, static_cast<const _Float16 *>(logits));
    const hipError_t status = hipGetLastError();
    if (status != hipSuccess) return status;
    // (a launch holds fewer than 2^32 threads)
    constexpr size_t kGroupsPerLaunch = size_t{1} << 22;
    for (size_t first = 0; first < b.groups; first += kGroupsPerLaunch) {
        const size_t groups = b.groups - first < kGroupsPerLaunch ? b.groups - first : kGroupsPerLaunch;
        const size_t row = first * b.beams, list = row * p.parts, out = first * b.keep;
        beam_pick_kernel<<<(uint32_t)groups, kPickWaves * kWave, 0, s>>>(
            entries + list * p.pitch, sums + list, scores + row, ended == nullptr ? nullptr : ended + row, (uint32_t)b.beams,
            p.parts, (uint32_t)b.keep, p.pitch,
            PickArgs{parents + out, tokens + out, new_scores + out, new_ended == nullptr ? nullptr : new_ended + out, end_token});
        const hipError_t launched = hipGetLastError();
        if (launched != hipSuccess) return launched;
    }
    return hipSuccess;
}

}  // namespace k
}  // namespace icsdk
