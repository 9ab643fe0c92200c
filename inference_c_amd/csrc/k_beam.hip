// One step's choice of a beam search over beams and vocabulary: of every group the
// `keep` candidates (beam, token) of largest score[b] + x[b, v] - log sum exp x[b, :].
//
// Within a beam the order is that of the logits, so a beam's own `keep` largest
// logits are all that can be chosen of it. beam_scan_kernel reads each row once, a wave
// per part of it, and leaves of each part the running sum of exp(x - max) and its
// largest logits in order; beam_pick_kernel, a workgroup per group, joins the sums of a
// row and takes the best of all parts' candidates by their scores.
//
// Scores are f64 from exact logits; of the log sums only the exponentials are f32,
// each off by 2^-23 or so in either direction, so that a sum of many is off by far less
// and two beams' candidates change places only where their scores are equal to 1e-8.
#include "kernels.hpp"
#include "kern_common.hpp"

namespace icsdk {
namespace k {
namespace {

constexpr uint32_t kMaxKeep = kBeamMaxKeep;   // a lane each at the end
static_assert(kMaxKeep == kWave);
constexpr uint32_t kTokenBits = 26;
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

// The want-th largest of the wave's keys (kSlots per lane, the first `slots` looked at;
// a key of 0 is none), or a smaller number above which there are exactly `want`: from
// the highest bit on, a bit is set where at least `want` keys reach it.
template <typename K, uint32_t kSlots>
__device__ inline K largest(const K (&key)[kSlots], uint32_t slots, uint32_t want) {
    K least = 0;
    for (K bit = K{1} << (8 * sizeof(K) - 1); bit != 0; bit >>= 1) {
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
    const void *logits;
    const uint32_t *ended;   // [rows] or null
    Entry *entries;          // [rows][parts][pitch]
    PartSum *sums;           // [rows][parts]
    uint32_t vocab, parts, per_part, keep, pitch;   // per_part: vectors
};

// exp(t) for t <= 0 (and NaN): log2 e in two pieces, so that the exponent is off by
// the rounding of one product alone.
__device__ inline float exp_below(float t) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(t, 1.925963033500001e-8f, t * 1.4426950216293335f));
}

template <typename T> constexpr uint32_t kVectors = sizeof(T) == 4 ? 2 : 1;   // of a lane, per tile: 8 logits
constexpr uint32_t kTile = 8 * kWave;
constexpr uint32_t kSpare = 2 * kMaxKeep;          // entries after which they are cut to the best
constexpr uint32_t kSlots = (kSpare + kTile) / kWave;

template <typename T>
__global__ __launch_bounds__(kWave) void beam_scan_kernel(ScanArgs a) {
    constexpr uint32_t E = Vec16<T>::N, U = kVectors<T>;
    __shared__ float logit[kSpare + kTile];
    __shared__ uint32_t token[kSpare + kTile];
    const uint32_t lane = threadIdx.x, part = blockIdx.x % a.parts, row = blockIdx.x / a.parts;
    if (a.ended != nullptr && a.ended[row] != 0) return;
    const T *x = static_cast<const T *>(a.logits);
    const float neg_inf = -__builtin_inff(), inf = __builtin_inff();
    // tokens lie in vectors from the row's first on, wherever in memory that is (a load
    // needs no alignment), so that rows alike have sums alike
    x += (uint64_t)row * a.vocab;
    const uint32_t vectors = (a.vocab + E - 1) / E;
    const uint32_t begin = min(part * a.per_part, vectors), end = min(begin + a.per_part, vectors);

    float now[U][E], m = neg_inf, s = 0.0f, least = neg_inf;
    uint32_t n = 0;   // entries
    auto load = [&](uint32_t at, float (&to)[U][E]) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t v = at + u * kWave + lane, from = v * E;
            if (v < end && from + E <= a.vocab) {
                T w[E];
                __builtin_memcpy(w, x + from, sizeof(w));
#pragma unroll
                for (uint32_t e = 0; e < E; ++e) to[u][e] = (float)w[e];
            } else {   // what is not the row's, or not the part's
#pragma unroll
                for (uint32_t e = 0; e < E; ++e) to[u][e] = v < end && from + e < a.vocab ? (float)x[from + e] : neg_inf;
            }
        }
    };
    // cuts the entries to the `keep` best, equal ones by their tokens
    auto cut = [&] {
        wave_order();
        float value[kSlots];
        uint32_t key[kSlots], id[kSlots];
        const uint32_t slots = (n + kWave - 1) / kWave;
#pragma unroll
        for (uint32_t i = 0; i < kSlots; ++i) {
            const uint32_t at = i * kWave + lane;
            key[i] = 0;
            id[i] = 0;
            if (i < slots && at < n) {
                value[i] = logit[at];
                key[i] = key_of(value[i]);
                id[i] = ~token[at];   // (not 0: a token has 26 bits)
            }
        }
        const uint32_t bound = largest(key, slots, a.keep);
        uint32_t over = 0, same = 0;
#pragma unroll
        for (uint32_t i = 0; i < kSlots; ++i)
            if (i < slots) {
                over += lanes(key[i] > bound);
                same += lanes(key[i] == bound);
            }
        uint32_t first_ids = 0;   // of those equal to the bound, what a token has to be
        if (over + same > a.keep) {
            uint32_t of[kSlots];
#pragma unroll
            for (uint32_t i = 0; i < kSlots; ++i) of[i] = key[i] == bound ? id[i] : 0;
            first_ids = largest(of, slots, a.keep - over);
        }
        wave_order();
        uint32_t to = 0;
        uint32_t lowest = 0xffffffffu;
#pragma unroll
        for (uint32_t i = 0; i < kSlots; ++i)
            if (i < slots) {
                const bool stays = key[i] > bound || (key[i] == bound && key[i] != 0 && id[i] >= first_ids);
                const uint32_t at = to + lanes_below(stays, lane);
                if (stays) {
                    logit[at] = value[i];
                    token[at] = ~id[i];
                    lowest = min(lowest, key[i]);
                }
                to += lanes(stays);
            }
        n = to;
        wave_order();
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) lowest = min(lowest, (uint32_t)__shfl_xor((int)lowest, d, kWave));
        if (n >= a.keep) least = from_key(lowest);
    };
    if (begin < end) load(begin, now);
    for (uint32_t at = begin; at < end; at += U * kWave) {
        float next[U][E];
        if (at + U * kWave < end) load(at + U * kWave, next);
        float top = neg_inf;
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
#pragma unroll
            for (uint32_t e = 0; e < E; ++e) top = fmaxf(top, now[u][e]);
        // the sum
        const float up = fmaxf(m, top);
        if (wave_any(up == inf)) {
            float add = 0.0f;
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
#pragma unroll
                for (uint32_t e = 0; e < E; ++e) {
                    const float y = now[u][e];
                    add += y == inf ? 1.0f : y != y ? y : up == inf ? 0.0f : exp_below(y - (up == neg_inf ? 0.0f : up));
                }
            s = (m == up ? s : m == neg_inf || up == inf ? s * 0.0f : s * exp_below(m - up)) + add;
        } else {
            const float base = up == neg_inf ? 0.0f : up;
            s *= exp_below(m - base);
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
#pragma unroll
                for (uint32_t e = 0; e < E; ++e) s += exp_below(now[u][e] - base);
        }
        m = up;
        // the candidates: larger than the least of `keep` ones before them (an equal one
        // comes after those), of the first tile those that reach the keep-th largest lane
        const uint32_t tops[1] = {top == neg_inf ? 0 : key_of(top)};
        const bool bounded = at == begin && lanes(tops[0] != 0) >= a.keep;
        const uint32_t reach = bounded ? largest(tops, 1, a.keep) : 0;
        if (wave_any(top > least)) {
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
#pragma unroll
                for (uint32_t e = 0; e < E; ++e) {
                    const float y = now[u][e];
                    const bool passes = y > least && (!bounded || key_of(y) >= reach);
                    if (!wave_any(passes)) continue;
                    const uint32_t to = n + lanes_below(passes, lane);
                    if (passes) {
                        logit[to] = y;
                        token[to] = (at + u * kWave + lane) * E + e;
                    }
                    n += lanes(passes);
                }
            if (n > kSpare || (n >= a.keep && least == neg_inf)) cut();
        }
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
#pragma unroll
            for (uint32_t e = 0; e < E; ++e) now[u][e] = next[u][e];
    }
    if (n > a.keep) cut();
    wave_order();
    // in order, each entry behind those that are larger (of equal ones, earlier)
    const size_t list = (size_t)row * a.parts + part;
    float mine = neg_inf;
    uint32_t id = 0, rank = lane;
    if (lane < n) {
        mine = logit[lane];
        id = token[lane];
        rank = 0;
        for (uint32_t i = 0; i < n; ++i) rank += logit[i] > mine || (logit[i] == mine && token[i] < id);
    }
    if (rank < a.pitch) a.entries[list * a.pitch + rank] = Entry{mine, id};
    const float top = wave_max(m);
    const double sum = wave_sum_f64((double)(s * (m == top ? 1.0f : exp_below(m - top))));
    if (lane == 0) a.sums[list] = PartSum{sum, top, 0};
}

// ---- of a group ----------------------------------------------------------------------

struct PickArgs {
    const Entry *entries;
    const PartSum *sums;
    const float *scores;
    const uint32_t *ended;
    uint32_t *parents, *tokens;
    float *new_scores;
    uint32_t *new_ended;
    uint32_t beams, parts, keep, pitch, end_token;
};

constexpr uint32_t kPickWaves = 8;
constexpr uint32_t kPickHeld = 192, kPickSlots = kPickHeld / kWave;   // entries of a wave: cut from 128 on
constexpr uint32_t kAhead = 4;                                        // entries of a list asked for at once

// A candidate: its score, and what goes before where scores are equal (the lower
// beam, the larger logit, the lower token), both as keys.
struct Candidate {
    uint64_t score, rest;
};
__device__ inline Candidate candidate(double score, uint32_t beam, float logit, uint32_t token) {
    return Candidate{key_of(score), (uint64_t)(kBeamMax - 1 - beam) << 58 | (uint64_t)key_of(logit) << kTokenBits |
                                        ((1u << kTokenBits) - 1 - token)};
}

__global__ __launch_bounds__(kPickWaves *kWave) void beam_pick_kernel(PickArgs a) {
    __shared__ Candidate held[kPickWaves][kPickHeld];
    __shared__ uint32_t count[kPickWaves];
    __shared__ uint64_t bound[kPickWaves];
    __shared__ double log_sum[kBeamMax];   // of a beam; NaN: it has no candidates
    __shared__ float most[kBeamMax], score[kBeamMax];
    __shared__ uint32_t over[kBeamMax];
    const uint32_t lane = threadIdx.x % kWave, wave = (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t group = blockIdx.x, first = group * a.beams;
    const float neg_inf = -__builtin_inff();
    // the beams' sums
    for (uint32_t b = wave; b < a.beams; b += kPickWaves) {
        const float sc = a.scores[first + b];
        const bool ended = a.ended != nullptr && a.ended[first + b] != 0;
        float top = neg_inf;
        double sum = 0.0;
        if (!ended) {
            const PartSum *const of = a.sums + (size_t)(first + b) * a.parts;
            for (uint32_t p = lane; p < a.parts; p += kWave) top = fmaxf(top, of[p].max);
            top = wave_max(top);
            for (uint32_t p = lane; p < a.parts; p += kWave)
                sum += of[p].sum * (of[p].max == top ? 1.0 : exp((double)of[p].max - (double)top));
            sum = wave_sum_f64(sum);
        }
        if (lane == 0) {
            log_sum[b] = log(sum);
            most[b] = top;
            score[b] = sc;
            over[b] = ended ? 1 : 0;
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
        const uint64_t to_reach = largest(sc, slots, a.keep);
        uint32_t above = 0, same = 0;
#pragma unroll
        for (uint32_t i = 0; i < kPickSlots; ++i) {
            above += lanes(sc[i] > to_reach);
            same += lanes(sc[i] == to_reach && sc[i] != 0);
        }
        uint64_t first_rest = 0;
        if (above + same > a.keep) {
            uint64_t of[kPickSlots];
#pragma unroll
            for (uint32_t i = 0; i < kPickSlots; ++i) of[i] = sc[i] == to_reach ? rest[i] : 0;
            first_rest = largest(of, slots, a.keep - above);
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
        if (n >= a.keep) least = lowest;
    };
    auto add = [&](bool passes, const Candidate &c) {
        const uint32_t at = n + lanes_below(passes, lane);
        if (passes) mine[at] = c;
        n += lanes(passes);
        if (n > kPickHeld - kWave) cut();
    };

    // the parts' lists, a lane each, in order of their logits: a list is done with its
    // first candidate that is not among the best so far
    const uint32_t lists = a.beams * a.parts;
    for (uint32_t l0 = wave * kWave; l0 < lists; l0 += kPickWaves * kWave) {
        const uint32_t list = min(l0 + lane, lists - 1), b = list / a.parts;
        bool going = l0 + lane < lists && over[b] == 0;
        const double sc = (double)score[b], sum = log_sum[b];
        const float top = most[b];
        const u32x4 *const from =
            reinterpret_cast<const u32x4 *>(a.entries + ((size_t)(first + b) * a.parts + (list - b * a.parts)) * a.pitch);
        for (uint32_t j0 = 0; j0 < a.keep; j0 += kAhead) {
            if (!wave_any(going)) break;
            u32x4 w[kAhead / 2];
#pragma unroll
            for (uint32_t i = 0; i < kAhead / 2; ++i)
                w[i] = going ? from[j0 / 2 + i] : u32x4{0xff800000u, 0, 0xff800000u, 0};
#pragma unroll
            for (uint32_t e = 0; e < kAhead; ++e) {
                const uint32_t bits = w[e / 2][e % 2 * 2], token = w[e / 2][e % 2 * 2 + 1];
                const float x = __builtin_bit_cast(float, bits);
                const double to_top = x == top ? 0.0 : (double)x - (double)top;
                const double s = sc + (to_top - sum);
                going = going && j0 + e < a.keep && x > neg_inf && s > -__builtin_inf();
                const Candidate c = candidate(s, b, x, token);
                if (j0 + e == 0) {
                    const uint64_t heads[1] = {going ? c.score : 0};
                    if (lanes(going) >= a.keep) {
                        const uint64_t reach = largest(heads, 1, a.keep);
                        least = reach > least ? reach : least;
                    }
                }
                going = going && c.score >= least;
                add(going, c);
            }
        }
    }
    if (n > a.keep) cut();
    if (lane == 0) {
        count[wave] = n;
        bound[wave] = least;
    }
    __syncthreads();
    if (wave != 0) return;
    // the waves' candidates, and those of the beams that have ended
    for (uint32_t w = 1; w < kPickWaves; ++w) least = bound[w] > least ? bound[w] : least;
    for (uint32_t w = 1; w < kPickWaves; ++w) {
        const Candidate c = held[w][lane];   // (of an entry that is not there, not used)
        add(lane < count[w] && c.score >= least, c);
    }
    if (a.ended != nullptr) {
        const uint32_t b = min(lane, a.beams - 1);
        add(lane < a.beams && over[b] != 0 && score[b] > neg_inf, candidate((double)score[b], b, 0.0f, a.end_token));
    }
    if (n > a.keep) cut();
    wave_order();
    const size_t out = (size_t)group * a.keep;
    Candidate c{};
    uint32_t rank = lane;
    if (lane < n) {
        c = mine[lane];
        rank = 0;
        for (uint32_t i = 0; i < n; ++i) {
            const Candidate other = mine[i];
            rank += other.score > c.score || (other.score == c.score && other.rest > c.rest);
        }
    }
    if (rank >= a.keep) return;
    const bool there = lane < n;
    const uint32_t token = there ? (1u << kTokenBits) - 1 - ((uint32_t)c.rest & ((1u << kTokenBits) - 1)) : a.end_token;
    a.parents[out + rank] = there ? kBeamMax - 1 - (uint32_t)(c.rest >> 58) : 0;
    a.tokens[out + rank] = token;
    a.new_scores[out + rank] = there ? (float)from_key(c.score) : neg_inf;
    if (a.new_ended != nullptr) a.new_ended[out + rank] = token == a.end_token ? 1 : 0;
}

// ---- plan and launch -------------------------------------------------------------------

constexpr uint32_t kWavesWanted = 2048;   // eight for every CU

struct Plan {
    uint32_t parts, per_part, pitch;
    size_t entry_bytes, sum_bytes;
};

Plan plan_of(size_t rows, size_t vocab, size_t keep, size_t elem) {
    Plan p;
    const size_t tile = kTile * elem / 16, tiles = (vocab + kTile - 1) / kTile;   // (of vectors)
    size_t parts = kWavesWanted / rows;
    parts = parts < 1 ? 1 : parts > kMaxParts ? kMaxParts : parts;
    const size_t most = (tiles + 1) / 2;   // two tiles each at least
    parts = parts > most ? most : parts;
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
    const Plan p = plan_of(b.groups * b.beams, b.vocab, b.keep, f32 ? 4 : 2);
    return p.entry_bytes + p.sum_bytes;
}

hipError_t beam_select(bool f32, const BeamShape &b, const void *logits, const float *scores, const uint32_t *ended,
                       uint32_t end_token, uint32_t *parents, uint32_t *tokens, float *new_scores, uint32_t *new_ended,
                       void *workspace, hipStream_t s) {
    const size_t rows = b.groups * b.beams;
    const Plan p = plan_of(rows, b.vocab, b.keep, f32 ? 4 : 2);
    Entry *const entries = static_cast<Entry *>(workspace);
    PartSum *const sums = reinterpret_cast<PartSum *>(static_cast<char *>(workspace) + p.entry_bytes);
    const ScanArgs scan{logits, ended, entries, sums, (uint32_t)b.vocab, p.parts, p.per_part, (uint32_t)b.keep, p.pitch};
    const uint32_t grid = (uint32_t)(rows * p.parts);
    if (f32) beam_scan_kernel<float><<<grid, kWave, 0, s>>>(scan);
    else beam_scan_kernel<_Float16><<<grid, kWave, 0, s>>>(scan);
    const hipError_t status = hipGetLastError();
    if (status != hipSuccess) return status;
    beam_pick_kernel<<<(uint32_t)b.groups, kPickWaves * kWave, 0, s>>>(
        PickArgs{entries, sums, scores, ended, parents, tokens, new_scores, new_ended, (uint32_t)b.beams, p.parts,
                 (uint32_t)b.keep, p.pitch, end_token});
    return hipGetLastError();
}

}  // namespace k
}  // namespace icsdk
