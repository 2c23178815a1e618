// Beam search's choice: fleet_beam_select (declaration in fleet_moe.h).
//
// First launch, a workgroup per 4,096 logits of a beam (16 a thread, in
// registers): their maximum, sum of exponentials, and n_out best. Second launch, a
// workgroup per group: each beam's log sum, and the n_out best of what its parts
// kept. Reading the logits bounds it (HBM for many beams; for few, the two
// launches' latency). Measured, 102,400 logits a beam: 32 groups of 8 beams, 16
// outputs each, 20 + 7 us (105 MB; the loads by themselves take 15.5); 4 beams,
// 4.9 + 5.2. (With 32 logits a thread 22.8 + 6.1 us where 16 took 22.0 + 7.)
//
// The best of many without sorting them: let T be a value that at least n_out of
// the threads' maxima reach. Every one of the n_out best is then >= T, and few
// others are, so the values >= T go to LDS and are ranked there by counting. Ranking
// uses the whole order (value, then index), so the outcome does not depend on the
// order in which they arrive. Where ties leave more than LDS holds, the best
// are taken one after the other.
//
// Sums: exponentials in fp32 (arguments <= 0, v_exp_f32), 16 of them added in fp32
// and the rest in 64 bits; scores are compared in 64 bits, because the log sums of
// beams that compete differ by less than a rounding of fp32. Where they differ by less than
// the sums' own error (doubt()), the sums of the beams in question are taken once more in
// 64 bits, for a subtraction a candidate of the others (the second launch 7.27 and 7.34 us).
#include <math.h>

#include <type_traits>

#include "moe_common.h"

namespace fleet_moe {
namespace beam {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kPer = 16;
constexpr int kPart = kThreads * kPer;
constexpr int kMaxOut = FLEET_BEAM_MAX_OUT;
constexpr int kMaxBeams = FLEET_BEAM_MAX_BEAMS;
constexpr int kHold = 1024;                    // values LDS holds for ranking

struct Params {
    const float* logits;
    int64_t ld;
    const float* scores;
    const uint8_t* finished;
    float* max;                 // [rows][parts]
    double* sum;                // [rows][parts], of exp(x - max)
    uint64_t* best;             // [rows][parts][n_out]: order key of x, ~token; 0: none
    float* out_scores;
    int32_t* parents;
    int32_t* tokens;
    uint8_t* out_finished;
    uint64_t per_beam;          // floor(2^44 / (parts * n_out)) + 1
    int n_beams, n_out, vocab, parts, eos;
};

// fp32 to uint32, in order; finite values and zeros only. Nothing maps to 0.
__device__ __forceinline__ uint32_t order32(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);          // -0 as +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unorder32(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t order64(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
    return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double unorder64(uint64_t k) {
    return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k));
}

// A beam that offers something; a logit that is offered.
__device__ __forceinline__ bool has_score(float s) { return s == s && s != -INFINITY; }

// The greatest T that at least k of the N * 64 words in v reach, to as many leading
// bits as leave at most k + 16 of them. Run by one wave.
template <int N>
__device__ __forceinline__ uint32_t reach_of(const uint32_t (&v)[N], int k) {
    uint32_t T = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = T | 1u << bit;
        int count = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) count += __popcll(__ballot(v[i] >= c));
        if (count >= k) {
            T = c;
            if (count <= k + (N > 1 ? 16 : 0)) break;
        }
    }
    return T;
}
// Of the kThreads words in `keys`; with kFours, for few outputs, of the 64 maxima of four
// each: where neighbours have nothing to do with each other hardly more values reach
// that T (of 4,096 for 16 outputs some 18 instead of 17), and each bit costs one comparison
// instead of four. (First launch 22.0 to 20.3 us; the second's neighbours are the best of
// one part, in order, and it went from 7.0 to 8.1.)
template <bool kFours>
__device__ __forceinline__ uint32_t reach(const uint32_t* keys, int k) {
    static_assert(kThreads == 4 * 64 && kMaxOut <= 64, "");
    const u32x4 w = reinterpret_cast<const u32x4*>(keys)[threadIdx.x & 63];
    if (kFours && k <= 16) {
        const uint32_t a = w.x > w.y ? w.x : w.y, b = w.z > w.w ? w.z : w.w;
        const uint32_t v[1] = {a > b ? a : b};
        return reach_of(v, k);
    }
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    return reach_of(v, k);
}

struct PartLds {
    __attribute__((aligned(16))) uint32_t top[kThreads];
    uint64_t hold[kHold];
    float max[kWaves];
    double sum[kWaves];
    uint64_t one[kWaves];
    uint32_t reach;
    int n;
};

__global__ __launch_bounds__(kThreads) void part_kernel(Params P) {
    __shared__ PartLds L;
    const int row = blockIdx.y, part = blockIdx.x, t = threadIdx.x;
    const int lane = t & 63, wave = t >> 6;
    const bool done = P.finished && P.finished[row];
    if (!has_score(P.scores[row]) | done) return;
    const float* x = P.logits + (int64_t)row * P.ld;
    const int base = part * kPart;
    const int n = P.vocab - base < kPart ? P.vocab - base : kPart;
    // thread t's value 4 i + j is at base + 1024 i + 4 t + j
    float v[kPer];
    const bool wide = ((uintptr_t)(x + base) & 15) == 0;
#pragma unroll
    for (int i = 0; i < kPer / 4; ++i) {
        const int at = i * 4 * kThreads + 4 * t;
        if (wide && at + 4 <= n) {
            const u32x4 w = ld_stream(reinterpret_cast<const u32x4*>(x + base + at));
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * i + j] = __uint_as_float(w[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[4 * i + j] = at + j < n ? ld_global(x + base + at + j) : -INFINITY;
        }
    }
    float top = -INFINITY, lowest = -INFINITY;
    asm("" : "+v"(lowest));                               // (or med3 becomes min and max)
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        // of three values with a NaN, med3 is the lesser of the others
        v[i] = __builtin_amdgcn_fmed3f(v[i], lowest, 3.402823466e38f);
        top = fmaxf(top, v[i]);
    }
    L.top[t] = top == -INFINITY ? 0 : order32(top);
    const float wmax = wave_max(top);
    if (lane == 0) L.max[wave] = wmax;
    if (t == 0) L.n = 0;
    __syncthreads();
    float m = L.max[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) m = fmaxf(m, L.max[i]);
    if (m != -INFINITY) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) s += __expf(v[i] - m);
        const double ws = wave_sum64((double)s);
        if (lane == 0) L.sum[wave] = ws;
    } else if (lane == 0) {
        L.sum[wave] = 0.0;
    }
    if (wave == 0) {
        const uint32_t T = reach<true>(L.top, P.n_out);
        if (lane == 0) L.reach = T > 0x00800000u ? T : 0x00800000u;     // order32(-FLT_MAX)
    }
    __syncthreads();
    const int64_t slot = (int64_t)row * P.parts + part;
    if (t == 0) {
        P.max[slot] = m;
        P.sum[slot] = (L.sum[0] + L.sum[1]) + (L.sum[2] + L.sum[3]);
    }
    const float least = unorder32(L.reach);               // -FLT_MAX or more: no -inf
    const auto key = [&](int i) {
        const int token = base + (i / 4) * 4 * kThreads + 4 * t + i % 4;
        return (uint64_t)order32(v[i]) << 32 | (uint32_t)~token;
    };
    uint64_t who[kPer];
    int hits = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        who[i] = __ballot(v[i] >= least);
        hits += __popcll(who[i]);
    }
    int at = 0;
    if (lane == 0 && hits) at = atomicAdd(&L.n, hits);
    at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        if (who[i] == 0) continue;
        const int mine = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(who[i] >> 32),
                                 __builtin_amdgcn_mbcnt_lo((uint32_t)who[i], 0));
        if (v[i] >= least && mine < kHold) L.hold[mine] = key(i);
        at += __popcll(who[i]);
    }
    __syncthreads();
    const int found = L.n;
    uint64_t* best = P.best + slot * P.n_out;
    if (found <= kHold) {
        for (int i = t; i < found; i += kThreads) {
            const uint64_t mine = L.hold[i];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < found; ++j) rank += L.hold[j] > mine;
            if (rank < P.n_out) best[rank] = mine;
        }
        for (int i = found + t; i < P.n_out; i += kThreads) best[i] = 0;
        return;
    }
    // too many ties: the greatest key below the last one, n_out times
    uint64_t last = ~0ull;
    for (int k = 0; k < P.n_out; ++k) {
        uint64_t mine = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint64_t c = v[i] != -INFINITY ? key(i) : 0;
            if (c < last && c > mine) mine = c;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t o = __shfl_xor((unsigned long long)mine, d);
            mine = o > mine ? o : mine;
        }
        if (lane == 0) L.one[wave] = mine;
        __syncthreads();
        last = L.one[0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) last = L.one[i] > last ? L.one[i] : last;
        if (t == 0) best[k] = last;
        __syncthreads();
    }
}

struct Best {
    uint64_t score;             // order64 of the 64-bit score; 0: none
    uint64_t key;               // of the logit and token
    int beam;
};
__device__ __forceinline__ bool ahead(const Best& a, const Best& b) {
    return (a.score > b.score) |
           ((a.score == b.score) &
            ((a.beam < b.beam) | ((a.beam == b.beam) & (a.key > b.key))));
}

// A group's candidates, the n_out best of every part of every beam: four a thread in
// registers, all their loads in flight at once. More than that (many beams, parts or
// outputs) are read once more.
constexpr int kGroupThreads = 1024;
constexpr int kGroupWaves = kGroupThreads / 64;
constexpr int kGroupPer = 4;
struct GroupLds {
    double lse[kMaxBeams];      // log of the sum of exp(x - max)
    float max[kMaxBeams], score[kMaxBeams];
    uint8_t kind[kMaxBeams];
    __attribute__((aligned(16))) uint32_t top[kThreads];
    uint64_t rank_score[kHold], key[kHold];
    uint8_t beam[kHold];
    uint16_t order[kHold];
    Best one[kGroupWaves];
    double sum[kGroupWaves];
    uint8_t doubt[kMaxBeams], any_doubt;    // beams whose log sums decide the order
    uint32_t reach;
    int n;
};
enum : uint8_t { kNothing, kItself, kTokens };

// How far apart scores of different beams have to be for their order to be certain. A part's
// sum is off by (2.5 D + 17) 2^-24 of itself at most: 2^-24 |d| from d = x - max, 1.5 *
// 2^-24 |d| from d * log2(e), 2^-23 from the exponential, 15 roundings of 2^-24 from the
// addition of 16; and D, the mean of |d| by weight, is log(kPart) at most (the entropy of
// the weights is D + log of the sum, which is 1 or more). That is 38 * 2^-24, less than
// 2^-18, for the log sums of each of the two, beside the roundings of the scores themselves.
__device__ __forceinline__ double doubt(double score) {
    return 0x1p-17 + fmin(fabs(score), 1.7976931348623157e308) * 0x1p-50;
}

// The least word of order64 that a score with one of T's word in its doubt can have.
__device__ __forceinline__ uint32_t below(uint32_t T) {
    if (T <= 0x00100000u) return T;                       // of the lowest finite score
    const double s = unorder64((uint64_t)T << 32);
    return (uint32_t)(order64(s - doubt(s)) >> 32);
}

// The log sums of the beams in doubt once more, exponentials and sums in 64 bits, from the
// logits: 40 us for a beam of 102,400, by one workgroup.
__device__ __forceinline__ void exact_sums(const Params& P, GroupLds& L, int row0) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    for (int b = 0; b < P.n_beams; ++b) {
        if (!L.doubt[b] || L.kind[b] != kTokens || L.max[b] == -INFINITY) continue;
        const float* x = P.logits + (int64_t)(row0 + b) * P.ld;
        const double max = (double)L.max[b];
        double s = 0.0;
        for (int i = t; i < P.vocab; i += kGroupThreads) {
            const float v = ld_global(x + i);
            if (has_score(v)) s += exp((double)fminf(v, 3.402823466e38f) - max);
        }
        s = wave_sum64(s);
        if (lane == 0) L.sum[wave] = s;
        __syncthreads();
        if (t == 0) {
            double all = 0.0;
            for (int i = 0; i < kGroupWaves; ++i) all += L.sum[i];
            L.lse[b] = log(all);
        }
        __syncthreads();
    }
}

__global__ __launch_bounds__(kGroupThreads) void group_kernel(Params P) {
    __shared__ GroupLds L;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int row0 = blockIdx.x * P.n_beams;
    const int each = P.parts * P.n_out;
    const int n = P.n_beams * each;
    // beam of candidate i: i * per_beam >> 44, exact for i < 64 * each <= 2^24
    const auto beam_of = [&](int i) { return (int)((uint64_t)(uint32_t)i * P.per_beam >> 44); };
    const uint64_t* best = P.best + (int64_t)row0 * each;
    uint64_t keys[kGroupPer];
#pragma unroll
    for (int k = 0; k < kGroupPer; ++k) {
        const int i = t + k * kGroupThreads;
        keys[k] = i < n ? ld_global(best + i) : 0;
    }
    for (int b = wave; b < P.n_beams; b += kGroupWaves) {
        const int row = row0 + b;
        // (a beam that kept nothing has whatever is there for its maxima and sums: not used)
        const float* max = P.max + (int64_t)row * P.parts;
        const double* sum = P.sum + (int64_t)row * P.parts;
        float own_max = lane < P.parts ? ld_global(max + lane) : -INFINITY;
        double own_sum = lane < P.parts ? ld_global(sum + lane) : 0.0;
        const float score = ld_global(P.scores + row);
        const bool done = P.finished && P.finished[row];
        for (int i = lane + 64; i < P.parts; i += 64) {
            const float x = ld_global(max + i);
            const double y = ld_global(sum + i);
            const float both = fmaxf(own_max, x);
            if (both != -INFINITY)
                own_sum = own_sum * exp((double)own_max - (double)both) +
                          y * exp((double)x - (double)both);
            own_max = both;
        }
        const uint8_t kind = !has_score(score) ? kNothing : done ? kItself : kTokens;
        const float m = wave_max(own_max);
        const double s = wave_sum64(
            own_max == -INFINITY ? 0.0 : own_sum * exp((double)own_max - (double)m));
        if (lane == 0) {
            L.lse[b] = log(s);
            L.max[b] = m;
            L.score[b] = score;
            L.kind[b] = kind;
            L.doubt[b] = 0;
        }
    }
    if (t == 0) L.any_doubt = 0;
    const auto candidate = [&](int i, uint64_t key) {
        Best c;
        c.beam = beam_of(i);
        c.key = key;
        c.score = 0;
        const uint8_t kind = L.kind[c.beam];
        const double score = (double)L.score[c.beam];
        if (kind == kItself && i == c.beam * each) {
            c.key = 1ull << 63 | (uint32_t)~(P.eos < 0 ? -1 : P.eos);
            c.score = order64(score);
        } else if (kind == kTokens && key) {
            const double x = unorder32((uint32_t)(key >> 32));
            c.score = order64(score + ((x - (double)L.max[c.beam]) - L.lse[c.beam]));
        }
        return c;
    };
    const auto put = [&](int k, const Best& c) {
        const int64_t at = (int64_t)blockIdx.x * P.n_out + k;
        const bool there = c.score != 0;
        const int row = row0 + c.beam, token = (int)~(uint32_t)c.key;
        P.out_scores[at] = there ? (float)unorder64(c.score) : -INFINITY;
        P.parents[at] = there ? row : -1;
        P.tokens[at] = there ? token : -1;
        if (P.out_finished)
            P.out_finished[at] = there && (L.kind[c.beam] == kItself ||
                                           (P.eos >= 0 && token == P.eos));
    };
    const auto live = [&] {
        return __popcll(__ballot(lane < P.n_beams && L.kind[lane] != kNothing));
    };
    constexpr int kHeld = kGroupPer * kGroupThreads;
    // Whether the order is in doubt. (Called twice, not a loop: as a loop it takes 128 instead of
    // 115 registers, and 8.0 us.)
    const auto choose = [&](auto again) __attribute__((always_inline)) {
        if (t == 0) L.n = 0;
        if (t < kThreads) L.top[t] = 0;
        __syncthreads();
        Best held[kGroupPer];
        uint64_t high = 0;
#pragma unroll
        for (int k = 0; k < kGroupPer; ++k) {
            const int i = t + k * kGroupThreads;
            held[k] = i < n ? candidate(i, keys[k]) : Best{0, 0, 0};
            high = held[k].score > high ? held[k].score : high;
        }
        for (int i = t + kHeld; i < n; i += kGroupThreads) {
            const uint64_t s = candidate(i, ld_global(best + i)).score;
            high = s > high ? s : high;
        }
        // (four threads share a word: reach() takes kThreads of them)
        atomicMax(&L.top[t % kThreads], (uint32_t)(high >> 32));
        __syncthreads();
        if (wave == 0) {
            const uint32_t T = reach<false>(L.top, P.n_out);
            if (lane == 0) L.reach = below(T);
        }
        __syncthreads();
        const uint32_t T = L.reach;
        const auto hold = [&](const Best& c) {
            if (c.score == 0 || (uint32_t)(c.score >> 32) < T) return;
            const int at = atomicAdd(&L.n, 1);
            if (at < kHold) {
                L.rank_score[at] = c.score;
                L.key[at] = c.key;
                L.beam[at] = (uint8_t)c.beam;
            }
        };
#pragma unroll
        for (int k = 0; k < kGroupPer; ++k) hold(held[k]);
        for (int i = t + kHeld; i < n; i += kGroupThreads) hold(candidate(i, ld_global(best + i)));
        __syncthreads();
        const int found = L.n;
        if (found <= kHold) {
            for (int i = wave; i < found; i += kGroupWaves) {
                const Best c{L.rank_score[i], L.key[i], L.beam[i]};
                int rank = 0;
                for (int j = lane; j - lane < found; j += 64)
                    rank += __popcll(__ballot(
                        j < found && ahead(Best{L.rank_score[j], L.key[j], L.beam[j]}, c)));
                if (lane == 0) {
                    L.order[rank] = (uint16_t)i;
                    if (rank < P.n_out) put(rank, c);
                }
            }
            for (int i = found + t; i < P.n_out; i += kGroupThreads) put(i, Best{0, 0, 0});
        } else if (again || live() < 2) {
            Best last{~0ull, ~0ull, -1};
            for (int k = 0; k < P.n_out; ++k) {
                Best top{0, 0, kMaxBeams};
                for (int i = t; i < n; i += kGroupThreads) {
                    const Best c = candidate(i, ld_global(best + i));
                    if (c.score != 0 && ahead(last, c) && ahead(c, top)) top = c;
                }
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const Best o{__shfl_xor((unsigned long long)top.score, d),
                                 __shfl_xor((unsigned long long)top.key, d),
                                 __shfl_xor(top.beam, d)};
                    if (ahead(o, top)) top = o;
                }
                if (lane == 0) L.one[wave] = top;
                __syncthreads();
                last = L.one[0];
#pragma unroll
                for (int i = 1; i < kGroupWaves; ++i)
                    if (ahead(L.one[i], last)) last = L.one[i];
                if (last.score == 0) last.beam = 0;
                if (t == 0) put(k, last);
                __syncthreads();
            }
        } else {
            // more ties than LDS holds, of any beams
            if (t < P.n_beams) L.doubt[t] = 1;
            if (t == 0) L.any_doubt = 1;
        }
        if constexpr (again) return false;
        __syncthreads();
        // neighbours in order, of different beams
        if (found <= kHold)
            for (int i = t; i + 1 < found; i += kGroupThreads) {
                const int a = L.order[i], b = L.order[i + 1];
                const double score = unorder64(L.rank_score[a]);
                if (L.beam[a] != L.beam[b] && score - unorder64(L.rank_score[b]) <= doubt(score))
                    L.doubt[L.beam[a]] = L.doubt[L.beam[b]] = L.any_doubt = 1;
            }
        __syncthreads();
        return L.any_doubt != 0;
    };
    if (choose(std::false_type{})) {
        exact_sums(P, L, row0);
        choose(std::true_type{});
    }
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

bool sizes_ok(int n_groups, int n_beams, int n_out, int vocab) {
    return n_groups >= 1 && n_beams >= 1 && n_beams <= kMaxBeams && n_out >= 1 &&
           n_out <= kMaxOut && (int64_t)n_groups * n_beams <= 65535 && vocab >= 1 &&
           vocab <= (1 << 24);
}
struct Layout {
    size_t sum, best, bytes;
    int parts;
};
Layout layout(int rows, int n_out, int vocab) {
    Layout l;
    l.parts = (vocab + kPart - 1) / kPart;
    const size_t n = (size_t)rows * l.parts;
    l.sum = up256(n * sizeof(float));
    l.best = l.sum + up256(n * sizeof(double));
    l.bytes = l.best + up256(n * n_out * sizeof(uint64_t));
    return l;
}

}  // namespace beam
}  // namespace fleet_moe

using namespace fleet_moe;

int fleet_moe_check_device(int min_cus);

extern "C" size_t fleet_beam_workspace_bytes(int32_t n_groups, int32_t n_beams, int32_t n_out,
                                             int32_t vocab) {
    if (!beam::sizes_ok(n_groups, n_beams, n_out, vocab)) return 0;
    return beam::layout(n_groups * n_beams, n_out, vocab).bytes;
}

extern "C" int fleet_beam_select(const float* logits, int64_t ld, const float* scores,
                                 const uint8_t* finished, int32_t n_groups, int32_t n_beams,
                                 int32_t n_out, int32_t vocab, int32_t eos, float* out_scores,
                                 int32_t* parents, int32_t* tokens, uint8_t* out_finished,
                                 void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (!logits || !scores || !out_scores || !parents || !tokens || !workspace ||
        (uintptr_t)logits % 4 || (uintptr_t)scores % 4 || (uintptr_t)out_scores % 4 ||
        (uintptr_t)parents % 4 || (uintptr_t)tokens % 4 || (uintptr_t)workspace % 256)
        return FLEET_MOE_ERR_ARG;
    if (!beam::sizes_ok(n_groups, n_beams, n_out, vocab) || ld < vocab ||
        ld > ((int64_t)1 << 40) || eos >= vocab)
        return FLEET_MOE_ERR_ARG;
    const beam::Layout l = beam::layout(n_groups * n_beams, n_out, vocab);
    if (workspace_bytes < l.bytes) return FLEET_MOE_ERR_WORKSPACE;
    if (int e = fleet_moe_check_device(1)) return e;
    char* ws = static_cast<char*>(workspace);
    beam::Params P{};
    P.logits = logits;
    P.ld = ld;
    P.scores = scores;
    P.finished = finished;
    P.max = reinterpret_cast<float*>(ws);
    P.sum = reinterpret_cast<double*>(ws + l.sum);
    P.best = reinterpret_cast<uint64_t*>(ws + l.best);
    P.out_scores = out_scores;
    P.parents = parents;
    P.tokens = tokens;
    P.out_finished = out_finished;
    P.n_beams = n_beams;
    P.n_out = n_out;
    P.vocab = vocab;
    P.parts = l.parts;
    P.eos = eos;
    P.per_beam = ((uint64_t)1 << 44) / ((uint64_t)l.parts * n_out) + 1;
    hipLaunchKernelGGL(beam::part_kernel, dim3(l.parts, n_groups * n_beams), dim3(beam::kThreads),
                       0, stream, P);
    hipLaunchKernelGGL(beam::group_kernel, dim3(n_groups), dim3(beam::kGroupThreads), 0, stream,
                       P);
    return (int)hipGetLastError();
}
