// Beam search's choice: fleet_beam_select (declaration in fleet_moe.h).
//
// First launch, a workgroup per 4,096 logits of a beam (16 a thread, in
// registers): their maximum, sum of exponentials, and n_out best. Second launch, a
// workgroup per group: each beam's log sum, and the n_out best of what its parts
// kept. Reading the logits bounds it (HBM for many beams; for few, the two
// launches' latency).
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
// beams that compete differ by less than a rounding of fp32.
#include <math.h>

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

// A beam that offers nothing, or only itself.
__device__ __forceinline__ bool has_score(float s) { return s == s && s != -INFINITY; }

// The greatest T that at least k of the kThreads words in `keys` reach, to as many
// leading bits as leave at most k + 16 of them. Run by one wave.
__device__ __forceinline__ uint32_t reach(const uint32_t* keys, int n, int k) {
    const int lane = threadIdx.x & 63;
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i * 64 + lane < n ? keys[i * 64 + lane] : 0;
    uint32_t T = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = T | 1u << bit;
        int count = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) count += __popcll(__ballot(v[i] >= c));
        if (count >= k) {
            T = c;
            if (count <= k + 16) break;
        }
    }
    return T;
}

struct PartLds {
    uint32_t top[kThreads];
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
    if ((P.finished && P.finished[row]) || !has_score(P.scores[row])) return;
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
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        v[i] = v[i] == v[i] ? fminf(v[i], 3.402823466e38f) : -INFINITY;
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
        const uint32_t T = reach(L.top, kThreads, P.n_out);
        if (lane == 0) L.reach = T ? T : 1;
    }
    __syncthreads();
    const int64_t slot = (int64_t)row * P.parts + part;
    if (t == 0) {
        P.max[slot] = m;
        P.sum[slot] = (L.sum[0] + L.sum[1]) + (L.sum[2] + L.sum[3]);
    }
    const uint32_t T = L.reach;
    const auto key = [&](int i) {
        const int token = base + (i / 4) * 4 * kThreads + 4 * t + i % 4;
        return (uint64_t)order32(v[i]) << 32 | (uint32_t)~token;
    };
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        if (v[i] != -INFINITY && order32(v[i]) >= T) {
            const int at = atomicAdd(&L.n, 1);
            if (at < kHold) L.hold[at] = key(i);
        }
    }
    __syncthreads();
    const int found = L.n;
    uint64_t* best = P.best + slot * P.n_out;
    if (found <= kHold) {
        for (int i = t; i < found; i += kThreads) {
            const uint64_t mine = L.hold[i];
            int rank = 0;
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
    if (a.score != b.score) return a.score > b.score;
    if (a.beam != b.beam) return a.beam < b.beam;
    return a.key > b.key;
}

struct GroupLds {
    double lse[kMaxBeams];      // log of the sum of exp(x - max)
    float max[kMaxBeams];
    uint32_t top[kThreads];
    uint64_t score[kHold], key[kHold];
    uint8_t beam[kHold];
    Best one[kWaves];
    uint32_t reach;
    int n;
};

__global__ __launch_bounds__(kThreads) void group_kernel(Params P) {
    __shared__ GroupLds L;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int row0 = blockIdx.x * P.n_beams;
    for (int b = wave; b < P.n_beams; b += kWaves) {
        const int row = row0 + b;
        if ((P.finished && P.finished[row]) || !has_score(P.scores[row])) continue;
        float m = -INFINITY;
        for (int i = lane; i < P.parts; i += 64) m = fmaxf(m, P.max[(int64_t)row * P.parts + i]);
        m = wave_max(m);
        double s = 0.0;
        if (m != -INFINITY)
            for (int i = lane; i < P.parts; i += 64) {
                const int64_t at = (int64_t)row * P.parts + i;
                s += P.sum[at] * exp((double)P.max[at] - (double)m);
            }
        s = wave_sum64(s);
        if (lane == 0) {
            L.lse[b] = log(s);
            L.max[b] = m;
        }
    }
    if (t == 0) L.n = 0;
    __syncthreads();
    // candidate i of the group: beam i / each, the rest its part and place
    const int each = P.parts * P.n_out;
    const int64_t n = (int64_t)P.n_beams * each;
    const auto candidate = [&](int64_t i) {
        Best c;
        c.beam = (int)(i / each);
        c.score = 0;
        const int row = row0 + c.beam;
        const float score = P.scores[row];
        c.key = 0;
        if (!has_score(score)) return c;
        if (P.finished && P.finished[row]) {
            if (i % each == 0) {
                c.key = 1ull << 63 | (uint32_t)~(P.eos < 0 ? -1 : P.eos);
                c.score = order64((double)score);
            }
            return c;
        }
        c.key = P.best[(int64_t)row * each + i % each];
        if (c.key == 0) return c;
        const double x = unorder32((uint32_t)(c.key >> 32));
        c.score = order64((double)score + ((x - (double)L.max[c.beam]) - L.lse[c.beam]));
        return c;
    };
    Best mine{0, 0, 0};
    for (int64_t i = t; i < n; i += kThreads) {
        const Best c = candidate(i);
        if (c.score > mine.score) mine = c;
    }
    L.top[t] = (uint32_t)(mine.score >> 32);
    __syncthreads();
    if (wave == 0) {
        const uint32_t T = reach(L.top, kThreads, P.n_out);
        if (lane == 0) L.reach = T;
    }
    __syncthreads();
    const uint32_t T = L.reach;
    for (int64_t i = t; i < n; i += kThreads) {
        const Best c = candidate(i);
        if (c.score == 0 || (uint32_t)(c.score >> 32) < T) continue;
        const int at = atomicAdd(&L.n, 1);
        if (at < kHold) {
            L.score[at] = c.score;
            L.key[at] = c.key;
            L.beam[at] = (uint8_t)c.beam;
        }
    }
    __syncthreads();
    const auto put = [&](int k, const Best& c) {
        const int64_t at = (int64_t)blockIdx.x * P.n_out + k;
        const bool there = c.score != 0;
        const int row = row0 + c.beam, token = (int)~(uint32_t)c.key;
        P.out_scores[at] = there ? (float)unorder64(c.score) : -INFINITY;
        P.parents[at] = there ? row : -1;
        P.tokens[at] = there ? token : -1;
        if (P.out_finished)
            P.out_finished[at] = there && ((P.finished && P.finished[row]) ||
                                           (P.eos >= 0 && token == P.eos));
    };
    const int found = L.n;
    if (found <= kHold) {
        for (int i = t; i < found; i += kThreads) {
            const Best c{L.score[i], L.key[i], L.beam[i]};
            int rank = 0;
            for (int j = 0; j < found; ++j) rank += ahead(Best{L.score[j], L.key[j], L.beam[j]}, c);
            if (rank < P.n_out) put(rank, c);
        }
        for (int i = found + t; i < P.n_out; i += kThreads) put(i, Best{0, 0, 0});
        return;
    }
    Best last{~0ull, ~0ull, -1};
    for (int k = 0; k < P.n_out; ++k) {
        Best top{0, 0, kMaxBeams};
        for (int64_t i = t; i < n; i += kThreads) {
            const Best c = candidate(i);
            if (c.score != 0 && ahead(last, c) && ahead(c, top)) top = c;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const Best o{__shfl_xor((unsigned long long)top.score, d),
                         __shfl_xor((unsigned long long)top.key, d), __shfl_xor(top.beam, d)};
            if (ahead(o, top)) top = o;
        }
        if (lane == 0) L.one[wave] = top;
        __syncthreads();
        last = L.one[0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i)
            if (ahead(L.one[i], last)) last = L.one[i];
        if (t == 0) put(k, last);
        __syncthreads();
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
    hipLaunchKernelGGL(beam::part_kernel, dim3(l.parts, n_groups * n_beams), dim3(beam::kThreads),
                       0, stream, P);
    hipLaunchKernelGGL(beam::group_kernel, dim3(n_groups), dim3(beam::kThreads), 0, stream, P);
    return (int)hipGetLastError();
}
