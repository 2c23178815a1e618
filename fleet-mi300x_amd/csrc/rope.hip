// Rotary positions: fleet_rope_rotate and fleet_cache_rotate (declarations in
// fleet_moe.h).
//
// A pair (a, b) of a head's values becomes (a cos - b sin, b cos + a sin), with the angle
// of its position and frequency; the bytes of x and out bound many tokens, a launch's
// latency few. An angle costs some seventy-five instructions and serves all heads of its token, so
// a thread takes the same four pairs of several heads where there are enough tokens. Measured: one
// token of 16 heads 2.6 us, 2,000 5.7; 8,001 whole heads of 192 fp32 values (197 MB) 39 us, a
// large copy's 5.1 TB/s.
#include <math.h>

#include "cache_pages.h"
#include "rope.h"

namespace fleet_moe {
namespace rope {

struct Params {
    fleet_rope r;
    const void* x;
    void* out;
    int64_t x_token, x_head, o_token, o_head;
    const int32_t* positions;   // or from the cache:
    const int32_t* lens;
    const int32_t* start;
    cache::Header* h;
    int n_seqs, max_pages;
    int n_tokens, n_heads, width, at;
    int items;                  // of a head: up to four pairs or 16 bytes of other values each
    int pairs;                  // items that are pairs
    int parts;                  // groups of heads
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

// Up to four neighbouring values, anywhere a value may lie: four are one load or store.
template <bool kStream>
__device__ __forceinline__ f32x4 load4(const float* p, int n) {
    if (n >= 4) return kStream ? ld_stream_at<4, f32x4>(p) : ld_global_at<4, f32x4>(p);
    f32x4 v{0.f, 0.f, 0.f, 0.f};
    if (n > 0) v[0] = ld_global(p);
    if (n > 1) v[1] = ld_global(p + 1);
    if (n > 2) v[2] = ld_global(p + 2);
    return v;
}
template <bool kStream>
__device__ __forceinline__ f32x4 load4(const uint16_t* p, int n) {
    const auto one = [&](int i) { return __uint_as_float((uint32_t)ld_global(p + i) << 16); };
    if (n >= 4) {
        const uint64_t w =
            kStream ? ld_stream_at<2, uint64_t>(p) : ld_global_at<2, uint64_t>(p);
        const uint32_t lo = (uint32_t)w, hi = (uint32_t)(w >> 32);
        return f32x4{bf_lo(lo), bf_hi(lo), bf_lo(hi), bf_hi(hi)};
    }
    f32x4 v{0.f, 0.f, 0.f, 0.f};
    if (n > 0) v[0] = one(0);
    if (n > 1) v[1] = one(1);
    if (n > 2) v[2] = one(2);
    return v;
}
template <bool kStream>
__device__ __forceinline__ void store4(float* p, const f32x4& v, int n) {
    if (n >= 4) {
        if (kStream) st_stream_at<4>(p, v);
        else st_global_at<4>(p, v);
        return;
    }
    if (n > 0) st_global(p, v[0]);
    if (n > 1) st_global(p + 1, v[1]);
    if (n > 2) st_global(p + 2, v[2]);
}
template <bool kStream>
__device__ __forceinline__ void store4(uint16_t* p, const f32x4& v, int n) {
    bf16x4 b;
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = (__bf16)v[i];
    const uint64_t w = __builtin_bit_cast(uint64_t, b);
    if (n >= 4) {
        if (kStream) st_stream_at<2>(p, w);
        else st_global_at<2>(p, w);
        return;
    }
    if (n > 0) st_global(p, (uint16_t)w);
    if (n > 1) st_global(p + 1, (uint16_t)(w >> 16));
    if (n > 2) st_global(p + 2, (uint16_t)(w >> 32));
}

// The position of a token, from the sequences' lengths, if it has one.
__device__ __forceinline__ bool cache_position(const Params& P, const int* start, int token,
                                               bool lead, int& pos) {
    int s = token, a = token, z = token + 1;
    if (P.start) {
        int lo = 0, hi = P.n_seqs;                        // the last s with start[s] <= token
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (start[mid] <= token) lo = mid;
            else hi = mid - 1;
        }
        if (lo >= P.n_seqs) return false;
        s = lo;
        a = start[s];
        z = start[s + 1];
        if (token < a || token >= z) return false;        // nobody's
    }
    const int len = cache::checked_len(ld_global(P.lens + s), P.max_pages);
    pos = len - (z - token);
    if (len >= 0 && pos >= 0) return true;
    if (lead) cache::raise(P.h, FLEET_MOE_ABORT_POSITION);
    return false;
}

constexpr int kThreads = 256;

// Values of 16 bytes (8 bytes a thread: 3,000 tokens of 128 heads of 192, bf16, 81 us where this
// takes 62).
template <class T>
__host__ __device__ constexpr int copied() { return 16 / (int)sizeof(T); }

// Thread (slot, item); a slot is a token and kHeads of its heads, an item up to four pairs,
// always four with kFours, or 16 bytes of the other values.
// (Seven waves a SIMD: with the 90 registers the compiler takes otherwise, five, 49 us.)
template <class T, int kHeads, bool kFours, bool kStream>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(7)))
void rope_kernel(Params P) {
    __shared__ int starts[cache::kMaxSeqs + 1];
    if (!P.positions && P.start) {
        for (int i = threadIdx.x; i <= P.n_seqs; i += kThreads)
            starts[i] = cache::clamp_row(ld_global(P.start + i), P.n_tokens);
        __syncthreads();
    }
    const int64_t id = wide_block() * kThreads + threadIdx.x;
    const int64_t slot = id / P.items;
    const int item = (int)(id - slot * P.items);
    const int64_t tok = slot / P.parts;
    if (tok >= P.n_tokens) return;
    const int token = (int)tok, head0 = (int)(slot - tok * P.parts) * kHeads;
    int pos = 0;
    if (P.positions) pos = ld_global(P.positions + token);
    else if (!cache_position(P, starts, token, item == 0 && head0 == 0, pos)) return;
    const T* x = static_cast<const T*>(P.x) + token * P.x_token;
    T* out = static_cast<T*>(P.out) + token * P.o_token;
    const int half = P.r.dim / 2;
    if (item < P.pairs) {
        const int p = 4 * item, n = kFours || half - p > 4 ? 4 : half - p;
        // (the pairs' first values and their second ones, or pairs as they are)
        const bool hin = P.r.halves_in, hout = P.r.halves_out;
        const int xa = P.at + (hin ? p : 2 * p), xb = hin ? xa + half : xa + 4;
        const int oa = P.at + (hout ? p : 2 * p), ob = hout ? oa + half : oa + 4;
        const int xn = kFours || hin ? n : 2 * n, xm = kFours || hin ? n : 2 * n - 4;
        const int on = kFours || hout ? n : 2 * n, om = kFours || hout ? n : 2 * n - 4;
        float2 cs[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            cs[i] = angle(ld_global(P.r.turns + (i < n ? p + i : p)), pos, P.r.magnitude);
        f32x4 a[kHeads], b[kHeads];
#pragma unroll
        for (int j = 0; j < kHeads; ++j)
            if (head0 + j < P.n_heads) {
                a[j] = load4<kStream>(x + (head0 + j) * P.x_head + xa, xn);
                b[j] = load4<kStream>(x + (head0 + j) * P.x_head + xb, xm);
            }
#pragma unroll
        for (int j = 0; j < kHeads; ++j) {
            if (head0 + j < P.n_heads) {
                // the pairs' values as they lie, apart; then the result as it is to lie
                const f32x4 u = hin ? a[j] : f32x4{a[j][0], a[j][2], b[j][0], b[j][2]};
                const f32x4 v = hin ? b[j] : f32x4{a[j][1], a[j][3], b[j][1], b[j][3]};
                f32x4 f, g;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    f[i] = fmaf(u[i], cs[i].x, -(v[i] * cs[i].y));
                    g[i] = fmaf(v[i], cs[i].x, u[i] * cs[i].y);
                }
                T* to = out + (head0 + j) * P.o_head;
                store4<kStream>(to + oa, hout ? f : f32x4{f[0], g[0], f[1], g[1]}, on);
                store4<kStream>(to + ob, hout ? g : f32x4{f[2], g[2], f[3], g[3]}, om);
            }
        }
    } else {
        // what is before the rotated part, and what is behind it, as it is
        constexpr int kCopied = copied<T>();
        const int front = (P.at + kCopied - 1) / kCopied, k = item - P.pairs;
        const int at = k < front ? kCopied * k : P.at + P.r.dim + kCopied * (k - front);
        const int n = (k < front ? P.at : P.width) - at;
        if (n >= kCopied) {
            u32x4 a[kHeads];
#pragma unroll
            for (int j = 0; j < kHeads; ++j)
                if (head0 + j < P.n_heads) {
                    const T* from = x + (head0 + j) * P.x_head + at;
                    a[j] = kStream ? ld_stream_at<sizeof(T), u32x4>(from)
                                   : ld_global_at<sizeof(T), u32x4>(from);
                }
#pragma unroll
            for (int j = 0; j < kHeads; ++j)
                if (head0 + j < P.n_heads) {
                    T* to = out + (head0 + j) * P.o_head + at;
                    if (kStream) st_stream_at<sizeof(T)>(to, a[j]);
                    else st_global_at<sizeof(T)>(to, a[j]);
                }
        } else {
            int i = at;
            if (sizeof(T) == 2 && n >= 4) {
                uint64_t a[kHeads];
#pragma unroll
                for (int j = 0; j < kHeads; ++j)
                    if (head0 + j < P.n_heads)
                        a[j] = ld_global_at<2, uint64_t>(x + (head0 + j) * P.x_head + i);
#pragma unroll
                for (int j = 0; j < kHeads; ++j)
                    if (head0 + j < P.n_heads) st_global_at<2>(out + (head0 + j) * P.o_head + i, a[j]);
                i += 4;
            }
            for (; i < at + n; ++i) {
                T a[kHeads];
#pragma unroll
                for (int j = 0; j < kHeads; ++j)
                    if (head0 + j < P.n_heads) a[j] = ld_global(x + (head0 + j) * P.x_head + i);
#pragma unroll
                for (int j = 0; j < kHeads; ++j)
                    if (head0 + j < P.n_heads) st_global(out + (head0 + j) * P.o_head + i, a[j]);
            }
        }
    }
}

}  // namespace rope
}  // namespace fleet_moe

using namespace fleet_moe;
using namespace fleet_moe::rope;

int fleet_moe_check_device(int min_cus);

int fleet_moe_check_rope(const fleet_rope* r) {
    if (!r || !r->turns || (uintptr_t)r->turns % 8 || r->dim < 2 || r->dim > FLEET_ROPE_MAX_DIM ||
        r->dim % 2 || (r->halves_in | 1) != 1 || (r->halves_out | 1) != 1 ||
        !(fabsf(r->magnitude) <= 3.402823466e38f))
        return FLEET_MOE_ERR_ARG;
    return 0;
}

// Results of that many bytes go by L2, and so do the values: what reads them next finds little of
// them there (with a copy of the result behind it, 98 MB 72.7 us, through L2 79.6; 49 MB 41.0
// and 39.4, the rotation alone 21.5 and 24.3).
constexpr int64_t kStreamed = 64 << 20;
template <class T>
static int launch_rope(Params& P, hipStream_t stream) {
    P.pairs = (P.r.dim / 2 + 3) / 4;
    P.items = P.pairs;
    if (P.out != P.x)                             // (in place, what is not rotated is there)
        P.items += (P.at + copied<T>() - 1) / copied<T>() +
                   (P.width - P.at - P.r.dim + copied<T>() - 1) / copied<T>();
    // Four heads a thread where that still leaves two workgroups a CU.
    const bool many = (int64_t)P.n_tokens * ((P.n_heads + 3) / 4) * P.items >= 512 * kThreads;
    P.parts = many ? (P.n_heads + 3) / 4 : P.n_heads;
    const int64_t n = (int64_t)P.n_tokens * P.parts * P.items;
    const int64_t grid = (n + kThreads - 1) / kThreads;
    if (grid > 65535 * kGridRow) return FLEET_MOE_ERR_ARG;
    const auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, wide_grid(grid), dim3(kThreads), 0, stream, P);
        return (int)hipGetLastError();
    };
    const int64_t values = (int64_t)P.n_tokens * P.n_heads * P.width;
    const bool large = many && values >= kStreamed / (int64_t)sizeof(T);
    if (P.r.dim / 2 % 4 == 0) {
        if (large) return launch(rope_kernel<T, 4, true, true>);
        return many ? launch(rope_kernel<T, 4, true, false>) : launch(rope_kernel<T, 1, true, false>);
    }
    if (large) return launch(rope_kernel<T, 4, false, true>);
    return many ? launch(rope_kernel<T, 4, false, false>) : launch(rope_kernel<T, 1, false, false>);
}

static int rotate(Params& P, bool f32, hipStream_t stream) {
    const int64_t most = (int64_t)1 << 32, w = P.width, t = P.n_tokens, n = P.n_heads;
    if (int e = fleet_moe_check_rope(&P.r)) return e;
    if (P.n_tokens < 0 || P.n_tokens > (1 << 28) || P.n_heads < 1 || P.n_heads > (1 << 16) ||
        P.at < 0 || P.width < P.r.dim || P.at > P.width - P.r.dim ||
        P.width > FLEET_ROPE_MAX_WIDTH)
        return FLEET_MOE_ERR_ARG;
    if (P.n_tokens == 0) return 0;
    const int size = f32 ? 4 : 2;
    if (!P.x || !P.out || (uintptr_t)P.x % size || (uintptr_t)P.out % size || P.x_token < 0 ||
        P.x_token > most || P.x_head < 0 || P.x_head > most || P.o_token < 0 || P.o_token > most ||
        P.o_head < 0 || P.o_head > most)
        return FLEET_MOE_ERR_ARG;
    // no two heads are written to one place
    if ((n > 1 && P.o_head < w) || (t > 1 && P.o_token < w) ||
        (n > 1 && t > 1 && P.o_token < (n - 1) * P.o_head + w &&
         P.o_head < (t - 1) * P.o_token + w))
        return FLEET_MOE_ERR_ARG;
    // in place, a head's values stay with the thread that reads them
    if (P.out == P.x && (P.r.halves_in != P.r.halves_out || (n > 1 && P.x_head != P.o_head) ||
                         (t > 1 && P.x_token != P.o_token)))
        return FLEET_MOE_ERR_ARG;
    if (int e = fleet_moe_check_device(1)) return e;
    return f32 ? launch_rope<float>(P, stream) : launch_rope<uint16_t>(P, stream);
}

static Params rope_params(const fleet_rope* rope, const void* x, int64_t x_token, int64_t x_head,
                          void* out, int64_t out_token, int64_t out_head, int32_t n_tokens,
                          int32_t n_heads, int32_t width, int32_t at) {
    Params P{};
    if (rope) P.r = *rope;
    P.x = x;
    P.out = out;
    P.x_token = x_token;
    P.x_head = x_head;
    P.o_token = out_token;
    P.o_head = out_head;
    P.n_tokens = n_tokens;
    P.n_heads = n_heads;
    P.width = width;
    P.at = at;
    return P;
}

extern "C" int fleet_rope_rotate(const fleet_rope* rope, const void* x, int32_t f32,
                                 int64_t x_token, int64_t x_head, void* out, int64_t out_token,
                                 int64_t out_head, const int32_t* positions, int32_t n_tokens,
                                 int32_t n_heads, int32_t width, int32_t at, hipStream_t stream) {
    if ((f32 | 1) != 1 || (uintptr_t)positions % 4 || (n_tokens > 0 && !positions))
        return FLEET_MOE_ERR_ARG;
    Params P = rope_params(rope, x, x_token, x_head, out, out_token, out_head, n_tokens, n_heads,
                           width, at);
    P.positions = positions;
    return rotate(P, f32, stream);
}

extern "C" int fleet_cache_rotate(const fleet_cache* cache, const fleet_rope* rope, const void* x,
                                  int32_t f32, int64_t x_token, int64_t x_head, void* out,
                                  int64_t out_token, int64_t out_head, const int32_t* start,
                                  int32_t n_tokens, int32_t n_heads, int32_t width, int32_t at,
                                  void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (int e = cache::check_cache(cache, workspace, workspace_bytes)) return e;
    if ((f32 | 1) != 1 || (uintptr_t)start % 4 || (!start && n_tokens != cache->n_seqs))
        return FLEET_MOE_ERR_ARG;
    Params P = rope_params(rope, x, x_token, x_head, out, out_token, out_head, n_tokens, n_heads,
                           width, at);
    P.lens = cache->lens;
    P.start = start;
    P.h = static_cast<cache::Header*>(workspace);
    P.n_seqs = cache->n_seqs;
    P.max_pages = cache->max_pages;
    return rotate(P, f32, stream);
}
