// The norms around a block, with its gate and its residual: fleet_residual_norm
// (declaration in fleet_moe.h).
//
//   u  = y, or y / rms(y) * post_norm        rms(v) = sqrt(mean(v^2) + eps)
//   x' = x + scale * gate * u
//   h  = x' / rms(x') * norm
//
// One pass: a row's values stay in registers from their load to h, so x, y and a gate of
// every token are read once, x' and h written once, and those bytes are the bound. All
// arithmetic is fp32; x' and h are each rounded once, and h is taken from x' before its
// rounding. Measured: a row of 2,048 values 2.6 us, 250 rows 4.5; 16,000 rows
// (328 MB, with a gate of every token) 61 us, 5.4 TB/s, where a large copy reaches 5.1.
#include <math.h>

#include "cache_pages.h"

namespace fleet_moe {
namespace norm {

struct Params {
    const void* x;
    const void* y;
    const uint16_t* post;
    const uint16_t* gate;
    const uint16_t* weight;
    void* x_out;
    uint16_t* h;
    float* h_f32;
    int64_t x_stride, y_stride, gate_stride;
    float scale, eps;
    int rows, width;
    bool x_f32, y_f32;
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pack(float a, float b) {
    bf16x2 v;
    v[0] = (__bf16)a;
    v[1] = (__bf16)b;
    return __builtin_bit_cast(uint32_t, v);
}

// A thread's values of a row: kN chunks of 8, chunk i from value 8 * (t + i * kThreads) on.
// A row's last chunk may be short; what is behind the row is 0. (A row may begin anywhere a
// value may: odd widths take 70 us where one value at a time took 200, of 3,000 rows of 8,191.)
template <int kThreads, int kN>
struct Row {
    static constexpr int kValues = 8 * kN;
    float v[kValues];

    // whole(i, at) for a chunk of v[i ..] at value `at`, one(i, at) for a value of a short one
    template <class F, class G>
    __device__ __forceinline__ static void each(int t, int width, F whole, G one) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int at = 8 * (t + i * kThreads);
            if (at + 8 <= width) {
                whole(8 * i, at);
            } else if (at < width) {
#pragma unroll
                for (int k = 0; k < 7; ++k)
                    if (at + k < width) one(8 * i + k, at + k);
            }
        }
    }
    __device__ __forceinline__ void load(const uint16_t* p, int t, int width) {
#pragma unroll
        for (auto& e : v) e = 0.f;
        each(t, width,
             [&](int i, int at) {
                 const u32x4 w = ld_global_at<2, u32x4>(p + at);
#pragma unroll
                 for (int k = 0; k < 4; ++k) {
                     v[i + 2 * k] = bf_lo(w[k]);
                     v[i + 2 * k + 1] = bf_hi(w[k]);
                 }
             },
             [&](int i, int at) { v[i] = __uint_as_float((uint32_t)ld_global(p + at) << 16); });
    }
    __device__ __forceinline__ void load(const float* p, int t, int width) {
#pragma unroll
        for (auto& e : v) e = 0.f;
        each(t, width,
             [&](int i, int at) {
                 const f32x4 a = ld_global_at<4, f32x4>(p + at);
                 const f32x4 b = ld_global_at<4, f32x4>(p + at + 4);
#pragma unroll
                 for (int k = 0; k < 4; ++k) {
                     v[i + k] = a[k];
                     v[i + 4 + k] = b[k];
                 }
             },
             [&](int i, int at) { v[i] = ld_global(p + at); });
    }
    __device__ __forceinline__ void store(uint16_t* p, int t, int width) const {
        each(t, width,
             [&](int i, int at) {
                 u32x4 w;
#pragma unroll
                 for (int k = 0; k < 4; ++k) w[k] = pack(v[i + 2 * k], v[i + 2 * k + 1]);
                 st_global_at<2>(p + at, w);
             },
             [&](int i, int at) { st_global(p + at, (uint16_t)pack(v[i], 0.f)); });
    }
    __device__ __forceinline__ void store(float* p, int t, int width) const {
        each(t, width,
             [&](int i, int at) {
                 st_global_at<4>(p + at, f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]});
                 st_global_at<4>(p + at + 4, f32x4{v[i + 4], v[i + 5], v[i + 6], v[i + 7]});
             },
             [&](int i, int at) { st_global(p + at, v[i]); });
    }
    __device__ __forceinline__ void load(const void* p, bool f32, int64_t at, int t, int width) {
        if (f32) load(static_cast<const float*>(p) + at, t, width);
        else load(static_cast<const uint16_t*>(p) + at, t, width);
    }
};

// The sum over the threads of a row, the same in all of them.
template <int kThreads>
__device__ __forceinline__ float row_sum(float v, float* lds) {
    v = wave_sum(v);
    if constexpr (kThreads > 64) {
        constexpr int kWaves = kThreads / 64;
        const int t = threadIdx.x;
        if ((t & 63) == 0) lds[t >> 6] = v;
        __syncthreads();
        v = wave_sum((t & 63) < kWaves ? lds[t & 63] : 0.f);
        __syncthreads();
    }
    return v;
}

// Divides a row by rms(row). Squares beyond fp32 are taken again of 2^-75 of the values: then
// the sum of 32,768 of the largest is below 2^122, and eps has the same 2^-150 (1e30 is 2% of the
// mean of 32,768 squares of 2^105). (A row with an infinity gets NaN there and zeros elsewhere, as
// the formula says.)
template <int kThreads, class R>
__device__ __forceinline__ void unit(R& r, int width, float eps, float* lds) {
    float s = 0.f;
#pragma unroll
    for (const float& e : r.v) s = fmaf(e, e, s);
    s = row_sum<kThreads>(s, lds);
    const bool large = !(s < 0x1p120f);
    if (large) {
        s = 0.f;
#pragma unroll
        for (const float& e : r.v) {
            const float d = e * 0x1p-75f;
            s = fmaf(d, d, s);
        }
        s = row_sum<kThreads>(s, lds);
        eps = eps * 0x1p-75f * 0x1p-75f;
    }
    float inv = 1.f / sqrtf(s / (float)width + eps);
    if (large) {                                          // (2^-75 in two steps: in range)
        inv *= 0x1p-37f;
#pragma unroll
        for (float& e : r.v) e *= 0x1p-38f;
    }
#pragma unroll
    for (float& e : r.v) e *= inv;
}

// kThreads threads a row, with 8 kN values each; a wave for narrow rows, four a workgroup and
// no barrier.
template <int kThreads, int kN>
__global__ __launch_bounds__(kThreads > 256 ? kThreads : 256) void norm_kernel(Params P) {
    __shared__ float lds[16];
    constexpr int kRows = kThreads > 256 ? 1 : 256 / kThreads;
    const int t = threadIdx.x % kThreads;
    const int64_t row = wide_block() * kRows + threadIdx.x / kThreads;
    if (row >= P.rows) return;
    const int w = P.width;
    Row<kThreads, kN> x, u, f;
    x.load(P.x, P.x_f32, row * P.x_stride, t, w);
    if (P.y) {
        u.load(P.y, P.y_f32, row * P.y_stride, t, w);
        if (P.post) {
            f.load(P.post, t, w);
            unit<kThreads>(u, w, P.eps, lds);
#pragma unroll
            for (int i = 0; i < 8 * kN; ++i) u.v[i] *= f.v[i];
        }
        if (P.gate) {
            f.load(P.gate + row * P.gate_stride, t, w);
#pragma unroll
            for (int i = 0; i < 8 * kN; ++i) u.v[i] *= f.v[i];
        }
#pragma unroll
        for (int i = 0; i < 8 * kN; ++i) x.v[i] = fmaf(P.scale, u.v[i], x.v[i]);
        if (P.x_out) {
            if (P.x_f32) x.store(static_cast<float*>(P.x_out) + row * w, t, w);
            else x.store(static_cast<uint16_t*>(P.x_out) + row * w, t, w);
        }
    }
    unit<kThreads>(x, w, P.eps, lds);
    if (P.weight) {
        f.load(P.weight, t, w);
#pragma unroll
        for (int i = 0; i < 8 * kN; ++i) x.v[i] *= f.v[i];
    }
    x.store(P.h + row * w, t, w);
    if (P.h_f32) {
#pragma unroll
        for (float& e : x.v) e = (float)(__bf16)e;
        x.store(P.h_f32 + row * w, t, w);
    }
}

}  // namespace norm
}  // namespace fleet_moe

using namespace fleet_moe;
using namespace fleet_moe::norm;

int fleet_moe_check_device(int min_cus);

template <int kThreads, int kN>
static int launch_norm(const Params& P, hipStream_t stream) {
    constexpr int kBlock = kThreads > 256 ? kThreads : 256, kRows = kBlock / kThreads;
    hipLaunchKernelGGL((norm_kernel<kThreads, kN>), wide_grid((P.rows + kRows - 1) / kRows),
                       dim3(kBlock), 0, stream, P);
    return (int)hipGetLastError();
}

extern "C" int fleet_residual_norm(const void* x, int32_t x_f32, int64_t x_stride, const void* y,
                                   int32_t y_f32, int64_t y_stride, const uint16_t* post_norm,
                                   const uint16_t* gate, int64_t gate_stride, float scale,
                                   const uint16_t* norm, float eps, void* x_out, uint16_t* h,
                                   float* h_f32, int32_t n_rows, int32_t width,
                                   hipStream_t stream) {
    if (n_rows < 0 || n_rows > FLEET_NORM_MAX_ROWS || width < 1 || width > FLEET_NORM_MAX_WIDTH ||
        (x_f32 | 1) != 1 || (y_f32 | 1) != 1 || !(eps >= 1e-30f) || !(eps <= 1e30f) ||
        !(fabsf(scale) <= 3.402823466e38f))
        return FLEET_MOE_ERR_ARG;
    if (!y && (post_norm || gate || x_out)) return FLEET_MOE_ERR_ARG;
    if (n_rows == 0) return 0;
    const int64_t most = (int64_t)1 << 32;
    if (!x || !h || x_stride < 0 || x_stride > most || y_stride < 0 || y_stride > most ||
        gate_stride < 0 || gate_stride > most || (uintptr_t)x % (x_f32 ? 4 : 2) ||
        (uintptr_t)y % (y_f32 ? 4 : 2) || (uintptr_t)x_out % (x_f32 ? 4 : 2) ||
        (uintptr_t)post_norm % 2 || (uintptr_t)gate % 2 || (uintptr_t)norm % 2 ||
        (uintptr_t)h % 2 || (uintptr_t)h_f32 % 4)
        return FLEET_MOE_ERR_ARG;
    // in place only where a row is written where it was read
    if (x_out == x && n_rows > 1 && x_stride != width) return FLEET_MOE_ERR_ARG;
    if (int e = fleet_moe_check_device(1)) return e;
    Params P{};
    P.x = x;
    P.y = y;
    P.post = post_norm;
    P.gate = gate;
    P.weight = norm;
    P.x_out = x_out;
    P.h = h;
    P.h_f32 = h_f32;
    P.x_stride = x_stride;
    P.y_stride = y_stride;
    P.gate_stride = gate_stride;
    P.scale = scale;
    P.eps = eps;
    P.rows = n_rows;
    P.width = width;
    P.x_f32 = x_f32;
    P.y_f32 = y_f32;
    // As few threads as hold a row, in steps that leave few of them without values: 300 MB in rows
    // of 1,000 values take 56 us, by 256 threads 83; of 1,500 78, by 256 108; of 2,048 62, by a wave
    // 75; of 3,500 69, by 512 96; of 6,000 67, by 256 with three chunks 74; of 10,000 59, by 1,024
    // with four 100; of 20,000 72, with four 75.
    if (width <= 512) return launch_norm<64, 1>(P, stream);
    if (width <= 1024) return launch_norm<64, 2>(P, stream);
    if (width <= 1536) return launch_norm<64, 3>(P, stream);
    if (width <= 2048) return launch_norm<256, 1>(P, stream);
    if (width <= 4096) return launch_norm<256, 2>(P, stream);
    if (width <= 8192) return launch_norm<512, 2>(P, stream);
    if (width <= 16384) return launch_norm<1024, 2>(P, stream);
    if (width <= 24576) return launch_norm<1024, 3>(P, stream);
    return launch_norm<1024, 4>(P, stream);
}
