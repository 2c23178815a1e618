// What the kernels that attend over the 8-bit cache share: the copies from a page to
// LDS, the operands of the matrix instructions that its bytes make, and the arithmetic of a
// running softmax.
#pragma once

#include <float.h>
#include <math.h>

#include <atomic>

#include "cache_pages.h"

namespace fleet_moe {
namespace cache {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

constexpr float kSlack = 8.f;
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;

// Blocks in LDS lie 64 bytes further apart than they are long, so that the two
// halves of a transposing read, from neighbouring blocks, fall into different banks.
constexpr int kBlockStep = kBlockBytes + 64;

// Copies kN times 1 KB from global memory to LDS, 16 bytes a lane: from `src` (the
// lane's) + 1024 i to `lds` + 1024 i + 16 lane (the offset counts on both sides). There
// is no register for the data, so none is in flight behind the compiler's back. In
// asm, because the compiler would wait for every copy in flight before each LDS read;
// wait_copies() orders them. kOnce: not kept in the caches.
template <int kN, bool kOnce>
__device__ __forceinline__ void copy_kb(const uint8_t* src, uint32_t lds) {
    static_assert(kN == 1 || kN == 4, "");
    if constexpr (kN == 4 && kOnce)
        asm volatile(
            "s_nop 0\n\t"
            "global_load_lds_dwordx4 %0, off nt\n\t"
            "global_load_lds_dwordx4 %0, off offset:1024 nt\n\t"
            "global_load_lds_dwordx4 %0, off offset:2048 nt\n\t"
            "global_load_lds_dwordx4 %0, off offset:%2 nt" ::"v"(src), "{m0}"(lds), "n"(3 * 1024)
            : "memory");
    else if constexpr (kN == 4)
        asm volatile(
            "s_nop 0\n\t"
            "global_load_lds_dwordx4 %0, off\n\t"
            "global_load_lds_dwordx4 %0, off offset:1024\n\t"
            "global_load_lds_dwordx4 %0, off offset:2048\n\t"
            "global_load_lds_dwordx4 %0, off offset:%2" ::"v"(src), "{m0}"(lds), "n"(3 * 1024)
            : "memory");
    else if constexpr (kOnce)
        asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(src), "{m0}"(lds)
                     : "memory");
    else
        asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(lds)
                     : "memory");
}
template <int kLeft>
__device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLeft) : "memory");
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
// The workgroup's barrier, without waiting for copies in flight.
__device__ __forceinline__ void barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

__device__ __forceinline__ bf16x8 widen(uint32_t lo, uint32_t hi, float slo, float shi) {
    u32x4 r;
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, slo, false));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, slo, true));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, shi, false));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, shi, true));
    return __builtin_bit_cast(bf16x8, r);
}

// The scale of a block, or of one that holds no position yet and may have any bytes: a
// power of two up to the largest that append writes.
constexpr uint32_t kMaxScale = 0x7b800000u;     // 2^120
__device__ __forceinline__ float any_scale(uint32_t w) {
    w &= 0x7f800000u;
    return __uint_as_float(w < kMaxScale ? w : kMaxScale);
}

// The codes of a word that stand for no finite value as zeros: NaN (0x7f, 0xff) and,
// with the largest scale, 256 and more, which are infinite in bf16.
__device__ __forceinline__ uint32_t drop_infinite(uint32_t w, bool largest) {
    const uint32_t n = ((w & 0x7f7f7f7fu) + (largest ? 0x08080808u : 0x01010101u)) & 0x80808080u;
    return w & ~(n | (n - (n >> 7)));
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }

__device__ __forceinline__ float xor16_max(float v) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v),
                                                    false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float xor32_max(float v) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v),
                                                    false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// A row's reference in the exponent: of a finite score that is infinite times the scale,
// all weights would be exp2(finite - infinity) = 0, as if nothing were seen.
__device__ __forceinline__ float reference(float scaled) {
    return scaled == INFINITY ? __uint_as_float(0x7fc00000u) : scaled;
}
// What the sums so far are multiplied by; with the reference -infinity there are none.
__device__ __forceinline__ float shrink_to(float ref, float was) {
    return was == -INFINITY ? 1.f : exp2_(was - ref);
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Four weights as bf16.
__device__ __forceinline__ uint2 weights(const float (&p)[4]) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    bf16x2 a, b;
    a[0] = (__bf16)p[0];
    a[1] = (__bf16)p[1];
    b[0] = (__bf16)p[2];
    b[1] = (__bf16)p[3];
    return make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
}

// The transposing read: 8 positions of one of the 16 dimensions of chunk i, from the LDS
// address `col` of the first block and column_at(): lane r of a group of 16 points at row
// r / 2 of 8, positions 4g .. 4g + 3 of two neighbouring blocks. (Addresses as numbers: then
// the chunk is the instruction's own offset, not two additions.)
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
__device__ __forceinline__ uint32_t column_at(int lane) {
    const int r = (lane & 15) >> 1;
    return (r < 4 ? 0 : kBlockStep) + (4 * (lane >> 4) + (r & 3)) * 16 + (lane & 1) * 8;
}
__device__ __forceinline__ i32x2 column(uint32_t col, int i) {
    return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(uintptr_t)(col + i * 256));
}

// A block's values that are not finite as zeros, by one wave. Such a value makes the
// score of every row of q infinite or NaN, and the weight of one that sees it NaN or 0; a
// row that does not see it has the weight 0, and must not meet 0 * NaN. (Its score tells:
// the wave looks at the scores before it hides those of positions that are not seen.)
__device__ __forceinline__ void clean(uint8_t* block, uint32_t scale, int lane) {
    const bool largest = any_scale(scale) == __uint_as_float(kMaxScale);
    for (int i = 0; i < kC / 64; ++i) {
        u32x4* at = reinterpret_cast<u32x4*>(block + i * 1024 + lane * 16);
        u32x4 v = *at;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = drop_infinite(v[j], largest);
        *at = v;
    }
}

// What their rounding leaves of them, as bf16.
__device__ __forceinline__ uint2 rest(const float (&p)[4], uint2 w) {
    const float r[4] = {p[0] - bf_lo(w.x), p[1] - bf_hi(w.x), p[2] - bf_lo(w.y),
                        p[3] - bf_hi(w.y)};
    return weights(r);
}

__device__ __forceinline__ uint32_t bf16x2_bits(float a, float b) {
    return bf16_bits(a) | bf16_bits(b) << 16;
}
__device__ __forceinline__ void put(uint16_t* out, const f32x4& o, float inv) {
    const uint64_t b = (uint64_t)bf16x2_bits(o[0] * inv, o[1] * inv) |
                       (uint64_t)bf16x2_bits(o[2] * inv, o[3] * inv) << 32;
    st_global(reinterpret_cast<uint64_t*>(out), b);
}
__device__ __forceinline__ float lse_of(float m, float sum) {
    return sum == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(sum)) * kLn2;
}
constexpr uint32_t kOnes = 0x3f803f80u;                   // bf16 1, 1

// More than 64 KB of dynamic LDS has to be asked for. (The LDS is dynamic so that
// the compiler keeps to the registers of two waves on a SIMD, and takes O as an
// operand of the matrix instructions from them; where it knows that LDS allows one
// only, it moves O to accumulation registers and back, 400 moves a step.)
template <auto Kernel, class Params>
static int launch(int64_t grid, int threads, size_t lds, const Params& P, hipStream_t stream) {
    if (lds > 64 * 1024) {
        static std::atomic<uint64_t> asked{0};  // once a device
        int dev = 0;
        hipError_t e = hipGetDevice(&dev);
        const uint64_t bit = dev < 64 ? 1ull << dev : 0;
        if (e == hipSuccess && !(asked.load() & bit)) {
            e = hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e == hipSuccess) asked.fetch_or(bit);
        }
        if (e != hipSuccess) return (int)e;
    }
    hipLaunchKernelGGL(Kernel, dim3((unsigned)grid), dim3(threads), lds, stream, P);
    return (int)hipGetLastError();
}

}  // namespace cache
}  // namespace fleet_moe
