// What the kernels that write or read rows of the 8-bit cache share: the block of 16
// positions that a workgroup takes, and the conversions of its values.
#pragma once

#include "cache_pages.h"

namespace fleet_moe {
namespace cache {

// Nine waves: wave w holds chunks 4w .. 4w + 3, so the last wave holds exactly
// k_pe and the others c, and a row's four chunks are 128 consecutive bytes.
constexpr int kRowThreads = kBlock * kChunks;
static_assert(kRowThreads == 9 * 64, "");

struct RowParams {
    fleet_cache c;
    uint16_t* rows;
    int64_t row_stride, layer_stride;
    const int32_t* start;
    Header* h;
    int n_rows, layer0, n_layers;
};

// The block of positions of a workgroup, and its rows.
struct BlockAt {
    int seq, row0, first, len;      // row0: the row of position `first`
    int base;                       // the block's first position
    int page;
};

template <bool kAppend>
__device__ __forceinline__ bool block_at(const RowParams& P, BlockAt& b) {
    const fleet_cache& c = P.c;
    const int64_t u = blockIdx.x;
    b.seq = find_seq(P.start, c.n_seqs, P.n_rows, u, 1, kBlock, 2);
    if (b.seq < 0) return false;
    const int a = P.start ? clamp_row(P.start[b.seq], P.n_rows) : b.seq;
    const int z = P.start ? clamp_row(P.start[b.seq + 1], P.n_rows) : b.seq + 1;
    if (z <= a || u < first_unit(a, b.seq, 1, kBlock, 2)) return false;
    b.len = checked_len(c.lens[b.seq], c.max_pages);
    b.first = b.len - (z - a);
    b.row0 = a;
    const bool lead = threadIdx.x == 0 && blockIdx.y == 0 &&
                      u == first_unit(a, b.seq, 1, kBlock, 2);
    if (b.len < 0 || b.first < 0) {
        if (lead) {
            // (without the room that a grow refused, there may be fewer positions than rows)
            const uint32_t refused = kAppend ? P.h->refused : 0;
            raise(P.h, refused ? refused : (uint32_t)FLEET_MOE_ABORT_POSITION);
        }
        if (b.len < 0) return false;
    }
    const int lo = b.first < 0 ? 0 : b.first;
    const int64_t base = (int64_t)(lo / kBlock + (u - first_unit(a, b.seq, 1, kBlock, 2))) * kBlock;
    if (base >= b.len) return false;
    b.base = (int)base;
    b.page = c.table[(int64_t)b.seq * c.max_pages + b.base / kPage];
    if ((unsigned)b.page >= (unsigned)c.n_pages) {
        if (threadIdx.x == 0) raise(P.h, FLEET_MOE_ABORT_BAD_PAGE);
        return false;
    }
    return true;
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Four values as e4m3 bytes, to nearest even, values beyond +-448 (infinities)
// to +-448.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    const auto sat = [](float v) { return v != v ? v : fminf(fmaxf(v, -448.f), 448.f); };
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(sat(a), sat(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(sat(c), sat(d), r, true);
}

// The two bf16 values (bits) of the low or high half of a word of codes, times a
// power of two: exact.
template <bool kHigh>
__device__ __forceinline__ uint32_t bf16x2(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t,
                              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, kHigh));
}

// 16 codes under a scale 2^-by as large.
__device__ __forceinline__ u32x4 rescaled(const u32x4& o, int by) {
    const float down = pow2(by < -126 ? -126 : by);
    u32x4 n;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = bf16x2<false>(o[i], 1.f), hi = bf16x2<true>(o[i], 1.f);
        n[i] = e4m3x4(bf_lo(lo) * down, bf_hi(lo) * down, bf_lo(hi) * down, bf_hi(hi) * down);
    }
    return n;
}

// The exponent of a block's scale as it was, within what append writes.
__device__ __forceinline__ int exp_of(uint32_t scale) {
    const int e = (int)(scale >> 23 & 255) - 127;
    return e < -110 ? -110 : e > 120 ? 120 : e;
}

}  // namespace cache
}  // namespace fleet_moe
