// Projected rows into the 8-bit cache: fleet_cache_append_latent (declaration in
// fleet_moe.h).
//
// A row of kv_a_proj, [c (512) | k_pe (64)] in bf16, becomes the cache's row
//   c / sqrt(mean(c^2) + eps) * norm,  k_pe rotated by its position,
// in fp32, and is rounded once, to the 8 bits of its block. A workgroup takes one block of
// 16 positions as fleet_cache_append does; beside it the 8 waves of c share their rows' sums of
// squares, and all waves compute an angle a thread (16 positions of 32 pairs) while the
// rows are on their way.
//
// One row for each of 17 sequences: 5.3 us, the latency of the loads before the rows (start,
// length, table), the angle and two barriers. 11,004 rows: 10.8 us (19 MB, 1.8 TB/s; a copy of as
// much takes 4): that latency once, with every workgroup of the call on the chip (70
// registers; with 83 only two workgroups a CU, 13.5), and 424 vector instructions a wave.
#include <math.h>

#include "cache_rows.h"
#include "rope.h"

namespace fleet_moe {
namespace cache {

struct LatentParams {
    RowParams r;
    fleet_rope rope;
    const uint16_t* norm;
    float eps;
};

// The least e with a <= 448 * 2^e for the magnitude bits a of a finite fp32, at least -110.
__device__ __forceinline__ int scale_exp32(uint32_t bits) {
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000);
    return e < -110 ? -110 : e;
}

__global__ __launch_bounds__(kRowThreads) void latent_kernel(LatentParams P) {
    constexpr int kPairs = (kRow - kC) / 2;
    __shared__ float2 cs[kBlock][kPairs + 1];
    __shared__ double squares[8][kBlock];
    __shared__ uint32_t most[8];
    const int t = threadIdx.x, lane = t & 63, wave = wave_bcast(t >> 6);
    const int tok = lane >> 2, part = lane & 3, chunk = 4 * wave + part;
    // what depends on no position is on its way first
    const double turns = ld_global(P.rope.turns + t % kPairs);
    u32x4 w[2];
    if (P.norm && wave < 8) {
        w[0] = ld_global(reinterpret_cast<const u32x4*>(P.norm + chunk * 16));
        w[1] = ld_global(reinterpret_cast<const u32x4*>(P.norm + chunk * 16) + 1);
    }
    BlockAt b;
    if (!block_at<true>(P.r, b)) return;
    const fleet_cache& c = P.r.c;
    const int holders = c.refs[b.page];
    const uint32_t refused = P.r.h->refused;
    uint8_t* page = c.pool + page_offset(b.page, c.n_pages, P.r.layer0, c.n_layers);
    const int blk = b.base % kPage / kBlock;
    u32x4* mine = reinterpret_cast<u32x4*>(page + blk * kBlockBytes) + chunk * kBlock + tok;
    uint32_t* scale = reinterpret_cast<uint32_t*>(page + kCodeBytes) + 2 * blk + (wave == 8);
    const int pos = b.base + tok;
    const bool fresh = pos >= b.first && pos < b.len;
    const bool aged = b.base < b.first;                   // older positions in the block
    // c: a lane's 16 values; k_pe: the 16 pairs of which it makes the first or second values
    u32x4 in[4] = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
    if (fresh) {
        const uint16_t* row = P.r.rows + (int64_t)(b.row0 + pos - b.first) * P.r.row_stride;
        if (wave < 8) {
            const u32x4* at = reinterpret_cast<const u32x4*>(row + chunk * 16);
            in[0] = ld_stream(at);
            in[1] = ld_stream(at + 1);
        } else {
            const bool halves = P.rope.halves_in;
            const u32x4* at = reinterpret_cast<const u32x4*>(row + kC + (part & 1) * (halves ? 16 : 32));
            const int second = halves ? kPairs / 8 : 2;
            in[0] = ld_global(at);
            in[1] = ld_global(at + 1);
            in[2] = ld_global(at + second);
            in[3] = ld_global(at + second + 1);
        }
    }
    const uint32_t was = aged ? ld_global(scale) : 0;
    if (t < kBlock * kPairs)
        cs[t / kPairs][t % kPairs] = rope::angle(turns, b.base + t / kPairs, P.rope.magnitude);
    float v[16];
    if (wave < 8) {
        // (64 bits: the squares of any finite bf16 fit, and cost what 32 cost)
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t x = in[i / 4][i % 4];
            v[2 * i] = bf_lo(x);
            v[2 * i + 1] = bf_hi(x);
            s = fma((double)v[2 * i], (double)v[2 * i], s);
            s = fma((double)v[2 * i + 1], (double)v[2 * i + 1], s);
        }
        s += __shfl_xor(s, 1);
        s += __shfl_xor(s, 2);
        if (part == 0) squares[wave][tok] = s;
    }
    __syncthreads();
    if (wave < 8) {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += squares[i][tok];
        s = s * (1.0 / kC) + (double)P.eps;
        // (good to 2^-24; where it is below the least fp32, the values take part of it)
        const double inv = __builtin_amdgcn_rsq(s);
        if (s > 0x1p200) {
            const float rms = (float)(inv * 0x1p64);
#pragma unroll
            for (float& x : v) x = x * 0x1p-64f * rms;
        } else {
            const float rms = (float)inv;
#pragma unroll
            for (float& x : v) x *= rms;
        }
        if (P.norm)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[2 * i] *= bf_lo(w[i / 4][i % 4]);
                v[2 * i + 1] *= bf_hi(w[i / 4][i % 4]);
            }
    } else {
        // first values (parts 0, 1) are p cos - q sin, second ones q cos + p sin
        const bool halves = P.rope.halves_in, second = part >= 2;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float2 a = cs[tok][(part & 1) * 16 + i];
            const uint32_t w0 = in[i / 8][i / 2 % 4], w1 = in[2 + i / 8][i / 2 % 4];
            const uint32_t both = in[i / 4][i % 4];
            const float p = halves ? (i % 2 ? bf_hi(w0) : bf_lo(w0)) : bf_lo(both);
            const float q = halves ? (i % 2 ? bf_hi(w1) : bf_lo(w1)) : bf_hi(both);
            v[i] = fmaf(second ? q : p, a.x, (second ? p : -q) * a.y);
        }
    }
    // the largest finite magnitude, as bits: they order as the values do (rows that are not new
    // are zeros here; a maximum leaves NaN out, and the infinities are rare)
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i += 2) top = fmaxf(fmaxf(top, fabsf(v[i])), fabsf(v[i + 1]));
    if (!(top < INFINITY)) {
        top = 0.f;
#pragma unroll
        for (const float& x : v) top = fabsf(x) < INFINITY ? fmaxf(top, fabsf(x)) : top;
    }
    uint32_t big = __float_as_uint(top);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_xor(big, d);
        big = o > big ? o : big;
    }
    if (wave < 8 && lane == 0) most[wave] = big;
    __syncthreads();
    if (wave < 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) big = most[i] > big ? most[i] : big;
    }
    // without room for the new positions the last ones are older rows
    if (refused || holders != 1) {
        if (t == 0) raise(P.r.h, refused ? refused : (uint32_t)FLEET_MOE_ABORT_BAD_PAGE);
        return;
    }
    int e = scale_exp32(big);
    const int e_old = exp_of(was);
    if (aged && e_old > e) e = e_old;
    const float inv = pow2(-e);
    if (fresh) {
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o[i] = e4m3x4(v[4 * i] * inv, v[4 * i + 1] * inv, v[4 * i + 2] * inv,
                          v[4 * i + 3] * inv);
        st_global(mine, o);
    } else if (aged && e > e_old && pos < b.first) {
        st_global(mine, rescaled(ld_global(mine), e_old - e));
    }
    if (lane == 0 && (wave == 0 || wave == 8)) st_global(scale, (uint32_t)(e + 127) << 23);
}

}  // namespace cache
}  // namespace fleet_moe

using namespace fleet_moe;
using namespace fleet_moe::cache;

int fleet_moe_check_device(int min_cus);
int fleet_moe_check_rope(const fleet_rope* r);

extern "C" int fleet_cache_append_latent(const fleet_cache* cache, int32_t layer,
                                         const uint16_t* rows, int64_t row_stride,
                                         const uint16_t* norm, float eps, const fleet_rope* rope,
                                         const int32_t* start, int32_t n_rows, void* workspace,
                                         size_t workspace_bytes, hipStream_t stream) {
    if (int e = check_cache(cache, workspace, workspace_bytes)) return e;
    if (int e = fleet_moe_check_rope(rope)) return e;
    if (layer < 0 || layer >= cache->n_layers || n_rows < 0 || n_rows > (1 << 28) ||
        (uintptr_t)start % 4 || (!start && n_rows != cache->n_seqs) ||
        rope->dim != kRow - kC || !rope->halves_out || (uintptr_t)norm % 16 ||
        !(eps >= 1e-30f) || !(eps <= 1e30f))
        return FLEET_MOE_ERR_ARG;
    if (n_rows == 0) return 0;
    if (!rows || (uintptr_t)rows % 16 || row_stride < kRow || row_stride % 8 ||
        row_stride > ((int64_t)1 << 32))
        return FLEET_MOE_ERR_ARG;
    if (int e = fleet_moe_check_device(1)) return e;
    LatentParams P{};
    P.r.c = *cache;
    P.r.rows = const_cast<uint16_t*>(rows);
    P.r.row_stride = row_stride;
    P.r.start = start;
    P.r.h = static_cast<Header*>(workspace);
    P.r.n_rows = n_rows;
    P.r.layer0 = layer;
    P.r.n_layers = 1;
    P.rope = *rope;
    P.norm = norm;
    P.eps = eps;
    const int64_t units = first_unit(n_rows, cache->n_seqs, 1, kBlock, 2);
    hipLaunchKernelGGL(latent_kernel, dim3((unsigned)units), dim3(kRowThreads), 0, stream, P);
    return (int)hipGetLastError();
}
