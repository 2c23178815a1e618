// Rows of the 8-bit cache: fleet_cache_append and fleet_cache_read (declarations
// in fleet_moe.h).
//
// A workgroup takes one block of 16 positions of one layer, in either direction:
// thread (position, chunk) moves 16 values, 32 bytes of a row and 16 of the block.
// A row is 1152 bytes on one side, 576 on the other. Many rows: read is bound by HBM; append
// also by its vector instructions, 282 a wave, scaling, clamping and converting most of them,
// which issue in 62% of the cycles (read's 92 in 14%): 1,000 rows of 27 layers take 15.5 and
// 14.2 us, a copy of as many bytes 10.8. A row for each sequence: latency, 4.7 us.
#include "cache_pages.h"

namespace fleet_moe {
namespace cache {

// Nine waves: wave w holds chunks 4w .. 4w + 3, so the last wave holds exactly
// k_pe and the others c, and a row's four chunks are 128 consecutive bytes.
constexpr int kRowThreads = kBlock * kChunks;
static_assert(kRowThreads == 9 * 64, "");

// Layers that a workgroup of read takes, their loads on their way together. (Rows of 27
// layers, with 1 / 2 / 3 / 7 of them, us: 300 rows 8.1 / 7.9 / 7.9 / 8.1, 1,000 14.7 / 14.2 /
// 13.8 / 11.7, 1,500 17.8 / 17.2 / 17.9 / 20.7, 8,000 79.8 / 72.8 / 76.0 / 82.6; seven are
// best only where they make one workgroup a CU. append is fastest with one: its
// instructions stay the same, with fewer waves to fill another's waits.)
constexpr int kRead = 2;

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

__global__ __launch_bounds__(kRowThreads) void append_kernel(RowParams P) {
    __shared__ unsigned most[8];
    BlockAt b;
    if (!block_at<true>(P, b)) return;
    const fleet_cache& c = P.c;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int tok = lane >> 2, chunk = 4 * wave + (lane & 3);
    const int layer = P.layer0 + (int)blockIdx.y;
    // (these are read beside the rows: their latency is the same)
    const int holders = c.refs[b.page];
    const uint32_t refused = P.h->refused;
    uint8_t* page = c.pool + page_offset(b.page, c.n_pages, layer, c.n_layers);
    const int blk = b.base % kPage / kBlock;
    u32x4* mine = reinterpret_cast<u32x4*>(page + blk * kBlockBytes) + chunk * kBlock + tok;
    uint32_t* scale = reinterpret_cast<uint32_t*>(page + kCodeBytes) + 2 * blk + (wave == 8);
    const int pos = b.base + tok;
    const bool fresh = pos >= b.first && pos < b.len;
    const bool aged = b.base < b.first;                   // older positions in the block
    u32x4 v[2] = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
    if (fresh) {
        const uint16_t* row = P.rows + blockIdx.y * P.layer_stride +
                              (int64_t)(b.row0 + pos - b.first) * P.row_stride + chunk * 16;
        v[0] = ld_stream(reinterpret_cast<const u32x4*>(row));
        v[1] = ld_stream(reinterpret_cast<const u32x4*>(row) + 1);
    }
    const uint32_t was = aged ? ld_global(scale) : 0;
    // the largest finite magnitude, as bf16 bits: they order as the values do
    unsigned big = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t w = v[i / 4][i % 4];
        const unsigned x = w & 0x7fff, y = w >> 16 & 0x7fff;
        big = x < 0x7f80 && x > big ? x : big;
        big = y < 0x7f80 && y > big ? y : big;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned o = __shfl_xor(big, d);
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
        if (t == 0) raise(P.h, refused ? refused : (uint32_t)FLEET_MOE_ABORT_BAD_PAGE);
        return;
    }
    int e = scale_exp(big);
    int e_old = (int)(was >> 23 & 255) - 127;
    e_old = e_old < -110 ? -110 : e_old > 120 ? 120 : e_old;
    if (aged && e_old > e) e = e_old;
    const float inv = pow2(-e);
    if (fresh) {
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w0 = v[i / 2][2 * i % 4], w1 = v[i / 2][2 * i % 4 + 1];
            o[i] = e4m3x4(bf_lo(w0) * inv, bf_hi(w0) * inv, bf_lo(w1) * inv, bf_hi(w1) * inv);
        }
        st_global(mine, o);
    } else if (aged && e > e_old && pos < b.first) {
        // older codes under the larger scale
        const u32x4 o = ld_global(mine);
        const float down = pow2(e_old - e < -126 ? -126 : e_old - e);
        u32x4 n;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = bf16x2<false>(o[i], 1.f), hi = bf16x2<true>(o[i], 1.f);
            n[i] = e4m3x4(bf_lo(lo) * down, bf_hi(lo) * down, bf_lo(hi) * down, bf_hi(hi) * down);
        }
        st_global(mine, n);
    }
    if (lane == 0 && (wave == 0 || wave == 8)) st_global(scale, (uint32_t)(e + 127) << 23);
}

// Rows want the wave's lanes in another order than the block: lane 4 tok + i has chunk i
// of the wave's four for a row, 128 consecutive bytes of four lanes; lane 16 i + tok loads
// them, 1 KB of consecutive bytes a wave (1,000 rows of 27 layers 15.5 to 14.5 us; for
// append's stores the same 15.5 and 15.8).
__device__ __forceinline__ u32x4 to_row_order(const u32x4& v, int lane) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r[i] = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * ((lane & 3) * 16 + (lane >> 2)),
                                                      (int)v[i]);
    return r;
}

__global__ __launch_bounds__(kRowThreads) void read_kernel(RowParams P) {
    BlockAt b;
    if (!block_at<false>(P, b)) return;
    const fleet_cache& c = P.c;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int tok = lane >> 2, chunk = 4 * wave + (lane & 3);
    const int y0 = (int)blockIdx.y * kRead;
    const int n = P.n_layers - y0 < kRead ? P.n_layers - y0 : kRead;
    const uint8_t* page = c.pool + page_offset(b.page, c.n_pages, P.layer0 + y0, c.n_layers);
    const int blk = b.base % kPage / kBlock;
    const int pos = b.base + tok;
    u32x4 o[kRead];
    float scale[kRead];
#pragma unroll
    for (int j = 0; j < kRead; ++j) {
        if (j >= n) break;
        o[j] = ld_stream(reinterpret_cast<const u32x4*>(page + j * kPageBytes + blk * kBlockBytes) +
                         wave * 4 * kBlock + lane);
        scale[j] = __uint_as_float(ld_global(
            reinterpret_cast<const uint32_t*>(page + j * kPageBytes + kCodeBytes) + 2 * blk +
            (wave == 8)));
    }
    uint16_t* row = P.rows + y0 * P.layer_stride +
                    (int64_t)(b.row0 + pos - b.first) * P.row_stride + chunk * 16;
    const bool there = pos >= b.first && pos < b.len;
#pragma unroll
    for (int j = 0; j < kRead; ++j) {
        if (j >= n) break;
        const u32x4 w = to_row_order(o[j], lane);
        if (there) {
            u32x4 v[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i / 2][2 * i % 4] = bf16x2<false>(w[i], scale[j]);
                v[i / 2][2 * i % 4 + 1] = bf16x2<true>(w[i], scale[j]);
            }
            u32x4* at = reinterpret_cast<u32x4*>(row + j * P.layer_stride);
            st_global(at, v[0]);
            st_global(at + 1, v[1]);
        }
    }
}

}  // namespace cache
}  // namespace fleet_moe

using namespace fleet_moe;
using namespace fleet_moe::cache;

int fleet_moe_check_device(int min_cus);

static int rows_call(bool append, const fleet_cache* cache, int32_t layer0, int32_t n_layers,
                     uint16_t* rows, int64_t row_stride, int64_t layer_stride,
                     const int32_t* start, int32_t n_rows, void* workspace,
                     size_t workspace_bytes, hipStream_t stream) {
    if (int e = check_cache(cache, workspace, workspace_bytes)) return e;
    if (layer0 < 0 || n_layers < 1 || n_layers > cache->n_layers - layer0)
        return FLEET_MOE_ERR_ARG;
    if (n_rows < 0 || n_rows > (1 << 28) || (uintptr_t)start % 4 ||
        (!start && n_rows != cache->n_seqs))
        return FLEET_MOE_ERR_ARG;
    if (n_rows == 0) return 0;
    if (!rows || (uintptr_t)rows % 16 || row_stride < kRow || row_stride % 8 ||
        row_stride > ((int64_t)1 << 32) || layer_stride % 8 || layer_stride < 0 ||
        layer_stride > ((int64_t)1 << 48) ||
        (n_layers > 1 && layer_stride < kRow) ||
        // rows of a layer behind each other, or the layers of a row
        (n_layers > 1 && layer_stride < (int64_t)(n_rows - 1) * row_stride + kRow &&
         row_stride < (int64_t)(n_layers - 1) * layer_stride + kRow))
        return FLEET_MOE_ERR_ARG;
    if (int e = fleet_moe_check_device(1)) return e;
    RowParams P{};
    P.c = *cache;
    P.rows = rows;
    P.row_stride = row_stride;
    P.layer_stride = layer_stride;
    P.start = start;
    P.h = static_cast<Header*>(workspace);
    P.n_rows = n_rows;
    P.layer0 = layer0;
    const int64_t units = first_unit(n_rows, cache->n_seqs, 1, kBlock, 2);
    P.n_layers = n_layers;
    const int each = append ? 1 : kRead;
    const dim3 grid((unsigned)units, (n_layers + each - 1) / each);
    if (append) hipLaunchKernelGGL(append_kernel, grid, dim3(kRowThreads), 0, stream, P);
    else hipLaunchKernelGGL(read_kernel, grid, dim3(kRowThreads), 0, stream, P);
    return (int)hipGetLastError();
}

extern "C" int fleet_cache_append(const fleet_cache* cache, int32_t layer0, int32_t n_layers,
                                  const uint16_t* rows, int64_t row_stride, int64_t layer_stride,
                                  const int32_t* start, int32_t n_rows, void* workspace,
                                  size_t workspace_bytes, hipStream_t stream) {
    return rows_call(true, cache, layer0, n_layers, const_cast<uint16_t*>(rows), row_stride,
                     layer_stride, start, n_rows, workspace, workspace_bytes, stream);
}

extern "C" int fleet_cache_read(const fleet_cache* cache, int32_t layer0, int32_t n_layers,
                                uint16_t* rows, int64_t row_stride, int64_t layer_stride,
                                const int32_t* start, int32_t n_rows, void* workspace,
                                size_t workspace_bytes, hipStream_t stream) {
    return rows_call(false, cache, layer0, n_layers, rows, row_stride, layer_stride, start,
                     n_rows, workspace, workspace_bytes, stream);
}
