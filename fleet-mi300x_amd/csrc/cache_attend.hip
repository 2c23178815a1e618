// Attention over the 8-bit latent cache: fleet_cache_attend (declaration in
// fleet_moe.h).
//
// The heads share one cache row, so the rows of the products are (token, head)
// pairs. With K the [positions][576] values of a range and Q the rows, a step is
//   S^T = K Q^T,  P = exp(S - max),  O^T += K[:, :512]^T P^T,
// with the running maximum and sum of each row. Both products are taken
// transposed: the 16x16 result of the first then holds, per lane, four positions of
// one row, which is what the second takes as its right operand once the order of
// positions inside the matrix instruction's k index is chosen to match (positions
// 4g .. 4g+3 of two blocks for lane group g), so P moves between lanes nowhere.
// The left operands are the page's bytes: K as 16-byte LDS reads, K^T as
// transposing ones (ds_read_b64_tr_b8: 16 lanes get 8 positions of 16 dimensions),
// each widened to bf16 with its block's scale, exactly (4 significant bits and a
// power of two).
//
// Roundings: q and the cache are exact in bf16, products and sums fp32. P is
// rounded to bf16 (the MFMA's operand; 2^-9 of each weight); its sum, by which
// the result is divided, is taken of the rounded values, so a common rounding of
// all weights cancels. lse comes from the unrounded sum.
#include "cache_pages.h"

namespace fleet_moe {
namespace cache {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

struct AttendParams {
    fleet_cache c;
    const uint16_t* q;
    const int32_t* start;
    uint16_t* out;
    float* lse;
    float* part;                // fp32 [tile][split][16][512], then [tile][split][16][2..]
    Header* h;
    int64_t q_stride;
    int layer, n_tokens, n_heads, window, sinks, splits, pad;
    float scale;                // times log2(e)
};

// 32 positions, the k of a 16x16x32 product, are a tile.
constexpr int kTile = 32;
constexpr int kRows = 16;
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr float kLn2 = 0.6931471805599453f;

// A workgroup's rows and the positions they see: sink tiles [0, n_sink), then
// tiles [main, main + n - n_sink).
struct Work {
    int seq, row0, rows;        // rows row0 .. of the sequence's `rows`
    int tok0;                   // its first token
    int len, n_new;
    int n_sink, main, n;
};

template <int R>
__device__ __forceinline__ bool find_work(const AttendParams& P, int64_t u, Work& w) {
    const fleet_cache& c = P.c;
    w.seq = find_seq(P.start, c.n_seqs, P.n_tokens, u, P.n_heads, R, P.pad);
    if (w.seq < 0) return false;
    const int a = P.start ? clamp_row(P.start[w.seq], P.n_tokens) : w.seq;
    const int z = P.start ? clamp_row(P.start[w.seq + 1], P.n_tokens) : w.seq + 1;
    if (z <= a) return false;
    w.tok0 = a;
    w.n_new = z - a;
    w.rows = w.n_new * P.n_heads;
    const int64_t r = (u - first_unit(a, w.seq, P.n_heads, R, P.pad)) * R;
    if (r >= w.rows) return false;
    w.row0 = (int)r;
    int len = c.lens[w.seq];
    w.len = checked_len(len, c.max_pages);
    // the positions of the tile's first and last token
    const int last_row = w.row0 + R - 1 < w.rows ? w.row0 + R - 1 : w.rows - 1;
    const int p0 = w.len - w.n_new + w.row0 / P.n_heads;
    const int p1 = w.len - w.n_new + last_row / P.n_heads;
    w.n_sink = w.main = w.n = 0;
    if (w.len < 0) {
        if (threadIdx.x == 0) raise(P.h, FLEET_MOE_ABORT_POSITION);
        return true;
    }
    if (p1 < 0) return true;
    const Seen s = seen_of(p0 < 0 ? 0 : p0, P.window, P.sinks);
    const int end = (p1 + kTile) / kTile;                 // p1 + 1 positions
    w.main = s.lo / kTile;
    const int sink = (s.sink + kTile - 1) / kTile;
    w.n_sink = sink < w.main ? sink : w.main;
    w.n = w.n_sink + end - w.main;
    return true;
}

// The share of one of `splits` workgroups in n tiles, whole rounds of the waves.
// Fewer tiles than that leave the last workgroups without any.
__device__ __forceinline__ int split_size(int n, int splits) {
    const int each = (n + splits - 1) / splits;
    return (each + kWaves - 1) / kWaves * kWaves;
}

// LDS, per wave two tiles of two blocks. The second block sits 64 bytes off, so
// that the two halves of a transposing read fall into different banks.
constexpr int kBlockStep = kBlockBytes + 64;
constexpr int kScaleAt = 2 * kBlockStep;
constexpr int kTileBytes = kScaleAt + 256;
struct AttendLds {
    union {
        __attribute__((aligned(16))) uint8_t tile[kWaves][2][kTileBytes];
        f32x4 sum[kWaves][kC / 16][64];
    };
    float stat[kWaves][3][kRows];
};

// Copies 16 bytes per lane from global memory to LDS, kN times 1 KB: lane's `src`
// + 1024 i to `lds` + 1024 i + 16 lane (the offset counts on both sides). There is
// no register for the data, so none is in flight behind the compiler's back. In asm,
// because the compiler would wait for every copy in flight before each LDS read;
// wait_copies() orders them.
template <int kN>
__device__ __forceinline__ void copy_kb(const uint8_t* src, uint32_t lds) {
    static_assert(kN == 1 || kN == 4, "");
    if constexpr (kN == 4)
        asm volatile(
            "s_nop 0\n\t"
            "global_load_lds_dwordx4 %0, off\n\t"
            "global_load_lds_dwordx4 %0, off offset:1024\n\t"
            "global_load_lds_dwordx4 %0, off offset:2048\n\t"
            "global_load_lds_dwordx4 %0, off offset:3072" ::"v"(src), "{m0}"(lds)
            : "memory");
    else
        asm volatile(
            "s_nop 0\n\t"
            "global_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(lds)
            : "memory");
}
// The same with 4 bytes per lane.
__device__ __forceinline__ void copy_words(const uint8_t* src, uint32_t lds) {
    asm volatile(
        "s_nop 0\n\t"
        "global_load_lds_dword %0, off" ::"v"(src), "{m0}"(lds)
        : "memory");
}
template <int kLeft>
__device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLeft) : "memory");
}
constexpr int kCopies = 2 * kBlockBytes / 1024 + 1;       // of a tile

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// One tile of a page's layer into LDS; `src` is the page's layer, half 0 or 1.
__device__ __forceinline__ void load_tile(const uint8_t* src, int half, uint32_t lds, int lane) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const uint8_t* at = src + (2 * half + b) * kBlockBytes + lane * 16;
        const uint32_t to = lds + b * kBlockStep;
        copy_kb<4>(at, to);
        copy_kb<4>(at + 4096, to + 4096);
        copy_kb<1>(at + 8192, to + 8192);
    }
    copy_words(src + kCodeBytes + (lane & 7) * 4, lds + kScaleAt);
}

__device__ __forceinline__ bf16x8 widen(uint32_t lo, uint32_t hi, float slo, float shi) {
    u32x4 r;
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, slo, false));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, slo, true));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, shi, false));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, shi, true));
    return __builtin_bit_cast(bf16x8, r);
}

// A block that holds no position yet may hold any bytes: its weights are zero, and
// with a scale in range so are the products.
__device__ __forceinline__ float any_scale(uint32_t w) {
    w &= 0x7f800000u;
    return __uint_as_float(w < 0x7b800000u ? w : 0x7b800000u);      // 2^120
}

// NaN codes (0x7f, 0xff) of a word as zeros.
__device__ __forceinline__ uint32_t drop_nan(uint32_t w) {
    const uint32_t n = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    return w & ~(n | (n - (n >> 7)));
}

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

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// 16 rows against a share of the positions. Four waves take the tiles in turn,
// each with its own maximum, sum and O^T (16 rows x 512 in 128 registers), from two
// buffers of its own that copies fill a tile ahead: no wave waits for another
// before the end. At 576 bytes per position for 16 rows the memory bounds it, the
// products take about a third of the time; the LDS (2 x 18 KB per wave) is sized
// for what has to be in flight.
__global__ __launch_bounds__(kThreads, 1) void attend_kernel(AttendParams P) {
    __shared__ AttendLds L;
    const int t = threadIdx.x, lane = t & 63, wave = wave_bcast(t >> 6);
    const int split = blockIdx.x % P.splits;
    Work w;
    if (!find_work<kRows>(P, blockIdx.x / P.splits, w)) return;
    const int each = split_size(w.n, P.splits);
    const int t0 = split * each;
    const int t1 = t0 + each < w.n ? t0 + each : w.n;
    if (split > 0 && t0 >= w.n) return;
    const bool whole = each >= w.n;             // no other workgroup has these rows

    // this lane's row, and what it sees
    const int g = lane >> 4, row = w.row0 + (lane & 15);
    const bool live = row < w.rows;
    const int tok = live ? row / P.n_heads : 0, head = live ? row % P.n_heads : 0;
    const int pos = live ? w.len - w.n_new + tok : -1;
    const Seen seen = seen_of(pos < 0 ? 0 : pos, P.window, P.sinks);
    bf16x8 q[2 * kChunks / 4];
#pragma unroll
    for (int i = 0; i < kChunks / 4; ++i) {
        u32x4 a{0, 0, 0, 0}, b{0, 0, 0, 0};
        if (live) {
            const u32x4* src = reinterpret_cast<const u32x4*>(
                P.q + (int64_t)(w.tok0 + tok) * P.q_stride + head * kRow + (4 * i + g) * 16);
            a = ld_global(src);
            b = ld_global(src + 1);
        }
        q[2 * i] = __builtin_bit_cast(bf16x8, a);
        q[2 * i + 1] = __builtin_bit_cast(bf16x8, b);
    }
    f32x4 acc[kC / 16];
#pragma unroll
    for (int i = 0; i < kC / 16; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    f32x4 ones = f32x4{0.f, 0.f, 0.f, 0.f};     // the sum of the rounded weights
    const u32x4 one_bits{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    float m = -INFINITY, l = 0.f;

    // the wave's tiles: t0 + wave, + kWaves, ..; lane k holds the page of the k-th
    // of the next 64
    const int32_t* table = P.c.table + (int64_t)w.seq * P.c.max_pages;
    const auto tile_of = [&](int i) { return i < w.n_sink ? i : w.main + i - w.n_sink; };
    int pages = 0, held = 0, asked = 0;         // `held` pages from the asked-th tile on
    const int mine = t1 - t0 - wave > 0 ? (t1 - t0 - wave + kWaves - 1) / kWaves : 0;
    const auto page_of = [&](int k) {           // of the wave's k-th tile
        if (k >= held) {
            asked = k;
            held = k + 64;
            const int i = k + lane;
            pages = i < mine ? ld_global(table + tile_of(t0 + wave + i * kWaves) / 2) : 0;
        }
        return __builtin_amdgcn_readlane(pages, k - asked);
    };
    const auto issue = [&](int k) {
        const int page = page_of(k);
        const int tile = tile_of(t0 + wave + k * kWaves);
        const int64_t at = page_offset(page, P.c.n_pages, P.layer, P.c.n_layers);
        load_tile(P.c.pool + (at < 0 ? 0 : at), tile & 1, lds_addr(L.tile[wave][k & 1]), lane);
        return at >= 0;
    };
    // bit k & 1: whether the tile in that buffer is one of the pool's
    int good = 0;
    if (mine > 0) good |= issue(0) ? 1 : 0;
    if (mine > 1) good |= issue(1) ? 2 : 0;
    for (int k = 0; k < mine; ++k) {
        if (k + 1 < mine) wait_copies<kCopies>();
        else wait_copies<0>();
        const uint8_t* buf = L.tile[wave][k & 1];
        const int tile = tile_of(t0 + wave + k * kWaves);
        const uint32_t* sc = reinterpret_cast<const uint32_t*>(buf + kScaleAt) + 4 * (tile & 1);
        const float sc0 = any_scale(sc[0]), sp0 = any_scale(sc[1]);
        const float sc1 = any_scale(sc[2]), sp1 = any_scale(sc[3]);

        f32x4 s0{0.f, 0.f, 0.f, 0.f}, s1{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kChunks / 4; ++i) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(buf + i * 1024 + lane * 16);
            const u32x4 b = *reinterpret_cast<const u32x4*>(buf + kBlockStep + i * 1024 + lane * 16);
            const float sa = i < kC / 64 ? sc0 : sp0, sb = i < kC / 64 ? sc1 : sp1;
            s0 = mfma(widen(a.x, a.y, sa, sa), q[2 * i], s0);
            s1 = mfma(widen(b.x, b.y, sb, sb), q[2 * i], s1);
            s0 = mfma(widen(a.z, a.w, sa, sa), q[2 * i + 1], s0);
            s1 = mfma(widen(b.z, b.w, sb, sb), q[2 * i + 1], s1);
        }
        float s[8];
        bool nan = false;
        const int base = tile * kTile + 4 * g;
        const bool ok = good >> (k & 1) & 1;
        if (!ok && lane == 0) raise(P.h, FLEET_MOE_ABORT_BAD_PAGE);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float v = (j < 4 ? s0[j & 3] : s1[j & 3]) * P.scale;
            const int p = base + (j & 3) + (j < 4 ? 0 : kBlock);
            nan |= v != v;
            s[j] = ok && p <= pos && (p >= seen.lo || p < seen.sink) ? v : -INFINITY;
        }
        float top = m;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, s[j]);
        top = xor32_max(xor16_max(top));
        const float base_m = top == -INFINITY ? 0.f : top;
        const float shrink = exp2_(m - base_m);
        if (__ballot(top != m)) {
            l *= shrink;
            ones *= shrink;
#pragma unroll
            for (int i = 0; i < kC / 16; ++i) acc[i] *= shrink;
        }
        m = top;
        u32x4 pb;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float a = exp2_(s[2 * j] - base_m), b = exp2_(s[2 * j + 1] - base_m);
            l += a + b;
            typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
            bf16x2 r;
            r[0] = (__bf16)a;
            r[1] = (__bf16)b;
            pb[j] = __builtin_bit_cast(uint32_t, r);
        }
        const bf16x8 p = __builtin_bit_cast(bf16x8, pb);
        ones = mfma(__builtin_bit_cast(bf16x8, one_bits), p, ones);
        // lane r of its group of 16 points at row r / 2 of 8: positions 4g .. 4g + 3 of
        // both blocks
        const int r8 = (lane & 15) >> 1;
        const uint8_t* col = buf + (r8 < 4 ? 0 : kBlockStep) + (4 * g + (r8 & 3)) * 16 +
                             (lane & 1) * 8;
        typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
        if (__ballot(nan) == 0) {
#pragma unroll
            for (int i = 0; i < kC / 16; ++i) {
                const i32x2 v = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                    (lds_i32x2*)(const __attribute__((address_space(3))) uint8_t*)(col + i * 256));
                acc[i] = mfma(widen((uint32_t)v.x, (uint32_t)v.y, sc0, sc1), p, acc[i]);
            }
        } else {
            // A NaN in a row: every row of q that sees it has a NaN weight, and
            // those that do not must not meet 0 * NaN.
#pragma unroll
            for (int i = 0; i < kC / 16; ++i) {
                const i32x2 v = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                    (lds_i32x2*)(const __attribute__((address_space(3))) uint8_t*)(col + i * 256));
                acc[i] = mfma(widen(drop_nan((uint32_t)v.x), drop_nan((uint32_t)v.y), sc0, sc1), p,
                              acc[i]);
            }
        }
        if (k + 2 < mine) {
            // every LDS read of this buffer has returned before it is filled again
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            const int bit = 1 << (k & 1);
            good = issue(k + 2) ? good | bit : good & ~bit;
        }
    }
    l = xor32_sum(xor16_sum(l));

    // The waves' results: each takes 128 of the 512 columns of all four.
    if (lane < kRows) {
        L.stat[wave][0][lane] = m;
        L.stat[wave][1][lane] = l;
        L.stat[wave][2][lane] = ones[0];
    }
    __syncthreads();                            // (and every wave is done with its tiles)
    const int n = lane & 15;
    float top = L.stat[0][0][n];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) top = fmaxf(top, L.stat[i][0][n]);
    const float base_m = top == -INFINITY ? 0.f : top;
    float sum = 0.f, rounded = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        const float f = exp2_(L.stat[i][0][n] - base_m);
        sum += f * L.stat[i][1][n];
        rounded += f * L.stat[i][2][n];
    }
    const float f = exp2_(m - base_m);
#pragma unroll
    for (int i = 0; i < kC / 16; ++i) L.sum[wave][i][lane] = acc[i] * f;
    __syncthreads();
    constexpr int kMine = kC / 16 / kWaves;
    f32x4 o[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int ch = wave * kMine + i;
        o[i] = (L.sum[0][ch][lane] + L.sum[1][ch][lane]) + (L.sum[2][ch][lane] + L.sum[3][ch][lane]);
    }
    if (whole) {
        if (!live) return;
        const int64_t at = (int64_t)(w.tok0 + tok) * P.n_heads + head;
        const float inv = rounded == 0.f ? 0.f : 1.f / rounded;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const uint64_t b = (uint64_t)(bf16_bits(o[i][0] * inv) | bf16_bits(o[i][1] * inv) << 16) |
                               (uint64_t)(bf16_bits(o[i][2] * inv) | bf16_bits(o[i][3] * inv) << 16)
                                   << 32;
            st_global(reinterpret_cast<uint64_t*>(P.out + at * kC + (wave * kMine + i) * 16 + 4 * g), b);
        }
        if (P.lse && wave == 0 && g == 0)
            P.lse[at] = sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
        return;
    }
    const int64_t slot = (int64_t)(blockIdx.x / P.splits) * P.splits + split;
    float* part = P.part + slot * kRows * kC;
#pragma unroll
    for (int i = 0; i < kMine; ++i)
        st_global(reinterpret_cast<f32x4*>(part + n * kC + (wave * kMine + i) * 16 + 4 * g), o[i]);
    if (wave == 0 && g == 0) {
        float* stat = P.part + (int64_t)kPartRows * kC + (slot * kRows + n) * 4;
        stat[0] = top;
        stat[1] = sum;
        stat[2] = rounded;
    }
}

// Joins the splits of a row: a workgroup per row, each thread four columns. The splits
// are read in order, so the result does not depend on timing.
constexpr int kJoinThreads = 128;
__global__ __launch_bounds__(kJoinThreads) void join_kernel(AttendParams P) {
    Work w;
    const int64_t u = blockIdx.x / kRows;
    const int n = blockIdx.x % kRows;
    if (!find_work<kRows>(P, u, w)) return;
    const int each = split_size(w.n, P.splits);
    if (each >= w.n) return;
    const int row = w.row0 + n;
    if (row >= w.rows) return;
    const int used = (w.n + each - 1) / each;
    const int64_t slot0 = u * P.splits;
    const f32x4* stat = reinterpret_cast<const f32x4*>(P.part + (int64_t)kPartRows * kC) +
                        slot0 * kRows + n;
    float top = -INFINITY;
    for (int i = 0; i < used; ++i) top = fmaxf(top, stat[(int64_t)i * kRows][0]);
    const float base_m = top == -INFINITY ? 0.f : top;
    float sum = 0.f, rounded = 0.f;
    f32x4 o{0.f, 0.f, 0.f, 0.f};
    const f32x4* part = reinterpret_cast<const f32x4*>(P.part + (slot0 * kRows + n) * kC) +
                        threadIdx.x;
#pragma unroll 8
    for (int i = 0; i < used; ++i) {
        const f32x4 st = stat[(int64_t)i * kRows];
        const float f = exp2_(st[0] - base_m);
        sum += f * st[1];
        rounded += f * st[2];
        o += part[(int64_t)i * kRows * kC / 4] * f;
    }
    const int64_t at = (int64_t)w.tok0 * P.n_heads + row;
    const float inv = rounded == 0.f ? 0.f : 1.f / rounded;
    const uint64_t b = (uint64_t)(bf16_bits(o[0] * inv) | bf16_bits(o[1] * inv) << 16) |
                       (uint64_t)(bf16_bits(o[2] * inv) | bf16_bits(o[3] * inv) << 16) << 32;
    st_global(reinterpret_cast<uint64_t*>(P.out + at * kC + threadIdx.x * 4), b);
    if (P.lse && threadIdx.x == 0)
        P.lse[at] = sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

}  // namespace cache
}  // namespace fleet_moe

using namespace fleet_moe;
using namespace fleet_moe::cache;

int fleet_moe_check_device(int min_cus);

extern "C" int fleet_cache_attend(const fleet_cache* cache, int32_t layer, const uint16_t* q,
                                  int64_t q_stride, const int32_t* start, int32_t n_tokens,
                                  int32_t n_heads, int32_t max_len, int32_t window, int32_t sinks,
                                  float scale, uint16_t* out, float* lse, void* workspace,
                                  size_t workspace_bytes, hipStream_t stream) {
    if (int e = check_cache(cache, workspace, workspace_bytes)) return e;
    if (layer < 0 || layer >= cache->n_layers || n_tokens < 0 || n_heads < 1 ||
        n_heads > FLEET_CACHE_MAX_HEADS || (int64_t)n_tokens * n_heads > (1 << 26) ||
        max_len < 0 || window < 0 || sinks < 0 || !(scale > 0.f) || !(scale <= 3.0e38f) ||
        (uintptr_t)start % 4 || (!start && n_tokens != cache->n_seqs))
        return FLEET_MOE_ERR_ARG;
    if (n_tokens == 0) return 0;
    if (!q || !out || (uintptr_t)q % 16 || (uintptr_t)out % 8 || (uintptr_t)lse % 4 ||
        q_stride < (int64_t)n_heads * kRow || q_stride % 8 || q_stride > ((int64_t)1 << 32))
        return FLEET_MOE_ERR_ARG;
    if (int e = fleet_moe_check_device(1)) return e;
    AttendParams P{};
    P.c = *cache;
    P.q = q;
    P.start = start;
    P.out = out;
    P.lse = lse;
    char* ws = static_cast<char*>(workspace);
    P.h = reinterpret_cast<Header*>(ws);
    P.part = reinterpret_cast<float*>(ws + parts_at(cache->n_seqs, cache->n_pages));
    P.q_stride = q_stride;
    P.layer = layer;
    P.n_tokens = n_tokens;
    P.n_heads = n_heads;
    P.window = window;
    P.sinks = sinks;
    P.scale = scale * 1.4426950408889634f;
    P.pad = n_heads % kRows != 0;
    const int64_t units = first_unit(n_tokens, cache->n_seqs, n_heads, kRows, P.pad);
    int64_t seen = (int64_t)cache->max_pages * kPage;
    if (max_len > 0 && max_len < seen) seen = max_len;
    if (window > 0 && (int64_t)window + sinks + n_tokens < seen) seen = (int64_t)window + sinks + n_tokens;
    const int64_t rounds = (seen + kTile * kWaves - 1) / (kTile * kWaves);
    int64_t splits = 512 / units;
    if (splits > rounds) splits = rounds;
    if (splits > 64) splits = 64;
    if (splits < 1) splits = 1;
    P.splits = (int)splits;
    hipLaunchKernelGGL(attend_kernel, dim3((unsigned)(units * splits)), dim3(kThreads), 0, stream,
                       P);
    if (splits > 1)
        hipLaunchKernelGGL(join_kernel, dim3((unsigned)(units * kRows)), dim3(kJoinThreads), 0,
                           stream, P);
    return (int)hipGetLastError();
}
