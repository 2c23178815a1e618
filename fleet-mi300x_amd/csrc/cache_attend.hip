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
// Roundings: q and the cache are exact in bf16, products and sums fp32. P is the MFMA's
// operand in bf16. With few rows it is two operands, P rounded and what that leaves, so its
// weights are good to 2^-16: the bytes of the pages bound that kernel, and the second
// product of the same widened K costs 0.1 of 55.7 us. With many rows the matrix instructions
// and their issue bound it, and P is rounded (by 2^-8 of a weight at most): the second operand
// took 250 to 349 us there, for an error against 64 bits of 1.7e-3 instead of 2.1e-3, of which
// the result's own rounding to bf16 is 1.7e-3. The sum by which the result is divided is
// taken of the same operands, so a common rounding of all weights cancels. lse comes from the
// unrounded sum.
#include <float.h>
#include <math.h>

#include <atomic>

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
    float* part;                // partial O, fp32 [slot][rows][512]
    f32x4* stat;                // [slot][rows]: reference, sum, rounded sum
    int4* meta;                 // [unit]: first slot, next workgroup, number of slots
    Header* h;
    int64_t q_stride;
    uint64_t per_head;          // head_divisor(n_heads)
    int layer, n_tokens, n_heads, window, sinks, pad, units;
    int shares;                 // workgroups, or splits of a unit
    float scale;                // times log2(e)
    float slack;                // kSlack as a score: finite, so that -infinity + slack is too
};

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr float kSlack = 8.f;
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;

__device__ __forceinline__ int token_of(const AttendParams& P, int row) {
    return token_of_row(row, P.per_head);
}

// A unit: up to R rows (token, head) of a sequence, and the steps of S positions
// that some of them see: the first n_sink steps from position 0 on, the others from
// step `main` on.
struct Work {
    int seq, row0, rows;        // rows row0 .. of the sequence's `rows`
    int tok0, n_new, len;       // its first token, its tokens, its positions
    int n_sink, main, n;
};
template <int S>
__device__ __forceinline__ int step_of(const Work& w, int i) {
    return i < w.n_sink ? i : w.main + i - w.n_sink;
}

// The steps of a unit: everything but the sequence's tokens and length set here.
template <int R, int S>
__device__ __forceinline__ void see(const AttendParams& P, Work& w) {
    w.n_sink = w.main = w.n = 0;
    const int last = w.row0 + R - 1 < w.rows ? w.row0 + R - 1 : w.rows - 1;
    const int p0 = w.len - w.n_new + token_of(P, w.row0);
    const int p1 = w.len - w.n_new + token_of(P, last);
    if (w.len < 0 || p1 < 0) return;
    const Seen s = seen_of(p0 < 0 ? 0 : p0, P.window, P.sinks);
    const int end = (p1 + S) / S;                         // steps of p1 + 1 positions
    w.main = s.lo / S;
    const int sink = (s.sink + S - 1) / S;
    w.n_sink = sink < w.main ? sink : w.main;
    w.n = w.n_sink + end - w.main;
}
__device__ __forceinline__ void open_seq(const AttendParams& P, int seq, Work& w) {
    const int a = P.start ? clamp_row(ld_global(P.start + seq), P.n_tokens) : seq;
    const int z = P.start ? clamp_row(ld_global(P.start + seq + 1), P.n_tokens) : seq + 1;
    w.seq = seq;
    w.row0 = 0;
    w.tok0 = a;
    w.n_new = z > a ? z - a : 0;
    w.rows = z < a ? -1 : w.n_new * P.n_heads;            // -1: not a start at all
    w.len = checked_len(ld_global(P.c.lens + seq), P.c.max_pages);
}

// A lane's row, and what it sees.
struct Row {
    bool live;
    int tok, head;              // of the sequence's; dead rows: the unit's first
    int pos;
    Seen seen;
};
__device__ __forceinline__ Row row_of(const AttendParams& P, const Work& w, int row) {
    Row r;
    r.live = row < w.rows;
    if (!r.live) row = w.row0;
    r.tok = token_of(P, row);
    r.head = row - r.tok * P.n_heads;
    r.pos = r.live && w.len >= 0 ? w.len - w.n_new + r.tok : -1;
    r.seen = seen_of(r.pos < 0 ? 0 : r.pos, P.window, P.sinks);
    return r;
}
// (no short cuts: three comparisons cost less than a branch)
__device__ __forceinline__ bool sees(const Row& r, int pos) {
    return (pos <= r.pos) & ((pos >= r.seen.lo) | (pos < r.seen.sink));
}
// Whether all rows of a wave see all of the positions [a, a + n): what they all see,
// apart from the dead ones.
struct Common {
    int pos, lo, sink;
    __device__ __forceinline__ explicit Common(const Row& r) {
        pos = r.live ? r.pos : 0x7fffffff;
        lo = r.live ? r.seen.lo : 0;
        sink = r.live ? r.seen.sink : 0x7fffffff;
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
            const int a = __shfl_xor(pos, d), b = __shfl_xor(lo, d), c = __shfl_xor(sink, d);
            pos = a < pos ? a : pos;
            lo = b > lo ? b : lo;
            sink = c < sink ? c : sink;
        }
        pos = wave_bcast(pos);
        lo = wave_bcast(lo);
        sink = wave_bcast(sink);
    }
    __device__ __forceinline__ bool all(int a, int n) const {
        return a + n - 1 <= pos && (a >= lo || a + n <= sink);
    }
};
// Its query as the right operand. The k order of the products is that of the bytes a
// lane of group g takes of a row: its chunks 4i + g, 16 values each, i = 0 .. 8, make
// two of 18 steps. Two waves share the products: wave `half` of them has those of i =
// half, 2 + half, 4 + half, 6 + half, and one step of i = 8, which is k_pe.
constexpr int kHalf = kChunks / 4;              // steps of a wave
__device__ __forceinline__ void load_q(const AttendParams& P, const Work& w, const Row& r, int g,
                                       int half, bf16x8 (&q)[kHalf]) {
    const uint16_t* src = P.q + (int64_t)(w.tok0 + r.tok) * P.q_stride + r.head * kRow + g * 16;
    const auto at = [&](int v) {
        return __builtin_bit_cast(bf16x8, ld_global(reinterpret_cast<const u32x4*>(src + v)));
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        q[2 * i] = at((2 * i + half) * 64);
        q[2 * i + 1] = at((2 * i + half) * 64 + 8);
    }
    q[8] = at(8 * 64 + half * 8);
}
__device__ __forceinline__ int64_t out_row(const AttendParams& P, const Work& w, int row) {
    return (int64_t)w.tok0 * P.n_heads + row;
}

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

// Pages of 64 steps, one per lane: the next ones, and the few before that a copy's
// step is ahead of the one whose scores are finished.
constexpr int kBehind = 4;
struct Pages {
    int held, from;
    int page;
};
template <int S>
__device__ __forceinline__ int page_of(const AttendParams& P, const Work& w, Pages& h, int i,
                                       int end, int lane) {
    if (i >= h.held) {
        h.from = i - kBehind;
        h.held = h.from + 64;
        const int mine = h.from + lane;
        h.page = mine >= 0 && mine < end
                     ? ld_global(P.c.table + (int64_t)w.seq * P.c.max_pages +
                                 step_of<S>(w, mine) * S / kPage)
                     : 0;
        // here, not at the use: there the compiler would wait, every step, for
        // whatever copies are in flight
        __builtin_amdgcn_s_waitcnt(0x0F70);     // vmcnt(0)
    }
    return __builtin_amdgcn_readlane(h.page, i - h.from);
}

// ---------------------------------------------------------------- few rows: the products
//
// A workgroup of four waves has 16 rows and takes 32 positions a step, two blocks, half a
// page. Wave (block, half) takes half of the 576 products of its block's scores, so
// that no wave widens what another does; the halves meet in LDS, where the first wave
// of each block makes the weights, while the other two issue the copies of a later step.
// Then each wave adds its 128 columns of O: 32 registers a lane, and no sum over waves
// at the end. Two workgroups share a CU, so that one's barriers and latencies are the
// other's time; a wave alone on a SIMD issues a vector instruction every six cycles,
// two every three.
constexpr int kFew = 16;        // rows
constexpr int kStep = 32;       // positions
constexpr int kRing = 4;        // steps in LDS: three on their way from HBM
constexpr int kCopies = 10;     // that a wave issues for a step: nine of 1 KB, and scales

struct FewLds {
    __attribute__((aligned(16))) uint8_t tile[kRing][2 * kBlockStep];
    uint32_t scale[kRing][4];   // c and k_pe of either block
    f32x4 half[2][64];          // half of the scores of a block, for the wave that weighs
    u32x4 p[2][2][64];          // [step parity][weights, their rests][lane]
    int flag[2][2];             // [step parity][block]
    float top[2][16], sum[2][16];
};
static_assert(sizeof(FewLds) <= 80 * 1024, "two workgroups share a CU");
static_assert(2 * kShares * kFew <= kPartRows, "a workgroup has two parts at most");

// Steps off .. off + cnt - 1 of a unit, and its results: to `out` and `lse`, or as the
// partial results of slot `slot` if that is not negative.
__device__ __forceinline__ void attend(const AttendParams& P, FewLds& L, const Work& w, int off,
                                       int cnt, int slot) {
    constexpr int kCols = kC / 16 / kWaves;     // of 16
    const int t = threadIdx.x, lane = t & 63, wave = wave_bcast(t >> 6);
    const int g = lane >> 4, n = lane & 15, blk = wave & 1, half = wave >> 1;
    const bool weighs = half == 0;              // the others copy

    const Row r = row_of(P, w, w.row0 + n);
    const Common common(r);
    bf16x8 q[kHalf];
    load_q(P, w, r, g, half, q);
    f32x4 acc[kCols], ones{0.f, 0.f, 0.f, 0.f}; // O, and the sum of the rounded weights
#pragma unroll
    for (auto& a : acc) a = f32x4{0.f, 0.f, 0.f, 0.f};
    // Every row's reference, as a score and as it is in the exponent: any score not far
    // below the maximum, because weights up to 2^kSlack are as exact as those up to 1,
    // and moving it costs a pass over O and a barrier. All waves keep all of them.
    float m = -INFINITY, ref = -INFINITY, l = 0.f;
    const float slack = P.slack;
    f32x4 z, next;              // the scores of the block, and the next step's
    bool stray = false;         // a score of the wave is not finite
    float p[4];
    Pages pages{0, 0, 0};
    if (cnt > 0) page_of<kStep>(P, w, pages, off, off + cnt, lane);
    // q is there before a copy is issued, also as far as the compiler counts
    __builtin_amdgcn_s_waitcnt(0x0F70);         // vmcnt(0)

    const auto issue = [&](int k) {
        const int page = page_of<kStep>(P, w, pages, off + k, off + cnt, lane);
        const int64_t base = page_offset(page, P.c.n_pages, P.layer, P.c.n_layers);
        const uint8_t* src = P.c.pool + (base < 0 ? 0 : base);
        const int b = k % kRing, part = step_of<kStep>(w, off + k) & 1;
        const uint8_t* from = src + (2 * part + blk) * kBlockBytes + lane * 16;
        const uint32_t to = lds_addr(L.tile[b]) + blk * kBlockStep;
        static_assert(kBlockBytes == 9 * 1024, "");
        copy_kb<4, true>(from, to);
        copy_kb<4, true>(from + 4096, to + 4096);
        copy_kb<1, true>(from + 8192, to + 8192);
        if (lane == 0) copy_kb<1, true>(src + kCodeBytes + part * 16, lds_addr(L.scale[b]));
    };
    const auto score = [&](int k) {
        const int b = k % kRing;
        const uint8_t* block = L.tile[b] + blk * kBlockStep + lane * 16;
        const float sc = any_scale(L.scale[b][2 * blk]), sp = any_scale(L.scale[b][2 * blk + 1]);
        // two chains: a product's result is not the next one's operand
        f32x4 y0{0.f, 0.f, 0.f, 0.f}, y1{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(block + (2 * i + half) * 1024);
            y0 = mfma(widen(a.x, a.y, sc, sc), q[2 * i], y0);
            y1 = mfma(widen(a.z, a.w, sc, sc), q[2 * i + 1], y1);
        }
        const uint2 a = *reinterpret_cast<const uint2*>(block + 8 * 1024 + half * 8);
        y0 = mfma(widen(a.x, a.y, sp, sp), q[8], y0);
        next = y0 + y1;
        if (!weighs) L.half[blk][lane] = next;
    };
    const auto weigh = [&](int k) {
        const float down = ref == -INFINITY ? 0.f : ref;
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = exp2_(fmaf(z[j], P.scale, -down));
        const uint2 w = weights(p);
        reinterpret_cast<uint2*>(&L.p[k & 1][0][lane])[blk] = w;
        reinterpret_cast<uint2*>(&L.p[k & 1][1][lane])[blk] = rest(p, w);
    };
    const auto finish = [&](int k) {
        z = next + L.half[blk][lane];
        const int page = page_of<kStep>(P, w, pages, off + k, off + cnt, lane);
        const bool ok = (unsigned)page < (unsigned)P.c.n_pages;
        const int base = step_of<kStep>(w, off + k) * kStep + blk * kBlock;
        const bool bad = !finite((z[0] + z[1]) + (z[2] + z[3]));
        if (!(ok && common.all(base, kBlock))) {
            asm volatile("");                   // a branch, not twenty instructions every step
            if (!ok && t == 0) raise(P.h, FLEET_MOE_ABORT_BAD_PAGE);
#pragma unroll
            for (int j = 0; j < 4; ++j) z[j] = (ok & sees(r, base + 4 * g + j)) ? z[j] : -INFINITY;
        }
        weigh(k);
        const float top = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
        stray = __ballot(bad) != 0;
        const bool high = __ballot(top > m + slack) != 0;
        if (lane == 0) L.flag[k & 1][blk] = stray | high;
    };
    // What is rare: a row's scores beyond its reference, or one that is not finite, in step k.
    const auto mend = [&](int k) {
        if (weighs) {
            float top = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
            top = xor32_max(xor16_max(top));
            if (lane < 16) L.top[blk][lane] = top;
            if (stray)
                clean(L.tile[k % kRing] + blk * kBlockStep, L.scale[k % kRing][2 * blk], lane);
        }
        barrier();
        const float to = fmaxf(m, fmaxf(L.top[0][n], L.top[1][n]));
        const float scaled = reference(to * P.scale);
        const float shrink = shrink_to(scaled, ref);
        m = to;
        ref = scaled;
        l *= shrink;
        ones *= shrink;
#pragma unroll
        for (auto& a : acc) a *= shrink;
        if (weighs) weigh(k);
        barrier();
    };
    // O over step k
    const auto add = [&](int k) {
        const int b = k % kRing;
        const bf16x8 pb = __builtin_bit_cast(bf16x8, L.p[k & 1][0][lane]);
        const bf16x8 pr = __builtin_bit_cast(bf16x8, L.p[k & 1][1][lane]);
        const float sa = any_scale(L.scale[b][0]), sb = any_scale(L.scale[b][2]);
        const uint32_t col = lds_addr(L.tile[b]) + wave * kCols * 256 + column_at(lane);
#pragma unroll
        for (int i = 0; i < kCols; ++i) {
            const i32x2 v = column(col, i);
            const bf16x8 a = widen((uint32_t)v.x, (uint32_t)v.y, sa, sb);
            acc[i] = mfma(a, pb, acc[i]);
            acc[i] = mfma(a, pr, acc[i]);
        }
        const bf16x8 one = __builtin_bit_cast(bf16x8, u32x4{kOnes, kOnes, kOnes, kOnes});
        ones = mfma(one, pb, ones);
        ones = mfma(one, pr, ones);
    };

    // The first step's copies are waited for here, the others' kRing - 2 steps after
    // they are issued.
    if (!weighs) {
        for (int k = 0; k < kRing - 1 && k < cnt; ++k) issue(k);
        if (cnt > 2) wait_copies<2 * kCopies>();
        else if (cnt > 1) wait_copies<kCopies>();
        else wait_copies<0>();
    }
    barrier();
    // Step k: behind barrier A the weights of k and the rows of k + 1 are there, behind
    // B both halves of the scores of k + 1.
    for (int k = -1; k < cnt; ++k) {
        const int flags = k >= 0 ? L.flag[k & 1][0] | L.flag[k & 1][1] : 0;
        if (k + 1 < cnt) score(k + 1);
        if (k >= 0) {
            if (wave_bcast(flags)) mend(k);
            if (weighs) l += (p[0] + p[1]) + (p[2] + p[3]);
            add(k);
        }
        if (k + 1 == cnt) break;
        barrier();                              // B
        // into the buffer of step k - 1
        if (!weighs && k >= 0 && k + kRing - 1 < cnt) issue(k + kRing - 1);
        if (weighs) finish(k + 1);
        // step k + 2; the one behind it may be on its way
        if (cnt - k > 3) wait_copies<kCopies>();
        else wait_copies<0>();
        barrier();                              // A
    }
    // the sums of the two blocks
    l = xor32_sum(xor16_sum(l));
    if (weighs && lane < 16) L.sum[blk][lane] = l;
    barrier();
    const int column0 = wave * kCols * 16 + 4 * g;
    const float sum = L.sum[0][n] + L.sum[1][n];
    if (slot < 0) {
        if (w.row0 + n < w.rows) {
            const int64_t to = out_row(P, w, w.row0 + n);
            const float inv = ones[0] == 0.f ? 0.f : 1.f / ones[0];
#pragma unroll
            for (int j = 0; j < kCols; ++j) put(P.out + to * kC + column0 + j * 16, acc[j], inv);
            if (P.lse && wave == 0 && g == 0) P.lse[to] = lse_of(ref, sum);
        }
    } else {
        const int64_t at = (int64_t)slot * kFew + n;
#pragma unroll
        for (int j = 0; j < kCols; ++j)
            st_global(reinterpret_cast<f32x4*>(P.part + at * kC + column0 + j * 16), acc[j]);
        if (wave == 0 && g == 0) st_global(P.stat + at, f32x4{ref, sum, ones[0], 0.f});
    }
}

// ---------------------------------------------------------------- few rows: the work

// Sequences with a token or two: 16 rows a unit. The bytes of the pages bound it (576 a
// position for 16 rows, 60 flops a byte), so the work is divided into equal shares of
// steps over all units, whatever their lengths: a workgroup takes a range of the
// concatenated steps, across units where it has to. A unit that several have a part
// in leaves partial results, which join_few_kernel adds in order.
//
// Measured, both launches: one sequence of 1,024 positions 12.6 us, of 65,536 29; 64 of
// 5,120 to 8,192 55 us, 4.5 TB/s of pages (the copies alone reach 5.8; the waves wait 42% of
// their time, and the matrix units are busy 22%).
// The steps of all units of a sequence, an empty unit as one.
__device__ __forceinline__ int seq_steps(const AttendParams& P, Work& w) {
    int n = 0;
    for (w.row0 = 0; w.row0 < w.rows; w.row0 += kFew) {
        see<kFew, kStep>(P, w);
        n += w.n > 0 ? w.n : 1;
    }
    return n;
}
__device__ __forceinline__ int lane_of(int v, int lane) {
    return __builtin_amdgcn_readlane(v, lane);
}
__device__ __forceinline__ Work lane_of(const Work& v, int lane) {
    Work w{};
    w.seq = lane_of(v.seq, lane);
    w.rows = lane_of(v.rows, lane);
    w.tok0 = lane_of(v.tok0, lane);
    w.n_new = lane_of(v.n_new, lane);
    w.len = lane_of(v.len, lane);
    return w;
}

// A range of n things in `shares` parts that differ by one at most.
struct Shares {
    int each, more;             // the first `more` have each + 1
    __device__ Shares(int n, int shares) : each(n / shares), more(n % shares) {}
    __device__ int first(int i) const { return i * each + (i < more ? i : more); }
    __device__ int holder(int at) const {
        const int big = more * (each + 1);
        return at < big ? at / (each + 1) : more + (at - big) / each;
    }
};

// A unit counts kSetup steps besides its own where shares are long: beginning one in
// the middle of a share takes as long (queries, page numbers and the first copies
// one after the other), so that workgroups with two units ended later than the
// others. 64 sequences of 5,120 to 8,192: 55.6 us, without it 59.5.
constexpr int kSetup = 6;

// How many shares. A share of few steps is short, but each is a part to join: n steps
// of a unit in parts of m take some m + n / 16 m of a step, least where m is a
// quarter of n's root. One workgroup a CU, two where each has 4 steps or more of its
// own (shorter ones wait for each other's first copies). Measured over 27 layers in
// turn, against 512 shares wherever there are as many steps: one sequence of 16,384
// positions 20 and 35 us, of 65,536 29 and 40; 16 of 1,000 16.9 and 21.4; 8 of 4,100
// 22.5 and 25.7 (with another workspace for every call 22.3 and 21); 64 of 1,500 the
// same 30.1, with one workgroup a CU 31.6.
__device__ __forceinline__ int shares_of(int total, int steps, int units, int most) {
    const int least = (int)(sqrtf((float)steps / (float)units) * 0.25f);
    if (steps < 4 * kShares && most > kShares / 2) most = kShares / 2;
    if (least > 1) total = (total + least - 1) / least;
    return total < most ? total : most;
}

// The total of all units' steps; its division (no share is empty: the join counts
// on it); and the unit in which workgroup wg's part begins, and where. Every
// wave for itself, a lane per sequence (or for several, then once more a lane for each
// of the one lane's): no barrier, and one round of loads for 64 sequences.
struct Place {
    int off, total, shares, setup;
};
__device__ __forceinline__ bool locate(const AttendParams& P, int wg, Work& w, Place& at) {
    const int lane = threadIdx.x & 63;
    const int each = (P.c.n_seqs + 63) / 64;
    Work mine{};
    int n = 0, units = 0;
    bool bad = false;
    for (int i = 0; i < each; ++i) {
        const int s = lane * each + i;
        if (s < P.c.n_seqs) {
            open_seq(P, s, mine);
            bad |= mine.rows < 0;
            n += seq_steps(P, mine);
            units += (mine.rows + kFew - 1) / kFew;
        }
    }
    // starts that decrease: more rows than there are, nothing is done
    if (__ballot(bad)) {
        if (wg == 0) {
            for (int i = threadIdx.x; i < P.units; i += kThreads) P.meta[i] = make_int4(0, 0, 0, 0);
            if (threadIdx.x == 0) raise(P.h, FLEET_MOE_ABORT_POSITION);
        }
        return false;
    }
    int incl = wave_incl_scan(n);
    const int plain = lane_of(incl, 63);
    at.setup = plain >= 2 * kSetup * P.shares ? kSetup : 0;
    n += at.setup * units;
    incl = wave_incl_scan(n);
    at.total = lane_of(incl, 63);
    at.shares = shares_of(at.total, plain, lane_of(wave_incl_scan(units), 63), P.shares);
    if (wg >= at.shares) return false;
    int off = Shares(at.total, at.shares).first(wg);
    int owner = __popcll(__ballot(incl <= off));
    off -= lane_of(incl - n, owner);
    if (each > 1) {
        const int s = owner * each + lane;
        mine.seq = s;
        n = 0;
        if (lane < each && s < P.c.n_seqs) {
            open_seq(P, s, mine);
            n = seq_steps(P, mine) + at.setup * ((mine.rows + kFew - 1) / kFew);
        }
        incl = wave_incl_scan(n);
        owner = __popcll(__ballot(incl <= off));
        off -= lane_of(incl - n, owner);
    }
    w = lane_of(mine, owner);
    for (w.row0 = 0;; w.row0 += kFew) {
        see<kFew, kStep>(P, w);
        const int all = (w.n > 0 ? w.n : 1) + at.setup;
        if (off < all) break;
        off -= all;
    }
    at.off = off;
    return true;
}

__global__ __launch_bounds__(kThreads, 2) void few_kernel(AttendParams P) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    FewLds& L = *reinterpret_cast<FewLds*>(lds);
    const int t = threadIdx.x, wg = blockIdx.x;
    Work w;
    Place place;
    if (!locate(P, wg, w, place)) return;
    const Shares share(place.total, place.shares);
    int at = share.first(wg), off = place.off;
    const int end = share.first(wg + 1);
    for (bool lead = true;; lead = false) {
        see<kFew, kStep>(P, w);
        const int all = (w.n > 0 ? w.n : 1) + place.setup;
        const int take = all - off < end - at ? all - off : end - at;
        // the unit's own steps among them
        const int from = off > place.setup ? off - place.setup : 0;
        const int to = off + take - place.setup < w.n ? off + take - place.setup : w.n;
        if (w.len < 0 && t == 0) raise(P.h, FLEET_MOE_ABORT_POSITION);
        const bool whole = take == all;
        // a workgroup has at most two parts: its first, and its last
        const int slot = 2 * wg + (lead ? 0 : 1);
        attend(P, L, w, from, to > from ? to - from : 0, whole ? -1 : slot);
        if (off == 0 && t == 0) {
            const int64_t u = first_unit(w.tok0, w.seq, P.n_heads, kFew, P.pad) + w.row0 / kFew;
            const int last = share.holder(at + all - 1);
            P.meta[u] = make_int4(slot, wg + 1, whole ? 1 : last - wg + 1, 0);
        }
        at += take;
        if (at >= end) return;
        // the next unit
        off = 0;
        w.row0 += kFew;
        while (w.row0 >= w.rows) {
            if (w.seq + 1 >= P.c.n_seqs) return;
            open_seq(P, w.seq + 1, w);
        }
        barrier();                              // LDS is free again
    }
}

// Adds the parts of a row, in order: a workgroup per row, four groups of threads
// with a quarter of the parts each, the first few loaded before their weights are
// known. Latency bounds it.
constexpr int kJoinGroups = 4;
constexpr int kJoinThreads = kC / 4 * kJoinGroups;
constexpr int kJoinAhead = 4;
template <int R>
__device__ __forceinline__ void join(const AttendParams& P, int64_t row_at, int row, int64_t slot0,
                                     int64_t rest, int64_t step, int count) {
    __shared__ f32x4 sum_o[kJoinGroups][kC / 4];
    __shared__ float factor[kShares];
    const int t = threadIdx.x % (kC / 4), part = threadIdx.x / (kC / 4);
    const int lane = threadIdx.x & 63;
    const auto slot = [&](int i) { return (i == 0 ? slot0 : rest + (i - 1) * step) * R + row; };
    const auto load = [&](int i) {
        return ld_global(reinterpret_cast<const f32x4*>(P.part + slot(i) * kC) + t);
    };
    f32x4 v[kJoinAhead];
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i)
        v[i] = part + i * kJoinGroups < count ? load(part + i * kJoinGroups)
                                              : f32x4{0.f, 0.f, 0.f, 0.f};
    // the parts' weights: a lane per part
    float top = -INFINITY;
    for (int i = lane; i < count; i += 64) top = fmaxf(top, ld_global(P.stat + slot(i))[0]);
    top = wave_max(top);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f, rounded = 0.f;
    for (int i = lane; i < count; i += 64) {
        const f32x4 st = ld_global(P.stat + slot(i));
        const float f = exp2_(st[0] - ref);
        if (threadIdx.x < 64) factor[i] = f;
        sum += f * st[1];
        rounded += f * st[2];
    }
    sum = wave_sum(sum);
    rounded = wave_sum(rounded);
    __syncthreads();
    f32x4 o{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i)
        if (part + i * kJoinGroups < count) o += v[i] * factor[part + i * kJoinGroups];
#pragma unroll 4
    for (int i = part + kJoinAhead * kJoinGroups; i < count; i += kJoinGroups)
        o += load(i) * factor[i];
    sum_o[part][t] = o;
    __syncthreads();
    if (part) return;
    o = (sum_o[0][t] + sum_o[1][t]) + (sum_o[2][t] + sum_o[3][t]);
    put(P.out + row_at * kC + 4 * t, o, rounded == 0.f ? 0.f : 1.f / rounded);
    if (P.lse && threadIdx.x == 0) P.lse[row_at] = lse_of(top, sum);
}

// The same by one wave, kJoinWave parts at a time: enough where a row has hardly more, and
// four rows share a workgroup. (96 units of two parts joined by a workgroup a row, 6,144
// of them, four for each place on the chip: 22 us; by a wave a row 6.)
constexpr int kJoinWave = 16, kWaveParts = 16;
template <int R>
__device__ __forceinline__ void join_wave(const AttendParams& P, int64_t row_at, int row,
                                          int64_t slot0, int64_t rest, int64_t step, int count) {
    const int lane = threadIdx.x & 63;
    const auto slot = [&](int i) { return (i == 0 ? slot0 : rest + (i - 1) * step) * R + row; };
    f32x4 v[kJoinWave][2];
    const auto load = [&](int i0) {
#pragma unroll
        for (int i = 0; i < kJoinWave; ++i) {
            if (i0 + i >= count) break;
            const f32x4* at = reinterpret_cast<const f32x4*>(P.part + slot(i0 + i) * kC) + lane;
            v[i][0] = ld_global(at);
            v[i][1] = ld_global(at + 64);
        }
    };
    load(0);
    float top = -INFINITY;
    for (int i = lane; i < count; i += 64) top = fmaxf(top, ld_global(P.stat + slot(i))[0]);
    top = wave_max(top);
    const float ref = top == -INFINITY ? 0.f : top;
    float f = 0.f, sum = 0.f, rounded = 0.f;
    f32x4 o[2]{{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    for (int i0 = 0;;) {
        if (i0 % 64 == 0) {                     // the weights of 64 parts, a lane each
            f32x4 st{-INFINITY, 0.f, 0.f, 0.f};
            if (i0 + lane < count) st = ld_global(P.stat + slot(i0 + lane));
            f = exp2_(st[0] - ref);
            sum += f * st[1];
            rounded += f * st[2];
        }
#pragma unroll
        for (int i = 0; i < kJoinWave; ++i) {
            if (i0 + i >= count) break;
            const float weight = __builtin_bit_cast(
                float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), i0 % 64 + i));
            o[0] += v[i][0] * weight;
            o[1] += v[i][1] * weight;
        }
        i0 += kJoinWave;
        if (i0 >= count) break;
        load(i0);
    }
    static_assert(64 % kJoinWave == 0, "");
    sum = wave_sum(sum);
    rounded = wave_sum(rounded);
    const float inv = rounded == 0.f ? 0.f : 1.f / rounded;
    put(P.out + row_at * kC + 4 * lane, o[0], inv);
    put(P.out + row_at * kC + 4 * lane + 256, o[1], inv);
    if (P.lse && lane == 0) P.lse[row_at] = lse_of(top, sum);
}

// The unit of number u, if there is one.
template <int R, int S>
__device__ __forceinline__ bool find_work(const AttendParams& P, int64_t u, Work& w) {
    const int seq = find_seq(P.start, P.c.n_seqs, P.n_tokens, u, P.n_heads, R, P.pad);
    if (seq < 0) return false;
    open_seq(P, seq, w);
    const int64_t r = (u - first_unit(w.tok0, seq, P.n_heads, R, P.pad)) * R;
    if (r < 0 || r >= w.rows) return false;
    w.row0 = (int)r;
    see<R, S>(P, w);
    return true;
}

template <bool kWave>
__global__ __launch_bounds__(kWave ? 256 : kJoinThreads) void join_few_kernel(AttendParams P) {
    constexpr int kRows = kWave ? 4 : 1;
    const int64_t u = blockIdx.x / (kFew / kRows);
    const int row = blockIdx.x % (kFew / kRows) * kRows + (kWave ? wave_bcast(threadIdx.x >> 6) : 0);
    int64_t to = u * kFew + row;                // where units follow each other without gaps
    const int4 m = P.meta[u];
    if (P.pad == 0) {
        // (what is not between the first and the last start is no unit of this call)
        const int a = P.start ? clamp_row(ld_global(P.start), P.n_tokens) : 0;
        const int z = P.start ? clamp_row(ld_global(P.start + P.c.n_seqs), P.n_tokens)
                              : P.n_tokens;
        if (to < (int64_t)a * P.n_heads || to >= (int64_t)z * P.n_heads) return;
    } else {
        Work w;
        if (!find_work<kFew, kStep>(P, u, w) || w.row0 + row >= w.rows) return;
        to = out_row(P, w, w.row0 + row);
    }
    if (m.z <= 1) return;
    if constexpr (kWave) join_wave<kFew>(P, to, row, m.x, 2 * (int64_t)m.y, 2, m.z);
    else join<kFew>(P, to, row, m.x, 2 * (int64_t)m.y, 2, m.z);
}

// ---------------------------------------------------------------- many rows

// Prompts, and whatever else has more than 32 rows for a sequence: 64 rows a unit, four
// tiles of 16, a page a step, eight waves. The products bound it, so the step is large
// (a barrier's latency counts once for 64 x 64 scores) and the widening is shared: wave
// (tile pair, half, block pair) takes half of the 576 products of 32 rows with 32
// positions, so that each widened K operand serves two tiles; it exchanges halves with
// its partner, makes the weights of one tile and 32 positions, and adds its 64 columns
// of O for all 64 rows over the whole page, where each widened V operand serves four
// tiles. 72 registers of q, 64 of O: two waves a SIMD.
//
// A workgroup per unit, or several with a share of the unit's steps where there are
// few units. A sequence's last units come before its first ones: a causal prompt's are
// the longest. The last sequence's come first, whatever its length; of several sequences that
// is not the longest first, and ends later (the case below after 110 pages' time, where
// longest first would end after 103 and the mean is 93).
//
// Measured: the last 500 tokens of four sequences of up to 4,096 positions 250 us, 840
// TFLOP/s of the 1,212 that a library product of 8,192 cubed reaches. A step takes
// 5,350 cycles with its part of a unit's begin and end, 2,210 of them matrix instructions;
// two waves a SIMD issue 494 instructions each (308 vector ones with the 69 matrix, 100
// scalar, 40 of LDS), and a wave is ready without being issued 39% of its time. The second round
// of 455 units leaves 15% of the chip idle. Tried: 32 rows and four
// waves, two workgroups a CU 363 us (the copies of 32 rows take a third of the time), 64
// rows and four waves 288, two groups of four waves half a step apart 305 where this took
// 280. A prompt of 384: 26 us.
constexpr int kMany = 64;       // rows
constexpr int kManyWaves = 8;
constexpr int kManyThreads = kManyWaves * 64;
constexpr int kManyRing = 3;
struct ManyLds {
    __attribute__((aligned(16))) uint8_t tile[kManyRing][4 * kBlockStep];
    uint32_t scale[kManyRing][8];
    f32x4 half[kManyWaves][2][64];  // half of the scores of a tile and two blocks
    u32x4 p[2][4][2][64];       // [step parity][tile][half of the page][lane]
    int flag[2][kManyWaves];
    float m[4][16], top[4][2][16], sum[4][2][16], rounded[4][2][16];
};
static_assert(sizeof(ManyLds) <= 160 * 1024, "");
static_assert(kShares / 2 * kMany <= kPartRows, "units are divided into kShares / 2 parts at most");

__global__ __launch_bounds__(kManyThreads, 1) void many_kernel(AttendParams P) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    ManyLds& L = *reinterpret_cast<ManyLds*>(lds);
    constexpr int kCols = kC / 16 / kManyWaves; // of 16
    const int t = threadIdx.x, lane = t & 63, wave = wave_bcast(t >> 6);
    const int g = lane >> 4, n = lane & 15;
    const int bp = wave & 1, half = wave >> 1 & 1, tp = wave >> 2;
    const int mine = 2 * tp + half;             // the tile whose weights this wave makes
    const int unit = P.units - 1 - blockIdx.x / P.shares, split = blockIdx.x % P.shares;
    Work w;
    if (!find_work<kMany, kPage>(P, unit, w)) return;
    const int each = (w.n + P.shares - 1) / P.shares;
    const int off = split * each;
    const int cnt = off + each < w.n ? each : w.n - off;
    if (split > 0 && cnt <= 0) return;
    const bool whole = each >= w.n;             // no other workgroup has these rows
    if (w.len < 0 && t == 0 && split == 0) raise(P.h, FLEET_MOE_ABORT_POSITION);

    const Row r = row_of(P, w, w.row0 + mine * 16 + n);
    const Common common(r);
    bf16x8 q[2][kHalf];                         // of `mine` and of the pair's other tile
    load_q(P, w, r, g, half, q[0]);
    load_q(P, w, row_of(P, w, w.row0 + (mine ^ 1) * 16 + n), g, half, q[1]);
    f32x4 acc[4][kCols];
#pragma unroll
    for (auto& a : acc)
#pragma unroll
        for (auto& b : a) b = f32x4{0.f, 0.f, 0.f, 0.f};
    // the sum of the rounded weights of tile wave & 3 and half of the page wave >> 2
    f32x4 ones{0.f, 0.f, 0.f, 0.f};
    // the references of the wave's tile (see attend())
    float m = -INFINITY, ref = -INFINITY, l = 0.f;
    const float slack = P.slack;
    f32x4 z[2];                                 // the scores of `mine` and the two blocks
    float p0[4], p1[4];
    bool stray = false;                         // a score of the wave is not finite
    if (t < 64) L.m[t >> 4][n] = -INFINITY;
    Pages pages{0, 0, 0};
    if (cnt > 0) page_of<kPage>(P, w, pages, off, off + cnt, lane);
    __builtin_amdgcn_s_waitcnt(0x0F70);         // vmcnt(0): see attend()

    // (b is k % kManyRing, counted: of a remainder the compiler makes two products and a
    // difference for every address)
    const auto issue = [&](int k, int b) {
        const int page = page_of<kPage>(P, w, pages, off + k, off + cnt, lane);
        const int64_t base = page_offset(page, P.c.n_pages, P.layer, P.c.n_layers);
        const uint8_t* src = P.c.pool + (base < 0 ? 0 : base);
        // a wave a block; the first the scales too
        const uint8_t* from = src + wave * kBlockBytes + lane * 16;
        const uint32_t to = lds_addr(L.tile[b]) + wave * kBlockStep;
        copy_kb<4, false>(from, to);
        copy_kb<4, false>(from + 4096, to + 4096);
        copy_kb<1, false>(from + 8192, to + 8192);
        if (wave == 0 && lane < 2)
            copy_kb<1, false>(src + kCodeBytes + lane * 16, lds_addr(L.scale[b]));
    };
    const auto score = [&](int b) {
        u32x4 c[2][4];
        uint2 e[2];
        uint32_t f[2][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint8_t* block = L.tile[b] + (2 * bp + j) * kBlockStep + lane * 16;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                c[j][i] = *reinterpret_cast<const u32x4*>(block + (2 * i + half) * 1024);
            e[j] = *reinterpret_cast<const uint2*>(block + 8 * 1024 + half * 8);
            f[j][0] = L.scale[b][2 * (2 * bp + j)];
            f[j][1] = L.scale[b][2 * (2 * bp + j) + 1];
        }
        __builtin_amdgcn_sched_barrier(0);      // every read on its way
        f32x4 y[2][2];                          // [tile][block]
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float sc = any_scale(f[j][0]), sp = any_scale(f[j][1]);
            y[0][j] = y[1][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const u32x4 a = c[j][i];
                const bf16x8 lo = widen(a.x, a.y, sc, sc), hi = widen(a.z, a.w, sc, sc);
                y[0][j] = mfma(lo, q[0][2 * i], y[0][j]);
                y[1][j] = mfma(lo, q[1][2 * i], y[1][j]);
                y[0][j] = mfma(hi, q[0][2 * i + 1], y[0][j]);
                y[1][j] = mfma(hi, q[1][2 * i + 1], y[1][j]);
            }
            const bf16x8 pe = widen(e[j].x, e[j].y, sp, sp);
            y[0][j] = mfma(pe, q[0][8], y[0][j]);
            y[1][j] = mfma(pe, q[1][8], y[1][j]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            z[j] = y[0][j];
            L.half[wave][j][lane] = y[1][j];
        }
    };
    const auto weigh = [&](int k) {
        const float down = ref == -INFINITY ? 0.f : ref;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            p0[j] = exp2_(fmaf(z[0][j], P.scale, -down));
            p1[j] = exp2_(fmaf(z[1][j], P.scale, -down));
        }
        const uint2 a = weights(p0), b = weights(p1);
        L.p[k & 1][mine][bp][lane] = u32x4{a.x, a.y, b.x, b.y};
    };
    const auto finish = [&](int k) {
#pragma unroll
        for (int j = 0; j < 2; ++j) z[j] += L.half[wave ^ 2][j][lane];
        const int page = page_of<kPage>(P, w, pages, off + k, off + cnt, lane);
        const bool ok = (unsigned)page < (unsigned)P.c.n_pages;
        const int base = step_of<kPage>(w, off + k) * kPage + bp * 32;
        const f32x4 both = z[0] + z[1];
        const bool bad = !finite((both[0] + both[1]) + (both[2] + both[3]));
        if (!(ok && common.all(base, 32))) {
            asm volatile("");                   // a branch, not forty instructions every step
            if (!ok && t == 0) raise(P.h, FLEET_MOE_ABORT_BAD_PAGE);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    z[j][i] = (ok & sees(r, base + kBlock * j + 4 * g + i)) ? z[j][i] : -INFINITY;
        }
        weigh(k);
        const float top = fmaxf(fmaxf(fmaxf(z[0][0], z[0][1]), fmaxf(z[0][2], z[0][3])),
                                fmaxf(fmaxf(z[1][0], z[1][1]), fmaxf(z[1][2], z[1][3])));
        stray = __ballot(bad) != 0;
        const bool high = __ballot(top > m + slack) != 0;
        if (lane == 0) L.flag[k & 1][wave] = stray | high;
    };
    // What is rare: a row's scores beyond its reference, or one that is not finite, in step k.
    const auto mend = [&](int k, int b) {
        float top = fmaxf(fmaxf(fmaxf(z[0][0], z[0][1]), fmaxf(z[0][2], z[0][3])),
                          fmaxf(fmaxf(z[1][0], z[1][1]), fmaxf(z[1][2], z[1][3])));
        top = xor32_max(xor16_max(top));
        if (lane < 16) L.top[mine][bp][lane] = top;
        if (stray && half == 0 && tp == 0)
            for (int j = 0; j < 2; ++j)
                clean(L.tile[b] + (2 * bp + j) * kBlockStep, L.scale[b][2 * (2 * bp + j)], lane);
        barrier();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float was = L.m[i][n];
            const float to = fmaxf(was, fmaxf(L.top[i][0][n], L.top[i][1][n]));
            const float shrink = shrink_to(to * P.scale, was * P.scale);
            if (i == mine) {
                m = to;
                ref = reference(to * P.scale);
                l *= shrink;
            }
            if (i == (wave & 3)) ones *= shrink;
#pragma unroll
            for (auto& a : acc[i]) a *= shrink;
        }
        weigh(k);
        barrier();
        if (bp == 0 && lane < 16) L.m[mine][lane] = m;
    };
    // O over step k
    const auto add = [&](int k, int b) {
        uint32_t first = lds_addr(L.tile[b]) + wave * kCols * 256 + column_at(lane);
        asm("" : "+v"(first));                // one address, the rest is offsets
        bf16x8 pb[2][4];
        i32x2 v[2][kCols];
        uint32_t f[2][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t col = first + 2 * h * kBlockStep;
#pragma unroll
            for (int i = 0; i < kCols; ++i) v[h][i] = column(col, i);
#pragma unroll
            for (int j = 0; j < 4; ++j) pb[h][j] = __builtin_bit_cast(bf16x8, L.p[k & 1][j][h][lane]);
            f[h][0] = L.scale[b][4 * h];
            f[h][1] = L.scale[b][4 * h + 2];
        }
        __builtin_amdgcn_sched_barrier(0);      // every read on its way
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float sa = any_scale(f[h][0]), sb = any_scale(f[h][1]);
#pragma unroll
            for (int i = 0; i < kCols; ++i) {
                const bf16x8 a = widen((uint32_t)v[h][i].x, (uint32_t)v[h][i].y, sa, sb);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j][i] = mfma(a, pb[h][j], acc[j][i]);
            }
        }
        ones = mfma(__builtin_bit_cast(bf16x8, u32x4{kOnes, kOnes, kOnes, kOnes}),
                    __builtin_bit_cast(bf16x8, L.p[k & 1][wave & 3][wave >> 2][lane]), ones);
    };

    if (tp == 0)
        for (int k = 0; k < kManyRing - 1 && k < cnt; ++k) issue(k, k);
    wait_copies<0>();
    barrier();
    if (cnt > 0) {
        score(0);
        barrier();
        finish(0);
    }
    // Step k: behind barrier A the weights of k and the rows of k + 1 are there, behind
    // B both halves of the scores of k + 1.
    int b = 0;                                  // of step k
    for (int k = 0; k < cnt; ++k) {
        const int b1 = b == kManyRing - 1 ? 0 : b + 1, b2 = b1 == kManyRing - 1 ? 0 : b1 + 1;
        wait_copies<0>();                       // step k + 1
        barrier();                              // A
        const int* f = L.flag[k & 1];
        const int flags = ((f[0] | f[1]) | (f[2] | f[3])) | ((f[4] | f[5]) | (f[6] | f[7]));
        if (tp == 0 && k + kManyRing - 1 < cnt) issue(k + kManyRing - 1, b2);      // where step k - 1 was
        if (wave_bcast(flags)) mend(k, b);
        l += ((p0[0] + p0[1]) + (p0[2] + p0[3])) + ((p1[0] + p1[1]) + (p1[2] + p1[3]));
        if (k + 1 < cnt) {
            score(b1);
            barrier();                          // B
            finish(k + 1);
        }
        add(k, b);
        b = b1;
        asm("" : "+s"(b));
    }
    // the sums of the blocks, and of the page's halves
    l = xor32_sum(xor16_sum(l));
    if (lane < 16) {
        L.sum[mine][bp][lane] = l;
        L.rounded[wave & 3][wave >> 2][lane] = ones[0];
        if (bp == 0) L.m[mine][lane] = m;
    }
    barrier();
    const int64_t slot = (int64_t)unit * P.shares + split;
    const int column0 = wave * kCols * 16 + 4 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = i * 16 + n;
        const float sum = L.sum[i][0][n] + L.sum[i][1][n];
        const float rounded = L.rounded[i][0][n] + L.rounded[i][1][n];
        const float scaled = L.m[i][n] * P.scale;
        if (whole) {
            if (w.row0 + row < w.rows) {
                const int64_t to = out_row(P, w, w.row0 + row);
                const float inv = rounded == 0.f ? 0.f : 1.f / rounded;
#pragma unroll
                for (int j = 0; j < kCols; ++j)
                    put(P.out + to * kC + column0 + j * 16, acc[i][j], inv);
                if (P.lse && wave == 0 && g == 0) P.lse[to] = lse_of(scaled, sum);
            }
        } else {
            const int64_t at = slot * kMany + row;
#pragma unroll
            for (int j = 0; j < kCols; ++j)
                st_global(reinterpret_cast<f32x4*>(P.part + at * kC + column0 + j * 16), acc[i][j]);
            if (wave == 0 && g == 0) st_global(P.stat + at, f32x4{scaled, sum, rounded, 0.f});
        }
    }
}

template <bool kWave>
__global__ __launch_bounds__(kWave ? 256 : kJoinThreads) void join_many_kernel(AttendParams P) {
    constexpr int kRows = kWave ? 4 : 1;
    const int64_t u = blockIdx.x / (kMany / kRows);
    const int row = blockIdx.x % (kMany / kRows) * kRows + (kWave ? wave_bcast(threadIdx.x >> 6) : 0);
    Work w;
    if (!find_work<kMany, kPage>(P, u, w) || w.row0 + row >= w.rows) return;
    const int each = (w.n + P.shares - 1) / P.shares;
    if (each >= w.n) return;
    const int count = (w.n + each - 1) / each;
    const int64_t to = out_row(P, w, w.row0 + row), first = u * P.shares;
    if constexpr (kWave) join_wave<kMany>(P, to, row, first, first + 1, 1, count);
    else join<kMany>(P, to, row, first, first + 1, 1, count);
}

}  // namespace cache
}  // namespace fleet_moe

using namespace fleet_moe;
using namespace fleet_moe::cache;

int fleet_moe_check_device(int min_cus);

// More than 64 KB of dynamic LDS has to be asked for. (The LDS is dynamic so that
// the compiler keeps to the registers of two waves on a SIMD, and takes O as an
// operand of the matrix instructions from them; where it knows that LDS allows one
// only, it moves O to accumulation registers and back, 400 moves a step.)
template <auto Kernel>
static int launch(int64_t grid, int threads, size_t lds, const AttendParams& P,
                  hipStream_t stream) {
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

extern "C" int fleet_cache_attend(const fleet_cache* cache, int32_t layer, const uint16_t* q,
                                  int64_t q_stride, const int32_t* start, int32_t n_tokens,
                                  int32_t n_heads, int32_t max_len, int32_t window, int32_t sinks,
                                  float scale, uint16_t* out, float* lse, void* workspace,
                                  size_t workspace_bytes, hipStream_t stream) {
    if (int e = check_cache(cache, workspace, workspace_bytes)) return e;
    if (layer < 0 || layer >= cache->n_layers || n_tokens < 0 || n_heads < 1 ||
        n_heads > FLEET_CACHE_MAX_HEADS || (int64_t)n_tokens * n_heads > kMaxRows ||
        max_len < 0 || window < 0 || sinks < 0 || !(scale > 0.f) || !(scale * kLog2e <= FLT_MAX) ||
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
    char* ws = static_cast<char*>(workspace) + parts_at(cache->n_seqs, cache->n_pages);
    P.h = static_cast<Header*>(workspace);
    P.part = reinterpret_cast<float*>(ws);
    P.stat = reinterpret_cast<f32x4*>(ws + kPartBytes);
    P.meta = reinterpret_cast<int4*>(ws + kPartBytes + kStatBytes);
    P.q_stride = q_stride;
    P.layer = layer;
    P.n_tokens = n_tokens;
    P.n_heads = n_heads;
    P.per_head = head_divisor(n_heads);
    P.window = window;
    P.sinks = sinks;
    P.scale = scale * kLog2e;
    P.slack = fminf(kSlack / P.scale, FLT_MAX);
    // positions that a row may see, as far as the host knows
    int64_t seen = (int64_t)cache->max_pages * kPage;
    if (max_len > 0 && max_len < seen) seen = max_len;
    if (window > 0 && (int64_t)window + sinks + n_tokens < seen)
        seen = (int64_t)window + sinks + n_tokens;
    const int64_t rows = (int64_t)n_tokens * n_heads;
    P.pad = n_heads % kFew != 0;
    const int64_t few = first_unit(n_tokens, cache->n_seqs, n_heads, kFew, P.pad);
    if (rows <= 2 * kFew * (int64_t)cache->n_seqs && few <= kMaxUnits &&
        2 * few * cache->max_pages < (1 << 30)) {
        P.units = (int)few;
        const int64_t steps = few * ((seen + kStep - 1) / kStep);
        P.shares = (int)(steps < kShares ? steps : kShares);
        if (int e = launch<few_kernel>(P.shares, kThreads, sizeof(FewLds), P, stream)) return e;
        // A wave a row where the mean is up to 16 parts (64 sequences of 4,000 positions 42
        // to 41 us, of 1,000 25.4 to 23.9; 16 of 1,000 the same), a workgroup a row for more.
        if (P.shares <= kWaveParts * few)
            return launch<join_few_kernel<true>>(few * (kFew / 4), 256, 0, P, stream);
        return launch<join_few_kernel<false>>(few * kFew, kJoinThreads, 0, P, stream);
    }
    P.pad = n_heads % kMany != 0;
    const int64_t units = first_unit(n_tokens, cache->n_seqs, n_heads, kMany, P.pad);
    P.units = (int)units;
    // Few units divide their pages, into parts of 4 or more, unless fewer than 8 pages
    // (2.4 us each) are saved: parts and join cost 6 us and, of 256 parts, 11 more.
    // Measured, divided and not: 64 tokens of 16 heads at the end of 8,192
    // positions 47 and 310 us, of 1,024 29 and 49; 384 at the end of 384, 33 and 28.
    const int64_t n_pages = (seen + kPage - 1) / kPage;
    int64_t splits = kShares / 2 / units;
    if (splits > (n_pages + 3) / 4) splits = (n_pages + 3) / 4;
    if (splits < 1 || n_pages - n_pages / splits < 8) splits = 1;
    P.shares = (int)splits;
    if (int e = launch<many_kernel>(units * P.shares, kManyThreads, sizeof(ManyLds), P, stream))
        return e;
    if (P.shares == 1) return 0;
    // (the same to a few percent from 4 parts to 16: 45.7 to 46.5 us of 8,192 positions)
    if (P.shares <= kWaveParts)
        return launch<join_many_kernel<true>>(units * (kMany / 4), 256, 0, P, stream);
    return launch<join_many_kernel<false>>(units * kMany, kJoinThreads, 0, P, stream);
}
