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
    float* part;                // partial O, fp32 [slot][rows][512]
    f32x4* stat;                // [slot][rows]: reference, sum, rounded sum
    int4* meta;                 // [unit]: first slot, next workgroup, number of slots
    Header* h;
    int64_t q_stride;
    uint64_t per_head;          // floor(2^40 / n_heads) + 1
    int layer, n_tokens, n_heads, window, sinks, pad, units;
    int shares;                 // workgroups, or splits of a unit
    float scale;                // times log2(e)
};

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr float kSlack = 8.f;
constexpr float kLn2 = 0.6931471805599453f;

// row / n_heads: exact for row < 2^33 (n_heads * per_head is over 2^40 by n_heads at most).
__device__ __forceinline__ int token_of(const AttendParams& P, int row) {
    return (int)((uint64_t)(uint32_t)row * P.per_head >> 40);
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
    w.rows = w.n_new * P.n_heads;
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
// Its query as the right operand: the k order of the products is that of the bytes
// a lane of group g takes of a row: chunks g, 4 + g, ..
template <int N>                // N of the 18 steps of 32 values, from `step` on
__device__ __forceinline__ void load_q(const AttendParams& P, const Work& w, const Row& r, int g,
                                       int step, bf16x8 (&q)[N]) {
    const uint16_t* src = P.q + (int64_t)(w.tok0 + r.tok) * P.q_stride + r.head * kRow + g * 16;
#pragma unroll
    for (int i = 0; i < N; ++i)
        q[i] = __builtin_bit_cast(bf16x8, ld_global(reinterpret_cast<const u32x4*>(
                                              src + (step + i) / 2 * 64 + (step + i) % 2 * 8)));
}
__device__ __forceinline__ int64_t out_row(const AttendParams& P, const Work& w, int row) {
    return (int64_t)w.tok0 * P.n_heads + row;
}

// Blocks in LDS lie 64 bytes further apart than they are long, so that the two
// halves of a transposing read, from neighbouring blocks, fall into different banks.
constexpr int kBlockStep = kBlockBytes + 64;

// Copies 16 bytes per lane from global memory to LDS, 1 KB in all: to `lds` + 16 lane.
// There is no register for the data, so none is in flight behind the compiler's
// back. In asm, because the compiler would wait for every copy in flight before each
// LDS read; wait_copies() orders them.
template <bool kOnce>           // read once: kept out of the caches
__device__ __forceinline__ void copy_kb(const uint8_t* src, uint32_t lds) {
    if constexpr (kOnce)
        asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(src), "{m0}"(lds)
                     : "memory");
    else
        asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(lds)
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

// The transposing read: 8 positions of one of the 16 dimensions of chunk i. `col`
// is what column_at() gives: lane r of a group of 16 points at row r / 2 of 8,
// positions 4g .. 4g + 3 of two neighbouring blocks.
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
__device__ __forceinline__ const uint8_t* column_at(const uint8_t* block, int lane) {
    const int r = (lane & 15) >> 1;
    return block + (r < 4 ? 0 : kBlockStep) + (4 * (lane >> 4) + (r & 3)) * 16 + (lane & 1) * 8;
}
__device__ __forceinline__ i32x2 column(const uint8_t* col, int i) {
    return __builtin_amdgcn_ds_read_tr8_b64_v2i32(
        (lds_i32x2*)(const __attribute__((address_space(3))) uint8_t*)(col + i * 256));
}

// A block's NaN codes as zeros, by one wave. A NaN in a row makes the score, and
// so the weight, of every row of q that sees it NaN; a row that does not see it
// has the weight 0, and must not meet 0 * NaN.
__device__ __forceinline__ void clean(uint8_t* block, int lane) {
    for (int i = 0; i < kC / 64; ++i) {
        u32x4* at = reinterpret_cast<u32x4*>(block + i * 1024 + lane * 16);
        u32x4 v = *at;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = drop_nan(v[j]);
        *at = v;
    }
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

// Pages of the next 64 steps, one per lane.
struct Pages {
    int held, from;
    int page;
};
template <int S>
__device__ __forceinline__ int page_of(const AttendParams& P, const Work& w, Pages& h, int i,
                                       int end, int lane) {
    if (i >= h.held) {
        h.from = i;
        h.held = i + 64;
        h.page = i + lane < end ? ld_global(P.c.table + (int64_t)w.seq * P.c.max_pages +
                                            step_of<S>(w, i + lane) * S / kPage)
                                : 0;
    }
    return __builtin_amdgcn_readlane(h.page, i - h.from);
}

// ---------------------------------------------------------------- few rows

// Sequences with a token or two: 16 rows a unit, 32 positions (two blocks, half a
// page) a step. The bytes of the pages bound it (576 a position for 16 rows, 60 flops
// a byte), so what matters is that they keep coming: four steps fit in LDS, two or
// three of them on their way, and two workgroups share a CU, so that one's
// barriers and latencies are the other's time. A block's scores are shared by two
// waves, half of the 576 products each; the first two waves add the halves up and
// make the weights while the other two issue the copies (a copy of 1 KB occupies the
// address unit for 24 cycles, so that holds a wave up). Then each wave adds its 128
// columns of O: 32 registers a lane, and no sum over waves at the end.
//
// The work is divided into equal shares of steps over all units, whatever their
// lengths: a workgroup takes a range of the concatenated steps, across units where it
// has to. A unit that several have a part in leaves partial results, which
// join_few_kernel adds in order.
constexpr int kDeep = 4;        // steps in LDS
constexpr int kStep = 32;       // positions
struct FewLds {
    __attribute__((aligned(16))) uint8_t tile[kDeep][2 * kBlockStep];
    uint32_t scale[kDeep][64];
    f32x4 half[2][64];          // the second half of a block's scores
    u32x4 p[2][64];             // [step parity][lane]
    float top[2][2][16];
    int flag[2][2];
    float sum[2][16];
};
static_assert(sizeof(FewLds) <= 80 * 1024, "two workgroups share a CU");
constexpr int kFew = 16;        // rows

constexpr int kStepCopies = 10; // of each of two waves: 9 KB of codes, and the scales
constexpr int kNeedMax = 1, kHasNan = 2;

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

// The total of all units' steps; its division (no share is empty: the join counts
// on it); and the unit in which workgroup wg's part begins, and where. Every
// wave for itself, a lane per sequence (or for several, then once more a lane for each
// of the one lane's): no barrier, and one round of loads for 64 sequences.
__device__ __forceinline__ bool locate(const AttendParams& P, int wg, Work& w, int& off, int& total,
                                       int& shares) {
    const int lane = threadIdx.x & 63;
    const int each = (P.c.n_seqs + 63) / 64;
    Work mine{};
    int n = 0;
    for (int i = 0; i < each; ++i) {
        const int s = lane * each + i;
        if (s < P.c.n_seqs) {
            open_seq(P, s, mine);
            n += seq_steps(P, mine);
        }
    }
    int incl = wave_incl_scan(n);
    total = lane_of(incl, 63);
    shares = total < P.shares ? total : P.shares;
    if (wg >= shares) return false;
    off = Shares(total, shares).first(wg);
    int owner = __popcll(__ballot(incl <= off));
    off -= lane_of(incl - n, owner);
    if (each > 1) {
        const int s = owner * each + lane;
        mine.seq = s;
        n = 0;
        if (lane < each && s < P.c.n_seqs) {
            open_seq(P, s, mine);
            n = seq_steps(P, mine);
        }
        incl = wave_incl_scan(n);
        owner = __popcll(__ballot(incl <= off));
        off -= lane_of(incl - n, owner);
    }
    w = lane_of(mine, owner);
    for (w.row0 = 0;; w.row0 += kFew) {
        see<kFew, kStep>(P, w);
        const int all = w.n > 0 ? w.n : 1;
        if (off < all) return true;
        off -= all;
    }
}

__global__ __launch_bounds__(kThreads, 2) void few_kernel(AttendParams P) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    FewLds& L = *reinterpret_cast<FewLds*>(lds);
    const int t = threadIdx.x, lane = t & 63, wave = wave_bcast(t >> 6);
    const int g = lane >> 4, n = lane & 15, blk = wave & 1;
    const bool first = wave < 2;
    const int wg = blockIdx.x;
    Work w;
    int off, total, shares;
    if (!locate(P, wg, w, off, total, shares)) return;
    const Shares share(total, shares);
    int at = share.first(wg);
    const int end = share.first(wg + 1);
    for (bool lead = true;; lead = false) {
        see<kFew, kStep>(P, w);
        const int all = w.n > 0 ? w.n : 1;
        const int take = all - off < end - at ? all - off : end - at;
        const int until = off + take < w.n ? off + take : w.n;
        const int cnt = until > off ? until - off : 0;
        const Row r = row_of(P, w, w.row0 + n);
        if (w.len < 0 && t == 0) raise(P.h, FLEET_MOE_ABORT_POSITION);

        constexpr int kHalf = kChunks / 4;      // steps of 32 values, of 18
        bf16x8 q[kHalf];
        load_q(P, w, r, g, first ? 0 : kHalf, q);
        constexpr int kCols = kC / 16 / kWaves;
        f32x4 acc[kCols];
#pragma unroll
        for (auto& a : acc) a = f32x4{0.f, 0.f, 0.f, 0.f};
        f32x4 ones{0.f, 0.f, 0.f, 0.f};         // the sum of the rounded weights
        f32x4 z;
        float m = -INFINITY, l = 0.f;
        float s[4], p[4];
        Pages pages{0, 0, 0};
        // copies step k: the last two waves
        const auto issue = [&](int k) {
            const int page = page_of<kStep>(P, w, pages, off + k, until, lane);
            const int64_t base = page_offset(page, P.c.n_pages, P.layer, P.c.n_layers);
            const uint8_t* src = P.c.pool + (base < 0 ? 0 : base);
            const int b = k % kDeep, half = step_of<kStep>(w, off + k) & 1;
            const uint8_t* from = src + (2 * half + blk) * kBlockBytes + lane * 16;
            const uint32_t to = lds_addr(L.tile[b]) + blk * kBlockStep;
#pragma unroll
            for (int i = 0; i < kBlockBytes / 1024; ++i) copy_kb<true>(from + i * 1024, to + i * 1024);
            copy_words(src + kCodeBytes + half * 16 + (lane & 3) * 4, lds_addr(L.scale[b]));
        };
        // this wave's half of its block's scores
        const auto score = [&](int k) {
            const int b = k % kDeep;
            const uint8_t* block = L.tile[b] + blk * kBlockStep + lane * 16;
            const float sc = any_scale(L.scale[b][2 * blk]);
            f32x4 z0{0.f, 0.f, 0.f, 0.f}, z1{0.f, 0.f, 0.f, 0.f};
            const auto chunk = [&](int i) { return *reinterpret_cast<const u32x4*>(block + i * 1024); };
            if (first) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const u32x4 a = chunk(i);
                    z0 = mfma(widen(a.x, a.y, sc, sc), q[2 * i], z0);
                    z1 = mfma(widen(a.z, a.w, sc, sc), q[2 * i + 1], z1);
                }
                const u32x4 a = chunk(4);
                z0 = mfma(widen(a.x, a.y, sc, sc), q[8], z0);
            } else {
                const float sp = any_scale(L.scale[b][2 * blk + 1]);
                u32x4 a = chunk(4);
                z0 = mfma(widen(a.z, a.w, sc, sc), q[0], z0);
#pragma unroll
                for (int i = 5; i < 8; ++i) {
                    a = chunk(i);
                    z1 = mfma(widen(a.x, a.y, sc, sc), q[2 * i - 9], z1);
                    z0 = mfma(widen(a.z, a.w, sc, sc), q[2 * i - 8], z0);
                }
                a = chunk(8);
                z1 = mfma(widen(a.x, a.y, sp, sp), q[7], z1);
                z0 = mfma(widen(a.z, a.w, sp, sp), q[8], z0);
            }
            z = z0 + z1;
            if (!first) L.half[blk][lane] = z;
        };
        // the weights of step k under the reference m: the first two waves
        const auto weigh = [&](int k) {
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = exp2_(s[j] - ref);
            reinterpret_cast<uint2*>(&L.p[k & 1][lane])[blk] = weights(p);
        };
        const auto finish = [&](int k) {
            z += L.half[blk][lane];
            float top = -INFINITY;
            bool nan = false;
            const int page = page_of<kStep>(P, w, pages, off + k, until, lane);
            const bool ok = (unsigned)page < (unsigned)P.c.n_pages;
            if (!ok && t == 0) raise(P.h, FLEET_MOE_ABORT_BAD_PAGE);
            const int base = step_of<kStep>(w, off + k) * kStep + blk * kBlock + 4 * g;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float v = z[j] * P.scale;
                nan |= v != v;
                const int pos = base + j;
                s[j] = ok && pos <= r.pos && (pos >= r.seen.lo || pos < r.seen.sink) ? v : -INFINITY;
                top = fmaxf(top, s[j]);
            }
            top = xor32_max(xor16_max(top));
            weigh(k);
            if (lane < 16) L.top[k & 1][blk][lane] = top;
            const int flag = (__ballot(top > m + kSlack) ? kNeedMax : 0) |
                             (__ballot(nan) ? kHasNan : 0);
            if (lane == 0) L.flag[k & 1][blk] = flag;
        };
        // Step k: behind barrier A the weights of k and the rows of k + 1 are there, behind
        // B both halves of the scores of k + 1.
        if (!first) {
            for (int k = 0; k < kDeep - 1 && k < cnt; ++k) issue(k);
            if (cnt > 2) wait_copies<2 * kStepCopies>();
            else if (cnt > 1) wait_copies<kStepCopies>();
            else wait_copies<0>();
        }
        barrier();
        for (int k = -1; k < cnt; ++k) {
            if (k + 1 < cnt) {
                score(k + 1);
                barrier();                      // B
                if (first) {
                    finish(k + 1);
                } else {
                    // into the buffer of step k - 1
                    if (k >= 0 && k + kDeep - 1 < cnt) issue(k + kDeep - 1);
                    // step k + 2; the one behind it may be on its way
                    if (cnt - k > 3) wait_copies<kStepCopies>();
                    else wait_copies<0>();
                }
            }
            if (k >= 0) {
                const int b = k % kDeep, par = k & 1;
                const bf16x8 pb = __builtin_bit_cast(bf16x8, L.p[par][lane]);
                const float sa = any_scale(L.scale[b][0]), sb = any_scale(L.scale[b][2]);
                const uint8_t* col = column_at(L.tile[b], lane) + wave * kCols * 256;
#pragma unroll
                for (int i = 0; i < kCols; ++i) {
                    const i32x2 v = column(col, i);
                    acc[i] = mfma(widen((uint32_t)v.x, (uint32_t)v.y, sa, sb), pb, acc[i]);
                }
                ones = mfma(__builtin_bit_cast(bf16x8, u32x4{kOnes, kOnes, kOnes, kOnes}), pb, ones);
            }
            if (k + 1 == cnt) break;
            barrier();                          // A
            const int par = (k + 1) & 1;
            const int any = wave_bcast(L.flag[par][0] | L.flag[par][1]);
            if (any) {
                // m is any reference not far below the maximum: weights up to 2^kSlack
                // are as exact as those up to 1, and moving it costs a pass over O and a
                // barrier
                if (any & kNeedMax) {
                    float to = m;
#pragma unroll
                    for (int i = 0; i < 2; ++i) to = fmaxf(to, L.top[par][i][n]);
                    const float shrink = to == -INFINITY ? 1.f : exp2_(m - to);
                    m = to;
                    l *= shrink;
                    ones *= shrink;
#pragma unroll
                    for (auto& a : acc) a *= shrink;
                    if (first) weigh(k + 1);
                }
                if ((any & kHasNan) && first)
                    clean(L.tile[(k + 1) % kDeep] + blk * kBlockStep, lane);
                barrier();
            }
            if (first) l += (p[0] + p[1]) + (p[2] + p[3]);
        }
        // the sums of the two blocks
        l = xor32_sum(xor16_sum(l));
        if (first && lane < 16) L.sum[blk][lane] = l;
        barrier();
        const float sum = L.sum[0][n] + L.sum[1][n];
        const bool whole = take == all;
        const int column0 = wave * kCols * 16 + 4 * g;
        if (whole) {
            if (r.live) {
                const int64_t to = out_row(P, w, w.row0 + n);
                const float inv = ones[0] == 0.f ? 0.f : 1.f / ones[0];
#pragma unroll
                for (int i = 0; i < kCols; ++i) put(P.out + to * kC + column0 + i * 16, acc[i], inv);
                if (P.lse && wave == 0 && g == 0) P.lse[to] = lse_of(m, sum);
            }
        } else {
            // a workgroup has at most two such: its first, and its last
            const int slot = 2 * wg + (lead ? 0 : 1);
            float* part = P.part + ((int64_t)slot * kFew + n) * kC + column0;
#pragma unroll
            for (int i = 0; i < kCols; ++i)
                st_global(reinterpret_cast<f32x4*>(part + i * 16), acc[i]);
            if (wave == 0 && g == 0) st_global(P.stat + slot * kFew + n, f32x4{m, sum, ones[0], 0.f});
        }
        if (off == 0 && t == 0) {
            const int64_t u = first_unit(w.tok0, w.seq, P.n_heads, kFew, P.pad) + w.row0 / kFew;
            const int last = share.holder(at + all - 1);
            P.meta[u] = make_int4(2 * wg + (lead ? 0 : 1), wg + 1, whole ? 1 : last - wg + 1, 0);
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
// with a quarter of the parts each.
constexpr int kJoinGroups = 4;
constexpr int kJoinThreads = kC / 4 * kJoinGroups;
template <int R>
__device__ __forceinline__ void join(const AttendParams& P, int64_t row_at, int row, int64_t slot0,
                                     int64_t rest, int64_t step, int count) {
    __shared__ f32x4 sum_o[kJoinGroups][kC / 4];
    const int t = threadIdx.x % (kC / 4), part = threadIdx.x / (kC / 4);
    const auto slot = [&](int i) { return (i == 0 ? slot0 : rest + (i - 1) * step) * R + row; };
    // the parts' weights: a lane per part
    __shared__ float factor[kShares];
    const int lane = threadIdx.x & 63;
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
#pragma unroll 4
    for (int i = part; i < count; i += kJoinGroups)
        o += ld_global(reinterpret_cast<const f32x4*>(P.part + slot(i) * kC) + t) * factor[i];
    sum_o[part][t] = o;
    __syncthreads();
    if (part) return;
    o = (sum_o[0][t] + sum_o[1][t]) + (sum_o[2][t] + sum_o[3][t]);
    put(P.out + row_at * kC + 4 * t, o, rounded == 0.f ? 0.f : 1.f / rounded);
    if (P.lse && threadIdx.x == 0) P.lse[row_at] = lse_of(top, sum);
}

// The unit of number u, if there is one.
template <int R, int S>
__device__ __forceinline__ bool find_work(const AttendParams& P, int64_t u, Work& w) {
    const int seq = find_seq(P.start, P.c.n_seqs, P.n_tokens, u, P.n_heads, R, P.pad);
    if (seq < 0) return false;
    open_seq(P, seq, w);
    const int64_t r = (u - first_unit(w.tok0, seq, P.n_heads, R, P.pad)) * R;
    if (r >= w.rows) return false;
    w.row0 = (int)r;
    see<R, S>(P, w);
    return true;
}

__global__ __launch_bounds__(kJoinThreads) void join_few_kernel(AttendParams P) {
    const int64_t u = blockIdx.x / kFew;
    Work w;
    if (!find_work<kFew, kStep>(P, u, w)) return;
    const int row = blockIdx.x % kFew;
    if (w.row0 + row >= w.rows) return;
    const int4 m = P.meta[u];
    if (m.z <= 1) return;
    join<kFew>(P, out_row(P, w, w.row0 + row), row, m.x, 2 * (int64_t)m.y, 2, m.z);
}

// ---------------------------------------------------------------- many rows

// Prompts, and whatever else has 64 rows or more for a sequence: 64 rows a unit, 32
// positions a step. The products bound it, so K is read from LDS by four waves that
// have 16 rows each, and each widened V operand serves all 64 rows: a wave takes
// the scores of its 16 rows, and adds its 128 columns of O for all 64 (128
// registers). One barrier a step: behind it are the weights of this step and the
// copies of the next, so the second product of a step and the first of the next
// fill the matrix pipes together; two workgroups share a CU.
struct ManyLds {
    __attribute__((aligned(16))) uint8_t tile[3][2 * kBlockStep];
    uint32_t scale[3][kWaves][64];
    u32x4 p[2][kWaves][64];     // [step parity][16 rows][lane]
    float shrink[2][kWaves][16];
    int flag[2][kWaves];
};
static_assert(sizeof(ManyLds) <= 80 * 1024, "two workgroups share a CU");
constexpr int kMany = 64;       // rows

__global__ __launch_bounds__(kThreads, 2) void many_kernel(AttendParams P) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    ManyLds& L = *reinterpret_cast<ManyLds*>(lds);
    const int t = threadIdx.x, lane = t & 63, wave = wave_bcast(t >> 6);
    const int g = lane >> 4, n = lane & 15;
    const int unit = P.units - 1 - blockIdx.x / P.shares, split = blockIdx.x % P.shares;
    Work w;
    if (!find_work<kMany, kStep>(P, unit, w)) return;
    const int each = (w.n + P.shares - 1) / P.shares;
    const int off = split * each;
    const int cnt = off + each < w.n ? each : w.n - off;
    if (split > 0 && cnt <= 0) return;
    const bool whole = each >= w.n;             // no other workgroup has these rows
    const Row r = row_of(P, w, w.row0 + wave * 16 + n);
    if (w.len < 0 && t == 0 && split == 0) raise(P.h, FLEET_MOE_ABORT_POSITION);

    bf16x8 q[kChunks / 2];
    load_q(P, w, r, g, 0, q);
    constexpr int kCols = kC / 16 / kWaves;     // of 16
    f32x4 acc[kWaves][kCols];
#pragma unroll
    for (auto& a : acc)
#pragma unroll
        for (auto& b : a) b = f32x4{0.f, 0.f, 0.f, 0.f};
    f32x4 ones{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    Pages pages{0, 0, 0};
    int good = 0;
    const auto issue = [&](int k) {
        const int page = page_of<kStep>(P, w, pages, off + k, off + cnt, lane);
        const int64_t base = page_offset(page, P.c.n_pages, P.layer, P.c.n_layers);
        const uint8_t* src = P.c.pool + (base < 0 ? 0 : base);
        const int half = step_of<kStep>(w, off + k) & 1;
        // eighteen pieces of 1 KB: two waves take five, two take four
        const uint32_t to = lds_addr(L.tile[k % 3]);
#pragma unroll
        for (int i = 0; i < 5; ++i) {
            const int piece = wave + kWaves * i;
            if (piece < 18)
                copy_kb<false>(src + half * 2 * kBlockBytes + piece * 1024 + lane * 16,
                           to + piece * 1024 + (piece >= 9 ? kBlockStep - kBlockBytes : 0));
        }
        copy_words(src + kCodeBytes + half * 16 + (lane & 3) * 4, lds_addr(L.scale[k % 3][wave]));
        const int bit = 1 << (k % 3);
        good = base >= 0 ? good | bit : good & ~bit;
        if (base < 0 && t == 0) raise(P.h, FLEET_MOE_ABORT_BAD_PAGE);
    };
    // the scores and weights of step k
    const auto score = [&](int k) {
        const uint8_t* buf = L.tile[k % 3];
        const float sc0 = any_scale(L.scale[k % 3][wave][0]), sp0 = any_scale(L.scale[k % 3][wave][1]);
        const float sc1 = any_scale(L.scale[k % 3][wave][2]), sp1 = any_scale(L.scale[k % 3][wave][3]);
        f32x4 z0{0.f, 0.f, 0.f, 0.f}, z1{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kChunks / 4; ++i) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(buf + i * 1024 + lane * 16);
            const u32x4 b = *reinterpret_cast<const u32x4*>(buf + kBlockStep + i * 1024 + lane * 16);
            const float sa = i < kC / 64 ? sc0 : sp0, sb = i < kC / 64 ? sc1 : sp1;
            z0 = mfma(widen(a.x, a.y, sa, sa), q[2 * i], z0);
            z1 = mfma(widen(b.x, b.y, sb, sb), q[2 * i], z1);
            z0 = mfma(widen(a.z, a.w, sa, sa), q[2 * i + 1], z0);
            z1 = mfma(widen(b.z, b.w, sb, sb), q[2 * i + 1], z1);
        }
        float s0[4], s1[4], top = m;
        bool nan = false;
        const bool ok = good >> (k % 3) & 1;
        const int base = step_of<kStep>(w, off + k) * kStep + 4 * g;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float a = z0[j] * P.scale, b = z1[j] * P.scale;
            const int pa = base + j, pb = base + kBlock + j;
            nan |= a != a || b != b;
            s0[j] = ok && pa <= r.pos && (pa >= r.seen.lo || pa < r.seen.sink) ? a : -INFINITY;
            s1[j] = ok && pb <= r.pos && (pb >= r.seen.lo || pb < r.seen.sink) ? b : -INFINITY;
            top = fmaxf(top, fmaxf(s0[j], s1[j]));
        }
        top = xor32_max(xor16_max(top));
        int flag = __ballot(nan) ? kHasNan : 0;
        if (__ballot(top > m + kSlack)) {
            flag |= kNeedMax;
            const float shrink = top == -INFINITY ? 1.f : exp2_(m - top);
            m = top;
            l *= shrink;
            ones *= shrink;
            if (lane < 16) L.shrink[k & 1][wave][lane] = shrink;
        }
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s0[j] = exp2_(s0[j] - ref);
            s1[j] = exp2_(s1[j] - ref);
        }
        l += ((s0[0] + s0[1]) + (s0[2] + s0[3])) + ((s1[0] + s1[1]) + (s1[2] + s1[3]));
        const uint2 a = weights(s0), b = weights(s1);
        const u32x4 p{a.x, a.y, b.x, b.y};
        L.p[k & 1][wave][lane] = p;
        if (lane == 0) L.flag[k & 1][wave] = flag;
        ones = mfma(__builtin_bit_cast(bf16x8, u32x4{kOnes, kOnes, kOnes, kOnes}),
                    __builtin_bit_cast(bf16x8, p), ones);
    };
    if (cnt > 0) issue(0);
    if (cnt > 1) issue(1);
    wait_copies<0>();
    barrier();
    if (cnt > 0) score(0);
    for (int k = 0; k < cnt; ++k) {
        wait_copies<0>();
        barrier();              // this step's weights, and the next one's tile
        if (k + 2 < cnt) issue(k + 2);          // where the tile before was
        const int any = wave_bcast((L.flag[k & 1][0] | L.flag[k & 1][1]) |
                                   (L.flag[k & 1][2] | L.flag[k & 1][3]));
        if (any) {
            if (any & kNeedMax) {
#pragma unroll
                for (int i = 0; i < kWaves; ++i) {
                    if (!(wave_bcast(L.flag[k & 1][i]) & kNeedMax)) continue;
                    const float f = L.shrink[k & 1][i][n];
#pragma unroll
                    for (auto& a : acc[i]) a *= f;
                }
            }
            if (any & kHasNan) {
                if (wave < 2) clean(L.tile[k % 3] + wave * kBlockStep, lane);
                barrier();
            }
        }
        const float sa = any_scale(L.scale[k % 3][wave][0]), sb = any_scale(L.scale[k % 3][wave][2]);
        bf16x8 p[kWaves];
#pragma unroll
        for (int i = 0; i < kWaves; ++i) p[i] = __builtin_bit_cast(bf16x8, L.p[k & 1][i][lane]);
        const uint8_t* col = column_at(L.tile[k % 3], lane) + wave * kCols * 256;
#pragma unroll
        for (int i = 0; i < kCols; ++i) {
            const i32x2 v = column(col, i);
            const bf16x8 a = widen((uint32_t)v.x, (uint32_t)v.y, sa, sb);
#pragma unroll
            for (int j = 0; j < kWaves; ++j) acc[j][i] = mfma(a, p[j], acc[j][i]);
        }
        if (k + 1 < cnt) score(k + 1);
    }
    // every wave needs the sums of all rows
    l = xor32_sum(xor16_sum(l));
    barrier();
    f32x4* stat = reinterpret_cast<f32x4*>(&L.p[0][0][0]);
    if (lane < 16) stat[wave * 16 + lane] = f32x4{m, l, ones[0], 0.f};
    barrier();
    const int64_t slot = (int64_t)unit * P.shares + split;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        const int row = i * 16 + n;
        const f32x4 st = stat[row];
        const int column0 = wave * (kC / kWaves) + 4 * g;
        if (whole) {
            if (w.row0 + row >= w.rows) continue;
            const int64_t at = out_row(P, w, w.row0 + row);
            const float inv = st[2] == 0.f ? 0.f : 1.f / st[2];
#pragma unroll
            for (int j = 0; j < kCols; ++j) put(P.out + at * kC + column0 + j * 16, acc[i][j], inv);
            if (P.lse && wave == 0 && g == 0) P.lse[at] = lse_of(st[0], st[1]);
        } else {
            float* part = P.part + (slot * kMany + row) * kC + column0;
#pragma unroll
            for (int j = 0; j < kCols; ++j)
                st_global(reinterpret_cast<f32x4*>(part + j * 16), acc[i][j]);
            if (wave == 0 && g == 0) st_global(P.stat + slot * kMany + row, st);
        }
    }
}

__global__ __launch_bounds__(kJoinThreads) void join_many_kernel(AttendParams P) {
    const int64_t u = blockIdx.x / kMany;
    Work w;
    if (!find_work<kMany, kStep>(P, u, w)) return;
    const int row = blockIdx.x % kMany;
    if (w.row0 + row >= w.rows) return;
    const int each = (w.n + P.shares - 1) / P.shares;
    if (each >= w.n) return;
    join<kMany>(P, out_row(P, w, w.row0 + row), row, u * P.shares,
                u * P.shares + 1, 1, (w.n + each - 1) / each);
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
template <class K>
static int launch(K kernel, int64_t grid, int threads, size_t lds, const AttendParams& P,
                  hipStream_t stream) {
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)lds);
        if (e != hipSuccess) return (int)e;
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), lds, stream, P);
    return (int)hipGetLastError();
}

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
    char* ws = static_cast<char*>(workspace) + parts_at(cache->n_seqs, cache->n_pages);
    P.h = static_cast<Header*>(workspace);
    P.part = reinterpret_cast<float*>(ws);
    P.stat = reinterpret_cast<f32x4*>(ws + kPartBytes);
    P.meta = reinterpret_cast<int4*>(ws + kPartBytes + kStatBytes);
    P.q_stride = q_stride;
    P.layer = layer;
    P.n_tokens = n_tokens;
    P.n_heads = n_heads;
    P.per_head = ((uint64_t)1 << 40) / n_heads + 1;
    P.window = window;
    P.sinks = sinks;
    P.scale = scale * 1.4426950408889634f;
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
        if (int e = launch(few_kernel, P.shares, kThreads, sizeof(FewLds), P, stream)) return e;
        return launch(join_few_kernel, few * kFew, kJoinThreads, 0, P, stream);
    }
    P.pad = n_heads % kMany != 0;
    const int64_t units = first_unit(n_tokens, cache->n_seqs, n_heads, kMany, P.pad);
    P.units = (int)units;
    int64_t splits = kShares / 2 / units;
    const int64_t most = (seen + 4 * kStep - 1) / (4 * kStep);
    if (splits > most) splits = most;
    P.shares = splits < 1 ? 1 : (int)splits;
    if (int e = launch(many_kernel, units * P.shares, kThreads, sizeof(ManyLds), P, stream)) return e;
    return P.shares > 1 ? launch(join_many_kernel, units * kMany, kJoinThreads, 0, P, stream) : 0;
}
