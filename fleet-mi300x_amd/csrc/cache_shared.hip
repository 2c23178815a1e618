// Attention of sequences that share their first pages: fleet_cache_share and
// fleet_cache_attend_shared (declarations in fleet_moe.h).
//
// Sequences of a group (a request's beams, requests behind one prompt) name the same pages
// first. The softmax of a row over its positions splits into parts of positions, each with a
// reference m, a sum l and a sum O of weighted rows, which are added as
//   O = sum_i 2^(m_i - m) O_i,  l = sum_i 2^(m_i - m) l_i,
// so the common pages are one part, in which the rows of all the group's sequences stand
// together: each page is read, widened and multiplied once for 64 rows, where
// fleet_cache_attend does it for every sequence's 16. What is a sequence's own is another part.
//
// A unit is up to 64 (token, head) rows and a range of pages: a group's rows over its
// common pages, or a sequence's rows over the pages behind them. The steps (a page each) of all
// units follow each other, and a workgroup a CU takes an equal share of them, across units
// where it has to, so that neither the groups' sizes nor the lengths leave a CU idle. The
// parts go to the caller's plan, and a second launch adds those of a row, in order.
//
// Measured, a layer, 16 heads, both launches in a graph: 4 sequences of 1,000 + 40 positions 13.5 us
// (latency: the unit, its queries and first page, the join); 64 behind 8,192, 500 own, 48.3
// (19 GFLOP, 15 us at a library's rate: eight pages a workgroup after a beginning of 8 us); 8
// groups of 16 behind 4,000, 300 own, 4 tokens each, 118 (76 GFLOP, 58 us); 2 of 128 behind
// 16,300, 1,000 own, 208 (153 GFLOP, 117 us). The large ones are bound by the instructions of a
// page, half as many matrix instructions again as the formula has, as weights are two operands: the
// matrix unit has 49% of the time, other vector instructions 33%.
#include <stddef.h>

#include "attend_tile.h"

namespace fleet_moe {
namespace cache {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;               // rows of a unit
constexpr int kGrid = kShares / 2;      // workgroups
constexpr int kGridWaves = 8;
constexpr int kGridThreads = kGridWaves * 64;
constexpr int kPageRing = 3;
constexpr float kRise = 12.f;           // (8: 64 sequences 49.7 us where this takes 48.5)

// The plan: what share found, and the parts of an attention.
struct PlanHeader {
    uint32_t remaps;            // the cache's when share was called
    int32_t pad;
    int32_t first, end;         // the attention's rows: none if its starts are not in order
    int32_t pads[60];
};
static_assert(sizeof(PlanHeader) == 256, "");
struct Group {
    int32_t first, end;         // sequences, from the first that holds anything
    int32_t pages;              // common to those that do
    int32_t pad;
};
struct Parts {                  // of a row and kind: part 0, part 1, part 1 + kPartStep, ..
    int32_t at, next, count;
    int32_t front;              // there are parts over common pages, too
};
constexpr int kPartStep = 2 * kTile;    // a workgroup has two slots
constexpr int64_t kMaxPlanRows = 1 << 20;

// Partial results lie in tiles of 16 rows as the matrix instructions leave them: [wave (64
// columns)][16 columns][lane (4 columns, row)], 32 KB, so that a wave's store is 1 KB of
// consecutive bytes (rows of 512 columns: 64 bytes of 16 rows each, 6,300 cycles a unit where
// this takes 3,100). Part `at` is row at % 16 of tile at / 16. Whole units have a tile for every 16
// rows of a sequence (or group, by its first sequence), split ones the slots behind those.
struct Plan {
    PlanHeader* h;
    Group* groups;              // [n_seqs]: a sequence's
    Parts* meta;                // [2][rows]: over the common pages, over its own
    f32x4* stat;                // [parts]
    f32x4* part;                // [parts / 16][8][4][64]
};
__host__ __device__ inline int64_t whole_parts(int n_seqs, int64_t rows) {
    return 16 * (rows / 16 + n_seqs + 1);
}
__host__ __device__ inline int64_t whole_part(int seq, int64_t first_row) {
    return 16 * (first_row / 16 + seq);
}
inline int64_t plan_parts(int n_seqs, int64_t rows) {
    return 2 * whole_parts(n_seqs, rows) + (int64_t)kGrid * kPartStep;
}
inline size_t plan_size(int n_seqs, int64_t rows) {
    return sizeof(PlanHeader) + up256((size_t)n_seqs * sizeof(Group)) +
           up256((size_t)rows * 2 * sizeof(Parts)) +
           (size_t)plan_parts(n_seqs, rows) * (16 + 4 * kC);
}
inline Plan plan_at(void* p, int n_seqs, int64_t rows) {
    char* c = static_cast<char*>(p);
    Plan r;
    r.h = reinterpret_cast<PlanHeader*>(c);
    c += sizeof(PlanHeader);
    r.groups = reinterpret_cast<Group*>(c);
    c += up256((size_t)n_seqs * sizeof(Group));
    r.meta = reinterpret_cast<Parts*>(c);
    c += up256((size_t)rows * 2 * sizeof(Parts));
    r.stat = reinterpret_cast<f32x4*>(c);
    r.part = reinterpret_cast<f32x4*>(c + (size_t)plan_parts(n_seqs, rows) * 16);
    return r;
}
// Where lane `lane`'s four of columns 64 wave + 16 j .. lie.
__device__ __forceinline__ f32x4* part_at(const Plan& p, int64_t tile, int wave, int j, int lane) {
    return p.part + ((tile * kGridWaves + wave) * 4 + j) * 64 + lane;
}

// ---------------------------------------------------------------- share

// A workgroup a group: the leading pages that all its sequences with positions name, as far as
// all of them have filled them. (An append writes no such page, so the number stays right
// until sequences move.) One without positions is by itself, whatever pages it gets later; where
// its tokens are between the group's, their rows are computed and not used.
constexpr int kShareThreads = 1024;
__global__ __launch_bounds__(kShareThreads) void share_kernel(fleet_cache c, const int32_t* groups,
                                                              int n_groups, int32_t* pages_out,
                                                              Plan plan, Header* h) {
    __shared__ int pages, lead;
    const int t = threadIdx.x;
    // offsets that do not increase from 0 to the sequences at most: no groups at all
    bool bad = false;
    for (int i = t; i <= n_groups; i += kShareThreads) {
        const int at = groups[i];
        bad |= at < 0 || at > c.n_seqs || (i > 0 && at < groups[i - 1]);
    }
    const bool none = __syncthreads_or(bad);
    const int first = none ? 0 : groups[blockIdx.x], end = none ? 0 : groups[blockIdx.x + 1];
    if (blockIdx.x == 0) {
        if (t == 0) plan.h->remaps = h->remaps;
        if (t == 0 && none) raise(h, FLEET_MOE_ABORT_POSITION);
        const int lo = none ? 0 : groups[0], hi = none ? 0 : groups[n_groups];
        for (int s = t; s < c.n_seqs; s += kShareThreads)
            if (s < lo || s >= hi) plan.groups[s] = Group{s, s + 1, 0, 0};
    }
    if (t == 0) {
        pages = 0x7fffffff;
        lead = 0x7fffffff;
    }
    __syncthreads();
    int held = 0;
    for (int s = first + t; s < end; s += kShareThreads) {
        const int len = checked_len(c.lens[s], c.max_pages);
        if (len > 0) {
            ++held;
            atomicMin(&pages, len / kPage);
            atomicMin(&lead, s);
        }
    }
    held = __syncthreads_count(held > 0);     // 0, 1, or more (not how many more)
    int most = pages;
    const int from = lead;
    if (held == 0 || end - first < 2) most = 0;
    __syncthreads();
    // 256 columns at a time, a row a wave, until one differs; 16 loads of a lane on their way
    const int lane = t & 63, wave = t >> 6;
    const int32_t* row = c.table + (int64_t)from * c.max_pages;
    constexpr int kCols = 4, kRows = 4, kWaves = kShareThreads / 64;
    for (int j0 = 0; j0 < most; j0 += 64 * kCols) {
        int mine[kCols];
        int differs = 0x7fffffff;
#pragma unroll
        for (int k = 0; k < kCols; ++k) {
            const int j = j0 + 64 * k + lane;
            mine[k] = j < most ? row[j] : 0;
            if (j < most && (unsigned)mine[k] >= (unsigned)c.n_pages) differs = j < differs ? j : differs;
        }
        for (int s0 = first + wave; s0 < end; s0 += kRows * kWaves) {
            int there[kRows][kCols], lens[kRows];
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const int s = s0 + r * kWaves;
                lens[r] = s < end ? c.lens[s] : 0;
#pragma unroll
                for (int k = 0; k < kCols; ++k) {
                    const int j = j0 + 64 * k + lane;
                    there[r][k] = s < end && j < most ? c.table[(int64_t)s * c.max_pages + j] : mine[k];
                }
            }
#pragma unroll
            for (int r = 0; r < kRows; ++r)
                if (checked_len(lens[r], c.max_pages) > 0)
#pragma unroll
                    for (int k = 0; k < kCols; ++k) {
                        const int j = j0 + 64 * k + lane;
                        if (there[r][k] != mine[k] && j < differs) differs = j;
                    }
        }
        if (differs < most) atomicMin(&pages, differs);
        __syncthreads();
        const int now = pages;
        __syncthreads();
        if (now < most) {
            most = now;
            break;
        }
    }
    for (int s = first + t; s < end; s += kShareThreads)
        plan.groups[s] = checked_len(c.lens[s], c.max_pages) > 0 ? Group{from, end, most, 0}
                                                                 : Group{s, s + 1, 0, 0};
    if (pages_out && t == 0) pages_out[blockIdx.x] = most;
}

// ---------------------------------------------------------------- the work

struct SharedParams {
    fleet_cache c;
    const uint16_t* q;
    const int32_t* start;
    uint16_t* out;
    float* lse;
    Plan plan;
    Header* h;
    int64_t q_stride;
    uint64_t per_head;          // head_divisor(n_heads)
    int layer, n_tokens, n_heads;
    float scale;                // times log2(e)
    float slack;                // kRise as a score: finite
};

__device__ __forceinline__ int start_of(const SharedParams& P, int s) {
    return P.start ? clamp_row(ld_global(P.start + s), P.n_tokens) : s;
}

// What a sequence adds to the steps: its group's rows over their common pages, if it is the
// group's first, and its own rows over what is behind them.
struct Item {
    int seq, tok0, n_new, len;
    int pages;                          // its group's, and
    int first, end, last;               // the sequences, and the token behind them
    int steps0, steps1;                 // of a unit, whether they see anything or not
};
// What is loaded for a sequence, all on its way together.
struct RawItem {
    i32x4 group;
    int at, behind, len;
};
__device__ __forceinline__ RawItem raw_of(const SharedParams& P, int seq) {
    RawItem r;
    const int32_t* starts = P.start ? P.start : P.c.lens;     // (any, where tokens are sequences)
    r.group = ld_global(reinterpret_cast<const i32x4*>(P.plan.groups + seq));
    r.at = ld_global(starts + seq);
    r.behind = ld_global(starts + seq + (P.start ? 1 : 0));
    r.len = ld_global(P.c.lens + seq);
    return r;
}
// All but `last`, which needs the group's end.
__device__ __forceinline__ Item item_of(const SharedParams& P, int seq, const RawItem& r, bool stale) {
    Item w;
    w.seq = seq;
    w.tok0 = P.start ? clamp_row(r.at, P.n_tokens) : seq;
    w.n_new = (P.start ? clamp_row(r.behind, P.n_tokens) : seq + 1) - w.tok0;  // (< 0: out of order)
    w.len = checked_len(r.len, P.c.max_pages);
    w.first = stale ? seq : r.group.x;
    w.end = stale ? seq + 1 : r.group.y;
    w.pages = stale ? 0 : r.group.z;
    w.last = w.tok0;
    w.steps0 = w.pages;
    const int own = w.len < 0 ? 0 : pages_of(w.len) - w.pages;
    w.steps1 = own > 1 ? own : 1;
    return w;
}
__device__ __forceinline__ bool leads(const Item& w) { return w.pages > 0 && w.seq == w.first; }
__device__ __forceinline__ Item lane_of(const Item& v, int lane) {
    static_assert(sizeof(Item) == 40, "");
    struct Words {
        int w[sizeof(Item) / 4];
    } x = __builtin_bit_cast(Words, v);
#pragma unroll
    for (int& i : x.w) i = __builtin_amdgcn_readlane(i, lane);
    return __builtin_bit_cast(Item, x);
}

// What the work is divided by: the time of a unit's beginning and end, and of a page, for units
// of up to 16 rows and of more, in 500 cycles (a page takes 3,250 and 5,500; with 24, 8 and 40, 11
// twelve calls of 13 to 290 us take 1.4% longer, their mean, with 20, 7 and 33, 11 1.5%).
// A workgroup does the pages whose time begins in its share.
struct Cost {
    int setup, page;
    // How many pages begin before `time`.
    __device__ __forceinline__ int begun(int time) const;
};
constexpr Cost kCost16{18, 6}, kCost64{36, 11};
__device__ __forceinline__ int Cost::begun(int time) const {
    const int t = time > setup ? time - setup : 0;        // (divided by constants)
    return page == kCost16.page ? (t + kCost16.page - 1) / kCost16.page
                                : (t + kCost64.page - 1) / kCost64.page;
}
// Units have 64 rows, or 16 where there are few pages: up to eight a workgroup of 16 rows take
// less time than the two of 64 rows, with a unit's beginning and the parts to be joined (16
// sequences of 4,100 positions 20.9 us, in 64 rows 30.0; up to eleven, 32 in eight groups would
// take 28.2 for 30.5).
constexpr int kFewSteps = 8 * kGrid;
struct Sizes {
    int rows0, units0, rows1, units1;
    int tile;
    __device__ __forceinline__ Sizes(const SharedParams& P, const Item& w, int rows) {
        tile = rows;
        rows0 = (w.last - w.tok0) * P.n_heads;
        rows1 = w.n_new > 0 ? w.n_new * P.n_heads : 0;
        const int shift = tile == kTile ? 6 : 4;
        units0 = (rows0 + tile - 1) >> shift;
        units1 = (rows1 + tile - 1) >> shift;
    }
    __device__ __forceinline__ Cost full() const { return tile == kTile ? kCost64 : kCost16; }
    // The time of unit k of either kind.
    __device__ __forceinline__ Cost cost(int rows, int k) const {
        return rows - k * tile <= 16 ? kCost16 : full();
    }
    __device__ __forceinline__ int time(int rows, int units, int pages) const {
        if (units == 0) return 0;
        const Cost z = cost(rows, units - 1);
        return (units - 1) * (full().setup + full().page * pages) + z.setup + z.page * pages;
    }
    __device__ __forceinline__ int front(const Item& w) const { return time(rows0, units0, w.steps0); }
    __device__ __forceinline__ int total(const Item& w) const {
        return front(w) + time(rows1, units1, w.steps1);
    }
    __device__ __forceinline__ int units() const { return units0 + units1; }
    __device__ __forceinline__ int steps(const Item& w) const {
        return units0 * w.steps0 + units1 * w.steps1;
    }
};
static_assert(kTile == 64, "");

// A range of n things in `shares` parts that differ by one at most.
struct Split {
    int each, more;             // the first `more` have each + 1
    __device__ Split(int n, int shares) : each(n / shares), more(n - each * shares) {}
    __device__ int first(int i) const { return i * each + (i < more ? i : more); }
    __device__ int holder(int at) const {
        const int big = more * (each + 1);
        return at < big ? at / (each + 1) : more + (at - big) / each;
    }
};

constexpr int kLeast = 11;
static_assert(kLeast >= kCost64.page && kLeast >= kCost16.page, "");
// How many workgroups take part. No share is shorter than a page's time (so that every one
// between a unit's first and last has a part of it), and few pages are left to many only as
// far as the parts are joined in less time than that saves (15: 4 sequences of 1,000 14.4 us, with
// 11 13.5).
__device__ __forceinline__ int shares_of(int total) {
    const int n = total / kLeast;
    return n < 1 ? total > 0 : n < kGrid ? n : kGrid;
}

// Up to 64 rows and the pages of a table row that they see.
struct Unit {
    int row0, rows;             // rows row0 .. of the sequence's or group's `rows`
    int tok0;                   // the token of row 0
    int base;                   // own pages: the position of that token
    int first, end;             // common pages: the group
    bool common, inside;
    const int32_t* table;       // from the first page on
    int page0;
    int n;                      // pages that some row may see
};

// The position of token `tok` (a lane's) of the sequences [first, end).
__device__ __forceinline__ int position_of(const SharedParams& P, int first, int end, int tok) {
    int s = tok;
    if (P.start) {
        const int lane = threadIdx.x & 63;
        s = first;              // and how many sequences end at tok or before
        for (int s0 = first; s0 < end; s0 += 64) {
            const int z = s0 + lane < end ? start_of(P, s0 + lane + 1) : 0x7fffffff;
            int n = 0;
#pragma unroll
            for (int j = 0; j < 64; ++j) n += __builtin_amdgcn_readlane(z, j) <= tok;
            s += n;
            if (!__ballot(n == 64)) break;
        }
    }
    if (s >= end) return -1;
    const int len = checked_len(ld_global(P.c.lens + s), P.c.max_pages);
    return len < 0 ? -1 : len - (start_of(P, s + 1) - tok);
}

// A lane's row.
struct TileRow {
    bool live;
    int tok, head, pos;         // dead rows: the unit's first
};
__device__ __forceinline__ TileRow tile_row(const SharedParams& P, const Unit& u, int row) {
    TileRow r;
    r.live = row < u.rows;
    if (!r.live) row = u.row0;
    const int t = token_of_row(row, P.per_head);
    r.tok = u.tok0 + t;
    r.head = row - t * P.n_heads;
    r.pos = -1;
    return r;
}

// The position that all rows of a wave see, apart from the dead ones.
__device__ __forceinline__ int common_position(const TileRow& r) {
    int v = r.live ? r.pos : 0x7fffffff;
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
        const int o = __shfl_xor(v, d);
        v = o < v ? o : v;
    }
    return wave_bcast(v);
}

struct PageLds {
    __attribute__((aligned(16))) uint8_t tile[kPageRing][4 * kBlockStep];
    u32x4 p[2][4][2][64];       // [step parity][tile][half of the page][lane], and what the
    u32x4 left[2][4][2][64];    // weights' rounding leaves (p, this and `half` hold the rest of
                                // the queries first)
    f32x4 half[kGridWaves][2][64];      // half of the scores of a tile and two blocks
    uint32_t scale[kPageRing][8];
    int flag[2][kGridWaves], units[2][kGridWaves], front[2];
    __attribute__((aligned(8))) uint8_t flags[2][kGridWaves];   // (64 rows) 1: a row's reference
                                // rises, 2: a score is not finite
    float m[4][16], top[4][2][16], sum[4][2][16], rounded[4][2][16];
    Item item;                  // what follows a unit, out of the registers meanwhile
    int at, off;
    __attribute__((aligned(8))) uint64_t work[2][kGridWaves];   // threads of locate() whose first
                                                                // and second sequence has units
};
static_assert(sizeof(PageLds) <= 160 * 1024, "");
static_assert(kPageRing == 3 && offsetof(PageLds, p) == sizeof(PageLds::tile) &&
                  offsetof(PageLds, left) == offsetof(PageLds, p) + sizeof(PageLds::p) &&
                  offsetof(PageLds, half) == offsetof(PageLds, left) + sizeof(PageLds::left) &&
                  kTile * (2 * kRow + 16) <= 4 * kBlockStep + sizeof(PageLds::p) +
                                                 sizeof(PageLds::left) + sizeof(PageLds::half),
              "");

// The sequence in whose steps workgroup wg begins, and where, into L: a thread a sequence, or
// two.
struct Place {
    int total, shares;
    int tile;                   // rows of a unit
    int wg;                     // the share of the workgroup
    bool stale;                 // sequences have moved since share: every one by itself
    bool inside;                // some token stands within its group's common pages
};
__device__ __forceinline__ bool locate(const SharedParams& P, PageLds& L, int wg, Place& at) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int each = P.c.n_seqs > kGridThreads ? 2 : 1;
    static_assert(kMaxSeqs <= 2 * kGridThreads, "");
    int n = 0, first = 0, units = 0, steps = 0, first16 = 0, some = 0;
    bool bad = false, inside = false;
    Item w{}, w1{};
    int* starts = reinterpret_cast<int*>(L.tile);         // [n_seqs + 1]
    const int seq = t * each, top = P.c.n_seqs - 1;
    RawItem r = raw_of(P, seq < top ? seq : top), r1{};
    if (each > 1) r1 = raw_of(P, seq + 1 < top ? seq + 1 : top);
    asm volatile("" ::: "memory");              // (the loads above first)
    at.stale = ld_global(&P.plan.h->remaps) != ld_global(&P.h->remaps);
    if (seq <= top) {
        w = item_of(P, seq, r, at.stale);
        starts[seq + 1] = w.tok0 + w.n_new;
        if (each > 1 && seq < top) {
            w1 = item_of(P, seq + 1, r1, at.stale);
            starts[seq + 2] = w1.tok0 + w1.n_new;
        }
    }
    barrier();
    if (seq <= top) {
        if (leads(w)) w.last = starts[w.end];
        if (leads(w1)) w1.last = starts[w1.end];
        first = Sizes(P, w, kTile).total(w);
        n = first + Sizes(P, w1, kTile).total(w1);
        const Sizes a(P, w, 16), b(P, w1, 16);
        // (used where the call has few steps; else it may wrap)
        first16 = (int)((uint32_t)a.units() * kCost16.setup + (uint32_t)a.steps(w) * kCost16.page);
        units = a.units() + b.units();
        some = (a.units() > 0 ? 1 : 0) | (b.units() > 0 ? 2 : 0);
        steps = a.steps(w) + b.steps(w1);
        bad = (w.n_new | w1.n_new) < 0;
        inside = (w.n_new > 0 && w.len - w.n_new < w.pages * kPage) ||
                 (w1.n_new > 0 && w1.len - w1.n_new < w1.pages * kPage);
    }
    const uint64_t works = __ballot(some & 1), works1 = __ballot(some & 2);
    int incl = wave_incl_scan(n);
    const int units_incl = wave_incl_scan(units), steps_incl = wave_incl_scan(steps);
    const int flags = (__ballot(bad) ? 1 : 0) | (__ballot(inside) ? 2 : 0);
    if (lane == 63) {
        L.flag[0][wave] = incl;
        L.flag[1][wave] = flags;
        L.units[0][wave] = units_incl;
        L.units[1][wave] = steps_incl;
        L.work[0][wave] = works;
        L.work[1][wave] = works1;
    }
    if (t == 0) {
        L.front[0] = first;
        L.front[1] = first16;
    }
    barrier();
    int before = 0, any = 0, all_units = 0, all_steps = 0, units_before = 0, steps_before = 0;
    at.total = 0;
#pragma unroll
    for (int i = 0; i < kGridWaves; ++i) {
        if (i < wave) {
            before += L.flag[0][i];
            units_before += L.units[0][i];
            steps_before += L.units[1][i];
        }
        at.total += L.flag[0][i];
        all_units += L.units[0][i];
        all_steps += L.units[1][i];
        any |= L.flag[1][i];
    }
    int most = wave_bcast(L.front[0]);          // (the first group's, which is the one as a rule)
    at.tile = kTile;
    if (wave_bcast(all_steps) <= kFewSteps) {
        // (a unit has a page at least: the times are small)
        const auto time = [](int u, int s) { return u * kCost16.setup + s * kCost16.page; };
        at.tile = 16;
        most = wave_bcast(L.front[1]);
        at.total = time(all_units, all_steps);
        before = time(units_before, steps_before);
        incl = time(units_incl, steps_incl);
        n = time(units, steps);
        first = first16;
    }
    at.total = wave_bcast(at.total);
    any = wave_bcast(any);
    at.inside = any & 2;
    if (wg == 0 && t == 0) {
        P.plan.h->first = any & 1 ? 0 : w.tok0 * P.n_heads;
        P.plan.h->end = any & 1 ? 0 : starts[P.c.n_seqs] * P.n_heads;
        if (any & 1) raise(P.h, FLEET_MOE_ABORT_POSITION);
    }
    if (any & 1) return false;
    at.shares = shares_of(at.total);
    if (wg >= at.shares) return false;
    // Workgroups that are one die's take shares that follow each other, so that they meet a
    // group's pages in one L2 (eight groups of 16 sequences with 4 tokens fetch 77 MB where they
    // took 239, 119 us and 121); not where a group has most of the work: the eight dies come to its
    // pages in turn then, unit after unit (16 sequences of 4,100 21.1 us, and 21.7).
    const bool spread = at.shares < kGrid || 2 * (int64_t)most > at.total;
    at.wg = spread ? wg : (wg & 7) * (kGrid / 8) + (wg >> 3);
    const int off = Split(at.total, at.shares).first(at.wg) - (before + incl - n);
    if (off >= 0 && off < first) {
        L.item = w;
        L.off = off;
    } else if (off >= first && off < n) {
        L.item = w1;
        L.off = off - first;
    }
    barrier();
    return true;
}

// The sequence after `seq` that has units, the same in all lanes; n_seqs if there is none.
// (Sequence by sequence, by what is in memory of them, the first and last of 1,024 took 349 us
// where this takes 14.8.)
__device__ __forceinline__ int next_with_work(const PageLds& L, int seq, int n_seqs, int lane) {
    const int each = n_seqs > kGridThreads ? 2 : 1;
    int next = n_seqs;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        // thread t of locate() has sequence t * each + j: from which t on
        const int from = seq < j ? 0 : (seq - j) / each + 1;
        uint64_t mine = lane < kGridWaves ? L.work[j][lane] : 0;
        if (64 * lane + 63 < from) mine = 0;
        else if (64 * lane < from) mine &= ~0ull << (from - 64 * lane);
        const uint64_t waves = __ballot(mine != 0);
        if (waves) {
            const int w = __builtin_ctzll(waves);
            const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)mine, w);
            const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(mine >> 32), w);
            const int s = (64 * w + __builtin_ctzll((uint64_t)hi << 32 | lo)) * each + j;
            next = s < next ? s : next;
        }
    }
    return next;
}

// Pages of 64 steps, one per lane, and which of them are not of the pool.
struct PageList {
    int held, from, page;
    uint64_t bad;
};
__device__ __forceinline__ void turn_to(const SharedParams& P, const Unit& u, PageList& h, int i,
                                        int end, int lane) {
    if (i < h.held) return;
    h.from = i - 4;             // (the steps whose scores are not finished yet)
    h.held = h.from + 64;
    const int mine = h.from + lane;
    const bool there = mine >= 0 && mine < end;
    h.page = there ? ld_global(u.table + mine) : 0;
    // here, not at the use: there the compiler would wait, every step, for
    // whatever copies are in flight
    __builtin_amdgcn_s_waitcnt(0x0F70);         // vmcnt(0)
    h.bad = __ballot(there && (unsigned)h.page >= (unsigned)P.c.n_pages);
}
__device__ __forceinline__ int page_of(const PageList& h, int i) {
    return __builtin_amdgcn_readlane(h.page, i - h.from);
}
__device__ __forceinline__ bool valid(const PageList& h, int i) {
    return !(h.bad >> (i - h.from) & 1);
}

// The queries of a unit go through LDS, where its later pages come: a lane's own loads of them, 16
// bytes of 16 rows at a time, took 12,000 cycles for 64 rows (a page's step takes 5,500). Rows
// lie 16 bytes further apart than they are long, so that the operands of 16 rows fall into
// different banks.
constexpr int kQueryStep = 2 * kRow + 16;
__device__ __forceinline__ uint8_t* query_at(PageLds& L, int place, int row) {
    return L.tile[place] + row * kQueryStep;
}
// A wave's rows; of dead ones the unit's first. (A lane a row's address.)
template <int kRows>
__device__ __forceinline__ void copy_q(const SharedParams& P, PageLds& L, const Unit& u, int place,
                                       int wave, int lane) {
    const int mine = u.row0 + wave * kRows + lane % kRows, row = mine < u.rows ? mine : u.row0;
    const int tok = token_of_row(row, P.per_head);
    const uint64_t from = (uint64_t)(uintptr_t)(P.q + (int64_t)(u.tok0 + tok) * P.q_stride +
                                                (row - tok * P.n_heads) * kRow);
    const uint32_t to = lds_addr(query_at(L, place, wave * kRows));
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)from, i);
        const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(from >> 32), i);
        const uint8_t* src = reinterpret_cast<const uint8_t*>((uint64_t)hi << 32 | lo) + lane * 16;
        copy_kb<1, false>(src, to + i * kQueryStep);
        if (lane < (2 * kRow - 1024) / 16)
            copy_kb<1, false>(src + 1024, to + i * kQueryStep + 1024);
    }
}
// A lane's row as the right operand. The k order of the products is that of the bytes a lane of
// group g takes of a cache row: its chunks 4i + g, 16 values each, i = 0 .. 8, make two of 18
// steps. Wave `half` has those of i = half, 2 + half, 4 + half, 6 + half, and one of i = 8.
constexpr int kTileHalf = kChunks / 4;          // steps of a wave
__device__ __forceinline__ void read_q(PageLds& L, int place, int row, int g, int half,
                                       bf16x8 (&q)[kTileHalf]) {
    const uint8_t* src = query_at(L, place, row) + g * 32;
    const auto at = [&](int v) {
        return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(src + 2 * v));
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        q[2 * i] = at((2 * i + half) * 64);
        q[2 * i + 1] = at((2 * i + half) * 64 + 8);
    }
    q[8] = at(8 * 64 + half * 8);
}

__device__ __forceinline__ void set_position(const SharedParams& P, const Unit& u, TileRow& r) {
    int pos = 0x7fffffff;                       // common pages, in front of every token
    if (!u.common) pos = u.base + r.tok - u.tok0;
    else if (u.inside) pos = position_of(P, u.first, u.end, r.tok);
    r.pos = r.live ? pos : -1;
}

// The copies of a page to place b of the ring: a wave of four a block, the first the scales too.
__device__ __forceinline__ void issue_page(const SharedParams& P, PageLds& L, int page, int b,
                                           int wave, int lane) {
    const int64_t base = page_offset(page, P.c.n_pages, P.layer, P.c.n_layers);
    const uint8_t* src = P.c.pool + (base < 0 ? 0 : base);
    const uint8_t* from = src + wave * kBlockBytes + lane * 16;
    const uint32_t to = lds_addr(L.tile[b]) + wave * kBlockStep;
    copy_kb<4, false>(from, to);
    copy_kb<4, false>(from + 4096, to + 4096);
    copy_kb<1, false>(from + 8192, to + 8192);
    if (wave == 0 && lane < 2)
        copy_kb<1, false>(src + kCodeBytes + lane * 16, lds_addr(L.scale[b]));
}

// Pages off .. off + cnt - 1 of a unit; its results to `out` and `lse` if `to_part` is negative,
// else as the parts to_part + row.
//
// Eight waves: wave (tile pair, half, block pair) takes half of the 576 products of 32 rows
// with 32 positions, so that a widened K operand serves two tiles; it exchanges halves with
// its partner, makes the weights of one tile and 32 positions, and adds its 64 columns of O
// for all rows over the whole page, where a widened V operand serves four tiles.
//
// The weights are two operands, bf16 and what that leaves: 16 bits, as in attend16, so that what
// a sequence gets does not lose bits when other requests make the units higher. (With the first
// alone a page takes 4,450 cycles, 64 sequences 44 us for 48, 256 177 for 208, and sums of weights
// that nearly cancel are lost.)
//
// A page takes 5,500 cycles, of which the matrix unit has 3,264 (102 instructions of 16 cycles of
// each of a SIMD's two waves).
//
// Three pages are in work in a step: the scores of page k + 2, the weights of page k + 1 and the
// products of page k, none of which needs another, so that matrix and vector instructions and
// reads of LDS run beside each other. The codes of V are read a page ahead, so that three places
// of the ring suffice. The LDS has room for one page's halves of scores: those of page k + 2 come
// behind a second barrier.
__device__ __forceinline__ void attend64(const SharedParams& P, PageLds& L, const Unit& u, int off,
                                         int cnt, int64_t to_part) {
    constexpr int kCols = kC / 16 / kGridWaves; // of 16
    // (fm_tid: no lane's index is kept in a register from one unit to the next)
    const int t = fm_tid(), lane = t & 63, wave = wave_bcast(t >> 6);
    const int g = lane >> 4, n = lane & 15;
    const int bp = wave & 1, half = wave >> 1 & 1, tp = wave >> 2;
    const int mine = 2 * tp + half;             // the tile whose weights this wave makes

    // (b is k % kPageRing, counted)
    PageList pages{0, 0, 0, 0};
    const auto issue = [&](int k, int b) {
        turn_to(P, u, pages, off + k, off + cnt, lane);
        issue_page(P, L, page_of(pages, off + k), b, wave, lane);
    };
    // the copies of the first two pages, a wave of four a block, and the queries', behind them
    if (cnt > 0) {
        turn_to(P, u, pages, off, off + cnt, lane);
        if (tp < cnt) issue_page(P, L, page_of(pages, off + tp), tp, wave & 3, lane);
        copy_q<kTile / kGridWaves>(P, L, u, kPageRing - 1, wave, lane);
    }
    TileRow r = tile_row(P, u, u.row0 + mine * 16 + n);
    set_position(P, u, r);
    const int common = common_position(r);
    f32x4 acc[4][kCols];
#pragma unroll
    for (auto& a : acc)
#pragma unroll
        for (auto& b : a) b = f32x4{0.f, 0.f, 0.f, 0.f};
    // the sum of the rounded weights of tile wave & 3 and half of the page wave >> 2
    f32x4 ones{0.f, 0.f, 0.f, 0.f};
    // Every row's reference, as a score and as it is in the exponent: any score not far below
    // the maximum, because weights up to 2^kRise are as exact as those up to 1, and moving
    // it costs a pass over O and two barriers.
    float m = -INFINITY, ref = -INFINITY, l = 0.f, sum = 0.f;
    const float slack = P.slack;
    f32x4 z[2];                                 // the scores of `mine` and the two blocks
    f32x4 own[2];                               // the wave's half of the next ones
    if (t < 64) L.m[t >> 4][n] = -INFINITY;
    // q is there, also as far as the compiler counts, and the pages are
    wait_copies<0>();
    barrier();
    bf16x8 q[2][kTileHalf];                     // of `mine` and of the pair's other tile
    read_q(L, kPageRing - 1, mine * 16 + n, g, half, q[0]);
    read_q(L, kPageRing - 1, (mine ^ 1) * 16 + n, g, half, q[1]);

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
            own[j] = y[0][j];
            L.half[wave][j][lane] = y[1][j];
        }
    };
    const auto weigh = [&](int k) {
        const float down = ref == -INFINITY ? 0.f : ref;
        float p0[4], p1[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            p0[j] = exp2_(fmaf(z[0][j], P.scale, -down));
            p1[j] = exp2_(fmaf(z[1][j], P.scale, -down));
        }
        const uint2 a = weights(p0), b = weights(p1), c = rest(p0, a), d = rest(p1, b);
        L.p[k & 1][mine][bp][lane] = u32x4{a.x, a.y, b.x, b.y};
        L.left[k & 1][mine][bp][lane] = u32x4{c.x, c.y, d.x, d.y};
        sum = ((p0[0] + p0[1]) + (p0[2] + p0[3])) + ((p1[0] + p1[1]) + (p1[2] + p1[3]));
    };
    // The scores of step k whole, hidden where they are not seen, and whether some are not finite.
    bool stray = false;
    const auto join = [&](int k) {
#pragma unroll
        for (int j = 0; j < 2; ++j) z[j] = own[j] + L.half[wave ^ 2][j][lane];
        turn_to(P, u, pages, off + k, off + cnt, lane);
        const bool ok = valid(pages, off + k);
        const int base = (u.page0 + off + k) * kPage + bp * 32;
        const f32x4 both = z[0] + z[1];
        stray = __ballot(!finite((both[0] + both[1]) + (both[2] + both[3]))) != 0;
        if (!(ok && base + 31 <= common)) {
            asm volatile("");                   // a branch, not forty instructions every step
            if (!ok && t == 0) raise(P.h, FLEET_MOE_ABORT_BAD_PAGE);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    z[j][i] = (ok & (base + kBlock * j + 4 * g + i <= r.pos)) ? z[j][i] : -INFINITY;
        }
    };
    const auto finish = [&](int k) {
        weigh(k);
        const float top = fmaxf(fmaxf(fmaxf(z[0][0], z[0][1]), fmaxf(z[0][2], z[0][3])),
                                fmaxf(fmaxf(z[1][0], z[1][1]), fmaxf(z[1][2], z[1][3])));
        const bool high = __ballot(top > m + slack) != 0;
        if (lane == 0) L.flags[k & 1][wave] = (stray ? 2 : 0) | (high ? 1 : 0);
    };
    // The codes of V of a page, and their scales
    i32x2 v[2][kCols];
    uint32_t f[2][2];
    const auto fetch = [&](int b) {
        uint32_t first = lds_addr(L.tile[b]) + wave * kCols * 256 + column_at(lane);
        asm("" : "+v"(first));                // one address, the rest is offsets
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < kCols; ++i) v[h][i] = column(first + 2 * h * kBlockStep, i);
            f[h][0] = L.scale[b][4 * h];
            f[h][1] = L.scale[b][4 * h + 2];
        }
    };
    // What is rare: a row's scores beyond its reference, or one that is not finite, in step k.
    const auto mend = [&](int k, bool strays) {
        // (its addresses are made here, not kept in registers through all steps)
        const int lane = fm_tid() & 63, n = lane & 15;
        float top = fmaxf(fmaxf(fmaxf(z[0][0], z[0][1]), fmaxf(z[0][2], z[0][3])),
                          fmaxf(fmaxf(z[1][0], z[1][1]), fmaxf(z[1][2], z[1][3])));
        top = xor32_max(xor16_max(top));
        if (lane < 16) L.top[mine][bp][lane] = top;
        if (strays) {
            // Such a value makes the score of every row infinite or NaN, and the weight of one
            // that sees it NaN or 0; a row that does not see it has the weight 0, and must not
            // meet 0 * NaN.
            const float most = __uint_as_float(kMaxScale);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < kCols; ++i) {
                    v[h][i].x = (int)drop_infinite((uint32_t)v[h][i].x, any_scale(f[h][0]) == most);
                    v[h][i].y = (int)drop_infinite((uint32_t)v[h][i].y, any_scale(f[h][1]) == most);
                }
        }
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
    const auto add = [&](int k) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            bf16x8 pb[4], pr[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                pb[j] = __builtin_bit_cast(bf16x8, L.p[k & 1][j][h][lane]);
                pr[j] = __builtin_bit_cast(bf16x8, L.left[k & 1][j][h][lane]);
            }
            const float sa = any_scale(f[h][0]), sb = any_scale(f[h][1]);
#pragma unroll
            for (int i = 0; i < kCols; ++i) {
                const bf16x8 a = widen((uint32_t)v[h][i].x, (uint32_t)v[h][i].y, sa, sb);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j][i] = mfma(a, pb[j], acc[j][i]);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j][i] = mfma(a, pr[j], acc[j][i]);
            }
        }
        const bf16x8 one = __builtin_bit_cast(bf16x8, u32x4{kOnes, kOnes, kOnes, kOnes});
        ones = mfma(one, __builtin_bit_cast(bf16x8, L.p[k & 1][wave & 3][wave >> 2][lane]), ones);
        ones = mfma(one, __builtin_bit_cast(bf16x8, L.left[k & 1][wave & 3][wave >> 2][lane]), ones);
    };

    if (cnt > 0) {
        barrier();                              // q has been read: its place is free
        if (tp == 0 && kPageRing - 1 < cnt) issue(kPageRing - 1, kPageRing - 1);
        score(0);
        barrier();
        join(0);
        finish(0);
        fetch(0);
        if (cnt > 1) {
            barrier();                          // the halves of step 0 have been read
            score(1);
        }
    }
    // Step k: behind the barrier the weights of k, both halves of the scores of k + 1 and the
    // rows of k + 2 are there.
    int b = 0;                                  // of step k
    for (int k = 0; k < cnt; ++k) {
        const int b1 = b == kPageRing - 1 ? 0 : b + 1, b2 = b1 == kPageRing - 1 ? 0 : b1 + 1;
        wait_copies<0>();
        barrier();
        const uint2 fl = *reinterpret_cast<const uint2*>(L.flags[k & 1]);
        asm volatile("" ::: "memory");          // (the copies' addresses while it is on its way)
        if (tp == 0 && k + kPageRing < cnt) issue(k + kPageRing, b);    // where step k was
        const int flags = wave_bcast((int)(fl.x | fl.y));
        if (flags) mend(k, flags & 0x02020202);
        l += sum;
        // Of a SIMD's two waves (w and w + 4) one makes its weights while the other multiplies.
        // (The asm keeps each in its place: the compiler would fetch both's operands before.)
        if (tp != 0) {
            asm volatile("; products first" ::: "memory");
            add(k);
            asm volatile("; products made" ::: "memory");
        }
        if (k + 1 < cnt) {
            join(k + 1);
            finish(k + 1);
        }
        if (tp == 0) {
            asm volatile("; products last" ::: "memory");
            add(k);
            asm volatile("; products made, too" ::: "memory");
        }
        if (k + 2 < cnt) {
            barrier();                          // the halves of step k + 1 have been read
            score(b2);
        }
        if (k + 1 < cnt) fetch(b1);
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
    const int column0 = wave * kCols * 16 + 4 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (u.row0 + i * 16 >= u.rows) break;
        const int row = i * 16 + n;
        const float sum = L.sum[i][0][n] + L.sum[i][1][n];
        const float rounded = L.rounded[i][0][n] + L.rounded[i][1][n];
        const float scaled = L.m[i][n] * P.scale;
        if (to_part >= 0) {
#pragma unroll
            for (int j = 0; j < kCols; ++j)
                st_global(part_at(P.plan, to_part / 16 + i, wave, j, lane), acc[i][j]);
            if (wave == 0 && g == 0)
                st_global(P.plan.stat + to_part + row, f32x4{scaled, sum, rounded, 0.f});
        } else if (u.row0 + row < u.rows) {
            const int64_t to = (int64_t)u.tok0 * P.n_heads + u.row0 + row;
            const float inv = rounded == 0.f ? 0.f : 1.f / rounded;
#pragma unroll
            for (int j = 0; j < kCols; ++j)
                put(P.out + to * kC + column0 + j * 16, acc[i][j], inv);
            if (P.lse && wave == 0 && g == 0) P.lse[to] = lse_of(scaled, sum);
        }
    }
}

// The same for a unit of 16 rows or fewer, a sequence's one token: wave (block, half) takes half
// of the 576 products of the rows with 16 positions, half 0 makes the weights, and every wave
// adds 64 columns of O. Here a page's bytes bound a step, not its products, so the weights are
// two operands, bf16 and what that leaves: 16 bits.
__device__ __forceinline__ void attend16(const SharedParams& P, PageLds& L, const Unit& u, int off,
                                         int cnt, int64_t to_part) {
    constexpr int kCols = kC / 16 / kGridWaves;
    const int t = fm_tid(), lane = t & 63, wave = wave_bcast(t >> 6);
    const int g = lane >> 4, n = lane & 15, blk = wave & 3, half = wave >> 2;
    const bool weighs = half == 1;              // the others copy

    PageList pages{0, 0, 0, 0};
    const auto issue = [&](int k, int b) {
        turn_to(P, u, pages, off + k, off + cnt, lane);
        issue_page(P, L, page_of(pages, off + k), b, wave, lane);
    };
    if (cnt > 0) {
        turn_to(P, u, pages, off, off + cnt, lane);
        if (!weighs)
            for (int k = 0; k < kPageRing - 1 && k < cnt; ++k) issue(k, k);
        copy_q<16 / kGridWaves>(P, L, u, kPageRing - 1, wave, lane);
    }
    TileRow r = tile_row(P, u, u.row0 + n);
    set_position(P, u, r);
    const int common = common_position(r);
    f32x4 acc[kCols], ones{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (auto& a : acc) a = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, ref = -INFINITY, l = 0.f;
    const float slack = P.slack;
    f32x4 z, next;
    bool stray = false;
    float p[4]{0.f, 0.f, 0.f, 0.f};
    wait_copies<0>();
    barrier();
    bf16x8 q[kTileHalf];
    read_q(L, kPageRing - 1, n, g, half, q);

    const auto score = [&](int b) {
        const uint8_t* block = L.tile[b] + blk * kBlockStep + lane * 16;
        const float sc = any_scale(L.scale[b][2 * blk]), sp = any_scale(L.scale[b][2 * blk + 1]);
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
        if (!weighs) L.half[blk][0][lane] = next;
    };
    const auto weigh = [&](int k) {
        const float down = ref == -INFINITY ? 0.f : ref;
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = exp2_(fmaf(z[j], P.scale, -down));
        const uint2 w = weights(p);
        reinterpret_cast<uint2*>(&L.p[k & 1][0][blk >> 1][lane])[blk & 1] = w;
        reinterpret_cast<uint2*>(&L.p[k & 1][1][blk >> 1][lane])[blk & 1] = rest(p, w);
    };
    const auto finish = [&](int k) {
        z = next + L.half[blk][0][lane];
        turn_to(P, u, pages, off + k, off + cnt, lane);
        const bool ok = valid(pages, off + k);
        const int base = (u.page0 + off + k) * kPage + blk * kBlock;
        const bool bad = !finite((z[0] + z[1]) + (z[2] + z[3]));
        if (!(ok && base + kBlock - 1 <= common)) {
            asm volatile("");                   // a branch, not twenty instructions every step
            if (!ok && lane == 0) raise(P.h, FLEET_MOE_ABORT_BAD_PAGE);
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = (ok & (base + 4 * g + i <= r.pos)) ? z[i] : -INFINITY;
        }
        weigh(k);
        const float top = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
        stray = __ballot(bad) != 0;
        const bool high = __ballot(top > m + slack) != 0;
        if (lane == 0) L.flag[k & 1][blk] = stray | high;
    };
    const auto mend = [&](int k, int b) {
        if (weighs) {
            float top = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
            top = xor32_max(xor16_max(top));
            if (lane < 16) L.top[blk][0][lane] = top;
            if (stray) clean(L.tile[b] + blk * kBlockStep, L.scale[b][2 * blk], lane);
        }
        barrier();
        const float to = fmaxf(m, fmaxf(fmaxf(L.top[0][0][n], L.top[1][0][n]),
                                        fmaxf(L.top[2][0][n], L.top[3][0][n])));
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
    const auto add = [&](int k, int b) {
        const uint32_t first = lds_addr(L.tile[b]) + wave * kCols * 256 + column_at(lane);
        const bf16x8 one = __builtin_bit_cast(bf16x8, u32x4{kOnes, kOnes, kOnes, kOnes});
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bf16x8 pb = __builtin_bit_cast(bf16x8, L.p[k & 1][0][h][lane]);
            const bf16x8 pr = __builtin_bit_cast(bf16x8, L.p[k & 1][1][h][lane]);
            const float sa = any_scale(L.scale[b][4 * h]), sb = any_scale(L.scale[b][4 * h + 2]);
#pragma unroll
            for (int i = 0; i < kCols; ++i) {
                const i32x2 v = column(first + 2 * h * kBlockStep, i);
                const bf16x8 a = widen((uint32_t)v.x, (uint32_t)v.y, sa, sb);
                acc[i] = mfma(a, pb, acc[i]);
                acc[i] = mfma(a, pr, acc[i]);
            }
            ones = mfma(one, pb, ones);
            ones = mfma(one, pr, ones);
        }
    };

    if (cnt > 0) {
        score(0);
        barrier();
        if (weighs) finish(0);
    }
    int b = 0;                                  // of step k; the barriers as in attend64()
    for (int k = 0; k < cnt; ++k) {
        const int b1 = b == kPageRing - 1 ? 0 : b + 1, b2 = b1 == kPageRing - 1 ? 0 : b1 + 1;
        wait_copies<0>();
        barrier();                              // A
        const int* f = L.flag[k & 1];
        const int flags = (f[0] | f[1]) | (f[2] | f[3]);
        if (!weighs && k + kPageRing - 1 < cnt) issue(k + kPageRing - 1, b2);
        if (wave_bcast(flags)) mend(k, b);
        if (weighs) l += (p[0] + p[1]) + (p[2] + p[3]);
        if (k + 1 < cnt) {
            score(b1);
            barrier();                          // B
            if (weighs) finish(k + 1);
        }
        add(k, b);
        b = b1;
        asm("" : "+s"(b));
    }
    l = xor32_sum(xor16_sum(l));
    if (weighs && lane < 16) L.sum[blk][0][lane] = l;
    barrier();
    const float sum = (L.sum[0][0][n] + L.sum[1][0][n]) + (L.sum[2][0][n] + L.sum[3][0][n]);
    if (to_part >= 0) {
#pragma unroll
        for (int j = 0; j < kCols; ++j)
            st_global(part_at(P.plan, to_part / 16, wave, j, lane), acc[j]);
        if (wave == 0 && g == 0)
            st_global(P.plan.stat + to_part + n, f32x4{ref, sum, ones[0], 0.f});
    } else if (u.row0 + n < u.rows) {
        const int64_t to = (int64_t)u.tok0 * P.n_heads + u.row0 + n;
        const float inv = ones[0] == 0.f ? 0.f : 1.f / ones[0];
        const int column0 = wave * kCols * 16 + 4 * g;
#pragma unroll
        for (int j = 0; j < kCols; ++j) put(P.out + to * kC + column0 + j * 16, acc[j], inv);
        if (P.lse && wave == 0 && g == 0) P.lse[to] = lse_of(ref, sum);
    }
}

__global__ __launch_bounds__(kGridThreads, 1) void shared_kernel(SharedParams P) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    PageLds& L = *reinterpret_cast<PageLds*>(lds);
    const int t = threadIdx.x;
    Place place;
    if (!locate(P, L, blockIdx.x, place)) return;
    const int wg = place.wg;
    const Split share(place.total, place.shares);
    const int64_t all_rows = (int64_t)P.n_tokens * P.n_heads;
    const int end = share.first(wg + 1);
    for (int at = share.first(wg);;) {
        const Item w = lane_of(L.item, 0);
        const int off = wave_bcast(L.off);
        barrier();                              // they are read
        // the unit at time `off` of the item
        const Sizes z(P, w, place.tile);
        const int front = z.front(w);
        Unit u;
        u.common = off < front;
        const int rows = u.common ? z.rows0 : z.rows1, steps = u.common ? w.steps0 : w.steps1;
        const int o = u.common ? off : off - front, whole_unit = z.full().setup + z.full().page * steps;
        const int units = u.common ? z.units0 : z.units1;
        const int k0 = o / whole_unit, k = k0 < units ? k0 : units - 1;
        const Cost cost = z.cost(rows, k);
        const int from = o - k * whole_unit, all = cost.setup + cost.page * steps;
        u.row0 = k * z.tile;
        u.rows = rows;
        u.tok0 = w.tok0;
        u.first = w.first;
        u.end = w.end;
        u.inside = place.inside;
        if (u.common) {
            u.base = 0;
            u.page0 = 0;
            u.n = w.steps0;
            u.table = P.c.table + (int64_t)w.first * P.c.max_pages;
        } else {
            u.base = w.len - w.n_new;
            u.page0 = w.pages;
            u.table = P.c.table + (int64_t)w.seq * P.c.max_pages + w.pages;
            // up to the position of the unit's last token
            const int last = u.row0 + z.tile - 1 < u.rows ? u.row0 + z.tile - 1 : u.rows - 1;
            const int p = u.base + token_of_row(last, P.per_head);
            u.n = w.len < 0 || p < 0 ? 0 : pages_of((int64_t)p + 1) - w.pages;
            if (w.len < 0 && t == 0) raise(P.h, FLEET_MOE_ABORT_POSITION);
        }
        // the steps that begin from here to the share's end
        const int take = all - from < end - at ? all - from : end - at;
        const auto step_at = [&](int time) {
            const int i = cost.begun(time);
            return i < steps ? i : steps;
        };
        const int lo = step_at(from), hi = step_at(from + take);
        // what comes next, out of the registers meanwhile
        if (wave_bcast(t >> 6) == kGridWaves - 1) {
            int o2 = off + take;
            Item next = w;
            if (end - at > take && o2 >= z.total(w)) {
                const int s = next_with_work(L, w.seq, P.c.n_seqs, t & 63);
                if (s < P.c.n_seqs) {
                    next = item_of(P, s, raw_of(P, s), place.stale);
                    if (leads(next)) next.last = start_of(P, next.end);
                    o2 = 0;
                }
            }
            if (t == kGridThreads - 64) {
                L.item = next;
                L.off = o2;
                L.at = at + take;
            }
        }
        if (hi > lo) {
            // where the part goes: a whole unit's to its rows, or to one of two slots
            const bool whole = lo == 0 && hi == steps;
            const int64_t row = (int64_t)u.tok0 * P.n_heads + u.row0;
            const int64_t wholes = whole_parts(P.c.n_seqs, all_rows), slots = 2 * wholes;
            const int64_t mine = whole_part(w.seq, (int64_t)u.tok0 * P.n_heads) + u.row0;
            const int64_t part =
                whole ? (u.common ? mine : w.pages > 0 ? wholes + mine : -1)
                      : slots + (int64_t)(2 * wg + (lo == 0 ? 1 : 0)) * kTile;
            if (lo == 0 && t < z.tile && u.row0 + t < u.rows) {
                const int last = at - from + cost.setup + (steps - 1) * cost.page;
                Parts m;
                m.at = (int)(part + t);
                m.next = (int)(slots + (int64_t)(wg + 1) * kPartStep + t);
                m.count = part < 0 ? 0 : whole ? 1 : share.holder(last) - wg + 1;
                m.front = !u.common && w.pages > 0;
                P.plan.meta[(u.common ? 0 : all_rows) + row + t] = m;
            }
            const int n = hi < u.n ? hi : u.n;
            if (z.tile == 16 || u.rows - u.row0 <= 16) attend16(P, L, u, lo, n > lo ? n - lo : 0, part);
            else attend64(P, L, u, lo, n > lo ? n - lo : 0, part);
        }
        barrier();                              // LDS is free again
        at = wave_bcast(L.at);
        if (at >= end) return;
    }
}

// Adds the parts of 16 rows, those over common pages first: lane (g, n) has four columns of row
// n. A wave 64 columns and all parts of their rows, or, where there are few rows of many parts, an
// eighth of the parts, and the workgroup's eight waves their sum (shared and joined, 64 sequences
// of 16 heads 48.5 us and 50.3 in one wave each; 256 sequences 209 us and 207).
constexpr int kJoinParts = 2;                   // on their way together (four: more registers,
                                                // the same time)
constexpr int64_t kManyRows = 2048;
template <bool kSplit>
__global__ __launch_bounds__(kGridThreads) void join_kernel(SharedParams P) {
    const int t = threadIdx.x, lane = t & 63, wave = wave_bcast(t >> 6);
    const int g = lane >> 4, n = lane & 15;
    const int64_t all_rows = (int64_t)P.n_tokens * P.n_heads;
    const int64_t block = kSplit ? blockIdx.x / kGridWaves : blockIdx.x;
    const int column = kSplit ? blockIdx.x % kGridWaves : wave;         // of 64
    const int64_t row = block * 16 + n;
    // all on its way together; rows that are nobody's have no parts of this call
    const int64_t safe = row < all_rows ? row : 0;
    i32x4 own = ld_global(reinterpret_cast<const i32x4*>(P.plan.meta + all_rows + safe));
    const i32x4 front = ld_global(reinterpret_cast<const i32x4*>(P.plan.meta + safe));
    const i32x2 rows = ld_global(reinterpret_cast<const i32x2*>(&P.plan.h->first));
    if (row < rows.x || row >= rows.y) own.z = 0;
    const int n0 = own.z > 0 && own.w ? front.z : 0, count = n0 + own.z;
    const auto part = [&](int i) -> int64_t {
        const bool mine = i >= n0;
        const int j = mine ? i - n0 : i;
        const int first = mine ? own.x : front.x, next = mine ? own.y : front.y;
        return j == 0 ? first : next + (int64_t)(j - 1) * kPartStep;
    };
    constexpr int kEach = kSplit ? kGridWaves : 1;
    float top = -INFINITY, sum = 0.f, rounded = 0.f;
    f32x4 o[4];
#pragma unroll
    for (auto& e : o) e = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int i0 = kSplit ? wave : 0; __ballot(i0 < count); i0 += kJoinParts * kEach) {
        f32x4 st[kJoinParts], v[kJoinParts][4];
#pragma unroll
        for (int k = 0; k < kJoinParts; ++k) {
            const int i = i0 + k * kEach;
            st[k] = f32x4{-INFINITY, 0.f, 0.f, 0.f};
#pragma unroll
            for (auto& e : v[k]) e = f32x4{0.f, 0.f, 0.f, 0.f};
            if (i < count) {
                const int64_t at = part(i);
                st[k] = ld_global(P.plan.stat + at);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    v[k][j] = ld_global(part_at(P.plan, at / 16, column, j, g * 16 + (int)(at & 15)));
            }
        }
        float to = top;
#pragma unroll
        for (const f32x4& s : st) to = fmaxf(to, s[0]);
        const float ref = to == -INFINITY ? 0.f : to, shrink = exp2_(top - ref);
        top = to;
        sum *= shrink;
        rounded *= shrink;
#pragma unroll
        for (auto& e : o) e *= shrink;
#pragma unroll
        for (int k = 0; k < kJoinParts; ++k) {
            const float f = exp2_(st[k][0] - ref);
            sum += f * st[k][1];
            rounded += f * st[k][2];
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] += v[k][j] * f;
        }
    }
    const auto finish = [&](int j, const f32x4& e) {
        if (count == 0) return;
        put(P.out + row * kC + column * 64 + j * 16 + 4 * g, e, rounded == 0.f ? 0.f : 1.f / rounded);
        if (P.lse && column == 0 && j == 0 && g == 0) P.lse[row] = lse_of(top, sum);
    };
    if constexpr (kSplit) {
        __shared__ f32x4 all[kGridWaves][4][64], stats[kGridWaves][16];
#pragma unroll
        for (int j = 0; j < 4; ++j) all[wave][j][lane] = o[j];
        if (g == 0) stats[wave][n] = f32x4{top, sum, rounded, 0.f};
        __syncthreads();
        if (wave >= 4) return;
        top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kGridWaves; ++i) top = fmaxf(top, stats[i][n][0]);
        const float ref = top == -INFINITY ? 0.f : top;
        sum = rounded = 0.f;
        f32x4 e{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kGridWaves; ++i) {
            const float f = exp2_(stats[i][n][0] - ref);
            sum += f * stats[i][n][1];
            rounded += f * stats[i][n][2];
            e += all[i][wave][lane] * f;
        }
        finish(wave, e);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) finish(j, o[j]);
    }
}

}  // namespace cache
}  // namespace fleet_moe

using namespace fleet_moe;
using namespace fleet_moe::cache;

int fleet_moe_check_device(int min_cus);

extern "C" size_t fleet_cache_plan_bytes(int32_t n_seqs, int32_t max_tokens, int32_t n_heads) {
    if (n_seqs < 1 || n_seqs > kMaxSeqs || max_tokens < 1 || n_heads < 1 ||
        n_heads > FLEET_CACHE_MAX_HEADS || (int64_t)max_tokens * n_heads > kMaxPlanRows)
        return 0;
    return plan_size(n_seqs, (int64_t)max_tokens * n_heads);
}

extern "C" int fleet_cache_share(const fleet_cache* cache, const int32_t* groups,
                                 int32_t n_groups, int32_t* pages, void* plan, size_t plan_bytes,
                                 void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (int e = check_cache(cache, workspace, workspace_bytes)) return e;
    if (!groups || (uintptr_t)groups % 4 || (uintptr_t)pages % 4 || n_groups < 1 ||
        n_groups > cache->n_seqs || !plan || (uintptr_t)plan % 256)
        return FLEET_MOE_ERR_ARG;
    if (plan_bytes < plan_size(cache->n_seqs, 0)) return FLEET_MOE_ERR_WORKSPACE;
    if (int e = fleet_moe_check_device(1)) return e;
    hipLaunchKernelGGL(share_kernel, dim3(n_groups), dim3(kShareThreads), 0, stream, *cache, groups,
                       n_groups, pages, plan_at(plan, cache->n_seqs, 0),
                       static_cast<Header*>(workspace));
    return (int)hipGetLastError();
}

extern "C" int fleet_cache_attend_shared(const fleet_cache* cache, int32_t layer,
                                         const uint16_t* q, int64_t q_stride,
                                         const int32_t* start, int32_t n_tokens, int32_t n_heads,
                                         float scale, uint16_t* out, float* lse, void* plan,
                                         size_t plan_bytes, void* workspace,
                                         size_t workspace_bytes, hipStream_t stream) {
    if (int e = check_cache(cache, workspace, workspace_bytes)) return e;
    const int64_t rows = (int64_t)n_tokens * n_heads;
    if (layer < 0 || layer >= cache->n_layers || n_tokens < 0 || n_heads < 1 ||
        n_heads > FLEET_CACHE_MAX_HEADS || rows > kMaxPlanRows || !(scale > 0.f) ||
        !(scale * kLog2e <= FLT_MAX) || (uintptr_t)start % 4 ||
        (!start && n_tokens != cache->n_seqs) || !plan || (uintptr_t)plan % 256)
        return FLEET_MOE_ERR_ARG;
    if (n_tokens == 0) return 0;
    if (!q || !out || (uintptr_t)q % 16 || (uintptr_t)out % 8 || (uintptr_t)lse % 4 ||
        q_stride < (int64_t)n_heads * kRow || q_stride % 8 || q_stride > ((int64_t)1 << 32))
        return FLEET_MOE_ERR_ARG;
    // the time of all units is counted in 32 bits
    if ((2 * (rows / kTile) + 2 * (int64_t)cache->n_seqs) *
            (kCost64.setup + kCost64.page * (int64_t)cache->max_pages) > 0x7fffffff)
        return FLEET_MOE_ERR_ARG;
    if (plan_bytes < plan_size(cache->n_seqs, rows)) return FLEET_MOE_ERR_WORKSPACE;
    if (int e = fleet_moe_check_device(1)) return e;
    SharedParams P{};
    P.c = *cache;
    P.q = q;
    P.start = start;
    P.out = out;
    P.lse = lse;
    P.plan = plan_at(plan, cache->n_seqs, rows);
    P.h = static_cast<Header*>(workspace);
    P.q_stride = q_stride;
    P.per_head = head_divisor(n_heads);
    P.layer = layer;
    P.n_tokens = n_tokens;
    P.n_heads = n_heads;
    P.scale = scale * kLog2e;
    P.slack = fminf(kRise / P.scale, FLT_MAX);
    if (int e = launch<shared_kernel>(kGrid, kGridThreads, sizeof(PageLds), P, stream)) return e;
    // (a call of many rows has few parts a row: a unit's share of the workgroups)
    if (rows >= kManyRows) return launch<join_kernel<false>>((rows + 15) / 16, kGridThreads, 0, P, stream);
    return launch<join_kernel<true>>((rows + 15) / 16 * kGridWaves, kGridThreads, 0, P, stream);
}
