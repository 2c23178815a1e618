// The layout of the paged 8-bit latent cache, and what its kernels share: the
// workspace, the checks of a cache's sizes and the mapping of workgroups onto
// ragged sequences.
//
// A block's codes lie [chunk][position][16 bytes] because that is how the
// attention's matrix instructions take them: a wave's 16-byte loads of a chunk
// are the operand of q . row directly (1 KB of consecutive bytes per
// instruction), and the transposing LDS read of the same bytes is the operand of
// p . c, so neither product needs the rows rearranged.
#pragma once

#include <stdint.h>

#if defined(__HIP__) || defined(__HIPCC__)
#include "moe_common.h"
#define FLEET_HD __host__ __device__ __forceinline__
#else
#define FLEET_HD inline
#endif

namespace fleet_moe {
namespace cache {

constexpr int kRow = 576;                     // values of a position
constexpr int kC = 512;                       // c, the part that is summed too
constexpr int kPage = 64, kBlock = 16;        // positions
constexpr int kChunks = kRow / 16;            // 16-byte chunks of a row
constexpr int kBlockBytes = kBlock * kRow;
constexpr int kCodeBytes = kPage * kRow;
constexpr int kPageBytes = kCodeBytes + 128;  // with the scales: fp32 [4][2]
constexpr int kMaxSeqs = 1024;
constexpr int kMaxLayers = 64;
constexpr int kMaxPages = 1 << 24;
constexpr int kMaxRowPages = 1 << 20;
constexpr int kMaxRows = 1 << 26;             // (token, head) rows of an attention

FLEET_HD int pages_of(int64_t n) { return (int)((n + kPage - 1) / kPage); }

// A sequence's length as the kernels use it, or -1 where the table cannot hold it.
FLEET_HD int checked_len(int len, int max_pages) {
    return len < 0 || pages_of(len) > max_pages ? -1 : len;
}

// Where a page's layer starts, or -1 for a page outside the pool.
FLEET_HD int64_t page_offset(int page, int n_pages, int layer, int n_layers) {
    return (unsigned)page < (unsigned)n_pages
               ? ((int64_t)page * n_layers + layer) * kPageBytes
               : (int64_t)-1;
}

// Ragged work: sequence s has rows [start[s], start[s+1]), each `mul` items, and
// `div` items make a unit. Units are numbered so that a unit's sequence follows
// from start alone: sequence s has the numbers from first_unit(start[s], s) up to
// first_unit(start[s+1], s + 1). `pad` extra numbers per sequence cover units that
// do not begin on a multiple of div: 1 where a sequence's first item opens a new
// unit, 2 where it may fall into the middle of one (append: blocks are aligned to
// positions, not to rows: n rows touch at most (n + 30) / 16 blocks).
FLEET_HD int64_t first_unit(int start, int s, int mul, int div, int pad) {
    return (int64_t)start * mul / div + (int64_t)pad * s;
}

// Bounds start entries that are not what the caller promised.
FLEET_HD int clamp_row(int v, int n_rows) { return v < 0 ? 0 : v > n_rows ? n_rows : v; }

// The token of a (token, head) row: row / n_heads without a division. per = floor(2^36 /
// n_heads) + 1 is over 2^36 / n_heads by one at most, so row * per is over row * 2^36 /
// n_heads by less than 2^26, which is less than the 2^36 / 128 to the next token; and
// row * per <= 2^26 * (2^36 + 1) keeps within 63 bits. So for every row < kMaxRows
// and n_heads <= 128.
FLEET_HD uint64_t head_divisor(int n_heads) { return ((uint64_t)1 << 36) / n_heads + 1; }
FLEET_HD int token_of_row(int row, uint64_t per) {
    return (int)((uint64_t)(uint32_t)row * per >> 36);
}

// The range of positions a token at `pos` sees: [0, sink) and [lo, pos].
struct Seen {
    int sink, lo;
};
FLEET_HD Seen seen_of(int pos, int window, int sinks) {
    Seen r;
    const int64_t lo = window > 0 ? (int64_t)pos - window + 1 : 0;
    r.lo = lo > 0 ? (int)lo : 0;
    r.sink = sinks < r.lo ? sinks : r.lo;
    return r;
}

// The least e with a <= 448 * 2^e for the bf16 magnitude bits a (finite), at
// least -110: 448 = 1.75 * 2^8.
FLEET_HD int scale_exp(unsigned bits) {
    const int e = (int)(bits >> 7) - 127 - 8 + ((bits & 127) > 96);
    return (bits >> 7) == 0 || e < -110 ? -110 : e;
}

#if defined(__HIP__) || defined(__HIPCC__)

// The workspace: a header, what grow's and compact's first launch leaves for the
// second, and the attention's partial results.
struct Header {
    uint32_t unused[2];
    uint32_t status;
    int32_t count;              // pages to copy
    int32_t used;               // the first page that compact may have moved
    uint32_t refused;           // why the last grow changed nothing, or 0: append writes only then
    uint32_t remaps;            // calls of remap: what was found of the table before is stale
    int32_t pad[57];
};
static_assert(sizeof(Header) == 256, "");
struct Copy {
    int32_t src, dst, chunks, pad;    // chunks: 16-byte pieces of the codes
};

__device__ __forceinline__ void raise(Header* h, uint32_t bit) { atomicOr(&h->status, bit); }

// What the attention's second launch joins: partial results (fp32 [512] a row), the
// rows' references and sums, and where a unit's lie.
constexpr int kShares = 512;           // workgroups: two a CU
constexpr int kMaxUnits = 4096;
constexpr int kPartRows = 1024 * 16;   // two parts of 16 rows a workgroup, or 64 rows of half as many
constexpr size_t kPartBytes = (size_t)kPartRows * kC * 4;
constexpr size_t kStatBytes = (size_t)kPartRows * 16;
constexpr size_t kMetaBytes = (size_t)kMaxUnits * 16;

__host__ __device__ inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
__host__ __device__ inline size_t copies_at() { return sizeof(Header); }
__host__ __device__ inline size_t list_at(int n_seqs, int n_pages) {
    const int moved = n_pages / 2 + 1, n = n_seqs > moved ? n_seqs : moved;
    return copies_at() + up256((size_t)n * sizeof(Copy));
}
__host__ __device__ inline size_t parts_at(int n_seqs, int n_pages) {
    return list_at(n_seqs, n_pages) + up256((size_t)n_pages * 4);
}
inline size_t workspace_size(int n_seqs, int n_pages) {
    return parts_at(n_seqs, n_pages) + kPartBytes + kStatBytes + kMetaBytes;
}

// The checks every call makes of a cache.
inline int check_cache(const fleet_cache* c, const void* workspace, size_t bytes) {
    if (!c || !c->pool || !c->table || !c->lens || !c->refs || !workspace) return FLEET_MOE_ERR_ARG;
    if ((uintptr_t)c->pool % 16 || (uintptr_t)c->table % 4 || (uintptr_t)c->lens % 4 ||
        (uintptr_t)c->refs % 4 || (uintptr_t)workspace % 256)
        return FLEET_MOE_ERR_ARG;
    if (c->n_pages < 1 || c->n_pages > kMaxPages || c->n_layers < 1 || c->n_layers > kMaxLayers ||
        c->n_seqs < 1 || c->n_seqs > kMaxSeqs || c->max_pages < 1 || c->max_pages > kMaxRowPages)
        return FLEET_MOE_ERR_ARG;
    return bytes < workspace_size(c->n_seqs, c->n_pages) ? FLEET_MOE_ERR_WORKSPACE : 0;
}

// The sequence of unit `u` (every lane the same): the last s with
// first_unit(start[s], s) <= u. 64 sequences a step, so one step for most.
__device__ __forceinline__ int find_seq(const int32_t* start, int n_seqs, int n_rows, int64_t u,
                                        int mul, int div, int pad) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int s0 = 0; s0 < n_seqs; s0 += 64) {
        const int s = s0 + lane;
        bool below = false;
        if (s < n_seqs) {
            const int at = start ? clamp_row(ld_global(start + s), n_rows) : s;
            below = first_unit(at, s, mul, div, pad) <= u;
        }
        const int c = __popcll(__ballot(below));
        n += c;
        if (c < 64) break;
    }
    return n - 1;
}
#endif

}  // namespace cache
}  // namespace fleet_moe
