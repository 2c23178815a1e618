// Pages of the 8-bit cache: reordering and forking sequences, growing them,
// moving pages together (declarations in fleet_moe.h).
//
// What these calls decide is a few hundred words (table rows, holder counts), so
// one workgroup decides and latency bounds it; what they move is megabytes per
// page (every layer), which a second launch of the whole chip copies. The order in
// which pages are taken is fixed (lowest free page first, sequences in order), so
// the outcome does not depend on the order of any atomic.
#include "cache_pages.h"

namespace fleet_moe {
namespace cache {

constexpr int kBook = 1024;                   // threads that keep the book: one per sequence
constexpr int kBookWaves = kBook / 64;
constexpr int kScan = 8;                      // pages per thread and step of a scan of refs

// Sums of v over the threads before this one, and over all. `lds` has
// kBookWaves + 1 words, and may be used again after the call.
__device__ __forceinline__ int block_scan(int v, int* lds, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int incl = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d);
        if (lane >= d) incl += o;
    }
    if (lane == 63) lds[wave] = incl;
    __syncthreads();
    if (threadIdx.x < 64) {
        int w = lane < kBookWaves ? lds[lane] : 0;
        const int own = w;
#pragma unroll
        for (int d = 1; d < kBookWaves; d <<= 1) {
            const int o = __shfl_up(w, d);
            if (lane >= d) w += o;
        }
        if (lane < kBookWaves) lds[lane] = w - own;
        if (lane == kBookWaves - 1) lds[kBookWaves] = w;
    }
    __syncthreads();
    const int before = lds[wave] + incl - v;
    total = lds[kBookWaves];
    __syncthreads();
    return before;
}

// ---------------------------------------------------------------- remap

// In place without a second table: a workgroup owns kCols columns of every row,
// takes them into LDS, and writes them back reordered; no other workgroup reads
// or writes them. lens is one column more, the first workgroup's.
constexpr int kCols = 16;
constexpr int kRemapThreads = 256;

__global__ __launch_bounds__(kRemapThreads) void remap_kernel(fleet_cache c,
                                                              const int32_t* parents, Header* h) {
    extern __shared__ int32_t lds[];
    int32_t* children = lds;                              // [n_seqs]
    int32_t* parent = lds + c.n_seqs;                     // [n_seqs]
    int32_t* slab = lds + 2 * c.n_seqs;                   // [n_seqs][kCols]
    const int t = threadIdx.x, col0 = blockIdx.x * kCols;
    const int cols = c.max_pages - col0 < kCols ? c.max_pages - col0 : kCols;
    for (int i = t; i < c.n_seqs; i += kRemapThreads) children[i] = 0;
    __syncthreads();
    bool bad = false;
    for (int i = t; i < c.n_seqs; i += kRemapThreads) {
        int p = parents[i];
        if (p < -1 || p >= c.n_seqs) {
            bad = true;
            p = -1;
        }
        parent[i] = p;
        if (p >= 0) atomicAdd(&children[p], 1);
    }
    if (bad && blockIdx.x == 0) raise(h, FLEET_MOE_ABORT_BAD_ID);
    for (int i = t; i < c.n_seqs * kCols; i += kRemapThreads) {
        const int s = i / kCols, k = i % kCols;
        slab[i] = k < cols ? c.table[(int64_t)s * c.max_pages + col0 + k] : -1;
    }
    __syncthreads();
    for (int i = t; i < c.n_seqs * kCols; i += kRemapThreads) {
        const int s = i / kCols, k = i % kCols;
        if (k >= cols) continue;
        // the pages of a row that has no child or several change their count
        const int page = slab[i];
        if (page >= 0 && children[s] != 1) {
            if (page < c.n_pages) atomicAdd(&c.refs[page], children[s] - 1);
            else raise(h, FLEET_MOE_ABORT_BAD_PAGE);
        }
        const int p = parent[s];
        if (p != s) c.table[(int64_t)s * c.max_pages + col0 + k] = p < 0 ? -1 : slab[p * kCols + k];
    }
    if (blockIdx.x != 0) return;
    if (t == 0) h->remaps += 1;
    __syncthreads();
    for (int i = t; i < c.n_seqs; i += kRemapThreads) slab[i] = c.lens[i];
    __syncthreads();
    for (int i = t; i < c.n_seqs; i += kRemapThreads)
        c.lens[i] = parent[i] < 0 ? 0 : slab[parent[i]];
}

// ---------------------------------------------------------------- grow

__global__ __launch_bounds__(kBook) void grow_kernel(fleet_cache c, const int32_t* n_new,
                                                     Header* h, Copy* copies, int32_t* list) {
    __shared__ int lastp[kMaxSeqs], first[kMaxSeqs], from[kMaxSeqs];
    __shared__ int scan[kBookWaves + 1];
    __shared__ int any_shared;
    __shared__ uint32_t stop;
    const int t = threadIdx.x;
    if (t == 0) any_shared = stop = 0;
    __syncthreads();
    int len = 0, add = 0, have = 0, want = 0, last = -1, refs = 0;
    bool open = false;
    if (t < c.n_seqs) {
        len = checked_len(c.lens[t], c.max_pages);
        add = n_new[t];
        uint32_t why = 0;
        if (len < 0 || add < 0) {
            why = FLEET_MOE_ABORT_POSITION;
        } else if ((int64_t)len + add > (int64_t)c.max_pages * kPage ||
                   (int64_t)len + add > 0x7fffffff) {
            why = FLEET_MOE_ABORT_NO_PAGE;
        } else {
            have = pages_of(len);
            want = pages_of((int64_t)len + add);
            open = add > 0 && len % kPage != 0;
            if (open) {
                last = c.table[(int64_t)t * c.max_pages + have - 1];
                if ((unsigned)last >= (unsigned)c.n_pages) why = FLEET_MOE_ABORT_BAD_PAGE;
                else refs = c.refs[last];
            }
        }
        if (why) atomicOr(&stop, why);
        if (refs > 1) any_shared = 1;
        lastp[t] = open ? last : -1;
    }
    __syncthreads();
    const auto refuse = [&](uint32_t why) {
        raise(h, why);
        h->refused = why;
        h->count = 0;
    };
    if (stop) {
        if (t == 0) refuse(stop);
        return;
    }
    // Sequences leave a shared page in order, each with a copy, until one holder
    // is left: the one that finds the count at 1 keeps the page.
    bool copy = false;
    if (any_shared && refs > 1) {
        int left = refs;
        for (int j = 0; j < t; ++j) left -= lastp[j] == last;
        copy = left > 1;
    }
    const int need = t < c.n_seqs ? want - have + copy : 0;
    int total, n_copies;
    const int before = block_scan(need, scan, total);
    const int nth = block_scan(copy ? 1 : 0, scan, n_copies);
    first[t] = before;
    from[t] = have - copy;
    // the lowest free pages, in order
    int found = 0;
    for (int64_t p0 = 0; p0 < c.n_pages && found < total; p0 += kBook * kScan) {
        const int64_t at = p0 + (int64_t)t * kScan;
        uint32_t free = 0;
#pragma unroll
        for (int k = 0; k < kScan; ++k)
            if (at + k < c.n_pages && c.refs[at + k] == 0) free |= 1u << k;
        int here;
        int j = found + block_scan(__popc(free), scan, here);
        for (; free && j < total; free &= free - 1) list[j++] = (int)(at + __ffs(free) - 1);
        found += here;
    }
    __syncthreads();
    if (found < total) {
        if (t == 0) refuse(FLEET_MOE_ABORT_NO_PAGE);
        return;
    }
    if (copy) {
        Copy k;
        k.src = last;
        k.dst = list[before];
        k.chunks = (len % kPage + kBlock - 1) / kBlock * (kBlockBytes / 16);
        k.pad = 0;
        copies[nth] = k;
        atomicSub(&c.refs[last], 1);
    }
    if (t == 0) {
        h->refused = 0;
        h->count = n_copies;
    }
    if (t < c.n_seqs && add > 0) c.lens[t] = len + add;
    // page j of the list goes to the sequence whose share holds j
    for (int j = t; j < total; j += kBook) {
        int lo = 0, hi = kMaxSeqs - 1;                    // first[lo] <= j, the last such
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (first[mid] <= j) lo = mid;
            else hi = mid - 1;
        }
        const int page = list[j];
        c.table[(int64_t)lo * c.max_pages + from[lo] + j - first[lo]] = page;
        c.refs[page] = 1;
    }
}

// ---------------------------------------------------------------- compact

__global__ __launch_bounds__(kBook) void compact_kernel(fleet_cache c, int32_t* n_used, Header* h,
                                                        Copy* moves, int32_t* new_page) {
    __shared__ int scan[kBookWaves + 1];
    const int t = threadIdx.x;
    int used = 0;
    for (int64_t p0 = 0; p0 < c.n_pages; p0 += kBook * kScan) {
        const int64_t at = p0 + (int64_t)t * kScan;
        int n = 0, here;
#pragma unroll
        for (int k = 0; k < kScan; ++k) n += at + k < c.n_pages && c.refs[at + k] != 0;
        block_scan(n, scan, here);
        used += here;
    }
    int holes = 0, movers = 0;
    for (int64_t p0 = 0; p0 < c.n_pages; p0 += kBook * kScan) {
        const int64_t at = p0 + (int64_t)t * kScan;
        uint32_t hole = 0, mover = 0;
#pragma unroll
        for (int k = 0; k < kScan; ++k) {
            if (at + k >= c.n_pages) continue;
            const bool held = c.refs[at + k] != 0;
            if (!held && at + k < used) hole |= 1u << k;
            if (held && at + k >= used) mover |= 1u << k;
        }
        int n_hole, n_mover;
        int i = holes + block_scan(__popc(hole), scan, n_hole);
        int j = movers + block_scan(__popc(mover), scan, n_mover);
        for (; hole; hole &= hole - 1) moves[i++].dst = (int)(at + __ffs(hole) - 1);
        for (; mover; mover &= mover - 1) moves[j++].src = (int)(at + __ffs(mover) - 1);
        holes += n_hole;
        movers += n_mover;
    }
    __syncthreads();
    // as many holes as movers: both are `used` less the used pages in front
    for (int j = t; j < movers; j += kBook) {
        const int src = moves[j].src, dst = moves[j].dst;
        moves[j].chunks = kCodeBytes / 16;
        new_page[src] = dst;
        c.refs[dst] = c.refs[src];
        c.refs[src] = 0;
    }
    if (t == 0) {
        h->count = movers;
        h->used = used;
        if (n_used) *n_used = used;
    }
}

// Copies the listed pages, a workgroup per page and layer, and after compact
// names the moved pages anew in the table. Bound by HBM, read and write.
constexpr int kCopyThreads = 256;

template <bool kTable>
__global__ __launch_bounds__(kCopyThreads) void copy_kernel(fleet_cache c, const Header* h,
                                                            const Copy* copies,
                                                            const int32_t* new_page) {
    const int t = threadIdx.x, count = h->count;
    if (count == 0) return;
    if constexpr (kTable) {
        const int used = h->used;
        const int64_t n = (int64_t)c.n_seqs * c.max_pages;
        for (int64_t i = (int64_t)blockIdx.x * kCopyThreads + t; i < n;
             i += (int64_t)gridDim.x * kCopyThreads) {
            const int p = c.table[i];
            if (p >= used && p < c.n_pages) c.table[i] = new_page[p];
        }
    }
    const int64_t units = (int64_t)count * c.n_layers;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const Copy k = copies[u / c.n_layers];
        const int layer = (int)(u % c.n_layers);
        const u32x4* src = reinterpret_cast<const u32x4*>(
            c.pool + page_offset(k.src, c.n_pages, layer, c.n_layers));
        u32x4* dst = reinterpret_cast<u32x4*>(
            c.pool + page_offset(k.dst, c.n_pages, layer, c.n_layers));
        constexpr int kAll = kCodeBytes / 16;
        constexpr int kSteps = kAll / kCopyThreads;           // 9, all in flight at once
        static_assert(kSteps * kCopyThreads == kAll, "");
        u32x4 v[kSteps], s;
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
            if (i * kCopyThreads + t < k.chunks) v[i] = ld_stream(src + i * kCopyThreads + t);
        if (t < 2) s = ld_stream(src + kAll + t);
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
            if (i * kCopyThreads + t < k.chunks) st_global(dst + i * kCopyThreads + t, v[i]);
        if (t < 2) st_global(dst + kAll + t, s);
    }
}

}  // namespace cache
}  // namespace fleet_moe

using namespace fleet_moe;
using namespace fleet_moe::cache;

int fleet_moe_check_device(int min_cus);

static int copy_grid(int64_t units) {
    return (int)(units < 1 ? 1 : units > 4096 ? 4096 : units);
}

extern "C" size_t fleet_cache_workspace_bytes(int32_t n_pages, int32_t n_seqs) {
    if (n_pages < 1 || n_pages > kMaxPages || n_seqs < 1 || n_seqs > kMaxSeqs) return 0;
    return workspace_size(n_seqs, n_pages);
}

extern "C" int fleet_cache_remap(const fleet_cache* cache, const int32_t* parents,
                                 void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (int e = check_cache(cache, workspace, workspace_bytes)) return e;
    if (!parents || (uintptr_t)parents % 4) return FLEET_MOE_ERR_ARG;
    if (int e = fleet_moe_check_device(1)) return e;
    const fleet_cache c = *cache;
    const size_t lds = (size_t)c.n_seqs * (kCols + 2) * 4;
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&remap_kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 kMaxSeqs * (kCols + 2) * 4);
        if (e != hipSuccess) return (int)e;
    }
    hipLaunchKernelGGL(remap_kernel, dim3((c.max_pages + kCols - 1) / kCols),
                       dim3(kRemapThreads), lds, stream, c, parents,
                       static_cast<Header*>(workspace));
    return (int)hipGetLastError();
}

extern "C" int fleet_cache_grow(const fleet_cache* cache, const int32_t* n_new, void* workspace,
                                size_t workspace_bytes, hipStream_t stream) {
    if (int e = check_cache(cache, workspace, workspace_bytes)) return e;
    if (!n_new || (uintptr_t)n_new % 4) return FLEET_MOE_ERR_ARG;
    if (int e = fleet_moe_check_device(1)) return e;
    const fleet_cache c = *cache;
    char* ws = static_cast<char*>(workspace);
    Header* h = reinterpret_cast<Header*>(ws);
    Copy* copies = reinterpret_cast<Copy*>(ws + copies_at());
    int32_t* list = reinterpret_cast<int32_t*>(ws + list_at(c.n_seqs, c.n_pages));
    hipLaunchKernelGGL(grow_kernel, dim3(1), dim3(kBook), 0, stream, c, n_new, h, copies, list);
    hipLaunchKernelGGL(copy_kernel<false>, dim3(copy_grid((int64_t)c.n_seqs * c.n_layers)),
                       dim3(kCopyThreads), 0, stream, c, h, copies, list);
    return (int)hipGetLastError();
}

extern "C" int fleet_cache_compact(const fleet_cache* cache, int32_t* n_used, void* workspace,
                                   size_t workspace_bytes, hipStream_t stream) {
    if (int e = check_cache(cache, workspace, workspace_bytes)) return e;
    if (n_used && (uintptr_t)n_used % 4) return FLEET_MOE_ERR_ARG;
    if (int e = fleet_moe_check_device(1)) return e;
    const fleet_cache c = *cache;
    char* ws = static_cast<char*>(workspace);
    Header* h = reinterpret_cast<Header*>(ws);
    Copy* moves = reinterpret_cast<Copy*>(ws + copies_at());
    int32_t* map = reinterpret_cast<int32_t*>(ws + list_at(c.n_seqs, c.n_pages));
    hipLaunchKernelGGL(compact_kernel, dim3(1), dim3(kBook), 0, stream, c, n_used, h, moves, map);
    hipLaunchKernelGGL(copy_kernel<true>, dim3(copy_grid((int64_t)c.n_pages / 2 * c.n_layers)),
                       dim3(kCopyThreads), 0, stream, c, h, moves, map);
    return (int)hipGetLastError();
}
