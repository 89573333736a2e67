// Pages of a paged key-value cache: allocation, copies, forks, frees and
// compaction, on the device and on the caller's stream, so that a scheduler
// needs no host read and a step with them can be captured in a graph.
//
// page_refs[p] counts the block_table entries that name page p; 0 is a free
// page.  Free pages are always given out lowest first, in the order of the rows
// or of the list, so the tables follow from the calls alone.  Calls that give
// out pages plan in one workgroup (what they look at is a few ints a page or
// row), check everything first and change nothing when something is wrong
// (the status word says what); the pages' contents then move in a second
// launch at the memory's rate.  Every page and row index is checked against its
// bounds before it is used.
//
// What bounds the copies is the memory (each byte is read and written once); the
// plans are a few dependent reads in one workgroup, which is latency.  Measured:
// 256 rows forked from 16 parents (half a page of 8 heads of 128, K and V, each):
// copies 32 us for 233 MB, plan 9, alloc and free 4 each; 796 of a pool's 1600
// pages compacted: moves 155 us, plan 7; a pool of 64 pages: 5 and 4.
#include <algorithm>

#include "fa_common.h"

namespace fa {

constexpr int kPgThreads = 1024, kPgCopyThreads = 256;
constexpr int kPgMaxRows = 1 << 18;        // rows whose bitmap fits a plan's LDS
constexpr int kPgSlice = 16 * kPgCopyThreads;  // 16-byte pieces of a page that a workgroup copies

// Exclusive sum of x over the workgroup's threads in order; total gets the sum of all.
__device__ __forceinline__ int pg_scan(int x, int &total) {
    __shared__ int part[kPgThreads / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int inc = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(inc, d);
        if (lane >= d) inc += y;
    }
    __syncthreads();  // the last call's reads are done
    if (lane == 63) part[wave] = inc;
    __syncthreads();
    int base = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kPgThreads / 64; ++w) {
        base += w < wave ? part[w] : 0;
        total += part[w];
    }
    return base + inc - x;
}

// The first `want` free pages, lowest first, to list; returns how many there are
// (the whole workgroup; a barrier follows the writes).
__device__ __forceinline__ int pg_free_pages(const fa_kvpages_args &a, int want, int32_t *list) {
    int found = 0;
    for (int p0 = 0; p0 < a.num_pages && found < want; p0 += kPgThreads) {
        const int p = p0 + threadIdx.x;
        const int is = p < a.num_pages && a.page_refs[p] == 0;
        int total;
        const int at = found + pg_scan(is, total);
        if (is && at < want) list[at] = p;
        found += total;
    }
    __syncthreads();
    return min(found, want);
}

__device__ __forceinline__ void pg_report(const fa_kvpages_args &a, int err) {
    if (threadIdx.x == 0 && a.status) atomicOr(a.status, err);
}

// Alloc: the table entries that the tokens [L, L + new) of each row need and lack.
__global__ __launch_bounds__(kPgThreads) void pg_alloc_kernel(const fa_kvpages_args a, int32_t *const list) {
    int need = 0, err = 0;
    auto row_need = [&](int r, int &first, int &last) {
        const int L = a.cache_seqlens[r], n = a.seqlens_new ? a.seqlens_new[r] : a.seqlen_new;
        first = 0;
        last = -1;
        if (L < 0 || n < 0 || int64_t(L) + n > int64_t(a.max_pages) * a.page_block_size) {
            err = 1;
            return 0;
        }
        if (n == 0) return 0;
        first = L / a.page_block_size;
        last = int((int64_t(L) + n - 1) / a.page_block_size);
        int c = 0;
        for (int j = first; j <= last; ++j) c += a.block_table[r * a.block_table_stride + j] < 0;
        return c;
    };
    int first, last, total;
    for (int r = threadIdx.x; r < a.rows; r += kPgThreads) need += row_need(r, first, last);
    if (__syncthreads_or(err)) return pg_report(a, 1);
    pg_scan(need, total);
    if (total == 0) return;
    if (pg_free_pages(a, total, list) < total) return pg_report(a, FA_KV_NO_PAGES);
    int given = 0;
    for (int r0 = 0; r0 < a.rows; r0 += kPgThreads) {
        const int r = r0 + threadIdx.x;
        first = 0;
        last = -1;
        const int c = r < a.rows ? row_need(r, first, last) : 0;
        int at = given + pg_scan(c, total);
        for (int j = first; j <= last; ++j) {
            int32_t &e = a.block_table[r * a.block_table_stride + j];
            if (e < 0) {
                const int p = list[at++];
                e = p;
                a.page_refs[p] = 1;
            }
        }
        given += total;
    }
}

// Copies pieces [piece0, piece0 + kPgSlice) of the first `tokens` tokens of page
// src to page dst, of K (which = 0) or V.  ONCE: the source is in no other copy, so
// the caches are asked to keep neither side (a pool of 1600 pages, half in use,
// compacted: 161 -> 155 us, 192 -> 168 after other work; a fork's sources, 16 children
// each, are better kept: 60 us against 73).
template <bool ONCE>
__device__ __forceinline__ void pg_copy(const fa_kvpages_args &a, int which, int64_t src, int64_t dst, int tokens,
                                        int piece0) {
    const fa_tensor &t = which ? a.v_cache : a.k_cache;
    const int per_head = a.head_bytes / 16, per_row = a.nheads_k * per_head;
    const int n = min(tokens * per_row, piece0 + kPgSlice);
    const char *s = (const char *)t.ptr + src * t.batch_stride;
    char *d = (char *)t.ptr + dst * t.batch_stride;
    const bool dense = t.head_stride == a.head_bytes && t.row_stride == int64_t(a.nheads_k) * a.head_bytes;
    auto at = [&](int i) -> int64_t {
        if (dense) return int64_t(i) * 16;
        const int row = i / per_row, x = i - row * per_row, h = x / per_head;
        return row * t.row_stride + h * t.head_stride + (x - h * per_head) * 16;
    };
    constexpr int U = 8;  // loads in flight
    for (int i = piece0 + threadIdx.x; i < n; i += U * kPgCopyThreads) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * kPgCopyThreads < n) {
                const u32x4 *p = reinterpret_cast<const u32x4 *>(s + at(i + u * kPgCopyThreads));
                v[u] = ONCE ? __builtin_nontemporal_load(p) : *p;
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * kPgCopyThreads < n) {
                u32x4 *p = reinterpret_cast<u32x4 *>(d + at(i + u * kPgCopyThreads));
                if constexpr (ONCE)
                    __builtin_nontemporal_store(v[u], p);
                else
                    *p = v[u];
            }
    }
}

// Copy: workgroup (pair, K or V, slice).  All pairs copy at once, so a pair whose
// source another writes, or whose destination is another's, is not copied.  (Every
// workgroup looks through the list for that: 500 pairs of 512 KB pages 208 us, 5.0
// TB/s; 1000 pairs of 32 KB 22 us; with 10000 such pairs it shows, 333 us, 3.9 TB/s.)
__global__ __launch_bounds__(kPgCopyThreads) void pg_copy_kernel(const fa_kvpages_args a, const int slices) {
    const int i = blockIdx.x / (2 * slices), part = blockIdx.x % (2 * slices);
    const int src = a.from[i], dst = a.to[i];
    int bad = src < 0 || src >= a.num_pages || dst < 0 || dst >= a.num_pages;
    if (src == dst && !bad) return;
    for (int j = threadIdx.x; j < a.n; j += kPgCopyThreads)
        bad |= j != i && (a.to[j] == dst || (a.from[j] != a.to[j] && (a.to[j] == src || a.from[j] == dst)));
    if (__syncthreads_or(bad)) {
        if (part == 0) pg_report(a, FA_KV_BAD_LIST);
        return;
    }
    pg_copy<false>(a, part / slices, src, dst, a.page_block_size, part % slices * kPgSlice);
}

// Fork, the plan: checks the list and gives each child whose parent's last page
// is partly filled a page; ws: [0] whether all is well, [1 + i] child i's page or
// -1, then the free pages.
__global__ __launch_bounds__(kPgThreads) void pg_fork_plan_kernel(const fa_kvpages_args a, int32_t *const ws) {
    extern __shared__ uint32_t seen[];  // a bit for each row: a child
    int32_t *fresh = ws + 1, *list = fresh + a.n;
    if (threadIdx.x == 0) ws[0] = 0;
    for (int i = threadIdx.x; i < (a.rows + 31) / 32; i += kPgThreads) seen[i] = 0;
    __syncthreads();
    int err = 0;
    for (int i = threadIdx.x; i < a.n; i += kPgThreads) {
        const int p = a.from[i], c = a.to[i];
        if (p < 0 || p >= a.rows || c < 0 || c >= a.rows) {
            err = FA_KV_BAD_LIST;
            continue;
        }
        if (atomicOr(&seen[c >> 5], 1u << (c & 31)) >> (c & 31) & 1) err = FA_KV_BAD_LIST;
        if (a.cache_seqlens[c] != 0 || (a.max_pages > 0 && a.block_table[c * a.block_table_stride] >= 0)) err = FA_KV_BAD_LIST;
        const int L = a.cache_seqlens[p];
        if (L < 0 || L > int64_t(a.max_pages) * a.page_block_size) err = FA_KV_BAD_LIST;
    }
    if (__syncthreads_or(err)) return pg_report(a, FA_KV_BAD_LIST);
    // No child is a parent, and every page that a parent uses is one of the cache: a wave a parent, once
    // for neighbours of the list that share it.
    __shared__ int parent[kPgThreads];
    for (int i0 = 0; i0 < a.n; i0 += kPgThreads) {
        const int i = i0 + threadIdx.x;
        bool other = false;
        int p = 0, parents;
        if (i < a.n) {
            p = a.from[i];
            other = i == i0 || a.from[i - 1] != p;
            if (seen[p >> 5] >> (p & 31) & 1) err = FA_KV_BAD_LIST;
        }
        const int at = pg_scan(other, parents);
        if (other) parent[at] = p;
        __syncthreads();
        for (int k = threadIdx.x >> 6; k < parents; k += kPgThreads / 64) {
            const int q = parent[k], pages = (a.cache_seqlens[q] + a.page_block_size - 1) / a.page_block_size;
            for (int j = threadIdx.x & 63; j < pages; j += 64) {
                const int e = a.block_table[q * a.block_table_stride + j];
                if (e < 0 || e >= a.num_pages) err = FA_KV_BAD_PAGE;
            }
        }
        __syncthreads();
    }
    const int bad_page = __syncthreads_or(err == FA_KV_BAD_PAGE), bad_list = __syncthreads_or(err == FA_KV_BAD_LIST);
    if (bad_page | bad_list) return pg_report(a, (bad_page ? FA_KV_BAD_PAGE : 0) | (bad_list ? FA_KV_BAD_LIST : 0));
    int want = 0, total;
    for (int i0 = 0; i0 < a.n; i0 += kPgThreads) {
        const int i = i0 + threadIdx.x;
        const int part = i < a.n && a.cache_seqlens[a.from[i]] % a.page_block_size != 0;
        const int at = want + pg_scan(part, total);
        if (i < a.n) fresh[i] = part ? at : -1;
        want += total;
    }
    if (pg_free_pages(a, want, list) < want) return pg_report(a, FA_KV_NO_PAGES);
    for (int i = threadIdx.x; i < a.n; i += kPgThreads)
        if (fresh[i] >= 0) {
            const int p = list[fresh[i]];
            fresh[i] = p;
            a.page_refs[p] = 1;
        }
    if (threadIdx.x == 0) ws[0] = 1;
}

// Fork: workgroup (child, 0): its row, its length and the shared pages' counts;
// (child, 1 + K or V and slice): the copy of the last page's tokens.
__global__ __launch_bounds__(kPgCopyThreads) void pg_fork_kernel(const fa_kvpages_args a, const int32_t *const ws,
                                                                 const int slices) {
    if (ws[0] == 0) return;
    const int i = blockIdx.x / (1 + 2 * slices), part = blockIdx.x % (1 + 2 * slices) - 1;
    const int parent = a.from[i], child = a.to[i], fresh = ws[1 + i];
    const int L = a.cache_seqlens[parent], full = L / a.page_block_size, rest = L - full * a.page_block_size;
    const int32_t *row = a.block_table + parent * a.block_table_stride;
    if (part >= 0) {
        if (fresh >= 0) pg_copy<false>(a, part / slices, row[full], fresh, rest, part % slices * kPgSlice);
        return;
    }
    int32_t *own = a.block_table + child * a.block_table_stride;
    for (int j = threadIdx.x; j < a.max_pages; j += kPgCopyThreads) {
        const int e = j < full ? row[j] : j == full ? fresh : -1;
        own[j] = e;
        if (j < full) atomicAdd(a.page_refs + e, 1);
    }
    if (threadIdx.x == 0) a.cache_seqlens[child] = L;
}

// Free: one workgroup a row.  The exchange takes each entry once, also when the
// list holds a row twice.
__global__ __launch_bounds__(kPgCopyThreads) void pg_free_kernel(const fa_kvpages_args a) {
    const int r = a.from[blockIdx.x];
    if (r < 0 || r >= a.rows) return pg_report(a, FA_KV_BAD_LIST);
    int32_t *row = a.block_table + r * a.block_table_stride;
    for (int j = threadIdx.x; j < a.max_pages; j += kPgCopyThreads) {
        const int e = atomicExch(row + j, -1);
        if (e >= 0 && e < a.num_pages) atomicSub(a.page_refs + e, 1);
    }
    if (threadIdx.x == 0) a.cache_seqlens[r] = 0;
}

// Compaction, the plan: with U pages in use, the k-th free page below U takes the
// k-th used page from U on.  ws: [0] the moves, then their sources and
// destinations (num_pages / 2 + 1 each), then each page's new place.
__global__ __launch_bounds__(kPgThreads) void pg_compact_plan_kernel(const fa_kvpages_args a, int32_t *const ws) {
    const int most = a.num_pages / 2 + 1;
    int32_t *src = ws + 1, *dst = src + most, *place = dst + most;
    int used = 0, total;
    for (int p = threadIdx.x; p < a.num_pages; p += kPgThreads) used += a.page_refs[p] > 0;
    pg_scan(used, total);
    const int U = total;
    int holes = 0, movers = 0;
    for (int p0 = 0; p0 < a.num_pages; p0 += kPgThreads) {
        const int p = p0 + threadIdx.x, refs = p < a.num_pages ? a.page_refs[p] : 0;
        const int hole = p < U && refs <= 0, mover = p >= U && p < a.num_pages && refs > 0;
        const int h = holes + pg_scan(hole, total);
        holes += total;
        const int m = movers + pg_scan(mover, total);
        movers += total;
        if (hole) dst[h] = p;
        if (mover) src[m] = p;
        if (p < a.num_pages) {
            place[p] = p;
            a.out_refs[p] = mover ? 0 : refs;
        }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < movers; k += kPgThreads) {
        place[src[k]] = dst[k];
        a.out_refs[dst[k]] = a.page_refs[src[k]];
    }
    if (threadIdx.x == 0) {
        ws[0] = movers;
        a.out_used[0] = U;
    }
}

// Compaction: the first table_wgs workgroups write the new table, the others
// take the moves' slices.  Sources lie from U on, destinations below, so no move
// reads what another writes.
__global__ __launch_bounds__(kPgCopyThreads) void pg_compact_kernel(const fa_kvpages_args a, const int32_t *const ws,
                                                                    const int slices, const int table_wgs) {
    const int most = a.num_pages / 2 + 1;
    const int32_t *src = ws + 1, *dst = src + most, *place = dst + most;
    if (int(blockIdx.x) < table_wgs) {
        const int64_t n = int64_t(a.rows) * a.max_pages;
        for (int64_t i = int64_t(blockIdx.x) * kPgCopyThreads + threadIdx.x; i < n; i += int64_t(table_wgs) * kPgCopyThreads) {
            const int64_t r = i / a.max_pages, j = i - r * a.max_pages;
            const int e = a.block_table[r * a.block_table_stride + j];
            a.out_table[r * a.out_table_stride + j] = e >= 0 && e < a.num_pages ? place[e] : e;
        }
        return;
    }
    const int64_t n = int64_t(ws[0]) * 2 * slices;
    for (int64_t w = blockIdx.x - table_wgs; w < n; w += gridDim.x - table_wgs) {
        const int k = int(w / (2 * slices)), part = int(w - int64_t(k) * 2 * slices);
        pg_copy<true>(a, part / slices, src[k], dst[k], a.page_block_size, part % slices * kPgSlice);
    }
}

static bool pg_cache_ok(const fa_tensor &t) {
    return t.ptr && !((reinterpret_cast<uintptr_t>(t.ptr) | uint64_t(t.batch_stride) | uint64_t(t.row_stride) |
                       uint64_t(t.head_stride)) & 15u);
}
// cache: the call moves pages; table: it has rows; n: a list of that many entries.
static int pg_check(const fa_kvpages_args *p, bool cache, bool table, int lists) {
    if (!p) return FA_ERR_INVALID_ARG;
    const fa_kvpages_args &a = *p;
    if (a.num_pages < 0 || a.page_block_size <= 0 || a.rows < 0 || a.max_pages < 0 || a.n < 0) return FA_ERR_INVALID_ARG;
    if (cache && (a.nheads_k <= 0 || a.head_bytes <= 0 || a.head_bytes % 16 || !pg_cache_ok(a.k_cache) || !pg_cache_ok(a.v_cache) ||
                  int64_t(a.page_block_size) * a.nheads_k * (a.head_bytes / 16) > INT32_MAX / 2))
        return FA_ERR_INVALID_ARG;
    if (table && (!a.block_table || !a.page_refs)) return FA_ERR_INVALID_ARG;
    if (a.n > 0 && ((lists >= 1 && !a.from) || (lists >= 2 && !a.to))) return FA_ERR_INVALID_ARG;
    return FA_OK;
}
static int pg_slices(const fa_kvpages_args &a) {
    const int64_t pieces = int64_t(a.page_block_size) * a.nheads_k * (a.head_bytes / 16);
    return int((pieces + kPgSlice - 1) / kPgSlice);
}
static int pg_workspace(const fa_kvpages_args &a, int64_t bytes) {
    return !a.ws || a.ws_bytes < bytes || (reinterpret_cast<uintptr_t>(a.ws) & 3u) ? FA_ERR_WORKSPACE : FA_OK;
}

}  // namespace fa

extern "C" size_t fa_kvpages_ws_bytes(const fa_kvpages_args *a) {
    if (!a || a->num_pages < 0 || a->n < 0) return 0;
    // alloc: a list of free pages; fork: 1 + 2 n; compaction: 1 + 2 (num_pages / 2 + 1) + num_pages.
    return 4 * (size_t(3) + 2 * size_t(a->num_pages) + 2 * size_t(a->n));
}

extern "C" int fa_kvpages_alloc(const fa_kvpages_args *args, void *stream) {
    using namespace fa;
    int rc = pg_check(args, false, true, 0);
    if (rc) return rc;
    const fa_kvpages_args &a = *args;
    if (!a.cache_seqlens || a.seqlen_new < 0) return FA_ERR_INVALID_ARG;
    if ((rc = pg_workspace(a, 4 * int64_t(a.num_pages)))) return rc;
    if (a.rows == 0) return FA_OK;
    hipLaunchKernelGGL(pg_alloc_kernel, dim3(1), dim3(kPgThreads), 0, reinterpret_cast<hipStream_t>(stream), a,
                       static_cast<int32_t *>(a.ws));
    return int(hipGetLastError());
}

extern "C" int fa_kvpages_copy(const fa_kvpages_args *args, void *stream) {
    using namespace fa;
    const int rc = pg_check(args, true, false, 2);
    if (rc) return rc;
    const fa_kvpages_args &a = *args;
    if (a.n == 0) return FA_OK;
    const int64_t grid = int64_t(a.n) * 2 * pg_slices(a);
    if (grid > 0x7fffffff) return FA_ERR_INVALID_ARG;
    hipLaunchKernelGGL(pg_copy_kernel, dim3(unsigned(grid)), dim3(kPgCopyThreads), 0,
                       reinterpret_cast<hipStream_t>(stream), a, pg_slices(a));
    return int(hipGetLastError());
}

extern "C" int fa_kvpages_fork(const fa_kvpages_args *args, void *stream) {
    using namespace fa;
    int rc = pg_check(args, true, true, 2);
    if (rc) return rc;
    const fa_kvpages_args &a = *args;
    if (!a.cache_seqlens) return FA_ERR_INVALID_ARG;
    if (a.rows > kPgMaxRows) return FA_ERR_INVALID_ARG;
    if ((rc = pg_workspace(a, 4 * (1 + 2 * int64_t(a.n))))) return rc;
    if (a.n == 0) return FA_OK;
    const int64_t grid = int64_t(a.n) * (1 + 2 * pg_slices(a));
    if (grid > 0x7fffffff) return FA_ERR_INVALID_ARG;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    int32_t *ws = static_cast<int32_t *>(a.ws);
    hipLaunchKernelGGL(pg_fork_plan_kernel, dim3(1), dim3(kPgThreads), size_t((a.rows + 31) / 32) * 4, s, a, ws);
    if ((rc = int(hipGetLastError()))) return rc;
    hipLaunchKernelGGL(pg_fork_kernel, dim3(unsigned(grid)), dim3(kPgCopyThreads), 0, s, a, ws, pg_slices(a));
    return int(hipGetLastError());
}

extern "C" int fa_kvpages_free(const fa_kvpages_args *args, void *stream) {
    using namespace fa;
    const int rc = pg_check(args, false, true, 1);
    if (rc) return rc;
    const fa_kvpages_args &a = *args;
    if (!a.cache_seqlens) return FA_ERR_INVALID_ARG;
    if (a.n == 0) return FA_OK;
    hipLaunchKernelGGL(pg_free_kernel, dim3(a.n), dim3(kPgCopyThreads), 0, reinterpret_cast<hipStream_t>(stream), a);
    return int(hipGetLastError());
}

extern "C" int fa_kvpages_compact(const fa_kvpages_args *args, void *stream) {
    using namespace fa;
    int rc = pg_check(args, true, true, 0);
    if (rc) return rc;
    const fa_kvpages_args &a = *args;
    if (!a.out_table || !a.out_refs || !a.out_used || a.out_table == a.block_table || a.out_refs == a.page_refs)
        return FA_ERR_INVALID_ARG;
    if ((rc = pg_workspace(a, 4 * (3 + 2 * int64_t(a.num_pages))))) return rc;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    int32_t *ws = static_cast<int32_t *>(a.ws);
    hipLaunchKernelGGL(pg_compact_plan_kernel, dim3(1), dim3(kPgThreads), 0, s, a, ws);
    if ((rc = int(hipGetLastError()))) return rc;
    const int64_t entries = int64_t(a.rows) * a.max_pages;
    const int table_wgs = int(std::min<int64_t>((entries + kPgCopyThreads - 1) / kPgCopyThreads, 256));
    const int64_t most = int64_t(a.num_pages / 2) * 2 * pg_slices(a);
    const int move_wgs = int(std::max<int64_t>(std::min<int64_t>(most, 8 * device_cus()), 1));
    hipLaunchKernelGGL(pg_compact_kernel, dim3(unsigned(table_wgs + move_wgs)), dim3(kPgCopyThreads), 0, s, a, ws,
                       pg_slices(a), table_wgs);
    return int(hipGetLastError());
}
