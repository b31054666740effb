/*
 * g4s_pages.hip -- the pages of a cache that beams share: one step of the
 * tables (fork, reorder, append, truncate, end), compaction, and page copies,
 * on gfx950.
 *
 * A state names each row's pages in a table and counts the rows that hold a
 * page.  A step reads one state and writes another: the new tables gather
 * their parents' rows, the new counts are counted over them, and free pages are
 * the ones that the old state does not hold.  Counts are integer atomics, so
 * their order does not show; pages are handed out in order of page, row and
 * slot, so results do not depend on it either.
 */
#include "g4s_pages.h"

#include <limits.h>

#include "g4s_device.h"

namespace g4s {

namespace {

constexpr int kB = 256;
constexpr int kCopyItems = 4; /* vectors per thread in flight */

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

/* ------------------------------------------------------------------- scans */

/* Per block of 1024 pages: its free pages counted, its live and free pages listed. */
__global__ __launch_bounds__(kB) void pages_scan_kernel(PagesArgs a)
{
    __shared__ int s_wave[kB / 64];
    const int tid = threadIdx.x, blk = blockIdx.x;
    if (blk == 0 && tid == 0) *a.ws.plan = PagePlan{};
    int live[4], in[4], mine = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int p = blk * kPageBlock + tid * 4 + q;
        in[q] = p < a.geo.n_pages;
        live[q] = in[q] && a.from.refs[p] > 0;
        mine += live[q];
    }
    int total;
    int at = block_exclusive_scan<kB>(mine, s_wave, total);
    int held = a.geo.n_pages - blk * kPageBlock;
    held = held < kPageBlock ? held : kPageBlock;
    uint16_t* list = a.ws.list + blk * kPageBlock;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int l = tid * 4 + q;
        if (!in[q]) continue;
        const int r = live[q] ? at : l - at;
        list[live[q] ? r : kPageBlock - 1 - r] = (uint16_t)l;
        a.ws.rank[blk * kPageBlock + l] = (uint16_t)r;
        at += live[q];
    }
    if (tid == 0) a.ws.nfree[blk] = held - total;
}

/* Free pages before each block, in global memory; returns how many there are. */
__device__ int scan_blocks(const PagesArgs& a, int* s_wave)
{
    int base = 0;
    for (int b0 = 0; b0 < a.blocks; b0 += kB) {
        const int b = b0 + (int)threadIdx.x;
        const int f = b < a.blocks ? a.ws.nfree[b] : 0;
        int total;
        const int pre = block_exclusive_scan<kB>(f, s_wave, total);
        if (b < a.blocks) a.ws.before[b] = base + pre;
        base += total;
    }
    if (threadIdx.x == 0) a.ws.before[a.blocks] = base;
    __syncthreads();
    return base;
}

/* The i-th free page (0 <= i < free pages), and the i-th live one. */
__device__ __forceinline__ int free_page(const PagesArgs& a, int i)
{
    int lo = 0, hi = a.blocks - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.ws.before[mid] <= i)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo * kPageBlock + a.ws.list[lo * kPageBlock + kPageBlock - 1 - (i - a.ws.before[lo])];
}
__device__ __forceinline__ int live_before(const PagesArgs& a, int blk)
{
    return blk * kPageBlock - a.ws.before[blk];
}
__device__ __forceinline__ int live_page(const PagesArgs& a, int i)
{
    int lo = 0, hi = a.blocks - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (live_before(a, mid) <= i)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo * kPageBlock + a.ws.list[lo * kPageBlock + i - live_before(a, lo)];
}

__device__ __forceinline__ void report(const PagesArgs& a, int code)
{
    atomicMin(&a.ws.plan->code, code);
}

/* A table entry is a page of the pool that the state holds. */
__device__ __forceinline__ bool page_ok(const PagesArgs& a, int p)
{
    return p >= 0 && p < a.geo.n_pages && a.from.refs[p] > 0;
}

__device__ __forceinline__ RowStep step_of(const PagesArgs& a, int r, int& parent)
{
    parent = a.parents[r];
    const int len = parent >= 0 && parent < a.from_rows ? a.from.lengths[parent] : 0;
    return row_step(parent, a.from_rows, len, a.grow ? a.grow[r] : 0, a.geo.page_tokens,
                    a.geo.max_slots);
}

/* ----------------------------------------------------------------- advance */

/* Tables gathered from the parents' rows, their pages counted. */
__global__ __launch_bounds__(kB) void pages_gather_kernel(PagesArgs a)
{
    const int r = blockIdx.y;
    const int slot = blockIdx.x * kB + threadIdx.x;
    int parent;
    const RowStep s = step_of(a, r, parent);
    bool fresh = false;
    if (slot < s.kept) {
        const int p = a.from.table[(int64_t)parent * a.geo.max_slots + slot];
        if (page_ok(a, p)) {
            a.to.table[(int64_t)r * a.geo.max_slots + slot] = p;
            fresh = atomicAdd(&a.ws.count[p], 1u) == 0u;
        } else {
            report(a, G4S_ERR_FORMAT);
        }
    }
    const int n = __popcll(__ballot(fresh));
    if ((threadIdx.x & 63) == 0 && n) atomicAdd(&a.ws.plan->distinct, n);
    if (s.bad && slot == 0) report(a, G4S_ERR_INVALID_ARGUMENT);
}

/* The page that row r goes on writing, or -1. */
__device__ __forceinline__ int written_page(const PagesArgs& a, const RowStep& s, int parent)
{
    if (s.tail == 0) return -1;
    const int p = a.from.table[(int64_t)parent * a.geo.max_slots + s.kept - 1];
    return page_ok(a, p) ? p : -1;
}

/* One workgroup: which rows copy the page they write, what each row takes, and who gets
 * which free page. */
__global__ __launch_bounds__(kB) void pages_plan_kernel(PagesArgs a)
{
    __shared__ int s_wave[kB / 64];
    __shared__ int before[G4S_PAGES_MAX_ROWS + 1]; /* pages taken before row r */
    __shared__ int kept[G4S_PAGES_MAX_ROWS];       /* its kept slots * 2 + whether it copies */
    __shared__ int s_code;
    const int tid = threadIdx.x;
    const int nfree = scan_blocks(a, s_wave);
    for (int r = tid; r < a.rows; r += kB) {
        int parent;
        const RowStep s = step_of(a, r, parent);
        const int w = written_page(a, s, parent);
        if (w >= 0) {
            atomicAdd(&a.ws.writers[w], 1u);
            atomicMin(&a.ws.first[w], r);
        }
    }
    __threadfence();
    __syncthreads();
    int64_t taken = 0;
    int copies = 0;
    for (int r0 = 0; r0 < a.rows; r0 += kB) {
        const int r = r0 + tid;
        int need = 0, copy = 0, total;
        if (r < a.rows) {
            int parent;
            const RowStep s = step_of(a, r, parent);
            const int w = written_page(a, s, parent);
            if (w >= 0)
                copy = !(ld_dev(&a.ws.count[w]) == ld_dev(&a.ws.writers[w]) &&
                         (int)ld_dev((const uint32_t*)&a.ws.first[w]) == r);
            need = s.fresh + copy;
            kept[r] = s.kept * 2 + copy;
        }
        const int pre = block_exclusive_scan<kB>(need, s_wave, total);
        if (r < a.rows) before[r] = (int)(taken + pre < INT_MAX ? taken + pre : INT_MAX);
        taken += total;
        block_exclusive_scan<kB>(copy, s_wave, total);
        copies += total;
    }
    if (tid == 0) before[a.rows] = (int)(taken < INT_MAX ? taken : INT_MAX);
    if (tid == 0) {
        int code = (int)ld_dev((const uint32_t*)&a.ws.plan->code);
        if (code == G4S_OK && taken > nfree) code = G4S_ERR_OUT_OF_MEMORY;
        s_code = code;
        a.status[0] = code;
        a.status[1] = code ? a.geo.n_pages
                           : a.geo.n_pages - (int)ld_dev((const uint32_t*)&a.ws.plan->distinct) -
                                 (int)taken;
        a.status[2] = code ? 0 : (int)taken;
        a.status[3] = code ? 0 : copies;
        a.ws.plan->code = code;
        a.ws.plan->jobs = code ? 0 : copies;
    }
    __syncthreads();
    const int code = s_code;
    int job = 0;
    for (int r0 = 0; r0 < a.rows; r0 += kB) {
        const int r = r0 + tid;
        int copy = 0, total, w = -1, tail = 0;
        if (r < a.rows) {
            int parent;
            const RowStep s = step_of(a, r, parent);
            w = written_page(a, s, parent);
            tail = s.tail;
            if (w >= 0) {
                a.ws.writers[w] = 0u;
                a.ws.first[w] = INT_MAX;
            }
            a.to.lengths[r] = code ? 0 : (int)s.length;
            copy = code ? 0 : kept[r] & 1;
        }
        const int at = job + block_exclusive_scan<kB>(copy, s_wave, total);
        if (copy) {
            atomicSub(&a.ws.count[w], 1u);
            a.ws.jobs[at] = PageJob{w, free_page(a, before[r]), tail};
        }
        job += total;
    }
    if (code) return;
    for (int k = tid; k < (int)taken; k += kB) {
        int lo = 0, hi = a.rows - 1; /* the row that takes free page k */
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (before[mid] <= k)
                lo = mid;
            else
                hi = mid - 1;
        }
        const int p = free_page(a, k);
        const int slot = (kept[lo] >> 1) - (kept[lo] & 1) + (k - before[lo]);
        a.to.table[(int64_t)lo * a.geo.max_slots + slot] = p;
        atomicAdd(&a.ws.count[p], 1u);
    }
}

/* ------------------------------------------------------------------ copies */

/* Segment `seg` (256 x kCopyItems vectors) of the first `tokens` tokens of a
 * page in one plane. */
template <typename T>
__device__ __forceinline__ void copy_segment(const g4s_page_geometry& g, const char* src, char* dst,
                                             int plane, int seg, const PageJob& job)
{
    const uint32_t per_part = (uint32_t)((int64_t)job.tokens * g.token_bytes / (int64_t)sizeof(T));
    const uint32_t total = per_part * (uint32_t)g.parts;
    const uint32_t i0 = (uint32_t)seg * (kB * kCopyItems) + threadIdx.x;
    T v[kCopyItems];
    int64_t off[kCopyItems];
#pragma unroll
    for (int q = 0; q < kCopyItems; ++q) {
        const uint32_t i = i0 + q * kB;
        if (i < total) {
            off[q] = page_offset(g, 0, 0, i, per_part, sizeof(T));
            v[q] = *reinterpret_cast<const T*>(src + page_offset(g, plane, job.src, 0, 1, 0) + off[q]);
        }
    }
#pragma unroll
    for (int q = 0; q < kCopyItems; ++q) {
        const uint32_t i = i0 + q * kB;
        if (i < total)
            __builtin_nontemporal_store(
                v[q], reinterpret_cast<T*>(dst + page_offset(g, plane, job.dst, 0, 1, 0) + off[q]));
    }
}

template <typename T>
__host__ __device__ inline int copy_segments(const g4s_page_geometry& g)
{
    const int64_t n = (int64_t)g.parts * g.page_tokens * g.token_bytes / (int64_t)sizeof(T);
    return (int)((n + kB * kCopyItems - 1) / (kB * kCopyItems));
}

template <typename T, typename JobF>
__device__ void copy_all(const g4s_page_geometry& g, const char* src, char* dst, int jobs, JobF job)
{
    const int segs = copy_segments<T>(g);
    const int64_t units = (int64_t)jobs * g.planes * segs;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int64_t pj = u / segs;
        const int plane = (int)(pj / jobs);
        copy_segment<T>(g, src, dst, plane, (int)(u - pj * segs), job((int)(pj - (int64_t)plane * jobs)));
    }
}

/* The new counts, and the copies. */
template <typename T>
__global__ __launch_bounds__(kB) void pages_finish_kernel(PagesArgs a)
{
    const bool ok = a.ws.plan->code == G4S_OK;
    for (int p = blockIdx.x * kB + threadIdx.x; p < a.geo.n_pages; p += gridDim.x * kB) {
        a.to.refs[p] = ok ? (int32_t)a.ws.count[p] : 0;
        a.ws.count[p] = 0u;
    }
    copy_all<T>(a.geo, a.pool, a.pool, a.ws.plan->jobs, [&](int j) { return a.ws.jobs[j]; });
}

template <typename T>
__global__ __launch_bounds__(kB) void pages_copy_kernel(g4s_page_geometry g, const char* src,
                                                        char* dst, int n, const int32_t* d_src,
                                                        const int32_t* d_dst,
                                                        const int32_t* d_tokens)
{
    copy_all<T>(g, src, dst, n, [&](int j) {
        PageJob job{d_src[j], d_dst[j], d_tokens ? d_tokens[j] : g.page_tokens};
        const bool in = job.src >= 0 && job.src < g.n_pages && job.dst >= 0 && job.dst < g.n_pages;
        if (!in || job.tokens < 0) job.tokens = 0;
        if (job.tokens > g.page_tokens) job.tokens = g.page_tokens;
        return job;
    });
}

/* ----------------------------------------------------------------- compact */

/* Tables and lengths are valid: nothing is written before that is known. */
__global__ __launch_bounds__(kB) void pages_check_kernel(PagesArgs a)
{
    const int r = blockIdx.y;
    const int slot = blockIdx.x * kB + threadIdx.x;
    const RowStep s = row_step(r, a.rows, a.from.lengths[r], 0, a.geo.page_tokens, a.geo.max_slots);
    if (s.bad && slot == 0) report(a, G4S_ERR_INVALID_ARGUMENT);
    if (slot < s.kept && !page_ok(a, a.from.table[(int64_t)r * a.geo.max_slots + slot]))
        report(a, G4S_ERR_FORMAT);
}

__global__ __launch_bounds__(kB) void pages_compact_plan_kernel(PagesArgs a)
{
    __shared__ int s_wave[kB / 64];
    const int tid = threadIdx.x;
    const int nfree = scan_blocks(a, s_wave);
    const int live = a.geo.n_pages - nfree;
    const int code = (int)ld_dev((const uint32_t*)&a.ws.plan->code);
    /* live pages below `live`: whole blocks, then the one it falls into */
    const int blk = live / kPageBlock;
    int mine = 0;
    for (int p = blk * kPageBlock + tid; p < live; p += kB) mine += a.from.refs[p] > 0;
    mine = block_sum_i32<kB>(mine, s_wave);
    if (tid == 0) {
        const int below = (blk < a.blocks ? live_before(a, blk) : live) + mine;
        a.ws.plan->live = live;
        a.ws.plan->below = below;
        a.ws.plan->jobs = code ? 0 : live - below;
        a.status[0] = code;
        a.status[1] = code ? a.geo.n_pages : nfree;
        a.status[2] = 0;
        a.status[3] = code ? 0 : live - below;
    }
}

template <typename T>
__global__ __launch_bounds__(kB) void pages_compact_kernel(PagesArgs a)
{
    const PagePlan plan = *a.ws.plan;
    const bool ok = plan.code == G4S_OK;
    const int at = blockIdx.x * kB + threadIdx.x, step = gridDim.x * kB;
    for (int p = at; p < a.geo.n_pages; p += step) {
        int refs = 0;
        if (ok && p < plan.live) {
            refs = a.from.refs[p];
            if (refs <= 0)
                refs = a.from.refs[live_page(
                    a, plan.below + a.ws.before[p / kPageBlock] + a.ws.rank[p])];
        }
        a.to.refs[p] = refs;
    }
    for (int r = at; r < a.rows; r += step) a.to.lengths[r] = ok ? a.from.lengths[r] : 0;
    const int64_t S = a.geo.max_slots, cells = ok ? a.rows * S : 0;
    for (int64_t c = at; c < cells; c += step) {
        const int r = (int)(c / S);
        const int used = (a.from.lengths[r] + a.geo.page_tokens - 1) / a.geo.page_tokens;
        if (c - r * S >= used) continue;
        int p = a.from.table[c];
        if (p >= plan.live)
            p = free_page(a, live_before(a, p / kPageBlock) + a.ws.rank[p] - plan.below);
        a.to.table[c] = p;
    }
    copy_all<T>(a.geo, a.pool, a.pool, plan.jobs, [&](int j) {
        return PageJob{live_page(a, plan.below + j), free_page(a, j), a.geo.page_tokens};
    });
}

__global__ __launch_bounds__(kB) void pages_init_kernel(PageWorkspace ws, int n)
{
    for (int p = blockIdx.x * kB + threadIdx.x; p < n; p += gridDim.x * kB) {
        ws.count[p] = 0u;
        ws.writers[p] = 0u;
        ws.first[p] = INT_MAX;
    }
}

/* Widest vectors that every address of a copy is a multiple of. */
uint64_t copy_bits(const g4s_page_geometry& g, const void* src, const void* dst)
{
    return (uint64_t)(uintptr_t)src | (uint64_t)(uintptr_t)dst | (uint64_t)g.token_bytes |
           (uint64_t)g.plane_stride | (uint64_t)g.page_stride;
}

constexpr int kMaxGrid = 1 << 20;

template <typename T>
unsigned copy_grid(const g4s_page_geometry& g, int64_t jobs, int64_t other)
{
    const int64_t units = jobs * g.planes * copy_segments<T>(g);
    const int64_t want = units > other ? units : other;
    return (unsigned)(want < 1 ? 1 : want > kMaxGrid ? kMaxGrid : want);
}

}  // namespace

hipError_t pages_init_launch(const PageWorkspace& ws, int32_t n_pages, hipStream_t stream)
{
    pages_init_kernel<<<256, kB, 0, stream>>>(ws, n_pages);
    return hipGetLastError();
}

#define G4S_BY_WIDTH(bits, CALL)    \
    do {                            \
        if (((bits) & 15) == 0)     \
            CALL(u32x4);            \
        else if (((bits) & 3) == 0) \
            CALL(uint32_t);         \
        else                        \
            CALL(uint8_t);          \
    } while (0)

hipError_t pages_advance_launch(const PagesArgs& a, hipStream_t stream)
{
    const dim3 cells((unsigned)((a.geo.max_slots + kB - 1) / kB), (unsigned)a.rows);
    pages_scan_kernel<<<(unsigned)a.blocks, kB, 0, stream>>>(a);
    pages_gather_kernel<<<cells, kB, 0, stream>>>(a);
    pages_plan_kernel<<<1, kB, 0, stream>>>(a);
    const int64_t other = (a.geo.n_pages + kB - 1) / kB;
#define G4S_CALL(T) \
    pages_finish_kernel<T><<<copy_grid<T>(a.geo, a.rows, other), kB, 0, stream>>>(a)
    G4S_BY_WIDTH(copy_bits(a.geo, a.pool, a.pool), G4S_CALL);
#undef G4S_CALL
    return hipGetLastError();
}

hipError_t pages_compact_launch(const PagesArgs& a, hipStream_t stream)
{
    const dim3 cells((unsigned)((a.geo.max_slots + kB - 1) / kB), (unsigned)a.rows);
    pages_scan_kernel<<<(unsigned)a.blocks, kB, 0, stream>>>(a);
    pages_check_kernel<<<cells, kB, 0, stream>>>(a);
    pages_compact_plan_kernel<<<1, kB, 0, stream>>>(a);
    const int64_t cell = (int64_t)a.rows * a.geo.max_slots;
    const int64_t other = ((cell > a.geo.n_pages ? cell : a.geo.n_pages) + kB - 1) / kB;
#define G4S_CALL(T) \
    pages_compact_kernel<T><<<copy_grid<T>(a.geo, a.geo.n_pages / 2, other), kB, 0, stream>>>(a)
    G4S_BY_WIDTH(copy_bits(a.geo, a.pool, a.pool), G4S_CALL);
#undef G4S_CALL
    return hipGetLastError();
}

hipError_t pages_copy_launch(const g4s_page_geometry& geo, const char* src, char* dst, int32_t n,
                             const int32_t* d_src, const int32_t* d_dst, const int32_t* d_tokens,
                             hipStream_t stream)
{
#define G4S_CALL(T)                                                                     \
    pages_copy_kernel<T><<<copy_grid<T>(geo, n, 1), kB, 0, stream>>>(geo, src, dst, n, d_src, \
                                                                     d_dst, d_tokens)
    G4S_BY_WIDTH(copy_bits(geo, src, dst), G4S_CALL);
#undef G4S_CALL
    return hipGetLastError();
}

}  // namespace g4s
