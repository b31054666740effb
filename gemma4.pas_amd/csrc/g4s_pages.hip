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
#include "g4s_launch.h"

namespace g4s {

namespace {

constexpr int kB = 256;
constexpr int kCopyItems = 4; /* vectors per thread in flight */

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

/* ------------------------------------------------------- tables and counts */

constexpr int kScanPages = 4 * kB; /* pages of a scanning workgroup */
constexpr int kGatherRows = 4;     /* rows of a gathering one, 256 slots of each */

__host__ __device__ inline int scan_groups(int n_pages)
{
    return (n_pages + kScanPages - 1) / kScanPages;
}
__host__ __device__ inline int slot_groups(int slots) { return (slots + kB - 1) / kB; }

/* The free pages of kScanPages pages, as bits. */
__device__ __forceinline__ void scan_pages(const PagesArgs& a, int group)
{
#pragma unroll
    for (int q = 0; q < kScanPages / kB; ++q) {
        const int p = group * kScanPages + q * kB + (int)threadIdx.x;
        const bool in = p < a.geo.n_pages;
        const uint64_t w = __ballot(in && a.from.refs[in ? p : 0] <= 0);
        if ((threadIdx.x & 63) == 0 && in) st_dev(&a.ws.free[p / 64], w);
    }
}

__device__ __forceinline__ void report(const PagesArgs& a, int code)
{
    atomicMin(&a.ws.plan->bad, code);
}

/* kGatherRows rows of the new tables, 256 slots of each, gathered from
 * their parents' rows, and their pages counted: neighbouring rows that share
 * a page count it at once.  CHECK: nothing but whether the tables are valid. */
template <bool CHECK>
__device__ __forceinline__ void gather_rows(const PagesArgs& a, int group)
{
    const int across = slot_groups(a.geo.max_slots);
    const int r0 = group / across * kGatherRows;
    const int slot = group % across * kB + (int)threadIdx.x;
    /* in stages, each loading for all the rows at once (from a valid place where a row has
     * nothing to load): row by row the loads would wait for each other */
    int parent[kGatherRows], grow[kGatherRows], length[kGatherRows], page[kGatherRows];
    int held[kGatherRows];
    RowStep step[kGatherRows];
#pragma unroll
    for (int q = 0; q < kGatherRows; ++q) {
        const int r = r0 + q < a.rows ? r0 + q : r0;
        parent[q] = a.parents ? a.parents[r] : r;
        grow[q] = a.grow ? a.grow[r] : 0;
    }
#pragma unroll
    for (int q = 0; q < kGatherRows; ++q)
        length[q] =
            a.from.lengths[parent[q] >= 0 && parent[q] < a.from_rows ? parent[q] : 0];
#pragma unroll
    for (int q = 0; q < kGatherRows; ++q) {
        step[q] = row_step(parent[q], a.from_rows, length[q], grow[q], a.geo.page_tokens,
                           a.geo.max_slots);
        const bool in = slot < step[q].kept;
        page[q] = a.from.table[in ? (int64_t)parent[q] * a.geo.max_slots + slot : 0];
    }
#pragma unroll
    for (int q = 0; q < kGatherRows; ++q)
        held[q] = a.from.refs[page[q] >= 0 && page[q] < a.geo.n_pages ? page[q] : 0];
    bool ours[kGatherRows]; /* the slot of a page that the row goes on writing is
                               the deciding workgroup's to write, alone: nothing orders plain
                               stores of two XCDs to one word within a launch */
#pragma unroll
    for (int q = 0; q < kGatherRows; ++q) {
        const bool in = r0 + q < a.rows && slot < step[q].kept;
        /* a table entry is a page of the pool that the state holds */
        const bool ok = page[q] >= 0 && page[q] < a.geo.n_pages && held[q] > 0;
        if (in && !ok) report(a, G4S_ERR_FORMAT);
        if (r0 + q < a.rows && step[q].bad && slot == 0) report(a, G4S_ERR_INVALID_ARGUMENT);
        page[q] = in && ok ? page[q] : -1;
        ours[q] = step[q].tail == 0 || slot != step[q].kept - 1;
        if (CHECK) continue;
        /* the row's step for the workgroup that decides, by the thread that holds
         * its last kept slot: one read there instead of four that depend on each other */
        if (r0 + q < a.rows && slot == (step[q].kept > 0 ? step[q].kept - 1 : 0)) {
            const int64_t r = r0 + q;
            st_dev(&a.ws.steps[3 * r],
                   (uint64_t)(uint32_t)step[q].fresh << 32 | (uint32_t)step[q].kept);
            st_dev(&a.ws.steps[3 * r + 1],
                   (uint64_t)(uint32_t)step[q].tail << 32 |
                       (uint32_t)(step[q].tail ? page[q] : -1));
            st_dev(&a.ws.steps[3 * r + 2], (uint64_t)step[q].length);
        }
    }
    if (CHECK) return;
    uint32_t fresh = 0, run = 0;
#pragma unroll
    for (int q = 0; q < kGatherRows; ++q) {
        if (page[q] >= 0 && ours[q])
            a.to.table[(int64_t)(r0 + q) * a.geo.max_slots + slot] = page[q];
        ++run;
        if (q + 1 == kGatherRows || page[q + 1] != page[q]) {
            if (page[q] >= 0) fresh += atomicAdd(&a.ws.count[page[q]], run) == 0u;
            run = 0;
        }
    }
    const int n = wave_sum_i32((int)fresh);
    if ((threadIdx.x & 63) == 0 && n) atomicAdd(&a.ws.plan->distinct, (uint32_t)n);
}

/* Free pages before this thread's share of the words, shares in thread order. */
struct FreeShare {
    int words, first; /* words of a share, and this thread's first */
    int before, total;
};
__device__ __forceinline__ FreeShare share_free(const PagesArgs& a, int* s_wave)
{
    FreeShare f;
    f.words = (a.words + kB - 1) / kB;
    f.first = f.words * (int)threadIdx.x;
    int n = 0;
    for (int w = 0; w < f.words; ++w)
        if (f.first + w < a.words) n += __popcll(ld_dev(&a.ws.free[f.first + w]));
    f.before = block_exclusive_scan<kB>(n, s_wave, f.total);
    return f;
}

/* The i-th set bit of w (0 <= i < its bits). */
__device__ __forceinline__ int nth_bit(uint64_t w, int i)
{
    int at = 0;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        const int n = __popcll(w & (((uint64_t)1 << d) - 1));
        if (i >= n) {
            i -= n;
            w >>= d;
            at += d;
        }
    }
    return at;
}

/* ----------------------------------------------------------------- advance */

/* Rows that go on writing one page, by page, in LDS: open addressing over twice the rows. */
struct Writers {
    int* page;  /* -1 = empty */
    int* rows;
    int* first;
    uint32_t mask;
};
__device__ __forceinline__ uint32_t find_writer(const Writers& t, int page, bool add)
{
    uint32_t at = (uint32_t)page * 2654435761u >> 7 & t.mask;
    for (;;) {
        const int k = add ? atomicCAS(&t.page[at], -1, page) : t.page[at];
        if (k == page || (add && k == -1)) return at;
        at = (at + 1) & t.mask;
    }
}

__host__ __device__ inline uint32_t writer_slots(int rows)
{
    uint32_t n = 64;
    while (n < 2u * (uint32_t)rows) n <<= 1;
    return n;
}
/* LDS words of the plan: four a row and one, three a slot of the writers. */
__host__ __device__ inline size_t plan_lds(int rows)
{
    return sizeof(int) * (4 * (size_t)rows + 1 + 3 * (size_t)writer_slots(rows));
}

/* A row's step as gather_rows left it, and how many rows hold the page it writes. */
struct RowRecord {
    int kept, fresh, page, tail, length, holders;
};
__device__ __forceinline__ RowRecord read_row(const PagesArgs& a, int r)
{
    const uint64_t slots = ld_dev(&a.ws.steps[3 * r]);
    const uint64_t written = ld_dev(&a.ws.steps[3 * r + 1]);
    const uint64_t length = ld_dev(&a.ws.steps[3 * r + 2]);
    RowRecord s{(int)(uint32_t)slots, (int)(slots >> 32), (int)(uint32_t)written,
                (int)(written >> 32), (int)length, 0};
    if (s.page >= 0) s.holders = (int)ld_dev(&a.ws.count[s.page]);
    return s;
}

/* Scan and gather, all side by side; the workgroup that ends last then decides
 * which rows copy the page they write, what each row takes, and who gets
 * which free page.  Bound by the chain of reads that each depend on the last (parent, length,
 * page, count): 8 us for one sequence of four beams, half of them the
 * gathering, 11 us for 192 rows of some 125 pages; three launches for the same took
 * 12 and 18. */
__global__ __launch_bounds__(kB) void pages_advance_kernel(PagesArgs a)
{
    extern __shared__ int lds[];
    __shared__ int s_wave[kB / 64];
    __shared__ int s_share[kB + 1]; /* free pages before each thread's share */
    __shared__ int s_flag, s_code;
    const int tid = threadIdx.x;
    const int scans = scan_groups(a.geo.n_pages);
    if ((int)blockIdx.x < scans)
        scan_pages(a, blockIdx.x);
    else
        gather_rows<false>(a, blockIdx.x - scans);
    if (!elect_last(&a.ws.plan->ticket, gridDim.x, &s_flag)) return;

    /* everything that comes from other workgroups at once, the first row of
     * each thread ahead of what it is needed for */
    const int bad = (int)ld_dev((const uint32_t*)&a.ws.plan->bad);
    const int distinct = (int)ld_dev(&a.ws.plan->distinct);
    RowRecord row{};
    if (tid < a.rows) row = read_row(a, tid);
    int* before = lds;            /* [rows + 1] pages taken before the row */
    int* kept = before + a.rows + 1; /* [rows] its kept slots * 2 + whether it copies */
    int* page = kept + a.rows;    /* [rows] the page it goes on writing, or -1 */
    int* tail = page + a.rows;    /* [rows] tokens in it */
    Writers w;
    w.page = tail + a.rows;
    const uint32_t slots = writer_slots(a.rows);
    w.mask = slots - 1;
    w.rows = w.page + slots;
    w.first = w.rows + slots;
    int held = 0; /* holders of the first row's page */
    for (uint32_t i = tid; i < slots; i += kB) {
        w.page[i] = -1;
        w.rows[i] = 0;
        w.first[i] = INT_MAX;
    }
    const FreeShare f = share_free(a, s_wave); /* (a barrier: the writers are empty) */
    s_share[tid] = f.before;
    if (tid == 0) s_share[kB] = f.total;
    for (int r = tid; r < a.rows; r += kB) {
        if (r != tid) row = read_row(a, r);
        a.to.lengths[r] = row.length; /* (0 instead on an error) */
        before[r] = row.fresh;
        kept[r] = row.kept * 2;
        page[r] = row.page;
        tail[r] = row.tail;
        if (row.page >= 0) {
            const uint32_t at = find_writer(w, row.page, true);
            atomicAdd(&w.rows[at], 1);
            atomicMin(&w.first[at], r);
        }
        if (r == tid) held = row.holders;
    }
    __syncthreads();
    int64_t taken = 0;
    int copies = 0;
    for (int r0 = 0; r0 < a.rows; r0 += kB) {
        const int r = r0 + tid;
        int need = 0, copy = 0, total;
        if (r < a.rows) {
            if (page[r] >= 0) {
                const uint32_t at = find_writer(w, page[r], false);
                const int n = r0 == 0 ? held : (int)ld_dev(&a.ws.count[page[r]]);
                copy = !(n == w.rows[at] && w.first[at] == r);
            }
            need = before[r] + copy;
            kept[r] += copy;
        }
        const int pre = block_exclusive_scan<kB>(need, s_wave, total);
        if (r < a.rows) before[r] = (int)(taken + pre < INT_MAX ? taken + pre : INT_MAX);
        taken += total;
        block_exclusive_scan<kB>(copy, s_wave, total);
        copies += total;
    }
    if (tid == 0) {
        const int code = bad != G4S_OK ? bad : taken > f.total ? G4S_ERR_OUT_OF_MEMORY : G4S_OK;
        s_code = code;
        a.status[0] = code;
        a.status[1] = code ? a.geo.n_pages : a.geo.n_pages - distinct - (int)taken;
        a.status[2] = code ? 0 : (int)taken;
        a.status[3] = code ? 0 : copies;
        a.ws.plan->code = code;
        a.ws.plan->jobs = code ? 0 : copies;
        st_dev((uint32_t*)&a.ws.plan->bad, 0u);
        st_dev(&a.ws.plan->distinct, 0u);
    }
    __syncthreads();
    if (s_code) {
        for (int r = tid; r < a.rows; r += kB) a.to.lengths[r] = 0;
        return;
    }
    int job = 0;
    for (int r0 = 0; r0 < a.rows; r0 += kB) {
        const int r = r0 + tid;
        const int copy = r < a.rows ? kept[r] & 1 : 0;
        int total;
        const int at = job + block_exclusive_scan<kB>(copy, s_wave, total);
        if (copy) {
            atomicSub(&a.ws.count[page[r]], 1u);
            a.ws.jobs[at].src = page[r];
            a.ws.jobs[at].tokens = tail[r];
            tail[r] = at; /* its job, for whoever hands out its first page */
        } else if (r < a.rows && page[r] >= 0) {
            a.to.table[(int64_t)r * a.geo.max_slots + (kept[r] >> 1) - 1] = page[r];
        }
        job += total;
    }
    __syncthreads();
    for (int k = tid; k < (int)taken; k += kB) {
        int lo = 0, hi = a.rows - 1; /* the row that takes free page k */
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (before[mid] <= k)
                lo = mid;
            else
                hi = mid - 1;
        }
        int from = 0, to = kB - 1; /* the share that it lies in */
        while (from < to) {
            const int mid = (from + to + 1) >> 1;
            if (s_share[mid] <= k)
                from = mid;
            else
                to = mid - 1;
        }
        int i = k - s_share[from], word = from * f.words;
        uint64_t bits = ld_dev(&a.ws.free[word]);
        for (int n; i >= (n = __popcll(bits)); i -= n) bits = ld_dev(&a.ws.free[++word]);
        const int p = word * 64 + nth_bit(bits, i);
        const int nth = k - before[lo];
        a.to.table[(int64_t)lo * a.geo.max_slots + (kept[lo] >> 1) - (kept[lo] & 1) + nth] = p;
        if (nth == 0 && (kept[lo] & 1)) a.ws.jobs[tail[lo]].dst = p;
        atomicAdd(&a.ws.count[p], 1u);
    }
}

/* ------------------------------------------------------------------ copies */

/* Copies are bound by memory: 1,501 pages of 16 x 16 KiB take 134 to 144 us by the card, 5.3 to
 * 5.0 TB/s, with streaming stores and a workgroup for each 16 KiB (where they took 134:
 * 170 us from a grid that stays resident, 145 without the streaming; two and eight
 * vectors a thread 136 and 268). */

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

/* Each job in a column of workgroups, its planes and segments in turn. */
template <typename T, typename JobF>
__device__ __forceinline__ void copy_all(const g4s_page_geometry& g, const char* src, char* dst,
                                         int jobs, JobF job)
{
    const int segs = copy_segments<T>(g);
    const uint32_t units = (uint32_t)g.planes * (uint32_t)segs;
    for (int64_t j = blockIdx.x; j < jobs; j += gridDim.x) {
        const PageJob it = job((int)j);
        for (uint32_t u = blockIdx.y; u < units; u += gridDim.y) {
            const uint32_t plane = u / (uint32_t)segs;
            copy_segment<T>(g, src, dst, (int)plane, (int)(u - plane * (uint32_t)segs), it);
        }
    }
}

/* The new counts, and the copies. */
template <typename T>
__global__ __launch_bounds__(kB) void pages_finish_kernel(PagesArgs a)
{
    const bool ok = a.ws.plan->code == G4S_OK;
    if (blockIdx.y == 0)
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

/* Scan and checks side by side: nothing is written before the tables are known to be valid.
 * The workgroup that ends last numbers the free pages. */
__global__ __launch_bounds__(kB) void pages_number_kernel(PagesArgs a)
{
    __shared__ int s_wave[kB / 64];
    __shared__ int s_flag;
    const int tid = threadIdx.x;
    const int scans = scan_groups(a.geo.n_pages);
    if ((int)blockIdx.x < scans)
        scan_pages(a, blockIdx.x);
    else
        gather_rows<true>(a, blockIdx.x - scans);
    if (!elect_last(&a.ws.plan->ticket, gridDim.x, &s_flag)) return;
    const FreeShare f = share_free(a, s_wave);
    const int live = a.geo.n_pages - f.total;
    /* free pages below `live`: as many live ones lie above and move down */
    int mine = 0;
    for (int w = 0, at = f.before; w < f.words; ++w) {
        const int word = f.first + w;
        if (word >= a.words) break;
        const uint64_t bits = ld_dev(&a.ws.free[word]);
        a.ws.before[word] = (uint32_t)at;
        at += __popcll(bits);
        const int in = live - word * 64;
        if (in > 0) mine += __popcll(in >= 64 ? bits : bits & (((uint64_t)1 << in) - 1));
    }
    const int holes = block_sum_i32<kB>(mine, s_wave);
    if (tid == 0) {
        const int code = (int)ld_dev((const uint32_t*)&a.ws.plan->bad);
        st_dev((uint32_t*)&a.ws.plan->bad, 0u);
        a.ws.plan->code = code;
        a.ws.plan->live = live;
        a.ws.plan->below = live - holes;
        a.ws.plan->jobs = code ? 0 : holes;
        a.status[0] = code;
        a.status[1] = code ? a.geo.n_pages : f.total;
        a.status[2] = 0;
        a.status[3] = code ? 0 : holes;
    }
}

/* Free pages before page p, and the i-th free and live page. */
__device__ __forceinline__ int free_before(const PagesArgs& a, int p)
{
    return (int)a.ws.before[p / 64] +
           __popcll(a.ws.free[p / 64] & (((uint64_t)1 << (p & 63)) - 1));
}
template <bool FREE>
__device__ __forceinline__ int nth_page(const PagesArgs& a, int i)
{
    auto before = [&](int w) { return FREE ? (int)a.ws.before[w] : w * 64 - (int)a.ws.before[w]; };
    int lo = 0, hi = a.words - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (before(mid) <= i)
            lo = mid;
        else
            hi = mid - 1;
    }
    const uint64_t bits = a.ws.free[lo];
    return lo * 64 + nth_bit(FREE ? bits : ~bits, i - before(lo));
}

template <typename T>
__global__ __launch_bounds__(kB) void pages_compact_kernel(PagesArgs a)
{
    const PagePlan plan = *a.ws.plan;
    const bool ok = plan.code == G4S_OK;
    if (blockIdx.y == 0) {
        const int at = blockIdx.x * kB + threadIdx.x, step = gridDim.x * kB;
        for (int p = at; p < a.geo.n_pages; p += step) {
            int refs = 0;
            if (ok && p < plan.live) {
                refs = a.from.refs[p];
                if (refs <= 0) refs = a.from.refs[nth_page<false>(a, plan.below + free_before(a, p))];
            }
            a.to.refs[p] = refs;
        }
        for (int r = at; r < a.rows; r += step) a.to.lengths[r] = ok ? a.from.lengths[r] : 0;
        const int64_t S = a.geo.max_slots, cells = ok ? a.rows * S : 0;
        for (int64_t c = at; c < cells; c += step) {
            const int r = (int)(c / S);
            if (c - r * S >= used_slots(a.from.lengths[r], a.geo.page_tokens)) continue;
            int p = a.from.table[c];
            if (p >= plan.live) p = nth_page<true>(a, p - free_before(a, p) - plan.below);
            a.to.table[c] = p;
        }
    }
    copy_all<T>(a.geo, a.pool, a.pool, plan.jobs, [&](int j) {
        return PageJob{nth_page<false>(a, plan.below + j), nth_page<true>(a, j),
                       a.geo.page_tokens};
    });
}

__global__ __launch_bounds__(kB) void pages_init_kernel(PageWorkspace ws, int n)
{
    for (int p = blockIdx.x * kB + threadIdx.x; p < n; p += gridDim.x * kB) ws.count[p] = 0u;
    if (blockIdx.x == 0 && threadIdx.x == 0) *ws.plan = PagePlan{};
}

/* Widest vectors that every address of a copy is a multiple of. */
uint64_t copy_bits(const g4s_page_geometry& g, const void* src, const void* dst)
{
    return (uint64_t)(uintptr_t)src | (uint64_t)(uintptr_t)dst | (uint64_t)g.token_bytes |
           (uint64_t)g.plane_stride | (uint64_t)g.page_stride;
}

/* At most `jobs` jobs: a workgroup for each, and as many side by side as its planes and
 * segments fill until there are kCopyGroups, some rounds of the device (a
 * compaction's workgroups each find their page first: 6,000 pages 154 us, with
 * 2^15 and 2^13 of them 164 and 157). */
constexpr int kCopyGroups = 1 << 14;

template <typename T>
dim3 copy_grid(const g4s_page_geometry& g, int64_t jobs, int64_t least)
{
    const int64_t units = (int64_t)g.planes * copy_segments<T>(g);
    int64_t x = jobs > least ? jobs : least;
    x = x < 1 ? 1 : x > kCopyGroups ? kCopyGroups : x;
    int64_t y = kCopyGroups / (jobs < 1 ? 1 : jobs);
    y = y > units ? units : y > 65535 ? 65535 : y;
    y = y < 1 ? 1 : y;
    const int64_t each = (units + y - 1) / y; /* as many for each */
    return dim3((unsigned)x, (unsigned)(each < 1 ? 1 : (units + each - 1) / each));
}

}  // namespace

hipError_t pages_init_launch(const PageWorkspace& ws, int32_t n_pages, hipStream_t stream)
{
    return launch(pages_init_kernel, 256, kB, 0, stream, ws, n_pages);
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

static unsigned first_grid(const PagesArgs& a)
{
    return (unsigned)(scan_groups(a.geo.n_pages) +
                      (a.rows + kGatherRows - 1) / kGatherRows * slot_groups(a.geo.max_slots));
}

hipError_t pages_advance_launch(const PagesArgs& a, hipStream_t stream)
{
    hipError_t e = launch(pages_advance_kernel, first_grid(a), kB, plan_lds(a.rows), stream, a);
    if (e != hipSuccess) return e;
    const int64_t least = (a.geo.n_pages + kB - 1) / kB;
#define G4S_CALL(T) \
    e = launch(pages_finish_kernel<T>, copy_grid<T>(a.geo, a.rows, least), kB, 0, stream, a)
    G4S_BY_WIDTH(copy_bits(a.geo, a.pool, a.pool), G4S_CALL);
#undef G4S_CALL
    return e;
}

hipError_t pages_compact_launch(const PagesArgs& a, hipStream_t stream)
{
    hipError_t e = launch(pages_number_kernel, first_grid(a), kB, 0, stream, a);
    if (e != hipSuccess) return e;
    const int64_t cell = (int64_t)a.rows * a.geo.max_slots;
    const int64_t least = ((cell > a.geo.n_pages ? cell : a.geo.n_pages) + kB - 1) / kB;
#define G4S_CALL(T)                                                                         \
    e = launch(pages_compact_kernel<T>, copy_grid<T>(a.geo, a.geo.n_pages / 2, least), kB, 0, \
               stream, a)
    G4S_BY_WIDTH(copy_bits(a.geo, a.pool, a.pool), G4S_CALL);
#undef G4S_CALL
    return e;
}

hipError_t pages_copy_launch(const g4s_page_geometry& geo, const char* src, char* dst, int32_t n,
                             const int32_t* d_src, const int32_t* d_dst, const int32_t* d_tokens,
                             hipStream_t stream)
{
    hipError_t e;
#define G4S_CALL(T)                                                                       \
    e = launch(pages_copy_kernel<T>, copy_grid<T>(geo, n, 1), kB, 0, stream, geo, src, dst, n, \
               d_src, d_dst, d_tokens)
    G4S_BY_WIDTH(copy_bits(geo, src, dst), G4S_CALL);
#undef G4S_CALL
    return e;
}

}  // namespace g4s
