/*
 * g4s_pages.h -- launch interface of the page kernels (g4s_pages.hip), and
 * the rules of a row's step and of addresses, which the host can run too.
 */
#ifndef G4S_PAGES_H
#define G4S_PAGES_H

#include <stdint.h>

#include "gemma4_beam.h"

#if defined(__HIPCC__)
#include <hip/hip_runtime.h>
#define G4S_PAGE_HD __host__ __device__ inline
#else
#define G4S_PAGE_HD inline
#endif

namespace g4s {

constexpr int64_t kMaxPageBytes = (int64_t)1 << 30;

/* What one row does in a step. */
struct RowStep {
    int64_t length; /* tokens afterwards */
    int32_t kept;   /* slots taken over from the parent */
    int32_t fresh;  /* slots behind them */
    int32_t tail;   /* tokens of the last kept page if the row goes on writing
                       it, else 0 */
    int32_t bad;    /* the row's parent or a length is not valid (a row
                       without tokens is returned) */
};

/* Slots of a row of `tokens` tokens.  A row may hold 2^31 - 1: the sum passes 32 bits. */
G4S_PAGE_HD int32_t used_slots(int64_t tokens, int32_t page_tokens)
{
    return (int32_t)((tokens + page_tokens - 1) / page_tokens);
}

G4S_PAGE_HD RowStep row_step(int32_t parent, int32_t from_rows, int32_t parent_length, int32_t grow,
                        int32_t page_tokens, int32_t max_slots)
{
    RowStep s{0, 0, 0, 0, 1};
    const int64_t room = (int64_t)page_tokens * max_slots;
    if (parent < -1 || parent >= from_rows) return s;
    const int64_t old = parent >= 0 ? parent_length : 0;
    if (old < 0 || old > room) return s;
    int64_t now = old + grow;
    if (now < 0) now = 0;
    if (now > room) return s;
    const int64_t keep = old < now ? old : now;
    s.length = now;
    s.kept = used_slots(keep, page_tokens);
    s.fresh = used_slots(now, page_tokens) - s.kept;
    s.tail = now > keep ? (int32_t)(keep % page_tokens) : 0;
    s.bad = 0;
    return s;
}

/* Byte offset of token-vector `i` (of `vec` bytes) of the first `tokens` tokens of
 * each part, counted through the parts of a page in one plane. */
G4S_PAGE_HD int64_t page_offset(const g4s_page_geometry& g, int32_t plane, int32_t page, uint32_t i,
                           uint32_t per_part, int32_t vec)
{
    const uint32_t part = i / per_part;
    return (int64_t)plane * g.plane_stride + (int64_t)page * g.page_stride +
           (int64_t)part * g.page_tokens * g.token_bytes + (int64_t)(i - part * per_part) * vec;
}

/* Whether the pages of the geometry lie within 64-bit offsets without overlap. */
G4S_PAGE_HD bool geometry_ok(const g4s_page_geometry& g)
{
    if (g.page_tokens < 1 || g.page_tokens > 65536 || g.n_pages < 1 ||
        g.n_pages > G4S_PAGES_MAX_PAGES || g.max_rows < 1 || g.max_rows > G4S_PAGES_MAX_ROWS ||
        g.max_slots < 1 || g.max_slots > G4S_PAGES_MAX_PAGES ||
        (int64_t)g.max_slots * g.page_tokens > INT32_MAX || g.planes < 0 ||
        g.planes > 65536)
        return false;
    if (g.planes == 0) return true;
    if (g.parts < 1 || g.token_bytes < 1 || g.token_bytes > kMaxPageBytes || g.parts > 65536 ||
        g.plane_stride < 0 || g.page_stride < 0)
        return false;
    const int64_t one = (int64_t)g.page_tokens * g.token_bytes; /* <= 2^46 */
    if (one > kMaxPageBytes || one * g.parts > kMaxPageBytes) return false;
    const int64_t page = one * g.parts;
    const int64_t limit = (int64_t)1 << 56;
    if (g.plane_stride > limit / g.planes || g.page_stride > limit / g.n_pages) return false;
    const bool inner_pages = (g.n_pages == 1 || g.page_stride >= page) &&
                             (g.planes == 1 ||
                              g.plane_stride >= (g.n_pages - 1) * g.page_stride + page);
    const bool inner_planes = (g.planes == 1 || g.plane_stride >= page) &&
                              (g.n_pages == 1 ||
                               g.page_stride >= (g.planes - 1) * g.plane_stride + page);
    return inner_pages || inner_planes;
}

/* Bytes from a pool's start to the end of its last page. */
G4S_PAGE_HD int64_t pool_extent(const g4s_page_geometry& g)
{
    if (g.planes == 0) return 0;
    return (g.planes - 1) * g.plane_stride + (g.n_pages - 1) * g.page_stride +
           (int64_t)g.parts * g.page_tokens * g.token_bytes;
}

#if defined(__HIPCC__)

struct PageJob {
    int32_t src, dst, tokens;
};

/* What the kernels of one call tell each other. */
struct PagePlan {
    uint32_t ticket;   /* 0 between calls, as the next two */
    int32_t bad;       /* the first error (the lowest status) */
    uint32_t distinct; /* pages taken over by some row */
    int32_t code;
    int32_t jobs;  /* pages to copy */
    int32_t live;  /* compact: live pages */
    int32_t below; /* compact: live pages among the first `live` */
};

struct PageWorkspace {
    uint32_t* count;  /* [n_pages] rows that hold the page; 0 between calls */
    uint64_t* free;   /* [words] a bit for each free page, 64 pages a word */
    uint32_t* before; /* [words + 1] compact: free pages before the word */
    PageJob* jobs;    /* [max_rows] */
    uint64_t* steps;  /* [max_rows][3]  kept and fresh slots; written page and its tokens; length */
    PagePlan* plan;
};

struct PagesArgs {
    g4s_page_geometry geo;
    g4s_page_state from, to;
    int32_t from_rows, rows;
    const int32_t* parents;
    const int32_t* grow;
    char* pool;
    int32_t* status;
    int32_t words;
    PageWorkspace ws;
};

hipError_t pages_init_launch(const PageWorkspace& ws, int32_t n_pages, hipStream_t stream);
hipError_t pages_advance_launch(const PagesArgs& a, hipStream_t stream);
hipError_t pages_compact_launch(const PagesArgs& a, hipStream_t stream);
hipError_t pages_copy_launch(const g4s_page_geometry& geo, const char* src, char* dst, int32_t n,
                             const int32_t* d_src, const int32_t* d_dst, const int32_t* d_tokens,
                             hipStream_t stream);

#endif

}  // namespace g4s

#endif
