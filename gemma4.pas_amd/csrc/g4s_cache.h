/*
 * g4s_cache.h -- launch interface of the kernels of the 8-bit cache
 * (g4s_append.hip, g4s_attend.hip), and the rules of places, addresses and scales,
 * which the host can run too.
 */
#ifndef G4S_CACHE_H
#define G4S_CACHE_H

#include <stdint.h>

#include "g4s_pages.h"
#include "gemma4_cache.h"

namespace g4s {

/* n / d for 0 <= n < 2^31 and 1 <= d <= 2^31: with s = ceil(log2 d) and
 * m = floor(2^(31+s) / d) + 1, m * d - 2^(31+s) is at most 2^s, so the error of
 * n * m / 2^(31+s) stays below 1 / d. */
struct Divisor {
    uint32_t m;
    int32_t s, d;
};
inline Divisor divisor(int32_t d)
{
    int s = 0;
    while (((int64_t)1 << s) < d) ++s;
    return Divisor{(uint32_t)((((uint64_t)1 << (31 + s)) / (uint32_t)d) + 1), 31 + s, d};
}
G4S_PAGE_HD int32_t divide(int32_t n, const Divisor& d)
{
    return (int32_t)(((uint64_t)(uint32_t)n * d.m) >> d.s);
}

/* The pool as the kernels see it. */
struct CachePool {
    int64_t plane_stride, page_stride;
    int32_t part_bytes, token_bytes; /* of a head in a page, of a token */
    int32_t n_pages, max_slots;
    Divisor page_tokens;
    Divisor scale_tokens;
    int32_t head_dim;
};

/* Most tokens of a row. */
G4S_PAGE_HD int64_t cache_room(const CachePool& p) { return (int64_t)p.max_slots * p.page_tokens.d; }

/* Bytes from a plane's start to token `place` of head `head`, its page known. */
G4S_PAGE_HD int64_t cache_offset(const CachePool& p, int32_t page, int32_t in_page, int32_t head)
{
    return (int64_t)page * p.page_stride + (int64_t)head * p.part_bytes +
           (int64_t)in_page * p.token_bytes;
}

/* Tokens of a row in a call, the first of the views, and the row's length; a
 * length outside the table gives bad = 1 and d_starts that do not fit the call no
 * tokens. */
struct RowTokens {
    int32_t start, count, length, bad;
};
G4S_PAGE_HD RowTokens row_tokens(const int32_t* starts, const int32_t* lengths, int32_t row,
                                 int32_t tokens, int64_t room)
{
    RowTokens r{row, 1, lengths[row], 0};
    if (starts) {
        r.start = starts[row];
        const int32_t end = starts[row + 1];
        r.count = r.start >= 0 && end > r.start && end <= tokens ? end - r.start : 0;
    }
    if (r.length < 0 || r.length > room) {
        r.length = 0;
        r.bad = 1;
    }
    return r;
}

/* Least e from kScaleLow to kScaleHigh with top <= 448 * 2^e.  448 = 0.875 * 2^9: with
 * top = m * 2^x and m in [0.5, 1), that is x - 9 for m <= 0.875 and one more above. */
constexpr int kScaleLow = -100, kScaleHigh = 119;
G4S_PAGE_HD int32_t scale_exponent(double top)
{
    if (!(top > 0.0)) return kScaleLow;
    union {
        double d;
        uint64_t u;
    } b{top};
    const int32_t field = (int32_t)(b.u >> 52) & 0x7FF; /* (subnormals end at kScaleLow too) */
    const uint64_t fraction = b.u & (((uint64_t)1 << 52) - 1);
    int32_t e = field - 1022 - 9 + (fraction > ((uint64_t)3 << 50) ? 1 : 0);
    e = e < kScaleLow ? kScaleLow : e;
    return e > kScaleHigh ? kScaleHigh : e;
}

/* Whether these bits are those of a scale, a number from 0 to 2^kScaleHigh.  Any code times that is finite in
 * bf16; what is not would be NaN after a product with a weight of 0, for queries that do not see it, too. */
G4S_PAGE_HD bool scale_ok(uint32_t bits) { return bits <= (uint32_t)(127 + kScaleHigh) << 23; }

/* n / d (n >= 0, d > 0), in 32 bits where they hold both. */
G4S_PAGE_HD int64_t quotient(int64_t n, int64_t d)
{
    if (((uint64_t)n | (uint64_t)d) >> 32) return n / d;
    return (int64_t)((uint32_t)n / (uint32_t)d);
}

/* Units of work shared out among `groups` workgroups, total >= groups: group w takes
 * units total * w / groups up to total * (w + 1) / groups, and unit x is the group's
 * that unit_group gives (the last w with total * w / groups < x + 1). */
G4S_PAGE_HD int64_t first_unit(int64_t total, int32_t w, int32_t groups)
{
    return quotient(total * w, groups);
}
G4S_PAGE_HD int32_t unit_group(int64_t x, int64_t total, int32_t groups)
{
    return (int32_t)quotient((x + 1) * groups - 1, total);
}

/* Dims that the attention's kernels are made for, at least head_dim. */
G4S_PAGE_HD int32_t attend_width(int32_t head_dim)
{
    return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : head_dim <= 256 ? 256 : 512;
}

/* Query columns (tokens x heads of a key head) that the rows' kernel takes in a pass over the tokens, and how it is
 * made for a width of heads: waves of a workgroup, tokens of a wave's step, and units of `waves` steps
 * that a workgroup takes at least where there are enough of them. */
constexpr int kCols = 16;
struct RowsShape {
    int32_t waves, tokens, units;
    G4S_PAGE_HD constexpr int32_t unit() const { return waves * tokens; }
};
G4S_PAGE_HD constexpr RowsShape rows_shape(int32_t width)
{
    return width <= 128 ? RowsShape{8, 64, 1} : width <= 256 ? RowsShape{4, 32, 2} : RowsShape{4, 16, 4};
}

/* Rows with more than one token and more than `few` columns (tokens x heads of a key head)
 * are the prompts' kernel's, the others the rows' kernel's, which takes 16 columns a pass over the
 * tokens.  Eight rows of some 3,500 tokens, 8 key heads with 4 heads of 128 dims (2 of 256, binary32):
 * 24 to 28 columns a row 48 (42) us by rows and 69 (53) by prompts, 32 to 36 columns 50 (44) and 87 (58).  Rows
 * on both sides (48 to 60 columns) cost both kernels, one behind the other: 111 (82) us, 88 (59) by
 * prompts alone. */
constexpr int kFewCols = 48;
G4S_PAGE_HD bool is_prompt(int32_t count, int32_t group, int32_t few)
{
    return (int64_t)count * group > few && (count > 1 || few == 0);
}

/* Units of `unit` tokens that places from .. end - 1 lie in: one at least, for the output. */
G4S_PAGE_HD int32_t place_units(int32_t from, int32_t end, int32_t unit)
{
    return end > from ? (int32_t)(((uint32_t)end + unit - 1) / unit) - from / unit : 1;
}
G4S_PAGE_HD int32_t column_blocks(int32_t cols) { return (cols + kCols - 1) / kCols; }

/* The most units of a call's rows: each block of a row's columns, for each key head, goes over the row's places.  A
 * row of the rows' kernel has one token, or (with d_starts) as many as `few` columns hold; rows that
 * are taken together have no more than each by itself. */
G4S_PAGE_HD int64_t most_units(int32_t rows, int32_t tokens, bool starts, int32_t kv_heads, int32_t group,
                               int32_t few, int64_t room, int32_t unit)
{
    int64_t cols = (int64_t)tokens * group < few ? (int64_t)tokens * group : few;
    cols = starts && cols > group ? cols : group;
    return (int64_t)rows * kv_heads * column_blocks((int32_t)cols) * ((room + unit - 1) / unit + 1);
}
/* Workgroups, of a grid, that share `total` units: one unit each while that leaves CUs without any, and
 * `units` at least of each otherwise (501 tokens of 256 dims: 11 us, 15 with two at least). */
G4S_PAGE_HD int32_t sharing_groups(int64_t total, int32_t units, int32_t ncu, int32_t grid)
{
    const int64_t one_each = total < ncu ? total : ncu, several = (total + units - 1) / units;
    const int64_t groups = several < one_each ? one_each : several;
    return (int32_t)(groups < grid ? groups : grid);
}

/* Where a row's slots of a grid begin: `times` columns a token, `unit` columns a slot.  A row of
 * n tokens has floor(n * times / unit) + extra slots at least. */
G4S_PAGE_HD int64_t share_begin(const int32_t* starts, int32_t row, int32_t times, int32_t unit,
                                int32_t extra)
{
    return (int64_t)(starts ? starts[row] : row) * times / unit + (int64_t)extra * row;
}

/* Vectors of `vec` bytes for tokens and heads, at `at` and strides in bytes, where heads lie within a
 * token's stride or tokens within a head's (strides of dimensions with one vector are 0). */
struct Vectors {
    uint64_t at;
    int64_t tokens, heads, token_stride, head_stride, vec;
    G4S_PAGE_HD int64_t head_end() const { return (heads - 1) * head_stride + vec; }
    G4S_PAGE_HD int64_t end() const { return (tokens - 1) * token_stride + head_end(); }
};
/* Whether two of them (of vectors as long) share memory.  Views of the same strides, as parts of each token's record
 * or of each head's, do where a vector of one does with a vector of the other; those of one token stride
 * and different head strides where their heads do; others where they begin and end say so. */
G4S_PAGE_HD bool vectors_meet(const Vectors& a, const Vectors& b)
{
    if (!a.at || !b.at || a.at >= b.at + (uint64_t)b.end() || b.at >= a.at + (uint64_t)a.end()) return false;
    const int64_t ts = a.tokens > 1 ? a.token_stride : b.token_stride;
    const int64_t hs = a.heads > 1 ? a.head_stride : b.head_stride;
    const bool same_ts = b.tokens == 1 || b.token_stride == ts, same_hs = b.heads == 1 || b.head_stride == hs;
    const int64_t gap = (int64_t)(b.at - a.at);
    if (same_ts && same_hs) {
        /* gap + (tokens apart) ts + (heads apart) hs, next to 0 in the outer stride, then in the inner one */
        const bool by_token = ts >= hs;
        const int64_t outer = by_token ? ts : hs, inner = by_token ? hs : ts;
        const int64_t out_a = by_token ? a.tokens : a.heads, out_b = by_token ? b.tokens : b.heads;
        const int64_t in_a = by_token ? a.heads : a.tokens, in_b = by_token ? b.heads : b.tokens;
        const int64_t o0 = outer ? -gap / outer : 0;
        for (int64_t o = o0 - 1; o <= o0 + 1; ++o) {
            if (o <= -out_a || o >= out_b) continue;
            const int64_t rest = gap + o * outer, i0 = inner ? -rest / inner : 0;
            for (int64_t i = i0 - 1; i <= i0 + 1; ++i) {
                const int64_t apart = rest + i * inner;
                if (i > -in_a && i < in_b && apart < a.vec && apart > -a.vec) return true;
            }
        }
        return false;
    }
    if (same_ts && ts > 0 && a.head_end() <= ts && b.head_end() <= ts) {
        const int64_t r = (gap % ts + ts) % ts;
        return r < a.head_end() || ts - r < b.head_end();
    }
    return true;
}

#if defined(__HIPCC__)

/* The row whose share holds slot x: the last one that begins at or before it.  Every lane
 * looks at one row of 64 stretches, then within a stretch, ... */
__device__ __forceinline__ int find_share(const int32_t* starts, int rows, int64_t x, int times,
                                          int unit, int extra)
{
    int lo = 0, n = rows;
    const int lane = threadIdx.x & 63;
    while (n > 1) {
        const int each = (n + 63) / 64;
        const bool at = lane * each < n &&
                        share_begin(starts, lo + lane * each, times, unit, extra) <= x;
        const uint64_t m = __ballot(at);
        const int last = m ? 63 - __clzll(m) : 0;
        lo += last * each;
        n = n - last * each < each ? n - last * each : each;
    }
    return lo;
}

struct CacheView {
    char* data;
    int64_t token_stride, head_stride; /* elements */
};

struct AppendArgs {
    CachePool pool;
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* starts;
    int32_t rows, tokens;
    CacheView q, k, v, q_out; /* data NULL: none */
    const int32_t* positions;
    const float* freqs;
    char* k_plane;
    char* v_plane;
    int32_t heads, kv_heads, rotary_dims, rotary_pairs;
};

/* Columns whose parts a launch of its own joins. */
struct AttendRecord {
    int32_t parts; /* 0: none */
    int32_t cols;
    int32_t col0, head0; /* first column, and first head of its key head */
    int32_t row, start;  /* several rows' (start -1), or a single one's first token */
};

/* Workspace of the attention: what several workgroups found for the same columns. */
struct AttendSpace {
    float* sums;       /* kAttendSums for each workgroup of the rows' kernel */
    float* stats;      /* kAttendStats */
    uint32_t* tickets; /* one; 0 between calls */
    AttendRecord* records; /* one: what the rows' kernel leaves to be joined */
    int32_t groups;    /* workgroups of the rows' kernel at most; of the prompts' kernel half as
                          many, with twice the space, split the tokens */
};
constexpr int kAttendSums = 16384, kAttendStats = 256;

struct AttendArgs {
    CachePool pool;
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* starts;
    int32_t rows, tokens;
    CacheView q, out;
    const char* k_plane;
    const char* v_plane;
    float* lse;
    float scale;
    int32_t window;
    int32_t heads, kv_heads;
    Divisor group;
    int32_t few; /* kFewCols, or 0: all rows are prompts */
    AttendSpace ws;
};

hipError_t append_launch(const AppendArgs& a, int32_t dtype, hipStream_t stream);

hipError_t attend_rows_launch(const AttendArgs& a, int32_t dtype, hipStream_t stream);
hipError_t attend_prompts_launch(const AttendArgs& a, int32_t dtype, hipStream_t stream);

int32_t attend_groups(int32_t ncu);
hipError_t attend_init_launch(const AttendSpace& ws, hipStream_t stream);

#endif

}  // namespace g4s

#endif
