/*
 * g4s_attend.hip -- attention over the pages of an 8-bit cache for rows with few queries
 * (the tokens of a decode step), on gfx950.
 *
 * Neighbouring rows of one token each that begin with the same page (the beams of a search, requests
 * with one prompt) are taken together, as far as 16 query columns hold them: as long as
 * their pages are the same a tile of keys and values is read once for all, from the first
 * page on that differs each row's tiles by themselves.  The work of a launch, counted in units of
 * NW x TT tokens of one such group and key head, is shared out evenly over the
 * workgroups, whatever the lengths; every workgroup finds its share from them by itself.  A wave
 * takes TT tokens of each unit with a softmax of its own; the waves join in LDS, and where several
 * workgroups have parts of one group and head, the one that ends last joins those, in their
 * order, so that results do not depend on who that is; many parts are joined by a launch of their own.
 *
 * Scores are products of the widened codes (exact in bf16) with the queries as matrix operands, K Q^T,
 * so that a lane holds scores of one column and multiplies them, as weights, with V^T without
 * an exchange.  All that is read is read once, one step ahead of its use: 131,071 tokens of 8 heads of 128
 * dims 61 us (4.4 TB/s; this card reads 6.1 at most), 64 rows of 3,000 to 5,000 tokens 100 us (4.7
 * TB/s; 5.4 between start and end).  What is left is the start (lengths and tables 2 to 8 us, queries 1 to 6, page, scales
 * and codes one behind the other 2 to 8) and the joins (3 to 8 us, 4 to 11 in their own launch): 12
 * searches of 4 beams over 3,800 tokens, 512 dims in binary32, 85 us, of which the steps are 26.
 */
#include "g4s_attend.h"
#include "g4s_launch.h"

namespace g4s {

namespace {

constexpr int kB = 256;
/* Bytes of parts that their last workgroup joins by itself: more are left to a launch of
 * their own (the 12 searches of 512 dims: 86 us, 100 without it; 192 rows with windows of 512: 38.5 and, all
 * joined by it, 41). */
constexpr int kJoinBytes = 96 << 10;

/* What the scan keeps of a row: its length (bad: -1), and the first page of one that may be taken
 * together with others (-1: none). */
struct RowInfo {
    int length, key;
    int differs; /* about the first slot whose page is not that of the row it is compared with */
};

/* The rows that begin with a row and are taken together, and the places that any of their
 * queries sees. */
struct Group {
    int rows;  /* of one token each; or -n: one row of n tokens; 0: none (taken by a row before it,
                  without tokens, or the prompts' kernel's) */
    int start; /* a single row's first token */
    int from, end;
    int shared; /* units of tokens of several rows that are likely to have the same pages */
};
constexpr int kNone = 0x7FFFFFFF;

/* Rows that are taken together at most: a power of two, of rows that begin at a multiple of it. */
__device__ __forceinline__ int group_rows(const AttendArgs& a)
{
    const int n = kCols / a.group.d;
    return n >= 16 ? 16 : n >= 8 ? 8 : n >= 4 ? 4 : n >= 2 ? 2 : 1;
}

template <int UNIT>
__device__ __forceinline__ int last_unit(const Group& p)
{
    return (int)(((uint32_t)p.end + UNIT - 1) / UNIT);
}
template <int UNIT>
__device__ __forceinline__ Group find_group(const AttendArgs& a, const RowInfo* info, int row)
{
    Group p{0, 0, 0, 0, 0};
    const int key = info[row].key, most = group_rows(a), in = row & (most - 1);
    if (key >= 0) {
        if (in > 0 && info[row - 1].key == key) return p;
        p.rows = 1;
        p.end = info[row].length;
        p.from = sees_from(a, p.end - 1);
        int differs = info[row].differs;
        for (int i = 1; in + i < most && row + i < a.rows && info[row + i].key == key; ++i) {
            const int n = info[row + i].length, f = sees_from(a, n - 1);
            p.end = n > p.end ? n : p.end;
            p.from = f < p.from ? f : p.from;
            differs = info[row + i].differs < differs ? info[row + i].differs : differs;
            ++p.rows;
        }
        if (p.rows > 1) {
            const int64_t t = (int64_t)differs * a.pool.page_tokens.d;
            const int n = t < p.end ? (int)t / UNIT : last_unit<UNIT>(p);
            p.shared = n > p.from / UNIT ? n - p.from / UNIT : 0;
            return p;
        }
    }
    const RowTokens r = row_tokens(a.starts, a.lengths, row, a.tokens, cache_room(a.pool));
    p.rows = is_prompt(r.count, a.group.d, a.few) ? 0 : -r.count;
    p.start = r.start;
    p.end = r.length;
    p.from = sees_from(a, r.length - r.count);
    return p;
}

/* Query columns (tokens x heads of a key head) of a group, and units of UNIT tokens of each of
 * its blocks of them: one at least, for the output.  Tokens whose pages several rows share
 * count once, the others for each row. */
__device__ __forceinline__ int group_cols(const AttendArgs& a, const Group& p)
{
    return (p.rows < 0 ? -p.rows : p.rows) * a.group.d;
}
template <int UNIT>
__device__ __forceinline__ int group_units(const Group& p)
{
    const int n = place_units(p.from, p.end, UNIT);
    return p.rows > 1 ? p.shared + (n - p.shared) * p.rows : n;
}

/* Where the pages of rows that may be taken together part from those of the longest of them, in
 * the slots that both see: a search that takes one of EACH + 1 stretches a step by the
 * pages at their ends, EACH lanes a row.  It finds the slot if pages that have parted never
 * meet again, and otherwise some slot; it only decides how work is shared out. */
template <int NW, int EACH>
__device__ __forceinline__ void find_partings(const AttendArgs& a, RowInfo* info)
{
    const int lane = threadIdx.x & (EACH - 1), most = group_rows(a);
    for (int r0 = 0; r0 < a.rows; r0 += NW * 64 / EACH) {
        const int r = r0 + (int)threadIdx.x / EACH;
        const int key = r < a.rows ? info[r].key : -1;
        int ref = r;
        if (key >= 0) {
            for (int i = r - 1; i >= (r & -most) && info[i].key == key; --i)
                if (info[i].length >= info[ref].length) ref = i;
            for (int i = r + 1; i < a.rows && (i & (most - 1)) != 0 && info[i].key == key; ++i)
                if (info[i].length > info[ref].length) ref = i;
        }
        int lo = 0, hi = 0; /* the first that differs is one of lo .. hi, hi meaning none */
        if (ref != r) {
            lo = divide(sees_from(a, info[ref].length - 1), a.pool.page_tokens);
            hi = divide(info[r].length - 1, a.pool.page_tokens) + 1;
        }
        const int end = hi;
        const int32_t* mine = a.table + (int64_t)(r < a.rows ? r : 0) * a.pool.max_slots;
        const int32_t* other = a.table + (int64_t)(ref < a.rows ? ref : 0) * a.pool.max_slots;
        while (__any(lo < hi)) {
            const int n = (hi - lo + EACH) / (EACH + 1); /* slots lo + n i - 1 are looked at */
            const int at = lo + n * (lane + 1) - 1;
            const bool differs = lo < hi && (at >= hi || mine[at] != other[at]);
            const uint32_t found = (uint32_t)(__ballot(differs) >> ((threadIdx.x & 63) & -EACH)) &
                                   ((1u << EACH) - 1);
            if (lo < hi) {
                const int k = found ? __builtin_ctz(found) : EACH;
                const int top = lo + n * (k + 1) - 1;
                if (found && top < hi) hi = top;
                lo += n * k;
            }
        }
        if (lane == 0 && key >= 0) info[r].differs = lo < end ? lo : kNone;
    }
}

/* info and groups [0 .. rows - 1], and the work of the groups before each row, in units,
 * in before[0 .. rows]. */
template <int NW, int UNIT>
__device__ __forceinline__ void scan_rows(const AttendArgs& a, RowInfo* info, Group* groups,
                                          int64_t* before, int64_t* s_wave)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int each = (a.rows + NW * 64 - 1) / (NW * 64);
    const int64_t room = cache_room(a.pool);
    for (int r = tid; r < a.rows; r += NW * 64) {
        const int page = a.table[(int64_t)r * a.pool.max_slots];
        const RowTokens t = row_tokens(a.starts, a.lengths, r, a.tokens, room);
        RowInfo i{t.bad ? -1 : t.length, -1, kNone};
        if (t.count == 1 && t.length > 0 && page >= 0 && page < a.pool.n_pages) i.key = page;
        info[r] = i;
    }
    lds_barrier();
    if (a.rows > 1 && group_rows(a) > 1) {
        if (a.rows <= NW * 4)
            find_partings<NW, 16>(a, info);
        else
            find_partings<NW, 4>(a, info);
        lds_barrier();
    }
    int64_t sum = 0;
    for (int i = 0; i < each; ++i) {
        const int r = tid * each + i;
        if (r >= a.rows) break;
        const Group p = find_group<UNIT>(a, info, r);
        const int blocks = column_blocks(group_cols(a, p));
        groups[r] = p;
        before[r + 1] = (int64_t)(blocks * a.kv_heads) * group_units<UNIT>(p);
        sum += before[r + 1];
    }
    /* (a row's units are below 2^39) */
    int64_t x = (int64_t)wave_inclusive_scan((int)(sum >> 16)) * 65536 +
                wave_inclusive_scan((int)(sum & 0xFFFF));
    if (a.rows > 64 * each) {
        if (lane == 63) s_wave[wave] = x;
        lds_barrier();
        for (int w = 0; w < wave; ++w) x += s_wave[w];
    }
    x -= sum;
    for (int i = 0; i < each; ++i) {
        const int r = tid * each + i;
        if (r >= a.rows) break;
        x += before[r + 1];
        before[r + 1] = x;
    }
    if (tid == 0) before[0] = 0;
    lds_barrier();
}

/* Dims that the waves join at once (LDS also holds 40 bytes for each of up to 2048 rows). */
template <int D, int NW>
constexpr int kPass = D * NW < 512 ? D : 512 / NW;

template <int DT, int D, int NW, int TT>
struct Shared {
    union {
        Frag q[D / 64][2][DT == G4S_DTYPE_F32 ? 3 : 1][64]; /* the queries, as lanes take them */
        float o[NW][kCols][kPass<D, NW> + 4];               /* the waves' sums */
    };
    int64_t offset[NW][2][TT];
    float scale[NW][2][2][TT];
    float m[NW][kCols], l[NW][kCols];
    float top[kCols], sum[kCols];
    int64_t out[kCols]; /* of each column: its first element of out, and its lse */
    int lse[kCols];
    int64_t wave[NW];
    int differs; /* the first slot whose page is not the same for all rows */
    int flag;
};

/* Dims of a lane in registers, VW words of four. */
template <int VW>
__device__ __forceinline__ void load_words(const char* p, uint32_t (&w)[VW])
{
    if constexpr (VW == 1) {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (VW == 2) {
        const u32x2_4 x = *reinterpret_cast<const u32x2_4*>(p);
        w[0] = x[0], w[1] = x[1];
    } else {
        const u32x4_4 x = *reinterpret_cast<const u32x4_4*>(p);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = x[k];
    }
}

/* Output of a column whose sums over all parts are known.  (One that sees nothing has no
 * maximum and no sum.) */
template <int DT>
__device__ __forceinline__ void put(const AttendArgs& a, int64_t out, int64_t lse, int dim, f32x4 v,
                                    float top, float sum)
{
    const bool none = top == -inf32() && sum == 0.0f;
    v = none ? f32x4{0, 0, 0, 0} : v * (1.0f / sum);
    if (dim < a.pool.head_dim) store4<DT>(a.out.data + (out + dim) * Elem<DT>::SIZE, v);
    if (dim == 0 && a.lse) a.lse[lse] = none ? -inf32() : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

/* rows_shape: tokens of a wave's step, as many as its registers hold beside the sums (16, 32 or 64); waves, of
 * which eight are a CU's (131,071 tokens of 128 dims: 61 us with workgroups of eight, which have half the
 * parts to join, and 65 of four; 12 rows of 3,800 of 512 dims 82 and 67, as their units are then twice as long);
 * and units that a workgroup takes at least where there are enough of them (1, 2 and 4 of them: 49, 39 and 44 us
 * for the windows of 256 dims, 89, 88 and 83 for the searches of 512). */
constexpr int kResident = 8;

template <int DT, int D>
__global__ __launch_bounds__(rows_shape(D).waves * 64, 2) void attend_rows_kernel(AttendArgs a, int joins)
{
    constexpr int NW = rows_shape(D).waves, TT = rows_shape(D).tokens;
    constexpr int UNIT = rows_shape(D).unit();
    constexpr int NB = TT / 16;                     /* blocks of 16 tokens of a step */
    constexpr int NJ = TT < 32 ? 4 : 8;             /* tokens of a lane in a product with V .. */
    constexpr int NH = TT / (4 * NJ);               /* .. of which a step has so many */
    constexpr int QP = DT == G4S_DTYPE_F32 ? 3 : 1; /* pieces of a query */
    constexpr int PP = DT == G4S_DTYPE_F32 ? 3 : 2; /* and of a weight */
    constexpr int KC = D / 64;                      /* 16-dim chunks of a lane of K and Q */
    constexpr int VW = D / 64;                      /* words of a lane of V */
    constexpr int VL = VW < 4 ? VW : 4;             /* of one load */
    constexpr int DB = D / 16;                      /* blocks of 16 dims, and dims of a lane */
    static_assert(2 * kCols * D <= kAttendSums && 4 * kCols <= kAttendStats, "two slots a workgroup");
    extern __shared__ char lds[];
    using S = Shared<DT, D, NW, TT>;
    S& s = *reinterpret_cast<S*>(lds);
    Group* group = reinterpret_cast<Group*>(lds + ((sizeof(S) + 15) & ~(size_t)15));
    int64_t* before = reinterpret_cast<int64_t*>(group + a.rows);
    RowInfo* info = reinterpret_cast<RowInfo*>(before + a.rows + 1);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m = lane & 15, g = lane >> 4;
    if (joins && tid == 0) a.ws.records[blockIdx.x].parts = 0;
    scan_rows<NW, UNIT>(a, info, group, before, s.wave);
    const int64_t total = before[a.rows];
    const int groups = sharing_groups(total, rows_shape(D).units, a.ws.groups / 2, (int)gridDim.x);
    if ((int)blockIdx.x >= groups) return;
    int64_t x = first_unit(total, blockIdx.x, groups);
    const int64_t x_end = first_unit(total, blockIdx.x + 1, groups);
    const float c = base_two(a.scale);
    const __amdgpu_buffer_rsrc_t space = shared_space(a.ws.sums, (uint32_t)a.ws.groups * kAttendSums * 4);

    while (x < x_end) {
        /* the last row whose units begin at or before x: each lane looks at one of 64 stretches */
        int lo = 0;
        for (int n = a.rows; n > 1;) {
            const int each = (n + 63) / 64;
            const uint64_t at = __ballot(lane * each < n && before[lane * each < n ? lo + lane * each : 0] <= x);
            const int last = 63 - __clzll(at | 1);
            lo += last * each;
            n = n - last * each < each ? n - last * each : each;
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        Group p = group[lo];
        p.rows = __builtin_amdgcn_readfirstlane(p.rows);
        p.start = __builtin_amdgcn_readfirstlane(p.start);
        p.from = __builtin_amdgcn_readfirstlane(p.from);
        p.end = __builtin_amdgcn_readfirstlane(p.end);
        p.shared = __builtin_amdgcn_readfirstlane(p.shared);
        const bool several = p.rows > 1; /* rows */
        const int all_cols = group_cols(a, p), blocks = column_blocks(all_cols);
        const int units = group_units<UNIT>(p), first = p.from / UNIT;
        const int64_t in_group = x - before[lo];
        const int item = __builtin_amdgcn_readfirstlane((int)quotient(in_group, units));
        const int u0 = __builtin_amdgcn_readfirstlane((int)(in_group - (int64_t)item * units));
        const int u1 = units - u0 < x_end - x ? units : u0 + (int)(x_end - x);
        const int head = blocks == 1 ? item : item / blocks;
        const int col0 = (item - head * blocks) * kCols;
        const int64_t item_first = x - u0; /* its first unit among all */
        x += u1 - u0;

        /* this lane's query column: token x head, or row x head */
        const int cols = all_cols - col0 < kCols ? all_cols - col0 : kCols;
        const bool has_col = m < cols;
        const int col = col0 + (has_col ? m : 0), nth = divide(col, a.group);
        const int qhead = head * a.group.d + col - nth * a.group.d;
        const int token0 = several ? (a.starts ? a.starts[lo + nth] : lo + nth) : p.start + nth;
        const int place = several ? info[lo + nth].length - 1 : p.end + p.rows + nth;
        const int from = sees_from(a, place);
        if (tid < kCols) {
            s.out[tid] = (int64_t)token0 * a.out.token_stride + (int64_t)qhead * a.out.head_stride;
            s.lse[tid] = token0 * a.heads + qhead;
        }
        {
            const char* q = a.q.data + ((int64_t)token0 * a.q.token_stride +
                                        (int64_t)qhead * a.q.head_stride) * Elem<DT>::SIZE;
            for (int k = wave; k < KC; k += NW) {
                const int d0 = k * 64 + g * 16;
                Frag f[2][QP];
                const bool in = d0 < a.pool.head_dim;
                const char* q0 = q + (int64_t)(in ? d0 : 0) * Elem<DT>::SIZE;
                load_query<DT>(q0, has_col && in, a.scale < 0.0f, f[0]);
                load_query<DT>(q0 + 8 * Elem<DT>::SIZE, has_col && in, a.scale < 0.0f, f[1]);
#pragma unroll
                for (int b = 0; b < QP; ++b) {
                    s.q[k][0][b][lane] = f[0][b];
                    s.q[k][1][b][lane] = f[1][b];
                }
            }
        }
        /* places that all queries see */
        int all_from = from, all_to = place;
        const bool multi = several || p.rows < -1;
        if (multi)
            for (int d = 1; d < kCols; d <<= 1) {
                const int f = __shfl_xor(all_from, d), t = __shfl_xor(all_to, d);
                all_from = f > all_from ? f : all_from;
                all_to = t < all_to ? t : all_to;
            }
        all_from = __builtin_amdgcn_readfirstlane(all_from);
        all_to = __builtin_amdgcn_readfirstlane(all_to);
        /* the part's tiles: first those of all rows, of which the ones before a_shared have the
         * same pages for all, and then units v0 .. v1 - 1 of single rows' tiles */
        const int once = several ? p.shared : units;
        const int s0 = u0 < once ? u0 : once, s1 = u1 < once ? u1 : once;
        const int v0 = u0 - s0, v1 = u1 - s1;
        const int t0 = (first + s0) * UNIT > p.from ? (first + s0) * UNIT : p.from;
        const int t1 = (uint32_t)(first + s1) * UNIT < (uint32_t)p.end ? (first + s1) * UNIT : p.end;
        const int a0 = t0 / TT, a1 = t1 > t0 ? (int)((uint32_t)(t1 + TT - 1) / TT) : a0;
        int a_shared = a1;
        int ref = lo; /* the longest row, whose table has every place */
        if (several) {
            for (int i = 1; i < p.rows; ++i)
                if (info[lo + i].length > info[ref].length) ref = lo + i;
            ref = __builtin_amdgcn_readfirstlane(ref);
            if (tid == 0) s.differs = p.end;
            lds_barrier();
            const int begin = t0 < t1 ? divide(t0, a.pool.page_tokens) : 0;
            const int end = t0 < t1 ? divide(t1 - 1, a.pool.page_tokens) + 1 : 0;
            for (int slot = begin + (tid >> 4); slot < end; slot += NW * 4) {
                if (m >= p.rows) break;
                const int last = info[lo + m].length - 1;
                if (slot < divide(sees_from(a, last), a.pool.page_tokens) ||
                    slot > divide(last, a.pool.page_tokens))
                    continue;
                if (a.table[(int64_t)(lo + m) * a.pool.max_slots + slot] !=
                    a.table[(int64_t)ref * a.pool.max_slots + slot])
                    atomicMin(&s.differs, slot);
            }
        }
        lds_barrier();
        if (several) {
            const int64_t t = (int64_t)s.differs * a.pool.page_tokens.d;
            const int n = t < p.end ? (int)t / TT : a1;
            a_shared = __builtin_amdgcn_readfirstlane(n < a0 ? a0 : n < a1 ? n : a1);
        }

        f32x4 o[DB];
#pragma unroll
        for (int i = 0; i < DB; ++i) o[i] = f32x4{0, 0, 0, 0};
        float base = -inf32(), sum = 0.0f;

        /* steps, every NW-th of them the wave's: a tile for all rows, behind those (i >= 0) a tile
         * for each row that sees it, tile by tile, and then the single rows' units */
        struct Step {
            int tile, i, row; /* row: the table that is read */
            int first, last;  /* first and last place that is read */
        };
        const uint32_t by_rows = several ? 0xFFFFFFFFu / (uint32_t)p.rows + 1u : 0u; /* i / rows = high(i * it) */
        const int mixed = several ? ((a1 - a_shared) * p.rows + NW - 1) & -NW : 0;
        auto settle = [&](Step& t) {
            if (t.i < 0) {
                t.row = ref;
                t.first = p.from;
                t.last = p.end - 1;
                if (t.tile < a_shared) return;
                t.i = t.tile - a_shared;
                t.tile = kNone;
                if (!several) return;
            }
            for (;; t.i += NW) {
                const int v = t.i < mixed ? t.i : v0 + (t.i - mixed) / NW;
                const int q = (int)__umulhi((uint32_t)v, by_rows);
                if (t.i < mixed) {
                    t.tile = a_shared + q;
                    if (t.tile >= a1) continue;
                } else {
                    t.tile = kNone;
                    if (v >= v1) return;
                    t.tile = (first + once + q) * NW + t.i % NW;
                }
                t.row = lo + v - q * p.rows;
                t.last = __builtin_amdgcn_readfirstlane(info[t.row].length - 1);
                t.first = sees_from(a, t.last);
                if (t.tile * TT <= t.last && t.tile * TT + TT > t.first) return;
            }
        };
        auto advance = [&](Step t) {
            if (t.i < 0)
                t.tile += NW;
            else
                t.i += NW;
            settle(t);
            return t;
        };
        /* the lane's token of a step: beyond the ends the one at the end stands in, which some
         * query sees */
        auto token = [&](const Step& t) {
            const int i = t.tile * TT + (lane & (TT - 1));
            return i < t.first ? t.first : i > t.last ? t.last : i;
        };
        auto find_page = [&](const Step& t) {
            return a.table[(int64_t)t.row * a.pool.max_slots + divide(token(t), a.pool.page_tokens)];
        };
        const char* const keys = a.k_plane + (int64_t)head * a.pool.part_bytes;
        const char* const values = a.v_plane + (int64_t)head * a.pool.part_bytes;
        /* where its tokens are, a token a lane, and the keys' and values' scales (by halves of the
         * lanes where there are 32) */
        struct Scales {
            float k = 0.0f, v = 0.0f;
        };
        auto locate = [&](const Step& t, int page, int b, Scales& scale) {
            const int i = token(t);
            const int in = i - divide(i, a.pool.page_tokens) * a.pool.page_tokens.d;
            const bool ok = page >= 0 && page < a.pool.n_pages;
            const int64_t off = (int64_t)(ok ? page : 0) * a.pool.page_stride + in * a.pool.token_bytes;
            const int in_block = in - divide(in, a.pool.scale_tokens) * a.pool.scale_tokens.d;
            const int64_t at = off - in_block * a.pool.token_bytes + a.pool.head_dim;
            if (TT == 64 || lane < 32) s.offset[wave][b][lane & (TT - 1)] = off;
            if constexpr (TT == 64) {
                scale.k = *reinterpret_cast<const float*>(keys + at);
                scale.v = *reinterpret_cast<const float*>(values + at);
            } else {
                scale.k = *reinterpret_cast<const float*>((lane < 32 ? keys : values) + at);
            }
            return (uint64_t)__ballot(!ok);
        };
        /* A token whose page or scale is none is widened under 1, and NaN for who sees it: `bad` with
         * those of the scales. */
        auto keep_scales = [&](int b, const Scales& scale, uint64_t bad) {
            const bool ok = !(bad >> lane & 1) && scale_ok(__float_as_uint(scale.k)) &&
                            (TT < 64 || scale_ok(__float_as_uint(scale.v)));
            if constexpr (TT == 64) {
                s.scale[wave][b][0][lane] = ok ? scale.k : 1.0f;
                s.scale[wave][b][1][lane] = ok ? scale.v : 1.0f;
                return bad | (uint64_t)__ballot(!ok);
            } else {
                s.scale[wave][b][lane >> 5][lane & (TT - 1)] = ok ? scale.k : 1.0f;
                const uint64_t none = __ballot(!ok);
                return bad | none | none >> 32;
            }
        };
        /* (dims behind head_dim, whose queries are 0 and whose sums are not kept, are read in
         * the last ones' place) */
        const int last_key = a.pool.head_dim - 16, last_value = a.pool.head_dim - 4 * VL;
        uint32_t kw[NB][KC][4], vw[NH][NJ][VW];
        auto load_keys = [&](int b) {
#pragma unroll
            for (int h = 0; h < NB; ++h) {
                const char* from = keys + s.offset[wave][b][h * 16 + m];
#pragma unroll
                for (int k = 0; k < KC; ++k) {
                    const int d0 = k * 64 + g * 16;
                    load_words<4>(from + (d0 < last_key ? d0 : last_key), kw[h][k]);
                }
            }
        };
        auto load_values = [&](int b) {
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const char* from = values + s.offset[wave][b][h * 32 + (j & 4) * 4 + g * 4 + (j & 3)];
#pragma unroll
                    for (int i = 0; i < VW; i += VL) {
                        const int d0 = m * DB + 4 * i;
                        uint32_t w[VL];
                        load_words<VL>(from + (d0 < last_value ? d0 : last_value), w);
#pragma unroll
                        for (int k = 0; k < VL; ++k) vw[h][j][i + k] = w[k];
                    }
                }
        };

        Step now{a0 + wave, -1, 0, 0, 0};
        settle(now);
        Step next = now;
        int buf = 0, page = 0;
        uint64_t bad = 0;
        if (now.tile != kNone) {
            Scales scale;
            bad = locate(now, find_page(now), 0, scale);
            wave_fence();
            load_keys(0);
            load_values(0);
            next = advance(now);
            if (next.tile != kNone) page = find_page(next);
            bad = keep_scales(0, scale, bad);
            wave_fence();
        }
        while (now.tile != kNone) {
            const bool more = next.tile != kNone;
            const uint64_t bad_now = bad;
            Scales scale;
            Step after = next;
            if (more) {
                bad = locate(next, page, buf ^ 1, scale);
                wave_fence();
                after = advance(next);
                if (after.tile != kNone) page = find_page(after);
            }

            f32x4 sc[NB];
            float ks[NB];
#pragma unroll
            for (int h = 0; h < NB; ++h) {
                ks[h] = s.scale[wave][buf][0][h * 16 + m];
                sc[h] = f32x4{0, 0, 0, 0};
            }
#pragma unroll
            for (int k = 0; k < KC; ++k) {
                Frag q[2][QP];
#pragma unroll
                for (int b = 0; b < QP; ++b) {
                    q[0][b] = s.q[k][0][b][lane];
                    q[1][b] = s.q[k][1][b][lane];
                }
#pragma unroll
                for (int h = 0; h < NB; ++h) {
                    Frag f[2];
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        f[w >> 1].w[(w & 1) * 2] = widen2<false>(kw[h][k][w], ks[h]);
                        f[w >> 1].w[(w & 1) * 2 + 1] = widen2<true>(kw[h][k][w], ks[h]);
                    }
#pragma unroll
                    for (int b = QP - 1; b >= 0; --b) {
                        sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[0].v, q[0][b].v, sc[h], 0, 0, 0);
                        sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[1].v, q[1][b].v, sc[h], 0, 0, 0);
                    }
                }
            }
            /* one chunk's queries are read ahead (all of them at once would take the registers) */
            __builtin_amdgcn_sched_group_barrier(0x100, NB + 2 * QP, 0);
#pragma unroll
            for (int k = 1; k < KC; ++k) {
                __builtin_amdgcn_sched_group_barrier(0x100, 2 * QP, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 2 * QP * NB, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, 2 * QP * NB, 0);
            if (more) load_keys(buf ^ 1);
            /* y[j] of half h: token h * 32 + (j & 4) * 4 + g * 4 + (j & 3) */
            const int tile0 = now.tile * TT;
            const bool alone = now.i >= 0;
            const bool partly = bad_now != 0 || tile0 < all_from || tile0 + TT - 1 > all_to || alone;
            bool nan_v = false;
            if (partly) {
                /* (bits, as a comparison for each score would hold a mask of lanes for each) */
                const bool mine = !alone || lo + nth == now.row;
                uint64_t seen = seen_bits(tile0, from, place, g * 4);
                seen = mine ? seen : 0;
#pragma unroll
                for (int h = 0; h < NB; ++h)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        sc[h][j] = where_bit(seen, h * 16 + j, sc[h][j], -inf32());
                if (bad_now != 0) {
                    const uint64_t wrong = (bad_now >> (g * 4)) & seen;
#pragma unroll
                    for (int h = 0; h < NB; ++h)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            sc[h][j] = where_bit(wrong, h * 16 + j, nan32(), sc[h][j]);
                }
                if (multi) {
                    uint32_t any = 0;
#pragma unroll
                    for (int h = 0; h < NH; ++h)
#pragma unroll
                        for (int j = 0; j < NJ; ++j)
#pragma unroll
                            for (int w = 0; w < VW; ++w) any |= nan_codes(vw[h][j][w]);
                    nan_v = __any(any != 0);
                }
            }
            /* exponents against the base that holds, and their largest */
            float y[NB][4], most = -inf32();
            const float old = base == -inf32() ? 0.0f : base;
#pragma unroll
            for (int h = 0; h < NB; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    y[h][j] = __builtin_fmaf(sc[h][j], c, -old);
                    most = fmaxf(most, y[h][j]);
                }
            most = column_max(most);
            if (__any(rebase(base, most))) {
                const bool moves = rebase(base, most);
                const float keep = moves && base != -inf32() ? __builtin_amdgcn_exp2f(-most) : 1.0f;
                if (moves) base = old + most;
                sum *= keep;
#pragma unroll
                for (int i = 0; i < DB; ++i) o[i] *= keep;
                const float b = base == -inf32() ? 0.0f : base;
#pragma unroll
                for (int h = 0; h < NB; ++h)
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[h][j] = __builtin_fmaf(sc[h][j], c, -b);
            }
            Frag pw[NH][PP];
#pragma unroll
            for (int h = 0; h < NB; ++h)
#pragma unroll
                for (int j = 0; j < 4; j += 2) {
                    const float e0 = __builtin_amdgcn_exp2f(y[h][j]);
                    const float e1 = __builtin_amdgcn_exp2f(y[h][j + 1]);
                    sum += e0 + e1;
                    Frag* f = pw[h >> 1];
                    const int w = (h & 1) * 2 + (j >> 1);
                    f[0].w[w] = pack_bf16(e0, e1);
                    /* (pieces of eight bits: three are the weight, two are off by 2^-16 at most, which a
                     * bf16 output's own rounding hides and which costs a product less; a
                     * single one is off by 2^-8, as much as that rounding) */
                    const float r0 = e0 - __uint_as_float(f[0].w[w] << 16);
                    const float r1 = e1 - __uint_as_float(f[0].w[w] & 0xFFFF0000u);
                    f[1].w[w] = pack_bf16(r0, r1);
                    if constexpr (PP == 3) {
                        f[2].w[w] = pack_bf16(r0 - __uint_as_float(f[1].w[w] << 16),
                                              r1 - __uint_as_float(f[1].w[w] & 0xFFFF0000u));
                    }
                }
            if (nan_v) {
                /* a NaN that some queries see and others do not (0 times NaN is NaN): the products
                 * go without it, and whoever sees one, counted by a product too, gets NaN */
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    Frag see;
#pragma unroll
                    for (int j = 0; j < NJ; j += 2) {
                        const f32x4 y = sc[h * 2 + (j >> 2)];
                        see.w[j >> 1] = (y[j & 3] == -inf32() ? 0u : 0x3F80u) |
                                        (y[(j & 3) + 1] == -inf32() ? 0u : 0x3F800000u);
                    }
                    float one[NJ];
#pragma unroll
                    for (int j = 0; j < NJ; ++j) one[j] = 1.0f;
#pragma unroll
                    for (int w = 0; w < VW; ++w) {
                        uint32_t is[NJ];
                        Frag f[4];
#pragma unroll
                        for (int j = 0; j < NJ; ++j) {
                            is[j] = nan_codes(vw[h][j][w]) * 0x38u; /* the code of 1 */
                            vw[h][j][w] = without_nan(vw[h][j][w]);
                        }
                        value_frags<NJ>(is, one, f);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const f32x4 n = multiply<NJ>(f[i], see, f32x4{0, 0, 0, 0});
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                o[w * 4 + i][r] = nan_where(o[w * 4 + i][r], n[r]);
                        }
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                float vs[NJ];
#pragma unroll
                for (int j = 0; j < NJ; ++j)
                    vs[j] = s.scale[wave][buf][1][h * 32 + (j & 4) * 4 + g * 4 + (j & 3)];
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    uint32_t word[NJ];
                    Frag f[4];
#pragma unroll
                    for (int j = 0; j < NJ; ++j) word[j] = vw[h][j][w];
                    value_frags<NJ>(word, vs, f);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int b = PP - 1; b >= 0; --b)
                            o[w * 4 + i] = multiply<NJ>(f[i], pw[h][b], o[w * 4 + i]);
                }
            }
            if (more) {
                load_values(buf ^ 1);
                bad = keep_scales(buf ^ 1, scale, bad);
            }
            wave_fence(); /* before what comes after the next tile takes the place of this one */
            buf ^= 1;
            now = next;
            next = after;
        }

        /* the waves join */
        sum = column_sum(sum);
        if (g == 0) {
            s.m[wave][m] = base;
            s.l[wave][m] = sum;
        }
        const bool whole = u0 == 0 && u1 == units;
        const int slot = 2 * (int)blockIdx.x + (u0 == 0);
        lds_barrier();
        if (tid < kCols) {
            float best = s.m[0][tid];
#pragma unroll
            for (int w = 1; w < NW; ++w) best = fmaxf(best, s.m[w][tid]);
            float all = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float f = s.m[w][tid] == -inf32() ? 0.0f : __builtin_amdgcn_exp2f(s.m[w][tid] - best);
                all += s.l[w][tid] * f;
                s.l[w][tid] = f;
            }
            const bool bad_row = !several && info[lo].length < 0;
            best = bad_row ? nan32() : best;
            all = bad_row ? nan32() : all;
            s.top[tid] = best;
            s.sum[tid] = all;
            if (!whole && tid < cols)
                st_dev(reinterpret_cast<uint64_t*>(a.ws.stats + (slot * kCols + tid) * 2),
                       (uint64_t)__float_as_uint(best) | (uint64_t)__float_as_uint(all) << 32);
        }
        constexpr int PD = kPass<D, NW>;
#pragma unroll 1
        for (int pass = 0; pass < D / PD; ++pass) {
            /* lanes with dims of this pass: a lane has DB in each of four rows */
            if (pass > 0) lds_barrier();
            constexpr int GP = PD / (4 * DB); /* lane groups of a pass */
            if (g / GP == pass && m < cols) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int i = 0; i < DB; i += 4)
                        *reinterpret_cast<f32x4*>(&s.o[wave][m][DB * ((g % GP) * 4 + r) + i]) =
                            f32x4{o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]};
            }
            lds_barrier();
            for (int i = tid; i < cols * (PD / 4); i += NW * 64) {
                const int k = i / (PD / 4), d0 = i % (PD / 4) * 4, dim = pass * PD + d0;
                f32x4 v = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < NW; ++w)
                    v += *reinterpret_cast<const f32x4*>(&s.o[w][k][d0]) * s.l[w][k];
                if (whole)
                    put<DT>(a, s.out[k], s.lse[k], dim, v, s.top[k], s.sum[k]);
                else
                    st_dev4(space, (uint32_t)((slot * kCols + k) * D + dim) * 4, v);
            }
        }
        if (!whole) {
            const int w_first = unit_group(item_first, total, groups);
            const int parts = unit_group(item_first + units - 1, total, groups) - w_first + 1;
            if (joins && parts * cols * D * 4 > kJoinBytes) {
                if (tid == 0 && u0 == 0)
                    a.ws.records[blockIdx.x] = AttendRecord{parts, cols, col0, head * a.group.d, lo,
                                                            several ? -1 : p.start};
            } else if (elect_last(&a.ws.tickets[w_first], (uint32_t)parts, &s.flag)) {
                /* the last of the workgroups that have a part of this item joins them */
                for (int i = tid; i < cols * (D / 4); i += NW * 64) {
                    const int k = i / (D / 4), dim = i % (D / 4) * 4;
                    if (dim >= a.pool.head_dim) continue;
                    Joined j;
                    constexpr int N = 8; /* parts in flight */
                    for (int w0 = 0; w0 < parts; w0 += N) {
                        float2 st[N];
                        f32x4 part[N];
#pragma unroll
                        for (int w = 0; w < N; ++w) {
                            const int n = w0 + w < parts ? w0 + w : parts - 1;
                            const int from = (2 * (w_first + n) + (n == 0)) * kCols + k;
                            const uint64_t u = ld_dev(reinterpret_cast<const uint64_t*>(a.ws.stats + from * 2));
                            st[w] = make_float2(__uint_as_float((uint32_t)u),
                                                __uint_as_float((uint32_t)(u >> 32)));
                            part[w] = ld_dev4(space, (uint32_t)(from * D + dim) * 4);
                        }
                        join(j, parts - w0, st, part);
                    }
                    put<DT>(a, s.out[k], s.lse[k], dim, j.v, j.top, j.sum);
                }
            }
        }
        lds_barrier(); /* the next part's columns and queries take the place of these */
    }
}

/* The parts that are left to it, joined: two columns a workgroup, four dims a thread, the parts dealt
 * out to as many threads as there are. */
constexpr int kJoinCols = 2;
template <int DT, int D>
__global__ __launch_bounds__(kB) void join_rows_kernel(AttendArgs a)
{
    constexpr int QUADS = kJoinCols * D / 4, DEAL = kB > QUADS ? kB / QUADS : 1;
    __shared__ f32x4 s_v[DEAL][QUADS];
    __shared__ float2 s_st[DEAL][QUADS];
    const AttendRecord r = a.ws.records[blockIdx.x];
    const int deal = threadIdx.x / QUADS, i = threadIdx.x % QUADS;
    const int k = blockIdx.y * kJoinCols + i / (D / 4), dim = i % (D / 4) * 4;
    if (r.parts == 0 || (int)blockIdx.y * kJoinCols >= r.cols) return;
    Joined j;
    constexpr int N = 8; /* parts in flight */
    const int col = k < r.cols ? k : 0;
    for (int w0 = deal; w0 < r.parts; w0 += N * DEAL) {
        float2 st[N];
        f32x4 part[N];
#pragma unroll
        for (int w = 0; w < N; ++w) {
            const int n = w0 + w * DEAL < r.parts ? w0 + w * DEAL : r.parts - 1;
            const int slot = 2 * ((int)blockIdx.x + n) + (n == 0);
            st[w] = *reinterpret_cast<const float2*>(a.ws.stats + (slot * kCols + col) * 2);
            part[w] = *reinterpret_cast<const f32x4*>(a.ws.sums + (int64_t)(slot * kCols + col) * D + dim);
        }
        join(j, (r.parts - w0 + DEAL - 1) / DEAL, st, part);
    }
    s_v[deal][i] = j.v;
    s_st[deal][i] = make_float2(j.top, j.sum);
    __syncthreads();
    if (deal > 0 || k >= r.cols) return;
    Joined all;
    float2 st[DEAL];
    f32x4 part[DEAL];
#pragma unroll
    for (int w = 0; w < DEAL; ++w) {
        st[w] = s_st[w][i];
        part[w] = s_v[w][i];
    }
    join(all, DEAL, st, part);
    const int c = r.col0 + k, nth = divide(c, a.group);
    const int token = r.start >= 0 ? r.start + nth : a.starts ? a.starts[r.row + nth] : r.row + nth;
    const int head = r.head0 + c - nth * a.group.d;
    put<DT>(a, (int64_t)token * a.out.token_stride + (int64_t)head * a.out.head_stride,
            (int64_t)token * a.heads + head, dim, all.v, all.top, all.sum);
}

template <int DT, int D>
hipError_t rows_launch(const AttendArgs& a, hipStream_t stream)
{
    constexpr int NW = rows_shape(D).waves, TT = rows_shape(D).tokens, UNIT = rows_shape(D).unit();
    const size_t lds = ((sizeof(Shared<DT, D, NW, TT>) + 15) & ~(size_t)15) + ((size_t)a.rows + 1) * 8 +
                       (size_t)a.rows * (sizeof(RowInfo) + sizeof(Group));
    /* no more workgroups than the rows can have use for */
    const int64_t most = most_units(a.rows, a.tokens, a.starts, a.kv_heads, a.group.d, a.few,
                                    cache_room(a.pool), UNIT);
    const int64_t units = (cache_room(a.pool) + UNIT - 1) / UNIT + 1;
    const int64_t together = kCols / a.group.d < 1 ? 1 : kCols / a.group.d < a.rows ? kCols / a.group.d : a.rows;
    const int resident = a.ws.groups / 2 * (kResident / NW);
    const int groups = most < resident ? (int)most : resident;
    /* the most that can be left to be joined of one item, of one row's tokens or of rows that are taken
     * together: a launch of its own is enqueued only where it may have something to do */
    const int64_t cols = (int64_t)a.tokens * a.group.d < kCols ? (int64_t)a.tokens * a.group.d : kCols;
    const int64_t share = groups / a.kv_heads + 2;
    const int64_t parts = units < share ? units : share;
    const int64_t parts_of_all = units * together < share ? units * together : share;
    const int64_t cols_of_all = together * a.group.d < kCols ? together * a.group.d : kCols;
    const int64_t one = parts * cols, all = parts_of_all * cols_of_all;
    const int joins = (one > all ? one : all) * D * 4 > kJoinBytes;
    hipError_t e = launch(attend_rows_kernel<DT, D>, groups, NW * 64, lds, stream, a, joins);
    if (e != hipSuccess || !joins) return e;
    return launch(join_rows_kernel<DT, D>, dim3((unsigned)groups, (unsigned)(kCols / kJoinCols)), kB, 0,
                  stream, a);
}

template <int DT>
hipError_t by_width(const AttendArgs& a, hipStream_t stream)
{
    switch (attend_width(a.pool.head_dim)) {
    case 64: return rows_launch<DT, 64>(a, stream);
    case 128: return rows_launch<DT, 128>(a, stream);
    case 256: return rows_launch<DT, 256>(a, stream);
    default: return rows_launch<DT, 512>(a, stream);
    }
}

__global__ void attend_init_kernel(uint32_t* tickets, int n)
{
    for (int i = blockIdx.x * kB + threadIdx.x; i < n; i += gridDim.x * kB) tickets[i] = 0u;
}

}  // namespace

int32_t attend_groups(int32_t ncu) { return 2 * ncu; }

hipError_t attend_init_launch(const AttendSpace& ws, hipStream_t stream)
{
    return launch(attend_init_kernel, 4, kB, 0, stream, ws.tickets, ws.groups);
}

hipError_t attend_rows_launch(const AttendArgs& a, int32_t dtype, hipStream_t stream)
{
    return dtype == G4S_DTYPE_F32 ? by_width<G4S_DTYPE_F32>(a, stream)
                                  : by_width<G4S_DTYPE_BF16>(a, stream);
}

}  // namespace g4s
