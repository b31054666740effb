/*
 * g4s_prompt.hip -- attention over the pages of an 8-bit cache for rows with many queries
 * (prompts and chunks of them), on gfx950.
 *
 * A workgroup takes NW x NT x 16 query columns (tokens x heads of one key head) and goes over the
 * tokens that they see in tiles of KT: all its threads widen the next tile's codes into LDS, keys as
 * [token][dim] and values as [dim][token], while its waves multiply the present one, each
 * for NT x 16 columns of its own with the softmax in registers: K Q^T leaves a lane scores of one column,
 * which are an operand of V^T P^T as they are.  The exponents' base moves only when a score passes it
 * by 2^8, so that the sums are seldom multiplied.  Where there are fewer columns than
 * workgroups the tokens are split too, and a second launch joins what the parts of a block
 * found, in their order.
 *
 * Four prompts of 4,000 tokens, 32 and 8 heads of 128 dims: 910 us, 646 TFLOP/s of the 1,260 that a large
 * bf16 product reaches here (three products for two, as the weights are in two pieces: 747 us with one).  No single
 * unit is the bound: vector instructions (exponentials, weights, widened codes) are issued in 57% of the cycles,
 * the matrix units work in 42%, LDS in 39% (18% of all on bank conflicts), and they hardly overlap.  256 tokens
 * behind 7,844, 8 and 2 heads of 256 dims: 53 us (314 TFLOP/s), of which the joining launch is 8 and start and
 * end 10: a wave's 16 columns are all that its registers hold beside their sums, so that LDS, busy in 51% of the
 * cycles (22% of all on conflicts), is read once for each 16.  Binary32 costs three times the products: the first
 * prompts 1.60 ms.  Dims between head_dim and the width that a kernel is made for are multiplied too.
 */
#include "g4s_attend.h"
#include "g4s_launch.h"

namespace g4s {

namespace {

/* Values lie in rows of KT tokens (2 KT bytes) without padding; their 16-byte pieces are
 * exchanged by the dim, so that neither eight dims at one place nor a thread's four times
 * two meet in one bank. */
template <int KT>
__device__ __forceinline__ int value_piece(int dim, int piece)
{
    return piece ^ ((dim ^ (dim >> 3)) & (KT / 8 - 1));
}

/* A block of a row's query columns for each key head, and the tiles of the tokens
 * that its queries see; no columns where a slot of the grid has none. */
struct Block {
    RowTokens r;
    int row, col0, cols;
    int from, end;    /* places that any of its queries sees */
    int first, tiles; /* tiles of them */
    int parts;        /* workgroups that share the tiles */
};
__device__ __forceinline__ Block find_block(const AttendArgs& a, int64_t x, int unit, int tile,
                                            int splits)
{
    Block b{};
    b.row = find_share(a.starts, a.rows, x, a.group.d, unit, 1);
    b.r = row_tokens(a.starts, a.lengths, b.row, a.tokens, cache_room(a.pool));
    const int64_t block = x - share_begin(a.starts, b.row, a.group.d, unit, 1);
    const int64_t all = (int64_t)b.r.count * a.group.d;
    if (!is_prompt(b.r.count, a.group.d, a.few) || block < 0 || block * unit >= all) return b;
    b.col0 = (int)(block * unit);
    b.cols = all - b.col0 < unit ? (int)(all - b.col0) : unit;
    const int before = b.r.length - b.r.count;
    b.from = sees_from(a, before + divide(b.col0, a.group));
    b.end = before + divide(b.col0 + b.cols - 1, a.group) + 1;
    b.first = b.from / tile;
    b.tiles = b.end > b.from ? (b.end + tile - 1) / tile - b.first : 0;
    b.parts = b.tiles < 2 ? 1 : b.tiles < splits ? b.tiles : splits;
    return b;
}

/* A query column: the token it is of, its head and place. */
struct Column {
    int nth, head, place;
};
__device__ __forceinline__ Column column(const AttendArgs& a, const RowTokens& r, int kv_head, int col)
{
    const int nth = divide(col, a.group);
    return Column{nth, kv_head * a.group.d + col - nth * a.group.d, r.length - r.count + nth};
}
template <int DT>
__device__ __forceinline__ void put(const AttendArgs& a, const RowTokens& r, const Column& c, int dim,
                                    f32x4 v)
{
    if (dim >= a.pool.head_dim) return;
    if (r.bad) v = f32x4{nan32(), nan32(), nan32(), nan32()};
    else if (c.place < 0) v = f32x4{0, 0, 0, 0};
    store4<DT>(a.out.data + ((int64_t)(r.start + c.nth) * a.out.token_stride +
                             (int64_t)c.head * a.out.head_stride + dim) * Elem<DT>::SIZE, v);
}
__device__ __forceinline__ void put_lse(const AttendArgs& a, const RowTokens& r, const Column& c,
                                        float top, float sum)
{
    if (a.lse)
        a.lse[(int64_t)(r.start + c.nth) * a.heads + c.head] =
            r.bad ? nan32() : c.place < 0 ? -inf32() : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

/* x, computed anew where it is used: what follows from it is not kept in registers over a
 * loop. */
__device__ __forceinline__ int again(int x)
{
    asm volatile("" : "+v"(x));
    return x;
}

constexpr int kSlotSums = 2 * kAttendSums, kSlotStats = 2 * kAttendStats;
constexpr int kJoin = 256; /* threads of a joining workgroup */

template <int D, int NW, int KT, int NV, int HALVES>
struct Shared {
    alignas(16) uint16_t k[2][KT][D + 8];
    alignas(16) uint16_t v[NV][D][KT];
    f32x4 part[HALVES == 2 ? NW : 0][KT / 16][64]; /* products of keys with half of the dims */
    int64_t offset[3][KT];
    float scale[3][2][KT];
    uint64_t bad[3];
    int nan; /* whether any value so far was one */
};

/* Waves that share columns, each with a part of their dims: one wave's registers do not hold the
 * queries and sums of 512 (256 tokens behind 7,844, weights in one piece: 112 us and, binary32, 140; alone 169
 * and 425.  Now 118 and 146). */
template <int D>
constexpr int kHalves = D > 256 ? 2 : 1;
/* LDS holds a third tile of values, so that waves may be a phase apart (the four prompts: 910 us, 950 in
 * step; binary32 1,596 and 1,669; with 64 dims 736 and 715, binary32 947 and 976). */
template <int D>
constexpr bool kLate = D <= 128;

/* `steps` reads of a matrix operand from LDS and `each` products with it, as the compiler is to lay
 * them out: kAhead reads ahead of their products.  Left to itself it reads everything first
 * and spills registers. */
constexpr int kAhead = 4;
template <int STEPS, int EACH>
__device__ __forceinline__ void lay_out()
{
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
    for (int i = 0; i < STEPS - kAhead; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, EACH * kAhead, 0);
}

template <int DT, int D, int NW, int NT, int KT>
__global__ __launch_bounds__(NW * 64, NW == 4 ? 2 : NW / 4) void attend_prompts_kernel(AttendArgs a, int splits)
{
    constexpr int QP = DT == G4S_DTYPE_F32 ? 3 : 1;
    constexpr int PP = DT == G4S_DTYPE_F32 ? 3 : 2;
    constexpr int HALVES = kHalves<D>, COLW = NW / HALVES, DW = D / HALVES; /* a wave's dims */
    constexpr int CB = COLW * NT * 16;
    constexpr int KS = DW / 32, DB = DW / 16, TB = KT / 16;
    constexpr int THREADS = NW * 64;
    constexpr bool LATE = kLate<D>;
    constexpr int NV = LATE ? 3 : 2;
    constexpr int KL = (KT * D / 16 + THREADS - 1) / THREADS; /* 16-code loads of a thread */
    /* values: units of 8 tokens x 4 codes, or of 4 where that would leave threads without any */
    constexpr int VT = KT * D / 32 >= THREADS ? 8 : 4;
    constexpr int VU = KT * D / 4 / VT;
    constexpr int VL = (VU + THREADS - 1) / THREADS;
    static_assert(CB * D <= kSlotSums && CB * 2 <= kSlotStats, "a slot a workgroup");
    extern __shared__ char lds[];
    auto& s = *reinterpret_cast<Shared<D, NW, KT, NV, HALVES>*>(lds);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int colw = wave % COLW, dim0 = wave / COLW * DW;
    const int m = lane & 15, g = lane >> 4;

    /* heads side by side; the last columns of a row, which see most, first */
    const int slots = (int)(gridDim.x / (uint32_t)a.kv_heads);
    const int head = (int)(blockIdx.x % (uint32_t)a.kv_heads), part = blockIdx.z;
    const int64_t x = slots - 1 - (int)(blockIdx.x / (uint32_t)a.kv_heads);
    const Block b = find_block(a, x, CB, KT, splits);
    if (b.cols == 0 || part >= b.parts) return;
    const RowTokens r = b.r;
    const int row = b.row, col0 = b.col0, cols = b.cols, parts = b.parts;
    const int from0 = b.from, end0 = b.end, t_first = b.first;
    const int n0 = (int)((int64_t)b.tiles * part / parts);
    const int n1 = (int)((int64_t)b.tiles * (part + 1) / parts);

    /* this lane's columns */
    int place[NT], from[NT];
    Frag q[NT][KS][QP];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int c = (colw * NT + t) * 16 + m;
        const bool has = c < cols;
        const Column at = column(a, r, head, col0 + (has ? c : 0));
        place[t] = at.place;
        from[t] = sees_from(a, at.place);
        const char* q0 = a.q.data + ((int64_t)(r.start + at.nth) * a.q.token_stride +
                                     (int64_t)at.head * a.q.head_stride) * Elem<DT>::SIZE;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const int d0 = dim0 + k * 32 + g * 8;
            const bool in = d0 < a.pool.head_dim;
            load_query<DT>(q0 + (int64_t)(in ? d0 : 0) * Elem<DT>::SIZE, has && in, a.scale < 0.0f,
                           q[t][k]);
        }
    }
    /* places that any and that all of the wave's queries see */
    const int wcol0 = colw * NT * 16;
    const int wcol1 = wcol0 + NT * 16 < cols ? wcol0 + NT * 16 : cols;
    const bool busy = wcol0 < cols;
    const int w_first = r.length - r.count + divide(col0 + (busy ? wcol0 : 0), a.group);
    const int w_last = r.length - r.count + divide(col0 + (busy ? wcol1 - 1 : 0), a.group);
    const int any_from = sees_from(a, w_first), all_from = sees_from(a, w_last);

    const float c = base_two(a.scale);
    f32x4 o[NT][DB];
    float base[NT], sum[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        base[t] = -inf32();
        sum[t] = 0.0f;
#pragma unroll
        for (int i = 0; i < DB; ++i) o[t][i] = f32x4{0, 0, 0, 0};
    }

    /* Where the tokens of a tile are, found by the first wave in three steps of a tile each, so that
     * it waits for none of them: their pages, their scales, and both to LDS. */
    const int32_t* pages = a.table + (int64_t)row * a.pool.max_slots;
    const bool locates = wave == 0;
    int page = 0, in_page = 0;
    float k_scale = 0.0f, v_scale = 0.0f;
    int64_t offset = 0;
    uint64_t wrong = 0;
    auto find_pages = [&](int n) {
        if (!locates || n >= n1) return;
        int t = (t_first + n) * KT + (lane & (KT - 1));
        t = t < from0 ? from0 : t >= end0 ? end0 - 1 : t;
        const int slot = divide(t, a.pool.page_tokens);
        in_page = t - slot * a.pool.page_tokens.d;
        page = pages[slot];
    };
    auto find_scales = [&](int n) {
        if (!locates || n >= n1) return;
        const bool ok = page >= 0 && page < a.pool.n_pages;
        offset = cache_offset(a.pool, ok ? page : 0, in_page, head);
        const int in_block = in_page - divide(in_page, a.pool.scale_tokens) * a.pool.scale_tokens.d;
        const int64_t at = offset - (int64_t)in_block * a.pool.token_bytes + a.pool.head_dim;
        k_scale = *reinterpret_cast<const float*>(a.k_plane + at);
        v_scale = *reinterpret_cast<const float*>(a.v_plane + at);
        wrong = __ballot(!ok);
    };
    auto keep_places = [&](int n) {
        if (!locates || n >= n1) return;
        const int b = n % 3, i = lane & (KT - 1);
        /* (a token whose page or scale is none is widened under 1, and NaN for who sees it) */
        const bool ok = !(wrong >> lane & 1) && scale_ok(__float_as_uint(k_scale)) &&
                        scale_ok(__float_as_uint(v_scale));
        s.offset[b][i] = offset;
        s.scale[b][0][i] = ok ? k_scale : 1.0f;
        s.scale[b][1][i] = ok ? v_scale : 1.0f;
        const uint64_t bad = __ballot(!ok);
        if (lane == 0) s.bad[b] = bad;
    };
    /* a unit's first token */
    auto unit_token = [](int i) { return VT == 8 ? i / 4 * 32 + i % 4 * 4 : i * 4; };
    uint32_t kw[KL][4], vw[VL][VT];
    auto load = [&](int n) {
        const int b = n % 3;
        const int tid = D > 128 ? again(threadIdx.x) : (int)threadIdx.x;
#pragma unroll
        for (int i = 0; i < KL; ++i) {
            const int u = tid + i * THREADS, t = u / (D / 16), d0 = u % (D / 16) * 16;
            if (KT * D / 16 % THREADS == 0 || u < KT * D / 16) {
                const u32x4_4 w = *reinterpret_cast<const u32x4_4*>(
                    a.k_plane + s.offset[b][t] + (d0 < a.pool.head_dim ? d0 : 0));
#pragma unroll
                for (int j = 0; j < 4; ++j) kw[i][j] = w[j];
            }
        }
#pragma unroll
        for (int i = 0; i < VL; ++i) {
            const int u = tid + i * THREADS, d0 = u % (D / 4) * 4;
            if (VU % THREADS == 0 || u < VU) {
                const int64_t* at = &s.offset[b][unit_token(u / (D / 4))];
                const char* from = a.v_plane + (d0 < a.pool.head_dim ? d0 : 0);
#pragma unroll
                for (int j = 0; j < VT; ++j)
                    vw[i][j] = *reinterpret_cast<const uint32_t*>(from + at[(j & 4) * 4 + (j & 3)]);
            }
        }
    };
    auto store = [&](int n) {
        const int b = n % 3, to = n & 1;
        const int tid = D > 128 ? again(threadIdx.x) : (int)threadIdx.x;
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < KL; ++i) {
            const int u = tid + i * THREADS, t = u / (D / 16), d0 = u % (D / 16) * 16;
            if (KT * D / 16 % THREADS == 0 || u < KT * D / 16) {
                const float ks = s.scale[b][0][t];
                u32x4 lo, hi;
                lo[0] = widen2<false>(kw[i][0], ks), lo[1] = widen2<true>(kw[i][0], ks);
                lo[2] = widen2<false>(kw[i][1], ks), lo[3] = widen2<true>(kw[i][1], ks);
                hi[0] = widen2<false>(kw[i][2], ks), hi[1] = widen2<true>(kw[i][2], ks);
                hi[2] = widen2<false>(kw[i][3], ks), hi[3] = widen2<true>(kw[i][3], ks);
                u32x4* at = reinterpret_cast<u32x4*>(&s.k[to][t][d0]);
                at[0] = lo;
                at[1] = hi;
            }
        }
        /* piece 4 h + g of a dim: tokens 4 g .. 4 g + 3 of 32 h and those 16 behind them, in the order
         * that a lane of the second product takes them */
#pragma unroll
        for (int i = 0; i < VL; ++i) {
            const int u = tid + i * THREADS, d0 = u % (D / 4) * 4, t = unit_token(u / (D / 4));
            if (VU % THREADS == 0 || u < VU) {
                float vs[VT];
                Frag f[4];
#pragma unroll
                for (int j = 0; j < VT; ++j) {
                    vs[j] = s.scale[b][1][t + (j & 4) * 4 + (j & 3)];
                    any |= nan_codes(vw[i][j]);
                }
                value_frags<VT>(vw[i], vs, f);
                const int piece = t / 32 * 4 + t % 16 / 4;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint16_t* to = &s.v[n % NV][d0 + j][value_piece<KT>(d0 + j, piece) * 8 + t % 32 / 16 * 4];
                    if constexpr (VT == 8) *reinterpret_cast<bf16x8*>(to) = f[j].v;
                    else *reinterpret_cast<uint2*>(to) = make_uint2(f[j].w[0], f[j].w[1]);
                }
            }
        }
        if (__any(any != 0) && lane == 0) s.nan = 1;
    };

    /* the sums of tile n's values; `nan`: some of them may be NaN, and not all queries see all of them */
    Frag pw[NT][TB / 2][PP];
    auto add_values = [&](int n, bool nan_v) {
        /* value_piece(i * 16 + m, h * 4 + g) is that of m and g, exchanged by 2 i and 4 h: few
         * addresses for all */
        const char* const v0 = reinterpret_cast<const char*>(&s.v[n % NV][dim0 + m][0]);
        const int piece = value_piece<KT>(m, g);
        auto value = [&](int i, int h) {
            const int p = piece ^ (((h * 4) ^ (i * 2)) & (KT / 8 - 1));
            Frag f;
            f.v = *reinterpret_cast<const bf16x8*>(v0 + p * 16 + i * 16 * KT * 2);
            return f;
        };
        if (!nan_v) {
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int h = 0; h < TB / 2; ++h) {
                    const Frag f = value(i, h);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int p = PP - 1; p >= 0; --p)
                            o[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.v, pw[t][h][p].v, o[t][i], 0, 0, 0);
                }
            lay_out<DB * TB / 2, NT * PP>();
        } else {
            /* a NaN that some queries see and others do not (0 times NaN is NaN): the
             * products go without it, and whoever sees one, counted by a product too,
             * gets NaN */
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int h = 0; h < TB / 2; ++h) {
                    Frag f = value(i, h), is;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        /* (an exponent of ones carries into the sign's bit) */
                        const uint32_t nan = ((((f.w[w] & 0x7F807F80u) + 0x00800080u) & 0x80008000u) >> 15) * 0xFFFFu;
                        f.w[w] &= ~nan;
                        is.w[w] = nan & 0x3F803F80u;
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        Frag see; /* 1 for the tokens that the column sees */
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const int at = (t_first + n) * KT + h * 32 + (w & 2) * 8 + g * 4 + (w & 1) * 2;
                            see.w[w] = (at >= from[t] && at <= place[t] ? 0x3F80u : 0u) |
                                       (at + 1 >= from[t] && at + 1 <= place[t] ? 0x3F800000u : 0u);
                        }
                        const f32x4 e = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            is.v, see.v, f32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            o[t][i][j] = nan_where(o[t][i][j], e[j]);
#pragma unroll
                        for (int p = PP - 1; p >= 0; --p)
                            o[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.v, pw[t][h][p].v, o[t][i], 0, 0, 0);
                    }
                }
        }
    };
    /* Half of the waves add a tile's values while the others, on the same SIMDs, multiply the next
     * tile's keys, and the other way round: matrix products of one beside the exponentials of the
     * other. */
    const bool late = LATE && wave >= NW / 2;
    int before = -1; /* a late wave's tile whose values are still to be added */
    bool before_nan = false;

    if (tid == 0) s.nan = 0;
    find_pages(n0);
    find_scales(n0);
    find_pages(n0 + 1);
    keep_places(n0);
    find_scales(n0 + 1);
    find_pages(n0 + 2);
    keep_places(n0 + 1);
    lds_barrier();
    if (n0 < n1) {
        load(n0);
        store(n0);
    }
    lds_barrier();
    for (int n = n0; n < n1; ++n) {
        if (n + 1 < n1) load(n + 1);
        find_scales(n + 2);
        find_pages(n + 3);
        const int t0 = (t_first + n) * KT;
        const int buf = n & 1;
        if (before >= 0) {
            add_values(before, before_nan);
            before = -1;
        }
        const bool sees = busy && t0 <= w_last && t0 + KT > any_from;
        f32x4 sc[NT][TB];
        if (sees) {
#pragma unroll
            for (int b = 0; b < TB; ++b) {
#pragma unroll
                for (int t = 0; t < NT; ++t) sc[t][b] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    const bf16x8 f = *reinterpret_cast<const bf16x8*>(&s.k[buf][b * 16 + m][dim0 + k * 32 + g * 8]);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int p = QP - 1; p >= 0; --p)
                            sc[t][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, q[t][k][p].v, sc[t][b], 0, 0, 0);
                }
            }
            lay_out<TB * KS, NT * QP>();
        }
        if constexpr (HALVES == 2) {
            static_assert(NT == 1, "one block of columns a wave");
            if (sees)
#pragma unroll
                for (int b = 0; b < TB; ++b) s.part[wave][b][lane] = sc[0][b];
            lds_barrier();
            if (sees)
#pragma unroll
                for (int b = 0; b < TB; ++b) sc[0][b] += s.part[wave ^ COLW][b][lane];
        }
        if (sees) {
            const uint64_t bad = s.bad[n % 3];
            const bool partly = bad != 0 || t0 < all_from || t0 + KT - 1 > w_first;
            const bool nan_v = partly && s.nan != 0;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if (partly) {
                    const uint64_t seen = seen_bits(t0, from[t], place[t], g * 4);
#pragma unroll
                    for (int b = 0; b < TB; ++b)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            sc[t][b][i] = where_bit(seen, b * 16 + i, sc[t][b][i], -inf32());
                    if (bad != 0) {
                        const uint64_t none = (bad >> (g * 4)) & seen;
#pragma unroll
                        for (int b = 0; b < TB; ++b)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                sc[t][b][i] = where_bit(none, b * 16 + i, nan32(), sc[t][b][i]);
                    }
                }
                /* exponents against the base that holds, and their largest */
                float y[TB * 4], now = -inf32();
                const float old = base[t] == -inf32() ? 0.0f : base[t];
#pragma unroll
                for (int i = 0; i < TB * 4; ++i) {
                    y[i] = __builtin_fmaf(sc[t][i >> 2][i & 3], c, -old);
                    now = fmaxf(now, y[i]);
                }
                now = column_max(now);
                if (__any(rebase(base[t], now))) {
                    const bool moves = rebase(base[t], now);
                    const float keep = moves && base[t] != -inf32() ? __builtin_amdgcn_exp2f(-now) : 1.0f;
                    if (moves) base[t] = old + now;
                    sum[t] *= keep;
#pragma unroll
                    for (int i = 0; i < DB; ++i) o[t][i] *= keep;
                    const float b = base[t] == -inf32() ? 0.0f : base[t];
#pragma unroll
                    for (int i = 0; i < TB * 4; ++i) y[i] = __builtin_fmaf(sc[t][i >> 2][i & 3], c, -b);
                }
#pragma unroll
                for (int i = 0; i < TB * 4; i += 2) {
                    const float e0 = __builtin_amdgcn_exp2f(y[i]), e1 = __builtin_amdgcn_exp2f(y[i + 1]);
                    sum[t] += e0 + e1;
                    Frag* f = pw[t][i >> 3];
                    const int w = (i & 7) >> 1;
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
            }
            if (late) {
                before = n;
                before_nan = nan_v;
            } else {
                add_values(n, nan_v);
            }
        }
        if (n + 1 < n1) store(n + 1);
        keep_places(n + 2);
        lds_barrier();
    }
    if (before >= 0) add_values(before, before_nan);

    /* what the workgroup found */
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        sum[t] = column_sum(sum[t]);
        const int k = (colw * NT + t) * 16 + m;
        if (k >= cols) continue;
        if (parts == 1) {
            const Column at = column(a, r, head, col0 + k);
            const float inv = 1.0f / sum[t];
#pragma unroll
            for (int i = 0; i < DB; ++i) put<DT>(a, r, at, dim0 + i * 16 + g * 4, o[t][i] * inv);
            if (g == 0 && dim0 == 0) put_lse(a, r, at, base[t], sum[t]);
            continue;
        }
        const int64_t slot = (x * a.kv_heads + head) * splits + part;
        float* to = a.ws.sums + slot * kSlotSums + (int64_t)k * D;
#pragma unroll
        for (int i = 0; i < DB; ++i) *reinterpret_cast<f32x4*>(to + dim0 + i * 16 + g * 4) = o[t][i];
        if (g == 0 && dim0 == 0)
            *reinterpret_cast<float2*>(a.ws.stats + slot * kSlotStats + k * 2) =
                make_float2(base[t], sum[t]);
    }
}

/* What the parts of each block of columns found, joined: four dims of a column a thread.  A launch of
 * its own, as a block's parts are up to 128 KiB each: one workgroup took 200 us to join 14 of them. */
template <int DT, int D, int CB, int KT>
__global__ __launch_bounds__(kJoin) void join_prompts_kernel(AttendArgs a, int splits)
{
    const int head = (int)(blockIdx.x % (uint32_t)a.kv_heads);
    const int64_t x = blockIdx.x / (uint32_t)a.kv_heads;
    const Block b = find_block(a, x, CB, KT, splits);
    if (b.cols == 0 || b.parts == 1) return;
    const int i = blockIdx.z * kJoin + threadIdx.x, k = i / (D / 4), dim = i % (D / 4) * 4;
    if (k >= b.cols || dim >= a.pool.head_dim) return;
    const int64_t slot = (x * a.kv_heads + head) * splits;
    const float* stats = a.ws.stats + slot * kSlotStats + k * 2;
    const float* sums = a.ws.sums + slot * kSlotSums + (int64_t)k * D + dim;
    Joined j;
    constexpr int N = 8; /* parts in flight */
    for (int w0 = 0; w0 < b.parts; w0 += N) {
        float2 st[N];
        f32x4 p[N];
#pragma unroll
        for (int w = 0; w < N; ++w) {
            const int64_t n = w0 + w < b.parts ? w0 + w : b.parts - 1;
            st[w] = *reinterpret_cast<const float2*>(stats + n * kSlotStats);
            p[w] = *reinterpret_cast<const f32x4*>(sums + n * kSlotSums);
        }
        join(j, b.parts - w0, st, p);
    }
    const Column at = column(a, b.r, head, b.col0 + k);
    put<DT>(a, b.r, at, dim, j.v * (1.0f / j.sum));
    if (dim == 0) put_lse(a, b.r, at, j.top, j.sum);
}

template <int DT, int D, int NW, int NT, int KT>
hipError_t prompts_launch(const AttendArgs& a, hipStream_t stream)
{
    constexpr int CB = NW / kHalves<D> * NT * 16;
    const int64_t slots = (int64_t)a.tokens * a.group.d / CB + a.rows;
    const int64_t items = slots * a.kv_heads;
    int64_t splits = a.ws.groups / 2 / items;
    splits = splits < 1 ? 1 : splits > 64 ? 64 : splits;
    /* (in x, as the other two hold 2^16 - 1 each) */
    const dim3 grid((unsigned)items, 1, (unsigned)splits);
    const hipError_t e = launch(attend_prompts_kernel<DT, D, NW, NT, KT>, grid, NW * 64,
                                sizeof(Shared<D, NW, KT, (kLate<D> ? 3 : 2), kHalves<D>>), stream, a, (int)splits);
    if (e != hipSuccess || splits == 1) return e;
    const dim3 join((unsigned)items, 1, (unsigned)(CB * D / 4 / kJoin));
    return launch(join_prompts_kernel<DT, D, CB, KT>, join, kJoin, 0, stream, a, (int)splits);
}

template <int DT>
hipError_t by_width(const AttendArgs& a, hipStream_t stream)
{
    constexpr bool F32 = DT == G4S_DTYPE_F32;
    /* (32 columns a wave where they fit: with 256 dims, in four waves, they take 146 us for the chunk instead of
     * 54; 64 dims in eight waves 742 us, in four 736) */
    switch (attend_width(a.pool.head_dim)) {
    case 64: return prompts_launch<DT, 64, 4, F32 ? 1 : 2, 64>(a, stream);
    case 128: return prompts_launch<DT, 128, 8, F32 ? 1 : 2, 64>(a, stream);
    case 256: return prompts_launch<DT, 256, 8, 1, 64>(a, stream);
    default: return prompts_launch<DT, 512, 8, 1, 32>(a, stream);
    }
}

}  // namespace

hipError_t attend_prompts_launch(const AttendArgs& a, int32_t dtype, hipStream_t stream)
{
    return dtype == G4S_DTYPE_F32 ? by_width<G4S_DTYPE_F32>(a, stream)
                                  : by_width<G4S_DTYPE_BF16>(a, stream);
}

}  // namespace g4s
