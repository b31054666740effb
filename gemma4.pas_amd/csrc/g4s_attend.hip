/*
 * g4s_attend.hip -- attention over the pages of an 8-bit cache for rows with few queries
 * (the tokens of a decode step), on gfx950.
 *
 * The work of a launch, counted in units of NW x 32 tokens of one row and key
 * head, is shared out evenly over the workgroups, whatever the rows' lengths;
 * every workgroup finds its share from the lengths by itself.  A wave takes 32 tokens of
 * each unit with a softmax of its own; the waves join in LDS, and where
 * several workgroups have parts of one row and head, the one that ends last joins
 * those, in their order, so that results do not depend on who that is.
 */
#include "g4s_attend.h"
#include "g4s_launch.h"

namespace g4s {

namespace {

constexpr int kTile = 32; /* tokens of a wave's step */
constexpr int kB = 256;
constexpr int kCols = 16; /* query columns of a workgroup's part */
constexpr int kPass = 128; /* dims that the waves join at once */

/* What a row asks for. */
struct Work {
    int start, count, length, bad; /* RowTokens */
    int cols, blocks;              /* query columns (tokens x heads of a key head), 16 of them a block */
    int from, first;               /* first place that any query sees, and its unit */
    int units;                     /* of each key head and block: one at least, for the output */
};
template <int UNIT>
__device__ __forceinline__ Work row_work(const AttendArgs& a, int row)
{
    const RowTokens r = row_tokens(a.starts, a.lengths, row, a.tokens, cache_room(a.pool));
    Work w{r.start, r.count, r.length, r.bad, 0, 0, 0, 0, 0};
    w.cols = r.count * a.group.d;
    if (is_prompt(r.count, a.group.d)) return w;
    w.blocks = (w.cols + kCols - 1) / kCols;
    const int64_t from = a.window > 0 ? (int64_t)r.length - r.count + 1 - a.window : 0;
    w.from = from > 0 ? (int)from : 0;
    w.first = w.from / UNIT;
    w.units = r.length > w.from ? (int)(((int64_t)r.length + UNIT - 1) / UNIT) - w.first : 1;
    return w;
}

/* Work of the rows before each row, in units, into before[0 .. rows]. */
template <int NW>
__device__ __forceinline__ void scan_work(const AttendArgs& a, int64_t* before, int64_t* s_wave)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int each = (a.rows + NW * 64 - 1) / (NW * 64);
    int64_t sum = 0;
    for (int i = 0; i < each; ++i) {
        const int r = tid * each + i;
        if (r >= a.rows) break;
        const Work w = row_work<NW * kTile>(a, r);
        before[r + 1] = (int64_t)w.units * w.blocks * a.kv_heads;
        sum += before[r + 1];
    }
    int64_t x = sum;
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t y = __shfl_up((long long)x, d);
        if (lane >= d) x += y;
    }
    if (lane == 63) s_wave[wave] = x;
    __syncthreads();
    x -= sum;
    for (int w = 0; w < wave; ++w) x += s_wave[w];
    for (int i = 0; i < each; ++i) {
        const int r = tid * each + i;
        if (r >= a.rows) break;
        x += before[r + 1];
        before[r + 1] = x;
    }
    if (tid == 0) before[0] = 0;
    __syncthreads();
}

/* A part of one row's tokens for one key head and 16 query columns. */
struct Part {
    int row, head, col0;
    Work w;
};

template <int DT, int D, int NW>
struct Shared {
    Frag q[D / 64][2][DT == G4S_DTYPE_F32 ? 3 : 1][64]; /* the queries, as lanes take them */
    int64_t offset[NW][kTile];
    float scale[NW][2][kTile];
    float m[NW][kCols], l[NW][kCols];
    float top[kCols], sum[kCols];
    float o[NW][kCols][kPass + 4];
    int64_t wave[NW];
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
#pragma unroll
        for (int i = 0; i < VW; i += 4) {
            const u32x4_4 x = *reinterpret_cast<const u32x4_4*>(p + 4 * i);
#pragma unroll
            for (int k = 0; k < 4; ++k) w[i + k] = x[k];
        }
    }
}

template <int DT, int D, int NW>
__global__ __launch_bounds__(NW * 64, 1) void attend_rows_kernel(AttendArgs a)
{
    constexpr int UNIT = NW * kTile;
    constexpr int QP = DT == G4S_DTYPE_F32 ? 3 : 1; /* pieces of a query */
    constexpr int PP = DT == G4S_DTYPE_F32 ? 2 : 1; /* and of a weight */
    constexpr int KC = D / 64;                      /* 16-dim chunks of a lane of K and Q */
    constexpr int VW = D / 64;                      /* words of a lane of V */
    constexpr int DB = D / 16;                      /* blocks of 16 dims, and dims of a lane */
    static_assert(2 * kCols * D <= kAttendSums && 4 * kCols <= kAttendStats, "two slots a workgroup");
    extern __shared__ char lds[];
    auto& s = *reinterpret_cast<Shared<DT, D, NW>*>(lds);
    int64_t* before = reinterpret_cast<int64_t*>(lds + ((sizeof(s) + 15) & ~(size_t)15));
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int m = lane & 15, g = lane >> 4;
    scan_work<NW>(a, before, s.wave);
    const int64_t total = before[a.rows];
    const int groups = total < gridDim.x ? (int)total : (int)gridDim.x;
    if ((int)blockIdx.x >= groups) return;
    int64_t x = first_unit(total, blockIdx.x, groups);
    const int64_t x_end = first_unit(total, blockIdx.x + 1, groups);
    /* to base two, and never 0: what is masked stays -inf.  (The scale's sign is in the queries.) */
    const float c = fmaxf(__builtin_fabsf(a.scale * kLog2e), 1e-37f);

    while (x < x_end) {
        Part p;
        {
            int lo = 0, hi = a.rows - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (before[mid] <= x)
                    lo = mid;
                else
                    hi = mid - 1;
            }
            p.row = lo;
        }
        p.w = row_work<UNIT>(a, p.row);
        const int64_t in_row = x - before[p.row];
        const int item = (int)(in_row / p.w.units);
        const int u0 = (int)(in_row - (int64_t)item * p.w.units);
        const int64_t left = x_end - x;
        const int u1 = p.w.units - u0 < left ? p.w.units : u0 + (int)left;
        p.head = item / p.w.blocks;
        p.col0 = (item - p.head * p.w.blocks) * kCols;
        const int64_t item_first = x - u0; /* its first unit among all */
        x += u1 - u0;

        /* this lane's query column */
        const int col = p.col0 + m;
        const int cols = p.w.cols - p.col0 < kCols ? p.w.cols - p.col0 : kCols;
        const bool has_col = m < cols;
        const int nth = has_col ? divide(col, a.group) : 0;
        const int qhead = p.head * a.group.d + (has_col ? col - nth * a.group.d : 0);
        const int place = p.w.length - p.w.count + nth; /* sees from .. place */
        const int64_t from64 = a.window > 0 ? (int64_t)place - a.window + 1 : 0;
        const int from = from64 > 0 ? (int)from64 : 0;
        {
            const char* at = a.q.data + ((p.w.start + nth) * a.q.token_stride +
                                         qhead * a.q.head_stride) * Elem<DT>::SIZE;
            for (int k = wave; k < KC; k += NW) {
                const int d0 = k * 64 + g * 16;
                Frag f[2][QP];
                const bool in = d0 < a.pool.head_dim;
                const char* q0 = at + (int64_t)(in ? d0 : 0) * Elem<DT>::SIZE;
                load_query<DT>(q0, has_col && in, a.scale < 0.0f, f[0]);
                load_query<DT>(q0 + 8 * Elem<DT>::SIZE, has_col && in, a.scale < 0.0f, f[1]);
#pragma unroll
                for (int b = 0; b < QP; ++b) {
                    s.q[k][0][b][lane] = f[0][b];
                    s.q[k][1][b][lane] = f[1][b];
                }
            }
            __syncthreads();
        }
        f32x4 o[DB];
#pragma unroll
        for (int i = 0; i < DB; ++i) o[i] = f32x4{0, 0, 0, 0};
        float top = -inf32(), sum = 0.0f;

        const int last_place = p.w.length - 1;
        const int full_from = p.w.count > 1 && a.window > 0
                                  ? (p.w.length - a.window > 0 ? p.w.length - a.window : 0)
                                  : p.w.from;                  /* all queries see from here .. */
        const int full_to = p.w.length - p.w.count;            /* .. to here */
        const int32_t* pages = a.table + (int64_t)p.row * a.pool.max_slots;
        const int end = p.w.length > p.w.from ? p.w.length : 0;
        for (int u = u0; u < u1; ++u) {
            const int t0 = (p.w.first + u) * UNIT + wave * kTile;
            if (t0 >= end || t0 + kTile <= p.w.from) continue;
            /* a token a lane, keys' and values' scales by halves; beyond the ends the one at
             * the end stands in, which some query sees */
            int t = t0 + (lane & 31);
            t = t < p.w.from ? p.w.from : t > last_place ? last_place : t;
            const int slot = divide(t, a.pool.page_tokens);
            const int in = t - slot * a.pool.page_tokens.d;
            int page = pages[slot];
            const bool ok = page >= 0 && page < a.pool.n_pages;
            if (!ok) page = 0;
            const uint32_t bad = (uint32_t)__ballot(!ok);
            const int64_t off = cache_offset(a.pool, page, in, p.head);
            const int in_block = in - divide(in, a.pool.scale_tokens) * a.pool.scale_tokens.d;
            const float scale = *reinterpret_cast<const float*>(
                (lane < 32 ? a.k_plane : a.v_plane) + off - (int64_t)in_block * a.pool.token_bytes +
                a.pool.head_dim);
            if (lane < 32) s.offset[wave][lane] = off;
            s.scale[wave][lane >> 5][lane & 31] = scale;
            wave_fence();

            uint32_t kw[2][KC][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const char* at = a.k_plane + s.offset[wave][h * 16 + m];
#pragma unroll
                for (int k = 0; k < KC; ++k) {
                    const int d0 = k * 64 + g * 16;
                    load_words<4>(at + (d0 < a.pool.head_dim ? d0 : 0), kw[h][k]);
                }
            }
            uint32_t vw[8][VW];
            const int vd = m * DB;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const char* at = a.v_plane + s.offset[wave][(j & 4) * 4 + g * 4 + (j & 3)];
                if constexpr (VW <= 4) {
                    load_words<VW>(at + (vd < a.pool.head_dim ? vd : 0), vw[j]);
                } else {
                    uint32_t w4[4];
#pragma unroll
                    for (int i = 0; i < VW; i += 4) {
                        load_words<4>(at + (vd + 4 * i < a.pool.head_dim ? vd + 4 * i : 0), w4);
#pragma unroll
                        for (int k = 0; k < 4; ++k) vw[j][i + k] = w4[k];
                    }
                }
            }

            f32x4 sc[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float ks = s.scale[wave][0][h * 16 + m];
                sc[h] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < KC; ++k) {
                    Frag f[2];
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        f[w >> 1].w[(w & 1) * 2] = widen2<false>(kw[h][k][w], ks);
                        f[w >> 1].w[(w & 1) * 2 + 1] = widen2<true>(kw[h][k][w], ks);
                    }
#pragma unroll
                    for (int b = QP - 1; b >= 0; --b) {
                        sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[0].v, s.q[k][0][b][lane].v, sc[h], 0, 0, 0);
                        sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[1].v, s.q[k][1][b][lane].v, sc[h], 0, 0, 0);
                    }
                }
            }
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = sc[j >> 2][j & 3];
            const bool partly = bad != 0 || t0 < full_from || t0 + kTile - 1 > full_to;
            bool nan_v = false;
            if (partly) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int i = (j & 4) * 4 + g * 4 + (j & 3);
                    const int at = t0 + i;
                    if (bad >> i & 1) y[j] = nan32();
                    if (at < from || at > place) y[j] = -inf32();
                }
                if (p.w.count > 1) {
                    bool any = false;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int w = 0; w < VW; ++w) any = any || has_nan(vw[j][w]);
                    nan_v = __any(any);
                }
            }
            float now = y[0];
#pragma unroll
            for (int j = 1; j < 8; ++j) now = fmaxf(now, y[j]);
            now = fmaxf(now, __shfl_xor(now, 16));
            now = fmaxf(now, __shfl_xor(now, 32));
            now = fmaxf(now, top);
            if (__any(now > top)) {
                const float keep = now > top ? __builtin_amdgcn_exp2f((top - now) * c) : 1.0f;
                sum *= keep;
#pragma unroll
                for (int i = 0; i < DB; ++i) o[i] *= keep;
                top = now;
            }
            const float base = top == -inf32() ? 0.0f : top * c;
            Frag pw[PP];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(y[j], c, -base));
                const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(y[j + 1], c, -base));
                sum += e0 + e1;
                pw[0].w[j >> 1] = pack_bf16(e0, e1);
                if constexpr (PP == 2) {
                    const float r0 = e0 - __uint_as_float(pw[0].w[j >> 1] << 16);
                    const float r1 = e1 - __uint_as_float(pw[0].w[j >> 1] & 0xFFFF0000u);
                    pw[1].w[j >> 1] = pack_bf16(r0, r1);
                }
            }
            float vs[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) vs[j] = s.scale[wave][1][(j & 4) * 4 + g * 4 + (j & 3)];
            if (nan_v) {
                /* a NaN that some queries see and others do not (0 times NaN is NaN): the products
                 * go without it, and whoever sees one, counted by a product too, gets NaN */
                Frag see;
#pragma unroll
                for (int j = 0; j < 8; j += 2)
                    see.w[j >> 1] = (y[j] == -inf32() ? 0u : 0x3F80u) |
                                    (y[j + 1] == -inf32() ? 0u : 0x3F800000u);
                const float one[8] = {1, 1, 1, 1, 1, 1, 1, 1};
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    uint32_t at[8];
                    Frag f[4];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        at[j] = nan_codes(vw[j][w]) * 0x38u; /* the code of 1 */
                        vw[j][w] = without_nan(vw[j][w]);
                    }
                    value_frags(at, one, f);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f32x4 n = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            f[i].v, see.v, f32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (n[r] > 0.0f) o[w * 4 + i][r] = nan32();
                    }
                }
            }
#pragma unroll
            for (int w = 0; w < VW; ++w) {
                uint32_t at[8];
                Frag f[4];
#pragma unroll
                for (int j = 0; j < 8; ++j) at[j] = vw[j][w];
                value_frags(at, vs, f);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int b = PP - 1; b >= 0; --b)
                        o[w * 4 + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            f[i].v, pw[b].v, o[w * 4 + i], 0, 0, 0);
            }
            wave_fence(); /* the next tile's offsets and scales take the place of these */
        }

        /* the waves join */
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (g == 0) {
            s.m[wave][m] = top == -inf32() ? top : top * c;
            s.l[wave][m] = sum;
        }
        __syncthreads();
        if (tid < kCols) {
            float best = s.m[0][tid];
            for (int w = 1; w < NW; ++w) best = fmaxf(best, s.m[w][tid]);
            float all = 0.0f;
            for (int w = 0; w < NW; ++w) {
                const float f = s.m[w][tid] == -inf32() ? 0.0f : __builtin_amdgcn_exp2f(s.m[w][tid] - best);
                all += s.l[w][tid] * f;
                s.l[w][tid] = f;
            }
            s.top[tid] = best;
            s.sum[tid] = all;
        }
        const bool whole = u0 == 0 && u1 == p.w.units;
        const int w_first = whole ? 0 : unit_group(item_first, total, groups);
        const int w_last = whole ? 0 : unit_group(item_first + p.w.units - 1, total, groups);
        const int64_t slot = 2 * (int64_t)blockIdx.x + (u0 == 0);
        for (int pass = 0; pass < (D + kPass - 1) / kPass; ++pass) {
            /* lanes with dims of this pass */
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d0 = DB * (g * 4 + r) - pass * kPass;
                if (d0 >= 0 && d0 < kPass) {
#pragma unroll
                    for (int i = 0; i < DB; i += 4)
                        *reinterpret_cast<f32x4*>(&s.o[wave][m][d0 + i]) =
                            f32x4{o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]};
                }
            }
            __syncthreads();
            constexpr int Q4 = (D < kPass ? D : kPass) / 4;
            for (int i = tid; i < cols * Q4; i += NW * 64) {
                const int k = i / Q4, d0 = i % Q4 * 4, dim = pass * kPass + d0;
                f32x4 v = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < NW; ++w)
                    v += *reinterpret_cast<const f32x4*>(&s.o[w][k][d0]) * s.l[w][k];
                if (!whole) {
                    uint64_t* to = reinterpret_cast<uint64_t*>(a.ws.sums + (slot * kCols + k) * D + dim);
                    st_dev(to, (uint64_t)__float_as_uint(v[0]) | (uint64_t)__float_as_uint(v[1]) << 32);
                    st_dev(to + 1, (uint64_t)__float_as_uint(v[2]) | (uint64_t)__float_as_uint(v[3]) << 32);
                } else if (dim < a.pool.head_dim) {
                    const int cc = p.col0 + k, n = divide(cc, a.group), qh = p.head * a.group.d + cc - n * a.group.d;
                    const bool empty = p.w.length - p.w.count + n < 0 && !p.w.bad;
                    const float inv = p.w.bad ? nan32() : empty ? 0.0f : 1.0f / s.sum[k];
                    v = empty ? f32x4{0, 0, 0, 0} : v * inv;
                    store4<DT>(a.out.data + ((p.w.start + n) * a.out.token_stride +
                                             qh * a.out.head_stride + dim) * Elem<DT>::SIZE, v);
                }
            }
            if (pass == 0 && tid < cols) {
                if (!whole) {
                    st_dev(reinterpret_cast<uint64_t*>(a.ws.stats + (slot * kCols + tid) * 2),
                           (uint64_t)__float_as_uint(s.top[tid]) | (uint64_t)__float_as_uint(s.sum[tid]) << 32);
                } else if (a.lse) {
                    const int cc = p.col0 + tid, n = divide(cc, a.group), qh = p.head * a.group.d + cc - n * a.group.d;
                    const bool empty = p.w.length - p.w.count + n < 0 && !p.w.bad;
                    a.lse[(int64_t)(p.w.start + n) * a.heads + qh] =
                        p.w.bad ? nan32() : empty ? -inf32()
                                : (s.top[tid] + __builtin_amdgcn_logf(s.sum[tid])) * kLn2;
                }
            }
            __syncthreads();
        }
        if (whole) continue;
        /* the last of the workgroups that have a part of this item joins them */
        const int parts = w_last - w_first + 1;
        if (!elect_last(&a.ws.tickets[w_first], (uint32_t)parts, &s.flag)) continue;
        auto part_slot = [&](int i) { return 2 * (int64_t)(w_first + i) + (i == 0); };
        for (int i = tid; i < cols * (D / 4); i += NW * 64) {
            const int k = i / (D / 4), dim = i % (D / 4) * 4;
            if (dim >= a.pool.head_dim) continue;
            float best = -inf32();
            for (int w = 0; w < parts; ++w)
                best = fmaxf(best, __uint_as_float((uint32_t)ld_dev(
                    reinterpret_cast<const uint64_t*>(a.ws.stats + (part_slot(w) * kCols + k) * 2))));
            float all = 0.0f;
            f32x4 v = f32x4{0, 0, 0, 0};
            for (int w = 0; w < parts; ++w) {
                const uint64_t st = ld_dev(
                    reinterpret_cast<const uint64_t*>(a.ws.stats + (part_slot(w) * kCols + k) * 2));
                const uint64_t* at = reinterpret_cast<const uint64_t*>(
                    a.ws.sums + (part_slot(w) * kCols + k) * D + dim);
                const uint64_t v0 = ld_dev(at), v1 = ld_dev(at + 1);
                const float tw = __uint_as_float((uint32_t)st), lw = __uint_as_float((uint32_t)(st >> 32));
                const float f = tw == -inf32() ? 0.0f : __builtin_amdgcn_exp2f(tw - best);
                all += lw * f;
                v += f32x4{__uint_as_float((uint32_t)v0), __uint_as_float((uint32_t)(v0 >> 32)),
                           __uint_as_float((uint32_t)v1), __uint_as_float((uint32_t)(v1 >> 32))} * f;
            }
            const int cc = p.col0 + k, n = divide(cc, a.group), qh = p.head * a.group.d + cc - n * a.group.d;
            const bool empty = p.w.length - p.w.count + n < 0;
            v = empty ? f32x4{0, 0, 0, 0} : v * (1.0f / all);
            store4<DT>(a.out.data + ((p.w.start + n) * a.out.token_stride + qh * a.out.head_stride +
                                     dim) * Elem<DT>::SIZE, v);
            if (dim == 0 && a.lse)
                a.lse[(int64_t)(p.w.start + n) * a.heads + qh] =
                    empty ? -inf32() : (best + __builtin_amdgcn_logf(all)) * kLn2;
        }
        __syncthreads();
    }
}

template <int DT, int D, int NW>
hipError_t rows_launch(const AttendArgs& a, hipStream_t stream)
{
    const size_t lds = ((sizeof(Shared<DT, D, NW>) + 15) & ~(size_t)15) + ((size_t)a.rows + 1) * 8;
    /* no more workgroups than the rows can have units */
    const int64_t blocks = (a.group.d + kCols - 1) / kCols;
    const int64_t units = (cache_room(a.pool) + NW * kTile - 1) / (NW * kTile) + 1;
    const int64_t most = (int64_t)a.rows * a.kv_heads * blocks * units;
    const int groups = most < a.ws.groups ? (int)most : a.ws.groups;
    return launch(attend_rows_kernel<DT, D, NW>, groups, NW * 64, lds, stream, a);
}

template <int DT>
hipError_t by_width(const AttendArgs& a, hipStream_t stream)
{
    switch (attend_width(a.pool.head_dim)) {
    case 64: return rows_launch<DT, 64, 8>(a, stream);
    case 128: return rows_launch<DT, 128, 8>(a, stream);
    case 256: return rows_launch<DT, 256, DT == G4S_DTYPE_F32 ? 4 : 8>(a, stream);
    default: return rows_launch<DT, 512, 4>(a, stream);
    }
}

__global__ void attend_init_kernel(uint32_t* tickets, int n)
{
    for (int i = blockIdx.x * kB + threadIdx.x; i < n; i += gridDim.x * kB) tickets[i] = 0u;
}

}  // namespace

int32_t attend_width(int32_t head_dim)
{
    return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : head_dim <= 256 ? 256 : 512;
}

int32_t attend_groups(int32_t ncu) { return ncu; }

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
