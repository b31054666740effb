/*
 * g4s_prompt.hip -- attention over the pages of an 8-bit cache for rows with many queries
 * (prompts and chunks of them), on gfx950.
 *
 * A workgroup takes NW x NT x 16 query columns (tokens x heads of one key head) and goes over the
 * tokens that they see in tiles of KT: all its threads widen the next tile's codes into LDS, keys as
 * [token][dim] and values as [dim][token], while its waves multiply the present one, each
 * for NT x 16 columns of its own with the softmax in registers.  Where there are fewer columns than
 * workgroups the tokens are split too, and the last workgroup of a block of columns joins what
 * the others found, in their order.
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

template <int D, int KT>
struct Shared {
    alignas(16) uint16_t k[2][KT][D + 8];
    alignas(16) uint16_t v[2][D][KT];
    int64_t offset[3][KT];
    float scale[3][2][KT];
    uint64_t bad[3];
    int nan[2];
    int flag;
};

template <int DT, int D, int NW, int NT, int KT>
__global__ __launch_bounds__(NW * 64, 1) void attend_prompts_kernel(AttendArgs a, int splits)
{
    constexpr int QP = DT == G4S_DTYPE_F32 ? 3 : 1;
    constexpr int PP = DT == G4S_DTYPE_F32 ? 2 : 1;
    constexpr int CB = NW * NT * 16;
    constexpr int KS = D / 32, DB = D / 16, TB = KT / 16;
    constexpr int THREADS = NW * 64;
    constexpr int KL = (KT * D / 16 + THREADS - 1) / THREADS; /* 16-code loads of a thread */
    constexpr int VL = (KT * D / 16 + THREADS - 1) / THREADS; /* 4 x 4-code loads */
    static_assert(CB * D <= kAttendSums && CB * 2 <= kAttendStats, "a slot a workgroup");
    extern __shared__ char lds[];
    auto& s = *reinterpret_cast<Shared<D, KT>*>(lds);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int m = lane & 15, g = lane >> 4;

    /* heads side by side; the last columns of a row, which see most, first */
    const int head = blockIdx.x, part = blockIdx.z;
    const int64_t x = (int64_t)gridDim.y - 1 - blockIdx.y;
    const int row = find_share(a.starts, a.rows, x, a.group.d, CB, 1);
    const RowTokens r = row_tokens(a.starts, a.lengths, row, a.tokens, cache_room(a.pool));
    const int64_t block = x - share_begin(a.starts, row, a.group.d, CB, 1);
    const int64_t all_cols = (int64_t)r.count * a.group.d;
    if (!is_prompt(r.count, a.group.d) || block < 0 || block * CB >= all_cols) return;
    const int col0 = (int)(block * CB);
    const int cols = all_cols - col0 < CB ? (int)(all_cols - col0) : CB;

    /* places that the block's queries see */
    const int first_place = r.length - r.count + divide(col0, a.group);
    const int last_place = r.length - r.count + divide(col0 + cols - 1, a.group);
    auto sees_from = [&](int place) {
        const int64_t f = a.window > 0 ? (int64_t)place - a.window + 1 : 0;
        return f > 0 ? (int)f : 0;
    };
    const int from0 = sees_from(first_place), end0 = last_place + 1;
    const int t_first = from0 / KT;
    const int tiles = end0 > from0 ? (end0 + KT - 1) / KT - t_first : 0;
    const int parts = splits == 1 || tiles < 2 ? 1 : tiles < splits ? tiles : splits;
    if (part >= parts) return;
    const int n0 = (int)((int64_t)tiles * part / parts), n1 = (int)((int64_t)tiles * (part + 1) / parts);

    /* this lane's columns */
    int place[NT], from[NT], nth[NT], qhead[NT];
    bool has[NT];
    Frag q[NT][KS][QP];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int c = (wave * NT + t) * 16 + m;
        has[t] = c < cols;
        const int col = col0 + (has[t] ? c : 0);
        nth[t] = divide(col, a.group);
        qhead[t] = head * a.group.d + col - nth[t] * a.group.d;
        place[t] = r.length - r.count + nth[t];
        from[t] = sees_from(place[t]);
        const char* at = a.q.data + ((int64_t)(r.start + nth[t]) * a.q.token_stride +
                                     (int64_t)qhead[t] * a.q.head_stride) * Elem<DT>::SIZE;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const int d0 = k * 32 + g * 8;
            load_query<DT>(at + (int64_t)d0 * Elem<DT>::SIZE, has[t] && d0 < a.pool.head_dim, q[t][k]);
        }
    }
    /* places that any and that all of the wave's queries see */
    const int wcol0 = wave * NT * 16;
    const int wcol1 = wcol0 + NT * 16 < cols ? wcol0 + NT * 16 : cols;
    const bool busy = wcol0 < cols;
    const int w_first = r.length - r.count + divide(col0 + (busy ? wcol0 : 0), a.group);
    const int w_last = r.length - r.count + divide(col0 + (busy ? wcol1 - 1 : 0), a.group);
    const int any_from = sees_from(w_first), all_from = sees_from(w_last);

    const float c = a.scale * kLog2e;
    f32x4 o[NT][DB];
    float top[NT], sum[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        top[t] = -inf32();
        sum[t] = 0.0f;
#pragma unroll
        for (int i = 0; i < DB; ++i) o[t][i] = f32x4{0, 0, 0, 0};
    }

    const int32_t* pages = a.table + (int64_t)row * a.pool.max_slots;
    /* tile n's tokens: where they are, by the first lanes */
    auto locate = [&](int n) {
        if (tid >= 64 || n >= n1) return;
        const int i = KT == 64 ? lane : lane & (KT - 1);
        int t = (t_first + n) * KT + i;
        t = t < from0 ? from0 : t >= end0 ? end0 - 1 : t;
        const int slot = divide(t, a.pool.page_tokens);
        const int in = t - slot * a.pool.page_tokens.d;
        int page = pages[slot];
        const bool ok = page >= 0 && page < a.pool.n_pages;
        if (!ok) page = 0;
        const int64_t off = cache_offset(a.pool, page, in, head);
        const int in_block = in - divide(in, a.pool.scale_tokens) * a.pool.scale_tokens.d;
        const int64_t sc = off - (int64_t)in_block * a.pool.token_bytes + a.pool.head_dim;
        const uint64_t bad = __ballot(!ok);
        const int b = n % 3;
        s.offset[b][i] = off;
        s.scale[b][0][i] = *reinterpret_cast<const float*>(a.k_plane + sc);
        s.scale[b][1][i] = *reinterpret_cast<const float*>(a.v_plane + sc);
        if (lane == 0) s.bad[b] = bad;
    };
    uint32_t kw[KL][4], vw[VL][4];
    auto load = [&](int n) {
        const int b = n % 3;
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
            const int u = tid + i * THREADS, t = u / (D / 4) * 4, d0 = u % (D / 4) * 4;
            if (KT * D / 16 % THREADS == 0 || u < KT * D / 16) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    vw[i][j] = *reinterpret_cast<const uint32_t*>(
                        a.v_plane + s.offset[b][t + j] + (d0 < a.pool.head_dim ? d0 : 0));
            }
        }
    };
    auto store = [&](int n) {
        const int b = n % 3, to = n & 1;
        bool any = false;
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
#pragma unroll
        for (int i = 0; i < VL; ++i) {
            const int u = tid + i * THREADS, t = u / (D / 4) * 4, d0 = u % (D / 4) * 4;
            if (KT * D / 16 % THREADS == 0 || u < KT * D / 16) {
                uint32_t lo[4], hi[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float vs = s.scale[b][1][t + j];
                    lo[j] = widen2<false>(vw[i][j], vs);
                    hi[j] = widen2<true>(vw[i][j], vs);
                    any = any || has_nan(vw[i][j]);
                }
                /* tokens 4 k .. 4 k + 3 of 32 (k = 0 .. 7) at quads 2 (k % 4) + k / 4: in the order that a
                 * lane of the second product takes them */
                const int k = t / 4 % 8, quad = t / 32 * 8 + (k & 3) * 2 + (k >> 2);
                const uint2 w[4] = {make_uint2(lows(lo[0], lo[1]), lows(lo[2], lo[3])),
                                    make_uint2(highs(lo[0], lo[1]), highs(lo[2], lo[3])),
                                    make_uint2(lows(hi[0], hi[1]), lows(hi[2], hi[3])),
                                    make_uint2(highs(hi[0], hi[1]), highs(hi[2], hi[3]))};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int dim = d0 + j, p = value_piece<KT>(dim, quad >> 1);
                    *reinterpret_cast<uint2*>(&s.v[to][dim][p * 8 + (quad & 1) * 4]) = w[j];
                }
            }
        }
        if (__any(any) && lane == 0) s.nan[to] = 1;
    };

    if (tid < 2) s.nan[tid] = 0;
    locate(n0);
    locate(n0 + 1);
    __syncthreads();
    if (n0 < n1) {
        load(n0);
        store(n0);
    }
    __syncthreads();
    for (int n = n0; n < n1; ++n) {
        if (n + 1 < n1) load(n + 1);
        locate(n + 2);
        const int t0 = (t_first + n) * KT;
        const int buf = n & 1;
        if (busy && t0 <= w_last && t0 + KT > any_from) {
            f32x4 sc[NT][TB];
#pragma unroll
            for (int b = 0; b < TB; ++b) {
#pragma unroll
                for (int t = 0; t < NT; ++t) sc[t][b] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    const bf16x8 f = *reinterpret_cast<const bf16x8*>(&s.k[buf][b * 16 + m][k * 32 + g * 8]);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int p = QP - 1; p >= 0; --p)
                            sc[t][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, q[t][k][p].v, sc[t][b], 0, 0, 0);
                }
            }
            const uint64_t bad = s.bad[n % 3];
            const bool partly = bad != 0 || t0 < all_from || t0 + KT - 1 > w_first;
            const bool nan_v = partly && s.nan[buf] != 0;
            Frag pw[NT][TB / 2][PP];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float now = -inf32();
#pragma unroll
                for (int b = 0; b < TB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[t][b][i] *= c;
                if (partly) {
#pragma unroll
                    for (int b = 0; b < TB; ++b)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int in = b * 16 + g * 4 + i, at = t0 + in;
                            if (bad >> in & 1) sc[t][b][i] = nan32();
                            if (at < from[t] || at > place[t]) sc[t][b][i] = -inf32();
                        }
                }
#pragma unroll
                for (int b = 0; b < TB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) now = fmaxf(now, sc[t][b][i]);
                now = fmaxf(now, __shfl_xor(now, 16));
                now = fmaxf(now, __shfl_xor(now, 32));
                now = fmaxf(now, top[t]);
                if (__any(now > top[t])) {
                    const float keep = now > top[t] ? __builtin_amdgcn_exp2f(top[t] - now) : 1.0f;
                    sum[t] *= keep;
#pragma unroll
                    for (int i = 0; i < DB; ++i) o[t][i] *= keep;
                    top[t] = now;
                }
                const float base = top[t] == -inf32() ? 0.0f : top[t];
#pragma unroll
                for (int b = 0; b < TB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        const float e0 = __builtin_amdgcn_exp2f(sc[t][b][i] - base);
                        const float e1 = __builtin_amdgcn_exp2f(sc[t][b][i + 1] - base);
                        sum[t] += e0 + e1;
                        Frag* f = pw[t][b >> 1];
                        const int w = (b & 1) * 2 + (i >> 1);
                        f[0].w[w] = pack_bf16(e0, e1);
                        if constexpr (PP == 2)
                            f[1].w[w] = pack_bf16(e0 - __uint_as_float(f[0].w[w] << 16),
                                                  e1 - __uint_as_float(f[0].w[w] & 0xFFFF0000u));
                    }
            }
            auto value = [&](int i, int h) {
                const int dim = i * 16 + m;
                Frag f;
                f.v = *reinterpret_cast<const bf16x8*>(&s.v[buf][dim][value_piece<KT>(dim, h * 4 + g) * 8]);
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
                            const uint32_t lo = (f.w[w] & 0x7FFFu) > 0x7F80u ? 0xFFFFu : 0u;
                            const uint32_t hi = (f.w[w] & 0x7FFF0000u) > 0x7F800000u ? 0xFFFF0000u : 0u;
                            f.w[w] &= ~(lo | hi);
                            is.w[w] = (lo | hi) & 0x3F803F80u;
                        }
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            Frag see; /* 1 for the tokens that the column sees */
#pragma unroll
                            for (int w = 0; w < 4; ++w) {
                                const int at = t0 + h * 32 + (w & 2) * 8 + g * 4 + (w & 1) * 2;
                                see.w[w] = (at >= from[t] && at <= place[t] ? 0x3F80u : 0u) |
                                           (at + 1 >= from[t] && at + 1 <= place[t] ? 0x3F800000u : 0u);
                            }
                            const f32x4 e = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                is.v, see.v, f32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (e[j] > 0.0f) o[t][i][j] = nan32();
#pragma unroll
                            for (int p = PP - 1; p >= 0; --p)
                                o[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.v, pw[t][h][p].v, o[t][i], 0, 0, 0);
                        }
                    }
            }
        }
        if (n + 1 < n1) store(n + 1);
        __syncthreads();
    }

    /* what the workgroup found */
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        sum[t] += __shfl_xor(sum[t], 16);
        sum[t] += __shfl_xor(sum[t], 32);
    }
    auto finish = [&](int nt, int qh, int dim, f32x4 v) {
        store4<DT>(a.out.data + ((int64_t)(r.start + nt) * a.out.token_stride +
                                 (int64_t)qh * a.out.head_stride + dim) * Elem<DT>::SIZE, v);
    };
    auto log_sum = [&](int nt, int qh, float best, float all, bool empty) {
        if (a.lse)
            a.lse[(int64_t)(r.start + nt) * a.heads + qh] =
                r.bad ? nan32() : empty ? -inf32() : (best + __builtin_amdgcn_logf(all)) * kLn2;
    };
    const int64_t item = x * gridDim.x + head;
    if (parts == 1) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (!has[t]) continue;
            const bool empty = !r.bad && place[t] < 0;
            const float inv = r.bad ? nan32() : 1.0f / sum[t];
#pragma unroll
            for (int i = 0; i < DB; ++i) {
                const int dim = i * 16 + g * 4;
                if (dim < a.pool.head_dim)
                    finish(nth[t], qhead[t], dim, empty ? f32x4{0, 0, 0, 0} : o[t][i] * inv);
            }
            if (g == 0) log_sum(nth[t], qhead[t], top[t], sum[t], empty);
        }
        return;
    }
    const int64_t slot0 = item * splits;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (!has[t]) continue;
        const int k = (wave * NT + t) * 16 + m;
        float* to = a.ws.sums + (slot0 + part) * kAttendSums + (int64_t)k * D;
#pragma unroll
        for (int i = 0; i < DB; ++i) {
            uint64_t* w = reinterpret_cast<uint64_t*>(to + i * 16 + g * 4);
            st_dev(w, (uint64_t)__float_as_uint(o[t][i][0]) | (uint64_t)__float_as_uint(o[t][i][1]) << 32);
            st_dev(w + 1, (uint64_t)__float_as_uint(o[t][i][2]) | (uint64_t)__float_as_uint(o[t][i][3]) << 32);
        }
        if (g == 0)
            st_dev(reinterpret_cast<uint64_t*>(a.ws.stats + (slot0 + part) * kAttendStats + k * 2),
                   (uint64_t)__float_as_uint(top[t]) | (uint64_t)__float_as_uint(sum[t]) << 32);
    }
    if (!elect_last(&a.ws.tickets[item], (uint32_t)parts, &s.flag)) return;
    for (int i = tid; i < cols * (D / 4); i += THREADS) {
        const int k = i / (D / 4), dim = i % (D / 4) * 4;
        if (dim >= a.pool.head_dim) continue;
        const int col = col0 + k, nt = divide(col, a.group);
        const int qh = head * a.group.d + col - nt * a.group.d;
        float best = -inf32(), all = 0.0f;
        f32x4 v = f32x4{0, 0, 0, 0};
        for (int w = 0; w < parts; ++w) {
            const uint64_t st = ld_dev(reinterpret_cast<const uint64_t*>(
                a.ws.stats + (slot0 + w) * kAttendStats + k * 2));
            const uint64_t* at = reinterpret_cast<const uint64_t*>(
                a.ws.sums + (slot0 + w) * kAttendSums + (int64_t)k * D + dim);
            const uint64_t v0 = ld_dev(at), v1 = ld_dev(at + 1);
            const float tw = __uint_as_float((uint32_t)st), lw = __uint_as_float((uint32_t)(st >> 32));
            const float now = fmaxf(best, tw);
            const float keep = best == -inf32() ? 0.0f : __builtin_amdgcn_exp2f(best - now);
            const float f = tw == -inf32() ? 0.0f : __builtin_amdgcn_exp2f(tw - now);
            best = now;
            all = all * keep + lw * f;
            v = v * keep + f32x4{__uint_as_float((uint32_t)v0), __uint_as_float((uint32_t)(v0 >> 32)),
                                 __uint_as_float((uint32_t)v1), __uint_as_float((uint32_t)(v1 >> 32))} * f;
        }
        const bool empty = r.length - r.count + nt < 0;
        finish(nt, qh, dim, empty ? f32x4{0, 0, 0, 0} : v * (1.0f / all));
        if (dim == 0) log_sum(nt, qh, best, all, empty);
    }
}

template <int DT, int D, int NW, int NT, int KT>
hipError_t prompts_launch(const AttendArgs& a, hipStream_t stream)
{
    constexpr int CB = NW * NT * 16;
    const int64_t slots = (int64_t)a.tokens * a.group.d / CB + a.rows;
    const int64_t items = slots * a.kv_heads;
    int64_t splits = a.ws.groups / items;
    splits = splits < 1 ? 1 : splits > 64 ? 64 : splits;
    const dim3 grid((unsigned)a.kv_heads, (unsigned)slots, (unsigned)splits);
    return launch(attend_prompts_kernel<DT, D, NW, NT, KT>, grid, NW * 64, sizeof(Shared<D, KT>),
                  stream, a, (int)splits);
}

template <int DT>
hipError_t by_width(const AttendArgs& a, hipStream_t stream)
{
    switch (attend_width(a.pool.head_dim)) {
    case 64: return prompts_launch<DT, 64, 8, 2, 64>(a, stream);
    case 128: return prompts_launch<DT, 128, 8, 2, 64>(a, stream);
    case 256: return prompts_launch<DT, 256, 4, 2, 64>(a, stream);
    default: return prompts_launch<DT, 512, 4, 1, 32>(a, stream);
    }
}

}  // namespace

hipError_t attend_prompts_launch(const AttendArgs& a, int32_t dtype, hipStream_t stream)
{
    return dtype == G4S_DTYPE_F32 ? by_width<G4S_DTYPE_F32>(a, stream)
                                  : by_width<G4S_DTYPE_BF16>(a, stream);
}

}  // namespace g4s
