/*
 * g4s_beam.hip -- selection over beams and vocabulary, and the reordering of
 * contiguous states, on gfx950.
 *
 * The reference keeps one token string (TModel.Generate,
 * src/Gemma4.Model.pas:2829-2938); a search needs, of W rows of V logits per
 * sequence, the n best sums  score + log softmax(softcap(x)).  The softcap
 * grows with x, so a row's best candidates are its largest logits: they are
 * selected on the logits themselves, and only those that can win are evaluated in
 * binary64.  One pass over the logits gives both the row's candidates and its
 * softmax denominator.
 */
#include "g4s_beam.h"

#include "g4s_select.h"

namespace g4s {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kB = kBeamBlock;
constexpr int kE = kBeamItems;
constexpr int kListCap = 512; /* candidates of a workgroup kept for ranking */
constexpr int kNMax = 2 * G4S_BEAM_MAX_BEAMS;
constexpr float kMasked = -1e30f; /* a logit not above it is no candidate */

__device__ __forceinline__ uint64_t entry_of(uint32_t key, uint32_t token)
{
    return ((uint64_t)key << 32) | (uint32_t)~token;
}
__device__ __forceinline__ uint32_t entry_key(uint64_t e) { return (uint32_t)(e >> 32); }
__device__ __forceinline__ uint32_t entry_token(uint64_t e) { return ~(uint32_t)e; }

using cr::exp_fast_d;

constexpr double kLog2e = 0x1.71547652b82fep+0;

__device__ __forceinline__ uint64_t d2u(double x) { return __builtin_bit_cast(uint64_t, x); }
__device__ __forceinline__ double u2d(uint64_t u) { return __builtin_bit_cast(double, u); }

/* cap * tanh(x / cap), off by some 2^-52 of the cap. */
template <int MODE>
__device__ __forceinline__ double softcap64(float x, const BeamSoftcap& c)
{
    if constexpr (MODE == kCapNone) return (double)x;
    const double cap = (double)c.cap;
    const double e = exp_fast_d(fmax(-2.0 * fabs((double)x) / cap, -80.0));
    return copysign(cap * ((1.0 - e) / (1.0 + e)), (double)x);
}

/* log(x) for x in [1, 2^60], off by less than 1e-12: one Newton step from binary32's. */
__device__ __forceinline__ double log64(double x)
{
    const double l = (double)(__builtin_amdgcn_logf((float)x) * 0x1.62e43p-1f);
    return l + (x * exp_fast_d(-l) - 1.0);
}

/* exp(y - top) for y <= top; an infinite top (no softcap, x = +inf) counts 1
 * for itself and leaves nothing for the rest. */
__device__ __forceinline__ double term64(double y, double top)
{
    const double d = y - top;
    return y == top ? 1.0 : (d < -1000.0 ? 0.0 : exp_fast_d(d));
}

/* v(x) / x of BeamSoftcap, where |x| <= limit. */
__device__ __forceinline__ double near_factor(double x, const BeamSoftcap& c)
{
    const double s = x * x;
    double h = c.q[9];
#pragma unroll
    for (int i = 8; i >= 0; --i) h = __builtin_fma(h, s, c.q[i]);
    return h;
}
template <int MODE>
__device__ __forceinline__ double value64(float x, const BeamSoftcap& c)
{
    if (MODE == kCapPoly && fabsf(x) <= c.limit) return (double)x * near_factor((double)x, c);
    return softcap64<MODE>(x, c) * kLog2e;
}

/* 2^t to binary32's accuracy, for t in [-2^20, 1]: what binary32 would round off
 * t (a millionth where t is near -20) is kept by splitting t first. */
__device__ __forceinline__ float pow2_of(double t)
{
    constexpr double kRound = 0x1.8p52; /* the sum's low word is the rounded integer */
    const double m = t + kRound;
    const float f = (float)(t - (m - kRound));
    return __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(f), (int)(uint32_t)d2u(m));
}

/* The term of one logit in its chunk's sum, 2^(v(x) - ref), ref = v(top). */
template <int MODE, bool NEAR>
__device__ __forceinline__ float term_of(float x, float top, double ref, const BeamSoftcap& c)
{
    if constexpr (MODE == kCapNone)
        return x == top ? 1.0f : pow2_of(fmax(((double)x - (double)top) * kLog2e, -1000.0));
    else if constexpr (MODE == kCapPoly && NEAR)
        return pow2_of(__builtin_fma((double)x, near_factor((double)x, c), -ref));
    else
        return pow2_of(fmax(value64<MODE>(x, c) - ref, -1000.0));
}

/* Sum over the 64 lanes, in every lane (all lanes active). */
__device__ __forceinline__ double wave_sum_f64(double v)
{
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
/* Sum over the workgroup, in thread 0. */
__device__ __forceinline__ double block_sum_f64(double v, double* s_wave)
{
    v = wave_sum_f64(v);
    if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x >> 6] = v;
    __syncthreads();
    double r = 0.0;
    if (threadIdx.x == 0)
#pragma unroll
        for (int w = 0; w < kB / 64; ++w) r += s_wave[w];
    return r;
}

struct TopShared {
    uint32_t tmax[kB];
    uint32_t hist[256];
    int misc[8];
    int scan[kB / 64];
    double red[kB / 64];
    int count;
    int flag;
    alignas(16) uint64_t list[kListCap]; /* in any order */
    alignas(16) uint64_t sorted[kNMax];
    double y[kNMax];
};

struct TopList {
    int listed; /* entries of sh.list */
    float top;  /* the largest candidate */
};

/* The workgroup's largest candidates into sh.list, at least the n best (n <= kNMax) or all
 * there are.  x: this thread's E logits, token(e) their tokens; entry(i),
 * i < count, reads all of them again, in an order that tokens of equal keys
 * rise in.
 *
 * The n-th largest of the threads' largest keys bounds the n-th largest key
 * from below, and for n well below the threads few elements beside the n best
 * reach it.  Where more reach it than the list holds (equal logits in
 * masses), the n-th largest key is selected exactly and of its copies the
 * first are taken; that way reads again what it needs, so that it costs the
 * usual one no registers. */
template <int E, typename TokenF, typename EntryF>
__device__ __forceinline__ TopList top_list(const float (&x)[E], float largest, TokenF token,
                                            int count, EntryF entry, int n, TopShared& sh)
{
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t mkey = cand_key(largest);
    sh.tmax[tid] = mkey;
    if (tid == 0) sh.count = 0;
    __syncthreads();
    uint32_t v[kB / 64];
    uint32_t top = 0u;
    int nz = 0;
#pragma unroll
    for (int q = 0; q < kB / 64; ++q) {
        v[q] = sh.tmax[lane + 64 * q];
        top = v[q] > top ? v[q] : top;
        nz += __popcll(__ballot(v[q] != 0u));
    }
    const uint32_t t = nz >= n ? wave_kth_bound<kB / 64>(v, n, 10) : 1u;
    TopList r;
    r.top = key2f(wave_max_u32(top));
    const float bound = t <= 1u ? -__builtin_inff() : key2f(t);
    if (mkey >= t && mkey != 0u) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (x[e] > kMasked && x[e] >= bound) {
                const int p = atomicAdd(&sh.count, 1);
                if (p < kListCap) sh.list[p] = entry_of(f2key(x[e]), token(e));
            }
    }
    __syncthreads();
    int cnt = sh.count;
    if (cnt > kListCap) {
        int gt, eq;
        auto key = [&](int i) { return entry_key(entry(i)); };
        const uint32_t kth = block_radix_kth<kB>(
            count, n, key, [&](int i) { return key(i) != 0u; }, sh.hist, sh.misc, &gt, &eq);
        if (tid == 0) sh.count = 0;
        __syncthreads();
        int taken = gt;
#pragma unroll 1
        for (int i0 = 0; i0 < count; i0 += kB) {
            const uint64_t c = i0 + tid < count ? entry(i0 + tid) : 0ull;
            if (entry_key(c) > kth) sh.list[atomicAdd(&sh.count, 1)] = c;
            const int same = c != 0ull && entry_key(c) == kth;
            int total;
            const int p = taken + block_exclusive_scan<kB>(same, sh.scan, total);
            if (same && p < n) sh.list[p] = c;
            taken += total;
        }
        cnt = n;
        __syncthreads();
    }
    r.listed = cnt;
    return r;
}

/* How many of the list's entries are better than `mine`. */
__device__ __forceinline__ int rank_in(const uint64_t* list, int cnt, uint64_t mine)
{
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < cnt; ++j) rank += list[j] > mine;
    return rank;
}

/* ------------------------------------------------------------------ chunks */

/* Sum of N (2 or 4) terms: in binary32, which rounds twice at most; such sums are added
 * in binary64.  The polynomial and the split of its result run in binary64
 * because that costs what binary32 does on this machine, and binary32 would
 * leave errors of 1e-6 in the terms of equal logits, which many rows of bf16 have
 * thousands of. */
template <int MODE, bool NEAR, bool MASK, int N>
__device__ __forceinline__ double sum_few(const float* x, float top, double ref,
                                          const BeamSoftcap& c)
{
    float t[N];
#pragma unroll
    for (int q = 0; q < N; ++q) {
        t[q] = term_of<MODE, NEAR>(x[q], top, ref, c);
        if constexpr (MASK) t[q] = x[q] > kMasked ? t[q] : 0.0f;
    }
    if constexpr (N == 2)
        return (double)(t[0] + t[1]);
    else
        return (double)((t[0] + t[1]) + (t[2] + t[3]));
}

/* This thread's part of the chunk's sum.  Most waves hold no masked logit and none
 * beyond the polynomial; the others read their logits again (read(e), element
 * e) rather than hold them through the longer way. */
template <int MODE, int E, typename ReadF>
__device__ __forceinline__ double sum_terms(const float (&x)[E], float least, float largest,
                                            float top, const BeamSoftcap& c, ReadF read)
{
    const double ref = value64<MODE>(top, c);
    const bool near = MODE == kCapNone || (least >= -c.limit && largest <= c.limit);
    double s = 0.0;
    if (MODE != kCapExact && __all(least > kMasked && near)) {
#pragma unroll
        for (int e = 0; e < E; e += 4) s += sum_few<MODE, true, false, 4>(&x[e], top, ref, c);
        if (__all(s == s)) return s; /* a NaN is not seen by minimum and maximum */
        s = 0.0;
    }
#pragma unroll 1
    for (int e = 0; e < E; e += 2) {
        const float v[2] = {read(e), read(e + 1)};
        s += sum_few<MODE, false, true, 2>(v, top, ref, c);
    }
    return s;
}

/* One workgroup per chunk of kBeamChunk logits: its n best candidates, ranked, and its part of
 * the softmax denominator. */
template <int MODE>
__device__ __forceinline__ void merge_row(const BeamSelectArgs& a, int row, TopShared& sh);
__device__ __forceinline__ void merge_sequence(const BeamSelectArgs& a, int b, TopShared& sh);

template <int DT, int MODE>
__global__ __launch_bounds__(kB) void beam_select_kernel(BeamSelectArgs a)
{
    constexpr int VW = Elem<DT>::VW;
    constexpr int NV = kE / VW;
    __shared__ TopShared sh;
    const int row = blockIdx.y, ch = blockIdx.x, tid = threadIdx.x;
    const int b = row / a.beams;
    const bool live = a.scores[row] > kMasked;
    if (live) {
        const char* base =
            static_cast<const char*>(a.logits) + (int64_t)row * a.row_stride * Elem<DT>::SIZE;
        const int64_t first = (int64_t)ch * kBeamChunk;
        float x[kE];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float v[VW];
            load_vec<DT>(base, first + (int64_t)(j * kB + tid) * VW, a.vocab, v);
#pragma unroll
            for (int i = 0; i < VW; ++i) x[j * VW + i] = v[i];
        }
        const int rest = a.vocab - (int)first;
        const int count = rest < kBeamChunk ? rest : kBeamChunk;
        auto token = [&](int e) {
            return (uint32_t)first + (uint32_t)(((e / VW) * kB + tid) * VW + e % VW);
        };
        auto read = [&](int e) {
            const int64_t i = token(e);
            return i < a.vocab ? load_elem<DT>(base, i) : -__builtin_inff();
        };
        auto entry = [&](int i) {
            const uint32_t key = cand_key(load_elem<DT>(base, first + i));
            return key ? entry_of(key, (uint32_t)first + (uint32_t)i) : 0ull;
        };
        float largest = x[0], least = x[0];
#pragma unroll
        for (int e = 1; e < kE; ++e) {
            largest = fmaxf(largest, x[e]);
            least = fminf(least, x[e]);
        }
        const TopList tl = top_list<kE>(x, largest, token, count, entry, a.n, sh);
        const int64_t at = (int64_t)row * a.chunks + ch;
        uint64_t* cand = a.ws.cand + at * a.n;
        for (int i = tid; i < tl.listed; i += kB) {
            const uint64_t e = sh.list[i];
            const int rank = rank_in(sh.list, tl.listed, e);
            if (rank < a.n) st_dev(&cand[rank], e);
        }
        double s = 0.0;
        if (tl.listed)
            s = sum_terms<MODE, kE>(x, least, largest, tl.top, a.cap, read);
        for (int i = tl.listed + tid; i < a.n; i += kB) st_dev(&cand[i], (uint64_t)0);
        s = block_sum_f64(s, sh.red);
        if (tid == 0) st_dev(&a.ws.sums[at], d2u(s));
        if (a.chunks > 1 && !elect_last(&a.ws.tickets[row], (uint32_t)a.chunks, &sh.flag)) return;
        if (a.chunks == 1) {
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
        }
        merge_row<MODE>(a, row, sh);
    } else {
        if (ch != 0) return;
        if (tid == 0 && a.lse) a.lse[row] = -__builtin_inff();
        for (int i = tid; i < a.n; i += kB) st_dev(&a.ws.best[(int64_t)row * a.n + i], (uint64_t)0);
    }
    if (a.beams > 1 &&
        !elect_last(&a.ws.tickets[a.batch * a.beams + b], (uint32_t)a.beams, &sh.flag))
        return;
    if (a.beams == 1) {
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
    }
    merge_sequence(a, b, sh);
}

/* -------------------------------------------------------------------- rows */

/* A row's n best and its normaliser from its chunks'. */
template <int MODE>
__device__ __forceinline__ void merge_row(const BeamSelectArgs& a, int row, TopShared& sh)
{
    constexpr int E = 8;
    const int tid = threadIdx.x;
    const uint64_t* cand = a.ws.cand + (int64_t)row * a.chunks * a.n;
    const int64_t total = (int64_t)a.chunks * a.n;
    int cnt = 0;
    /* tiles of candidates beside the best of those before; the chunks' lists
     * lie in token order, so copies of one key do too */
    for (int64_t base = 0; base < total;) {
        const int64_t rest = cnt + total - base;
        const int count = rest < E * kB ? (int)rest : E * kB;
        auto entry = [&](int i) {
            return i < cnt ? sh.sorted[i] : ld_dev(&cand[base + i - cnt]);
        };
        float x[E];
        uint32_t tok[E];
        float largest = -__builtin_inff();
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = e * kB + tid;
            const uint64_t c = e * kB < count && i < count ? entry(i) : 0ull;
            x[e] = c ? key2f(entry_key(c)) : -__builtin_inff();
            tok[e] = entry_token(c);
            largest = fmaxf(largest, x[e]);
        }
        const TopList tl = top_list<E>(
            x, largest, [&](int e) { return tok[e]; }, count, entry, a.n, sh);
        base += count - cnt;
        __syncthreads();
        for (int i = tid; i < tl.listed; i += kB) {
            const uint64_t e = sh.list[i];
            const int rank = rank_in(sh.list, tl.listed, e);
            if (rank < a.n) sh.sorted[rank] = e;
        }
        cnt = tl.listed < a.n ? tl.listed : a.n;
        __syncthreads();
    }
    /* the chunks' sums relative to their largest logit, which leads each list */
    const double top =
        cnt ? softcap64<MODE>(key2f(entry_key(sh.sorted[0])), a.cap) : -__builtin_inf();
    double s = 0.0;
    for (int c = tid; c < a.chunks; c += kB) {
        const uint64_t first = ld_dev(&cand[(int64_t)c * a.n]);
        const double sum = u2d(ld_dev(&a.ws.sums[(int64_t)row * a.chunks + c]));
        if (first) s += sum * term64(softcap64<MODE>(key2f(entry_key(first)), a.cap), top);
    }
    for (int i = tid; i < cnt; i += kB) sh.y[i] = softcap64<MODE>(key2f(entry_key(sh.sorted[i])), a.cap);
    s = block_sum_f64(s, sh.red); /* (a barrier: y is complete) */
    for (int i = tid; i < a.n; i += kB) {
        uint64_t e = i < cnt ? sh.sorted[i] : 0ull;
        double y = -__builtin_inf();
        if (e) {
            /* where tanh saturates its last bit may waver: the list may not rise */
            y = top;
            for (int j = 1; j <= i; ++j) y = fmin(y, sh.y[j]);
            /* beside an infinite largest logit the rest have probability 0 */
            if (top == __builtin_inf() && y != top) e = 0ull;
        }
        st_dev(&a.ws.best[(int64_t)row * a.n + i], e);
        st_dev(&a.ws.y[(int64_t)row * a.n + i], d2u(y));
    }
    if (tid == 0) {
        const double ls = log64(s);
        st_dev(&a.ws.norm[2 * row], d2u(top));
        st_dev(&a.ws.norm[2 * row + 1], d2u(ls));
        if (a.lse) a.lse[row] = cnt ? (float)(top + ls) : -__builtin_inff();
    }
}

/* --------------------------------------------------------------- sequences */

/* The n best of the sequence's W sorted lists: a candidate's rank is the
 * number of better ones, found in each list by bisection. */
__device__ __forceinline__ void merge_sequence(const BeamSelectArgs& a, int b, TopShared& sh)
{
    extern __shared__ double sc[]; /* [W][n] scores, -inf = none */
    const int tid = threadIdx.x;
    const int W = a.beams, n = a.n, total = W * n;
    const uint64_t* best = a.ws.best + (int64_t)b * total;
    const uint64_t* ys = a.ws.y + (int64_t)b * total;
    int found = 0;
    for (int i = tid; i < total; i += kB) {
        const int w = i / n;
        double s = -__builtin_inf();
        if (ld_dev(&best[i])) {
            const uint64_t* norm = a.ws.norm + 2 * ((int64_t)b * W + w);
            const double top = u2d(ld_dev(&norm[0])), y = u2d(ld_dev(&ys[i]));
            s = (double)a.scores[b * W + w] + ((y == top ? 0.0 : y - top) - u2d(ld_dev(&norm[1])));
            ++found;
        }
        sc[i] = s;
    }
    found = block_sum_i32<kB>(found, sh.scan);
    int32_t* parents = a.parents + (int64_t)b * n;
    int32_t* tokens = a.tokens + (int64_t)b * n;
    float* out = a.out + (int64_t)b * n;
    for (int i = tid; i < total; i += kB) {
        const double s = sc[i];
        if (s == -__builtin_inf()) continue;
        const int w = i / n;
        int rank = i - w * n;
        for (int o = 0; o < W && rank < n; ++o) {
            if (o == w) continue;
            /* of equal scores those of the lower beam come first */
            int lo = 0, hi = n;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                const double t = sc[o * n + mid];
                if (t > s || (t == s && o < w))
                    lo = mid + 1;
                else
                    hi = mid;
            }
            rank += lo;
        }
        if (rank < n) {
            parents[rank] = b * W + w;
            tokens[rank] = (int32_t)entry_token(ld_dev(&best[i]));
            out[rank] = (float)s;
        }
    }
    for (int i = found + tid; i < n; i += kB) {
        parents[i] = -1;
        tokens[i] = -1;
        out[i] = -__builtin_inff();
    }
}

/* ----------------------------------------------------------------- reorder */

/* One thread holds the bytes of one column of all of a sequence's rows: it
 * reads the parents' and then writes, so in place no row is overwritten
 * before it was read, and nothing has to be kept elsewhere. */
template <typename T, int WMAX>
__global__ __launch_bounds__(kB) void beam_reorder_kernel(BeamReorderArgs a)
{
    const int64_t col = (int64_t)blockIdx.x * kB + threadIdx.x;
    const int W = a.beams;
    const int64_t groups = (int64_t)a.batch * a.planes;
    const bool inplace = a.src == a.dst;
    if (col >= a.row_bytes / (int64_t)sizeof(T)) return;
    for (int64_t g = blockIdx.y; g < groups; g += gridDim.y) {
        const int64_t plane = g / a.batch;
        const int b = (int)(g - plane * a.batch);
        const int64_t at =
            plane * a.plane_stride + (int64_t)b * W * a.row_stride + col * (int64_t)sizeof(T);
        T v[WMAX];
#pragma unroll
        for (int r = 0; r < WMAX; ++r)
            if (r < W) {
                const int p = a.parents[b * W + r] - b * W;
                const bool ok = p >= 0 && p < W;
                const int from = ok ? p : r;
                if (!inplace || from != r)
                    v[r] = *reinterpret_cast<const T*>(a.src + at + (int64_t)from * a.row_stride);
            }
#pragma unroll
        for (int r = 0; r < WMAX; ++r)
            if (r < W) {
                const int p = a.parents[b * W + r] - b * W;
                const bool ok = p >= 0 && p < W;
                const int from = ok ? p : r;
                if (!inplace || from != r)
                    *reinterpret_cast<T*>(a.dst + at + (int64_t)r * a.row_stride) = v[r];
            }
    }
}

template <typename T>
hipError_t reorder_with(const BeamReorderArgs& a, hipStream_t stream)
{
    const int64_t cols = a.row_bytes / (int64_t)sizeof(T);
    const int64_t groups = (int64_t)a.batch * a.planes;
    const dim3 grid((unsigned)((cols + kB - 1) / kB), (unsigned)(groups < 65535 ? groups : 65535));
    if (a.beams <= 4)
        beam_reorder_kernel<T, 4><<<grid, kB, 0, stream>>>(a);
    else if (a.beams <= 8)
        beam_reorder_kernel<T, 8><<<grid, kB, 0, stream>>>(a);
    else if (a.beams <= 16)
        beam_reorder_kernel<T, 16><<<grid, kB, 0, stream>>>(a);
    else if (a.beams <= 32)
        beam_reorder_kernel<T, 32><<<grid, kB, 0, stream>>>(a);
    else
        beam_reorder_kernel<T, 64><<<grid, kB, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace

/* tanh(z) / z as a polynomial in z^2 for |z| <= 1.25: |z| times its error is below
 * 5.4e-10 (weighted least squares at Chebyshev nodes, reweighted towards the
 * least maximum). */
BeamSoftcap beam_softcap(float cap)
{
    static const double q[10] = {0x1.ffffffbcad3ecp-1,  -0x1.555539c5a4875p-2,
                                 0x1.110dd56c82b34p-3,  -0x1.b9c2e07c36e05p-5,
                                 0x1.63abfe7705209p-6,  -0x1.161fef1075584p-7,
                                 0x1.8c273d5cd2dc4p-9,  -0x1.c8e7e314ad0f9p-11,
                                 0x1.650da776b43d8p-13, -0x1.0e9af9dea189cp-16};
    BeamSoftcap c{};
    c.cap = cap;
    if (!(cap > 0.0f)) {
        c.mode = kCapNone;
        return c;
    }
    const double d = (double)cap;
    c.mode = cap >= 1e-12f && cap <= 128.0f ? kCapPoly : kCapExact;
    double scale = kLog2e;
    for (int i = 0; i < 10; ++i) {
        c.q[i] = q[i] * scale;
        scale /= d * d;
    }
    c.limit = (float)(1.25 * d);
    return c;
}

template <int DT>
static void select_launch(const BeamSelectArgs& a, hipStream_t stream)
{
    const dim3 grid((unsigned)a.chunks, (unsigned)(a.batch * a.beams));
    const size_t lds = sizeof(double) * a.beams * a.n;
    if (a.cap.mode == kCapNone)
        beam_select_kernel<DT, kCapNone><<<grid, kB, lds, stream>>>(a);
    else if (a.cap.mode == kCapPoly)
        beam_select_kernel<DT, kCapPoly><<<grid, kB, lds, stream>>>(a);
    else
        beam_select_kernel<DT, kCapExact><<<grid, kB, lds, stream>>>(a);
}

hipError_t beam_select_launch(const BeamSelectArgs& a, int32_t dtype, hipStream_t stream)
{
    if (dtype == G4S_DTYPE_F32)
        select_launch<0>(a, stream);
    else
        select_launch<1>(a, stream);
    return hipGetLastError();
}

hipError_t beam_reorder_launch(const BeamReorderArgs& a, hipStream_t stream)
{
    const uint64_t bits = (uint64_t)(uintptr_t)a.src | (uint64_t)(uintptr_t)a.dst |
                          (uint64_t)a.plane_stride | (uint64_t)a.row_stride |
                          (uint64_t)a.row_bytes;
    /* 64 beams of 16 bytes would not stay in registers: 4 bytes from 17 beams on */
    if ((bits & 15) == 0 && a.beams <= 16) return reorder_with<u32x4>(a, stream);
    if ((bits & 3) == 0) return reorder_with<uint32_t>(a, stream);
    return reorder_with<uint8_t>(a, stream);
}

}  // namespace g4s
