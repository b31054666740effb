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

#include "g4s_launch.h"
#include "g4s_select.h"

namespace g4s {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));

constexpr int kB = 256;
constexpr int kListCap = 512; /* candidates of a workgroup kept for ranking */
constexpr int kNMax = 2 * G4S_BEAM_MAX_BEAMS;
/* Bits of a bound below the keys' common prefix: with values of both signs
 * four of the mantissa, with any others more.  Six let so many elements pass that lists overflow
 * (38 us where these take 18); sixteen cost 0.4 us. */
constexpr int kBoundBits = 13;
constexpr float kMasked = -1e30f; /* a logit not above it is no candidate */

__device__ __forceinline__ uint64_t entry_of(uint32_t key, uint32_t token)
{
    return ((uint64_t)key << 32) | (uint32_t)~token;
}
__device__ __forceinline__ uint32_t entry_key(uint64_t e) { return (uint32_t)(e >> 32); }
__device__ __forceinline__ uint32_t entry_token(uint64_t e) { return ~(uint32_t)e; }

using cr::exp_fast_d;

constexpr double kLog2e = 0x1.71547652b82fep+0;
constexpr double kLn2 = 0x1.62e42fefa39efp-1;

__device__ __forceinline__ uint64_t d2u(double x) { return __builtin_bit_cast(uint64_t, x); }
__device__ __forceinline__ double u2d(uint64_t u) { return __builtin_bit_cast(double, u); }

/* cap * tanh(x / cap).  kCapPoly (caps of up to 80): off by some 2^-52 of the cap,
 * below 1e-13.  kCapExact, whatever the cap: by less than 2^-49 of the value itself, since 1 - e
 * would leave nothing of a logit far below its cap. */
template <int MODE>
__device__ __forceinline__ double softcap64(float x, const BeamSoftcap& c)
{
    if constexpr (MODE == kCapNone) return (double)x;
    const double cap = (double)c.cap;
    if constexpr (MODE == kCapExact) return cap * cr::tanh_fast_d((double)x / cap);
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

/* 2^v(x): near, the term of a logit with |x| <= limit; far, of any unmasked one, relative to
 * ref (0 but where the softcap leaves binary32's range). */
template <int MODE>
__device__ __forceinline__ float near_term(float x, const BeamSoftcap& c)
{
    const double xd = (double)x;
    return pow2_of(xd * (MODE == kCapNone ? kLog2e : near_factor(xd, c)));
}
template <int MODE>
__device__ __forceinline__ float far_term(float x, double ref, const BeamSoftcap& c)
{
    const double v = value64<MODE>(x, c);
    return v == ref ? 1.0f : pow2_of(fmax(v - ref, -1000.0));
}

/* Sum over the 64 lanes, in every lane (all lanes active). */
__device__ __forceinline__ double wave_sum_f64(double v)
{
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
/* Sum over the workgroup, in thread 0. */
template <int BLOCK>
__device__ __forceinline__ double block_sum_f64(double v, double* s_wave)
{
    v = wave_sum_f64(v);
    if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x >> 6] = v;
    __syncthreads();
    double r = 0.0;
    if (threadIdx.x == 0)
#pragma unroll
        for (int w = 0; w < BLOCK / 64; ++w) r += s_wave[w];
    return r;
}

template <int BLOCK>
struct SelectShared {
    uint32_t tmax[BLOCK];
    uint32_t hist[256];
    int misc[8];
    int scan[BLOCK / 64];
    double red[BLOCK / 64];
    int count[3]; /* candidates that a tile listed, the tiles in turn */
    int flag;
    uint32_t far[BLOCK / 64][kBeamMaxTiles / 32]; /* tiles that a wave left for later */
    alignas(16) uint64_t list[kListCap]; /* candidates, in any order */
    alignas(16) uint64_t sorted[kNMax];
    double y[kNMax];
};

/* How many of the list's entries are better than `mine`. */
__device__ __forceinline__ int rank_in(const uint64_t* list, int cnt, uint64_t mine)
{
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < cnt; ++j) rank += list[j] > mine;
    return rank;
}

/* A lower bound of the n-th largest logit of the workgroup's tile, from the threads'
 * largest keys in sh.tmax: -inf where fewer than n threads hold a candidate. */
template <int BLOCK>
__device__ __forceinline__ float tile_bound(int n, SelectShared<BLOCK>& sh)
{
    const int lane = threadIdx.x & 63;
    uint32_t v[BLOCK / 64];
    int nz = 0;
#pragma unroll
    for (int q = 0; q < BLOCK / 64; ++q) {
        v[q] = sh.tmax[lane + 64 * q];
        nz += __popcll(__ballot(v[q] != 0u));
    }
    const uint32_t t = nz >= n ? wave_kth_bound<BLOCK / 64>(v, n, kBoundBits) : 0u;
    return t == 0u ? -__builtin_inff() : key2f(t);
}

/* The workgroup's best candidates so far: `listed` entries of sh.list, among
 * them the n best (n <= kNMax) or all there are.  No later logit that is not above `floor`
 * can be among the n best: n listed ones are at or above it, and of equal
 * logits the earlier come first. */
struct Best {
    float floor = kMasked;
    float before = kMasked; /* the floor before the last tile */
    int listed = 0;
    int tile = 0;
};

/* A tile's candidates join the list; a barrier a tile.  x(e), e < E: this thread's
 * logits, token(e) their tokens; none is above `largest`, and one is `sure` or
 * larger unless that is -inf.
 *
 * The first tile lists what reaches tile_bound, few elements beside the n
 * best for n well below the threads; later ones what is above the floor, and
 * where more lanes than n hold such, what reaches their wave's n-th lane.  The
 * count of a tile is looked at behind the next one's barrier (list_settle), so
 * its word must stay until the one after. */
template <int BLOCK, int E, typename ValueF, typename TokenF>
__device__ __forceinline__ void list_tile(Best& best, float largest, float sure, ValueF x,
                                          TokenF token, int n, SelectShared<BLOCK>& sh)
{
    const int at = best.tile % 3;
    if (threadIdx.x == 0) sh.count[(best.tile + 1) % 3] = 0;
    best.before = best.floor;
    float bound = -__builtin_inff();
    if (best.tile == 0) {
        bound = tile_bound<BLOCK>(n, sh);
    } else if (__popcll(__ballot(sure > best.floor)) > n) {
        const uint32_t key[1] = {cand_key(sure)};
        bound = key2f(wave_kth_bound<1>(key, n, kBoundBits));
    }
    if (__any(largest > best.floor && largest >= bound)) {
        /* few elements pass: by eights, most of which no lane takes further (and
         * one after another, or they would hold registers together) */
#pragma unroll
        for (int e0 = 0; e0 < E; e0 += 8) {
            float m = x(e0);
#pragma unroll
            for (int e = e0 + 1; e < e0 + 8; ++e) m = fmaxf(m, x(e));
            if (__any(m > best.floor && m >= bound)) {
#pragma unroll
                for (int e = e0; e < e0 + 8; ++e) {
                    const float v = x(e);
                    if (v > best.floor && v >= bound) {
                        const int p = best.listed + atomicAdd(&sh.count[at], 1);
                        if (p < kListCap) sh.list[p] = entry_of(f2key(v), token(e));
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (best.tile == 0 && bound > best.floor) best.floor = bound;
    ++best.tile;
}

/* Behind a barrier, after a tile: entry(i), i < count, are all of its candidates, in token
 * order, read again.  Where they were more than the list holds (equal logits
 * in masses), the tile's n-th largest key is selected exactly and of its
 * copies the first are taken.  A list that has grown is cut down to its n
 * best, whose last is the new floor. */
template <int BLOCK, typename EntryF>
__device__ __forceinline__ void list_settle(Best& best, int count, EntryF entry, int n,
                                            SelectShared<BLOCK>& sh)
{
    const int tid = threadIdx.x;
    int* word = &sh.count[(best.tile - 1) % 3];
    int cnt = best.listed + *word;
    if (cnt > kListCap) {
        __syncthreads();
        if (tid == 0) *word = 0;
        auto key = [&](int i) {
            const uint64_t c = entry(i);
            return c && key2f(entry_key(c)) > best.before ? entry_key(c) : 0u;
        };
        int gt, eq;
        const uint32_t kth = block_radix_kth<BLOCK>(
            count, n, key, [&](int i) { return key(i) != 0u; }, sh.hist, sh.misc, &gt, &eq);
        int taken = gt;
#pragma unroll 1
        for (int i0 = 0; i0 < count; i0 += BLOCK) {
            const uint64_t c = i0 + tid < count ? entry(i0 + tid) : 0ull;
            const uint32_t k = entry_key(c);
            if (k > kth) sh.list[best.listed + atomicAdd(word, 1)] = c;
            const int same = c != 0ull && k == kth;
            int total;
            const int p = taken + block_exclusive_scan<BLOCK>(same, sh.scan, total);
            if (same && p < n) sh.list[best.listed + p] = c;
            taken += total;
        }
        best.floor = key2f(kth);
        cnt = best.listed + n;
        __syncthreads();
    }
    if (cnt >= 2 * n + 32 || cnt > kListCap - kNMax) {
        for (int i = tid; i < cnt; i += BLOCK) {
            const uint64_t e = sh.list[i];
            const int rank = rank_in(sh.list, cnt, e);
            if (rank < n) sh.sorted[rank] = e;
        }
        __syncthreads();
        cnt = n;
        for (int i = tid; i < n; i += BLOCK) sh.list[i] = sh.sorted[i];
        best.floor = key2f(entry_key(sh.sorted[n - 1]));
    }
    best.listed = cnt;
}

/* The list's n best into sh.sorted (behind a barrier); returns how many. */
template <int BLOCK>
__device__ __forceinline__ int list_sort(const Best& best, int n, SelectShared<BLOCK>& sh)
{
    for (int i = threadIdx.x; i < best.listed; i += BLOCK) {
        const uint64_t e = sh.list[i];
        const int rank = rank_in(sh.list, best.listed, e);
        if (rank < n) sh.sorted[rank] = e;
    }
    __syncthreads();
    return best.listed < n ? best.listed : n;
}

/* ------------------------------------------------------------------ chunks */

template <int MODE, int BLOCK>
__device__ void merge_row(const BeamSelectArgs& a, int row, SelectShared<BLOCK>& sh);
template <int MODE, int BLOCK>
__device__ void end_row(const BeamSelectArgs& a, int row, int cnt, double sum,
                        SelectShared<BLOCK>& sh);
template <int BLOCK>
__device__ void merge_sequence(const BeamSelectArgs& a, int b, SelectShared<BLOCK>& sh,
                               double* sc);

template <int DT>
__device__ __forceinline__ u32x4 load_raw(const char* row, int64_t e0, int vocab)
{
    if (e0 + Elem<DT>::VW <= vocab)
        return *reinterpret_cast<const u32x4*>(row + e0 * Elem<DT>::SIZE);
    float v[Elem<DT>::VW];
#pragma unroll
    for (int i = 0; i < Elem<DT>::VW; ++i)
        v[i] = e0 + i < vocab ? load_elem<DT>(row, e0 + i) : -__builtin_inff();
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r[i] = DT == 0 ? __float_as_uint(v[i])
                       : (__float_as_uint(v[2 * i % Elem<DT>::VW]) >> 16) |
                             (__float_as_uint(v[(2 * i + 1) % Elem<DT>::VW]) & 0xFFFF0000u);
    return r;
}
/* Element e of the vectors r. */
template <int DT, int NV>
__device__ __forceinline__ float raw_value(const u32x4 (&r)[NV], int e)
{
    if constexpr (DT == 0) return __uint_as_float(r[e / 4][e % 4]);
    const uint32_t w = r[e / 8][e % 8 / 2];
    return __uint_as_float(e & 1 ? w & 0xFFFF0000u : w << 16);
}

typedef __attribute__((address_space(3))) const float LdsFloat;

/* The vectors as new values: what was unpacked from them before is unpacked
 * again rather than held in registers. */
template <int NV>
__device__ __forceinline__ void forget(u32x4 (&r)[NV])
{
#pragma unroll
    for (int j = 0; j < NV; ++j) __asm__ volatile("" : "+v"(r[j]));
}

/* Sum of four terms: in binary32, which rounds twice; such sums are added in
 * binary64.  A row's sum, and so lse, is off by less than 2.6e-7 of itself: these two
 * roundings 2^-23, a term's exponential 8.4e-8 (v_exp_f32 over [-1/2, 1/2], every value
 * measured) and its argument's rounding 1.1e-8, the polynomial 5.4e-10 of the cap, at most 4.4e-8. */
__device__ __forceinline__ double sum_four(const float (&t)[4])
{
    return (double)((t[0] + t[1]) + (t[2] + t[3]));
}

/* One workgroup per chunk of a row, which it takes tile by tile, the next one
 * loading while one is worked on: its n best candidates, ranked, and its part of the softmax
 * denominator.
 *
 * A term is 2^v(x), v(x) = log2(e) cap tanh(x/cap), without a reference: the
 * softcap keeps it within binary32 (so do logits within +-80 where there is
 * no cap).  v is a polynomial evaluated in binary64, whose instructions
 * issue as binary32's other than multiply-add do on this machine (4.7 against 2.7
 * cycles measured), and its fraction alone goes through binary32's exponential:
 * binary32 throughout leaves errors of 1e-6 in the terms of equal logits, and rows of
 * bf16 have thousands of those.  bf16 logits in long rows of a batch need no
 * arithmetic: their terms are looked up (TABLE), 30 KiB in LDS that hold the
 * terms of all values from 2^-24 to 64.
 *
 * The workgroup that ends last in a row merges its chunks, the one that ends
 * last in a sequence its rows.
 *
 * 512 rows of 262,144 bf16 logits: 72 us, 3.7 TB/s, bound by neither side alone: the
 * vector units issue for 38 us of it (11 instructions a logit), memory would take 43, and the
 * start and the end of the workgroups, 17 us, overlap nothing.  Without the table
 * 181 us (issue), with the binary64 softmax throughout 841.  64 binary32 rows: 36 us,
 * 11 of them the terms' issue, 20 the start and the merges.  Four rows:
 * 17 us, all of it latency.
 *
 * The longer ways: with half of the logits at -1e4 or -1e9, which are not masked, four binary32
 * rows take 23 us, 64 85 and 512 bf16 rows 423; without a cap 20, 59 and 306; with a cap
 * above 80, evaluated in a second pass, 23, 76 to 86 and 450 to 525. */
template <int DT, int MODE, bool TABLE, int BLOCK>
__global__ __launch_bounds__(BLOCK, 4) void beam_select_kernel(BeamSelectArgs a)
{
    constexpr int VW = Elem<DT>::VW;
    constexpr int TILE = TABLE ? kBeamTableTile : kBeamTile;
    constexpr int NV = TILE / BLOCK / VW;
    constexpr int E = NV * VW;
    extern __shared__ double dyn[]; /* terms; then the sequence's scores */
    __shared__ SelectShared<BLOCK> sh;
    const int row = blockIdx.y, ch = blockIdx.x, tid = threadIdx.x;
    const int b = row / a.beams;
    const bool live = a.scores[row] > kMasked;
    if (live) {
        const char* base =
            static_cast<const char*>(a.logits) + (int64_t)row * a.row_stride * Elem<DT>::SIZE;
        int first = ch * a.tiles * TILE; /* of the tile; chunks start within the row */
        const int64_t stop = (int64_t)first + (int64_t)a.tiles * TILE;
        const int end = stop < a.vocab ? (int)stop : a.vocab;
        u32x4 r[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j)
            r[j] = load_raw<DT>(base, (int64_t)first + (j * BLOCK + tid) * VW, a.vocab);
        if constexpr (TABLE) {
            float* table = reinterpret_cast<float*>(dyn);
            for (int i = tid; i < 2 * kBeamTableHalf / 4; i += BLOCK)
                reinterpret_cast<u32x4*>(table)[i] = reinterpret_cast<const u32x4*>(a.ws.table)[i];
            /* (complete behind the first tile's barrier) */
        }
        for (int i = tid & 63; i < kBeamMaxTiles / 32; i += 64) sh.far[tid / 64][i] = 0u;
        if (tid < 3) sh.count[tid] = 0;
        Best best;
        double s = 0.0;
        bool redo = MODE == kCapExact;
        /* unmasked and beyond what the table or the polynomial serves */
        auto is_far = [&](float v) {
            return v > kMasked && (TABLE ? fabsf(v) >= 64.0f : fabsf(v) > a.cap.limit);
        };
        /* the tile at `from` is all listed */
        auto settle = [&](int from) {
            list_settle<BLOCK>(
                best, a.vocab - from < TILE ? a.vocab - from : TILE,
                [&](int i) {
                    const uint32_t key = cand_key(load_elem<DT>(base, (int64_t)from + i));
                    return key ? entry_of(key, (uint32_t)(from + i)) : 0ull;
                },
                a.n, sh);
        };
        for (int tile = 0; first < end; first += TILE, ++tile) {
            u32x4 next[NV];
            if (first + TILE < end) {
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    next[j] = load_raw<DT>(base, (int64_t)first + TILE + (j * BLOCK + tid) * VW,
                                           a.vocab);
            }
            auto value = [&](int e) { return raw_value<DT, NV>(r, e); };
            auto offset = [&](int e) { return ((e / VW) * BLOCK + tid) * VW + e % VW; };
            float largest, sure, least;
            bool plain; /* every logit unmasked and within the way's limit */
            if constexpr (TABLE) {
                /* as 16-bit integers: the largest of the positive ones, the smallest
                 * magnitude of negative ones alone, the largest magnitude */
                i16x2 up = __builtin_bit_cast(i16x2, r[0][0]);
                u16x2 low = __builtin_bit_cast(u16x2, r[0][0]), wide = low;
#pragma unroll
                for (int i = 1; i < 4 * NV; ++i) {
                    const uint32_t w = r[i / 4][i % 4];
                    up = __builtin_elementwise_max(up, __builtin_bit_cast(i16x2, w));
                    low = __builtin_elementwise_min(low, __builtin_bit_cast(u16x2, w));
                    wide = __builtin_elementwise_max(wide, __builtin_bit_cast(u16x2, w));
                }
                const int u = up.x > up.y ? up.x : up.y;
                const uint32_t l = low.x < low.y ? low.x : low.y;
                const uint32_t m = wide.x > wide.y ? wide.x : wide.y;
                const uint32_t negative = m >> 15 ? m & 0x7FFFu : 0u;
                const uint32_t most = u > (int)negative ? (uint32_t)u : negative;
                largest = sure = __uint_as_float((u >= 0 ? (uint32_t)u : l) << 16);
                if (most > 0x7F80u) { /* a NaN: nothing known */
                    largest = __builtin_inff();
                    sure = -__builtin_inff();
                }
                plain = __all(most < (uint32_t)kBeamTableHigh);
            } else {
                largest = least = value(0);
#pragma unroll
                for (int e = 1; e < E; ++e) {
                    largest = fmaxf(largest, value(e));
                    least = fminf(least, value(e));
                }
                sure = largest;
                plain = __all(least >= -a.cap.limit && largest <= a.cap.limit);
            }
            if constexpr (DT == 1) forget(r);
            if (tile == 0) sh.tmax[tid] = cand_key(sure);
            __syncthreads();
            if (tile > 0) settle(first - TILE);
            list_tile<BLOCK, E>(
                best, largest, sure, value, [&](int e) { return (uint32_t)(first + offset(e)); },
                a.n, sh);
            if constexpr (DT == 1) forget(r);

            if constexpr (MODE != kCapExact) {
                /* most waves; then those with masked logits or NaNs (which minimum
                 * and maximum do not see); then, behind the loop, so that
                 * it costs the others no registers, those with logits beyond the limit */
                double part = 0.0;
                bool far = false;
                if constexpr (TABLE) {
                    const uint32_t table = (uint32_t)(uintptr_t)(LdsFloat*)dyn;
                    if (plain) {
                        u16x2 four = (u16x2)4;
                        const u16x2 start = (u16x2)(uint16_t)(table - 4 * kBeamTableLow);
                        __asm__("" : "+v"(four)); /* multiplied and added at once */
#pragma unroll
                        for (int i = 0; i < 4 * NV; i += 2) {
                            float t[4];
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                /* byte addresses modulo 2^16, where the parts may
                                 * overflow: 4 (max(magnitude, low) - low) + table, and
                                 * half the table further where negative */
                                const uint32_t w = r[(i + q) / 4][(i + q) % 4];
                                u16x2 m = __builtin_bit_cast(u16x2, w & 0x7FFF7FFFu);
                                u16x2 neg = __builtin_bit_cast(
                                    u16x2, __builtin_bit_cast(i16x2, w) >> 15);
                                __asm__("" : "+v"(neg)); /* a factor, no selection */
                                m = __builtin_elementwise_max(m, (u16x2)kBeamTableLow);
                                m = m * four + start;
                                m = neg * (u16x2)(uint16_t)(-4 * kBeamTableHalf) + m;
                                const uint32_t at = __builtin_bit_cast(uint32_t, m);
                                t[2 * q] = *(LdsFloat*)(uintptr_t)(at & 0xFFFFu);
                                t[2 * q + 1] = *(LdsFloat*)(uintptr_t)(at >> 16);
                            }
                            part += sum_four(t);
                            if (i % 4 == 2) __builtin_amdgcn_sched_barrier(0);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < E; e += 4) {
                            float t[4];
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const float v = value(e + q);
                                const uint32_t bits = __float_as_uint(v) >> 16;
                                uint32_t m = bits & 0x7FFFu;
                                far |= is_far(v);
                                const bool here = v > kMasked && !is_far(v);
                                m = m < (uint32_t)kBeamTableLow ? kBeamTableLow : m;
                                m = m >= (uint32_t)kBeamTableHigh ? kBeamTableHigh - 1 : m;
                                m += (bits >> 15) * kBeamTableHalf - kBeamTableLow;
                                const float u = *(LdsFloat*)(uintptr_t)(table + 4 * m);
                                t[q] = here ? u : 0.0f;
                            }
                            part += sum_four(t);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                } else {
                    bool done = plain;
                    if (done) {
#pragma unroll
                        for (int e = 0; e < E; e += 4) {
                            float t[4];
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                t[q] = near_term<MODE>(value(e + q), a.cap);
                            part += sum_four(t);
                        }
                        done = __all(part == part);
                    }
                    if (!done) {
                        part = 0.0;
                        forget(r);
#pragma unroll
                        for (int e = 0; e < E; e += 4) {
                            float t[4];
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const float v = value(e + q);
                                far |= is_far(v);
                                t[q] = near_term<MODE>(v, a.cap);
                                t[q] = v > kMasked && !is_far(v) ? t[q] : 0.0f;
                            }
                            part += sum_four(t);
                        }
                    }
                }
                if (__any(far)) {
                    redo = true;
                    if ((tid & 63) == 0) sh.far[tid / 64][tile / 32] |= 1u << (tile & 31);
                }
                s += part;
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) r[j] = next[j];
        }
        if constexpr (MODE == kCapPoly) {
            __syncthreads();
#pragma unroll 1
            for (int t = 0; t < a.tiles; ++t) {
                if (!(sh.far[tid / 64][t / 32] >> (t & 31) & 1u)) continue;
                const int64_t from = ((int64_t)ch * a.tiles + t) * TILE;
                auto at = [&](int e) { return from + ((e / VW) * BLOCK + tid) * VW + e % VW; };
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    r[j] = load_raw<DT>(base, at(j * VW), a.vocab);
                uint32_t which = 0;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    which |= is_far(raw_value<DT, NV>(r, e)) ? 1u << e : 0u;
                while (__any(which != 0u))
                    if (which) {
                        const int e = __builtin_ctz(which);
                        which &= which - 1;
                        s += (double)far_term<MODE>(load_elem<DT>(base, at(e)), 0.0, a.cap);
                    }
            }
        }
        __syncthreads();
        settle(first - TILE);
        __syncthreads();
        const int cnt = list_sort<BLOCK>(best, a.n, sh);
        double ref = 0.0;
        if (MODE != kCapPoly && __syncthreads_or(redo && cnt)) {
            /* relative to the chunk's largest logit, in a second pass */
            const float top = key2f(entry_key(sh.sorted[0]));
            ref = value64<MODE>(top, a.cap);
            s = 0.0;
#pragma unroll 1
            for (int i = ch * a.tiles * TILE + tid; i < end; i += BLOCK) {
                const float v = load_elem<DT>(base, i);
                if (v > kMasked)
                    s += v == top ? 1.0 : (double)far_term<MODE>(v, ref, a.cap);
            }
        }
        s = block_sum_f64<BLOCK>(s, sh.red);
        if (a.chunks == 1) {
            if (cnt)
                s *= term64(ref * kLn2,
                            value64<MODE>(key2f(entry_key(sh.sorted[0])), a.cap) * kLn2);
            end_row<MODE, BLOCK>(a, row, cnt, s, sh);
        } else {
            const int64_t at = (int64_t)row * a.chunks + ch;
            for (int i = tid; i < a.n; i += BLOCK)
                st_dev(&a.ws.cand[at * a.n + i], i < cnt ? sh.sorted[i] : (uint64_t)0);
            if (tid == 0) {
                st_dev(&a.ws.sums[2 * at], d2u(s));
                st_dev(&a.ws.sums[2 * at + 1], d2u(ref));
            }
        }
    }
    /* a dead row's workgroups arrive too: the last of a sequence may overwrite
     * its scores, which all of them must have read */
    if (a.chunks > 1 && !elect_last(&a.ws.tickets[row], (uint32_t)a.chunks, &sh.flag)) return;
    if (!live) {
        if (tid == 0 && a.lse) a.lse[row] = -__builtin_inff();
        for (int i = tid; i < a.n; i += BLOCK)
            st_dev(&a.ws.best[(int64_t)row * a.n + i], (uint64_t)0);
    } else if (a.chunks > 1) {
        merge_row<MODE, BLOCK>(a, row, sh);
    }
    if (a.beams > 1 &&
        !elect_last(&a.ws.tickets[a.batch * a.beams + b], (uint32_t)a.beams, &sh.flag))
        return;
    if (a.beams == 1) {
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
    }
    merge_sequence<BLOCK>(a, b, sh, dyn);
}

/* -------------------------------------------------------------------- rows */

/* A row's n best and its normaliser from its chunks'. */
template <int MODE, int BLOCK>
__device__ __forceinline__ void merge_row(const BeamSelectArgs& a, int row,
                                          SelectShared<BLOCK>& sh)
{
    constexpr int E = 8;
    const int tid = threadIdx.x;
    const uint64_t* cand = a.ws.cand + (int64_t)row * a.chunks * a.n;
    const int total = a.chunks * a.n;
    if (tid < 3) sh.count[tid] = 0;
    /* one chunk's sum a thread, on its way while the candidates are merged */
    const uint64_t* sums = a.ws.sums + (int64_t)row * a.chunks * 2;
    double sum = 0.0, ref = 0.0;
    if (tid < a.chunks) {
        sum = u2d(ld_dev(&sums[2 * tid]));
        ref = u2d(ld_dev(&sums[2 * tid + 1]));
    }
    Best best;
    int base = 0;
    /* the chunks' lists lie in token order, so copies of one key do too */
    auto count = [&](int from) { return total - from < E * BLOCK ? total - from : E * BLOCK; };
    auto settle = [&](int from) {
        list_settle<BLOCK>(
            best, count(from), [&](int i) { return ld_dev(&cand[from + i]); }, a.n, sh);
    };
    for (; base < total; base += E * BLOCK) {
        float x[E];
        uint32_t tok[E];
        float largest = -__builtin_inff();
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = e * BLOCK + tid;
            const uint64_t c =
                e * BLOCK < count(base) && i < count(base) ? ld_dev(&cand[base + i]) : 0ull;
            x[e] = c ? key2f(entry_key(c)) : -__builtin_inff();
            tok[e] = entry_token(c);
            largest = fmaxf(largest, x[e]);
        }
        if (base == 0) sh.tmax[tid] = cand_key(largest);
        __syncthreads();
        if (base) settle(base - E * BLOCK);
        list_tile<BLOCK, E>(
            best, largest, largest, [&](int e) { return x[e]; }, [&](int e) { return tok[e]; },
            a.n, sh);
    }
    __syncthreads();
    settle(base - E * BLOCK);
    __syncthreads();
    const int cnt = list_sort<BLOCK>(best, a.n, sh);
    /* the chunks' sums relative to the row's largest logit */
    const double vtop = cnt ? value64<MODE>(key2f(entry_key(sh.sorted[0])), a.cap) : 0.0;
    double s = 0.0;
    for (int c = tid; c < a.chunks;) {
        if (sum > 0.0) s += sum * term64(ref * kLn2, vtop * kLn2);
        c += BLOCK;
        if (c < a.chunks) {
            sum = u2d(ld_dev(&sums[2 * c]));
            ref = u2d(ld_dev(&sums[2 * c + 1]));
        }
    }
    end_row<MODE, BLOCK>(a, row, cnt, block_sum_f64<BLOCK>(s, sh.red), sh);
}

/* The row's cnt best candidates in sh.sorted; sum, in thread 0: its terms relative to the
 * largest. */
template <int MODE, int BLOCK>
__device__ __forceinline__ void end_row(const BeamSelectArgs& a, int row, int cnt, double sum,
                                        SelectShared<BLOCK>& sh)
{
    const int tid = threadIdx.x;
    for (int i = tid; i < cnt; i += BLOCK)
        sh.y[i] = softcap64<MODE>(key2f(entry_key(sh.sorted[i])), a.cap);
    __syncthreads();
    const double top = cnt ? sh.y[0] : -__builtin_inf();
    for (int i = tid; i < a.n; i += BLOCK) {
        uint64_t e = i < cnt ? sh.sorted[i] : 0ull;
        double y = -__builtin_inf();
        if (e) {
            /* where tanh saturates its last bit may waver: the list may not rise */
            y = top;
#pragma unroll 8
            for (int j = 1; j <= i; ++j) y = fmin(y, sh.y[j]);
            /* beside an infinite largest logit the rest have probability 0 */
            if (top == __builtin_inf() && y != top) e = 0ull;
        }
        st_dev(&a.ws.best[(int64_t)row * a.n + i], e);
        st_dev(&a.ws.y[(int64_t)row * a.n + i], d2u(y));
    }
    if (tid == 0) {
        const double ls = log64(sum);
        st_dev(&a.ws.norm[2 * row], d2u(top));
        st_dev(&a.ws.norm[2 * row + 1], d2u(ls));
        if (a.lse) a.lse[row] = cnt ? (float)(top + ls) : -__builtin_inff();
    }
}

/* --------------------------------------------------------------- sequences */

/* The n best of the sequence's W sorted lists: a candidate's rank is the
 * number of better ones, counted, or found in each list by bisection. */
template <int BLOCK>
__device__ __forceinline__ void merge_sequence(const BeamSelectArgs& a, int b,
                                               SelectShared<BLOCK>& sh, double* sc)
{
    /* sc: [W][n] scores, -inf = none */
    const int tid = threadIdx.x;
    const int W = a.beams, n = a.n, total = W * n;
    const uint64_t* best = a.ws.best + (int64_t)b * total;
    const uint64_t* ys = a.ws.y + (int64_t)b * total;
    int found = 0;
    uint64_t mine = 0ull; /* this thread's first candidate */
    for (int i = tid; i < total; i += BLOCK) {
        const int w = i / n;
        const uint64_t* norm = a.ws.norm + 2 * ((int64_t)b * W + w);
        const uint64_t e = ld_dev(&best[i]);
        const double y = u2d(ld_dev(&ys[i]));
        const double top = u2d(ld_dev(&norm[0])), ls = u2d(ld_dev(&norm[1]));
        double s = -__builtin_inf();
        if (e) { /* (of a dead row nothing else was written) */
            s = (double)a.scores[b * W + w] + ((y == top ? 0.0 : y - top) - ls);
            ++found;
        }
        if (i == tid) mine = e;
        sc[i] = s;
    }
    found = block_sum_i32<BLOCK>(found, sh.scan);
    int32_t* parents = a.parents + (int64_t)b * n;
    int32_t* tokens = a.tokens + (int64_t)b * n;
    float* out = a.out + (int64_t)b * n;
    for (int i = tid; i < total; i += BLOCK) {
        const double s = sc[i];
        if (s == -__builtin_inf()) continue;
        const int w = i / n;
        int rank = 0;
        if (total <= 64) {
            /* few: counted (0.5 us less for 32); of equal scores those of the lower beam,
             * and within a beam the earlier, come first */
#pragma unroll 4
            for (int j = 0; j < total; ++j) rank += sc[j] > s || (sc[j] == s && j < i);
        } else {
            rank = i - w * n;
            for (int o = 0; o < W && rank < n; ++o) {
                if (o == w) continue;
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
        }
        if (rank < n) {
            parents[rank] = b * W + w;
            tokens[rank] = (int32_t)entry_token(i == tid ? mine : ld_dev(&best[i]));
            out[rank] = (float)s;
        }
    }
    for (int i = found + tid; i < n; i += BLOCK) {
        parents[i] = -1;
        tokens[i] = -1;
        out[i] = -__builtin_inff();
    }
}

/* ----------------------------------------------------------------- reorder */

/* One thread holds the bytes of one column of all of a sequence's rows: it
 * reads the parents' and then writes, so in place no row is overwritten
 * before it was read, and nothing has to be kept elsewhere.  Bound by memory: 64 rows
 * of 1.5 MB in eight planes into another buffer take 214 us, 5.4 TB/s; the
 * streaming stores are worth a tenth (242 us without).  A parent that several
 * rows share is read from cache, so its loads are not streaming (256 us). */
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
                const uint32_t p = (uint32_t)a.parents[b * W + r] - (uint32_t)(b * W);
                const int from = p < (uint32_t)W ? (int)p : r;
                if (!inplace || from != r)
                    v[r] = *reinterpret_cast<const T*>(a.src + at + (int64_t)from * a.row_stride);
            }
#pragma unroll
        for (int r = 0; r < WMAX; ++r)
            if (r < W) {
                const uint32_t p = (uint32_t)a.parents[b * W + r] - (uint32_t)(b * W);
                const int from = p < (uint32_t)W ? (int)p : r;
                if (!inplace || from != r)
                    __builtin_nontemporal_store(
                        v[r], reinterpret_cast<T*>(a.dst + at + (int64_t)r * a.row_stride));
            }
    }
}

template <typename T>
hipError_t reorder_with(const BeamReorderArgs& all, hipStream_t stream)
{
    /* a launch has fewer than 2^32 threads across, and more would be cut off
     * without an error: longer rows (odd ones of 4 GiB) go column range by column range */
    constexpr int64_t kMost = (int64_t)1 << 31;
    const int64_t cols = all.row_bytes / (int64_t)sizeof(T);
    const int64_t groups = (int64_t)all.batch * all.planes;
    for (int64_t first = 0; first < cols; first += kMost) {
        BeamReorderArgs a = all;
        const int64_t n = cols - first < kMost ? cols - first : kMost;
        a.src += first * (int64_t)sizeof(T);
        a.dst += first * (int64_t)sizeof(T);
        a.row_bytes = n * (int64_t)sizeof(T);
        const dim3 grid((unsigned)((n + kB - 1) / kB), (unsigned)(groups < 65535 ? groups : 65535));
        hipError_t e;
        if (a.beams <= 4)
            e = launch(beam_reorder_kernel<T, 4>, grid, kB, 0, stream, a);
        else if (a.beams <= 8)
            e = launch(beam_reorder_kernel<T, 8>, grid, kB, 0, stream, a);
        else if (a.beams <= 16)
            e = launch(beam_reorder_kernel<T, 16>, grid, kB, 0, stream, a);
        else if (a.beams <= 32)
            e = launch(beam_reorder_kernel<T, 32>, grid, kB, 0, stream, a);
        else
            e = launch(beam_reorder_kernel<T, 64>, grid, kB, 0, stream, a);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
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
        c.limit = 80.0f;
        return c;
    }
    const double d = (double)cap;
    c.mode = cap >= 1e-12f && cap <= 80.0f ? kCapPoly : kCapExact;
    double scale = kLog2e;
    for (int i = 0; i < 10; ++i) {
        c.q[i] = q[i] * scale;
        scale /= d * d;
    }
    c.limit = (float)(1.25 * d);
    return c;
}

namespace {

template <int MODE>
__global__ __launch_bounds__(kB) void beam_init_kernel(BeamWorkspace ws, BeamSoftcap cap,
                                                       int tickets)
{
    const int at = blockIdx.x * kB + threadIdx.x;
    for (int i = at; i < tickets; i += gridDim.x * kB) ws.tickets[i] = 0u;
    for (int i = at; i < 2 * kBeamTableHalf; i += gridDim.x * kB) {
        const uint32_t mag = i % kBeamTableHalf;
        const float x = mag ? __uint_as_float((mag + kBeamTableLow) << 16) : 0.0f;
        const double y = softcap64<MODE>(i < kBeamTableHalf ? x : -x, cap);
        ws.table[i] = (float)exp_fast_d(y);
    }
}

template <int DT, int MODE>
hipError_t select_launch(const BeamSelectArgs& a, const BeamPlan& plan, hipStream_t stream)
{
    const dim3 grid((unsigned)a.chunks, (unsigned)(a.batch * a.beams));
    const size_t scores = sizeof(double) * a.beams * a.n;
    if constexpr (DT == 1 && MODE != kCapExact) {
        if (plan.table) {
            const size_t table = sizeof(float) * 2 * kBeamTableHalf;
            return launch(beam_select_kernel<DT, MODE, true, 512>, grid, 512,
                          table > scores ? table : scores, stream, a);
        }
    }
    return launch(beam_select_kernel<DT, MODE, false, kB>, grid, kB, scores, stream, a);
}

}  // namespace

BeamPlan beam_plan(int32_t vocab, int32_t rows, int32_t dtype, int32_t mode, int32_t ncu)
{
    BeamPlan p{};
    /* Looking terms up takes loading the table (30 KiB a workgroup) and tiles of four times
     * the size.  It pays from about half such a tile a CU on: 8 rows of 262,144 take 18.5 us
     * with it and 20.5 without, 64 rows 25 and 34, 256 rows 46 and 83 (4 rows 18.6 and 17.3);
     * 48 rows of 50,000 18.8 and 18.5, 64 rows 19.2 and 20.0.  Rows of less than three tiles,
     * whose last is up to half of the work and may be all but empty, need three times as much:
     * 64 rows of 33,000 take 19.6 us with it and 17.8 without, 192 rows 24.7 and 24.0, 512
     * rows 24.9 and 41.5; 128 rows of 45,000 22.4 and 21.6, 160 rows 22.3 and 24.7.  Rows that do
     * not fill two tiles are better without: 2,048 rows of 8,000 take 64 us with it and
     * 37 without, of 16,000 59 and 56.  What the rule leaves is 6 per cent at most, where either
     * way fills a round of the device by a little (192 rows of 100,003: 42.8 and 40.4). */
    const int64_t half = (int64_t)ncu * kBeamTableTile / 2;
    p.table = dtype == G4S_DTYPE_BF16 && mode != kCapExact && vocab >= 2 * kBeamTableTile &&
              (int64_t)rows * vocab >= (vocab >= 3 * kBeamTableTile ? half : 3 * half);
    const int32_t tile = p.table ? kBeamTableTile : kBeamTile;
    const int32_t all = (vocab + tile - 1) / tile;
    /* a row's workgroups: the fewest tiles that some CU takes one after another, its workgroups
     * side by side counted as if in turn from `full` on, where they fill it; the start and end
     * of a workgroup cost about a tile (two with a table: 160 rows of 50,000 in four
     * workgroups a row take 37 us, in two 27) */
    const int64_t full = p.table ? 2 : 3;
    int64_t least = INT64_MAX;
    for (int32_t tiles = 1; tiles <= all; ++tiles) {
        const int32_t chunks = (all + tiles - 1) / tiles;
        if (chunks > 1 && (int64_t)rows * chunks > beam_max_chunks(vocab, rows, ncu)) continue;
        int64_t each = ((int64_t)rows * chunks + ncu - 1) / ncu;
        if (each < full) each = full;
        const int64_t cost = each * (tiles + (p.table ? 2 : 1));
        if (cost < least) {
            least = cost;
            p.chunks = chunks;
            p.tiles = tiles;
        }
    }
    return p;
}

int64_t beam_max_chunks(int32_t vocab, int32_t rows, int32_t ncu)
{
    const int64_t every = (int64_t)((vocab + kBeamTile - 1) / kBeamTile) * rows;
    const int64_t most = (int64_t)8 * ncu > rows ? (int64_t)8 * ncu : rows;
    return most < every ? most : every;
}

hipError_t beam_init_launch(const BeamWorkspace& ws, const BeamSoftcap& cap, int32_t tickets,
                            hipStream_t stream)
{
    if (cap.mode == kCapNone)
        return launch(beam_init_kernel<kCapNone>, 64, kB, 0, stream, ws, cap, tickets);
    return launch(beam_init_kernel<kCapPoly>, 64, kB, 0, stream, ws, cap, tickets);
}

hipError_t beam_select_launch(const BeamSelectArgs& a, const BeamPlan& plan, int32_t dtype,
                              hipStream_t stream)
{
    const bool f32 = dtype == G4S_DTYPE_F32;
    if (a.cap.mode == kCapNone)
        return f32 ? select_launch<0, kCapNone>(a, plan, stream)
                   : select_launch<1, kCapNone>(a, plan, stream);
    if (a.cap.mode == kCapPoly)
        return f32 ? select_launch<0, kCapPoly>(a, plan, stream)
                   : select_launch<1, kCapPoly>(a, plan, stream);
    return f32 ? select_launch<0, kCapExact>(a, plan, stream)
               : select_launch<1, kCapExact>(a, plan, stream);
}

hipError_t beam_reorder_launch(const BeamReorderArgs& a, hipStream_t stream)
{
    const uint64_t bits = (uint64_t)(uintptr_t)a.src | (uint64_t)(uintptr_t)a.dst |
                          (uint64_t)a.plane_stride | (uint64_t)a.row_stride |
                          (uint64_t)a.row_bytes;
    /* 64 beams of 16 bytes would not stay in registers: 4 bytes from 17 beams on, which
     * move 2.1 to 2.6 TB/s (352,944-byte rows of 16 x 17 beams in eight planes 552 us; of
     * 16 x 16 beams by 16 bytes 244).  Rows of odd sizes: 0.6 to 0.8 TB/s */
    if ((bits & 15) == 0 && a.beams <= 16) return reorder_with<u32x4>(a, stream);
    if ((bits & 3) == 0) return reorder_with<uint32_t>(a, stream);
    return reorder_with<uint8_t>(a, stream);
}

}  // namespace g4s
