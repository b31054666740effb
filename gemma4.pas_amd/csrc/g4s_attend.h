/*
 * g4s_attend.h -- what the attention kernels share: tiles of 32 tokens in matrix
 * registers, the softmax between them, and the joining of partial results.
 *
 * Products are taken as S^T = K Q^T and O^T = V^T P^T in 16x16x32 bf16 matrix
 * instructions.  A lane l (m = l % 16, g = l / 16) then has, for query column m of
 * a tile of 32 tokens, the scores of tokens 4 g + i and 16 + 4 g + i (i = 0 .. 3), and
 * these eight are what the second product wants from it, if its eight tokens
 * are taken in that order on both sides: weights go from one product to the
 * next without leaving their lane.  A lane's dims of O^T are (D / 16) (4 g + r) + i:
 * consecutive ones.
 */
#ifndef G4S_ATTEND_H
#define G4S_ATTEND_H

#include "g4s_cache.h"
#include "g4s_device.h"

namespace g4s {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_4 __attribute__((ext_vector_type(2), aligned(4)));

__device__ __forceinline__ float inf32() { return __builtin_inff(); }
__device__ __forceinline__ float nan32() { return __builtin_nanf(""); }

/* The largest, and the sum, of a column's four lanes (l, l + 16, l + 32, l + 48), in each of them: rows
 * of lanes are exchanged in registers, a shuffle through LDS takes ten times as long. */
__device__ __forceinline__ float column_max(float x)
{
    const uint32_t u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float column_sum(float x)
{
    const uint32_t u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(__uint_as_float(a[0]) + __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

/* What products are multiplied by, to base two (the scale's sign is in the queries).  Never 0, as what is
 * masked stays -inf; the least number in its place makes 2^-21 of the largest product. */
__device__ __forceinline__ float base_two(float scale)
{
    return fmaxf(__builtin_fabsf(scale * kLog2e), 0x1p-149f);
}

/* The first place that a query at `place` (which may be negative) sees. */
__device__ __forceinline__ int sees_from(const AttendArgs& a, int place)
{
    const int from = a.window > 0 ? (int)((uint32_t)place - (uint32_t)a.window + 1u) : 0;
    return from > 0 && a.window <= place ? from : 0;
}

/* Bit i: whether token tile0 + shift + i is one of first .. last. */
__device__ __forceinline__ uint64_t seen_bits(int tile0, int first, int last, int shift)
{
    const int lo = first - tile0, hi = last - tile0; /* as places of the tile */
    const uint64_t from = lo <= 0 ? ~(uint64_t)0 : lo > 63 ? 0 : ~(uint64_t)0 << lo;
    const uint64_t to = hi >= 63 ? ~(uint64_t)0 : hi < 0 ? 0 : ~(uint64_t)0 >> (63 - hi);
    return (from & to) >> shift;
}
/* x where bit i is set, `other` where it is not. */
__device__ __forceinline__ float where_bit(uint64_t bits, int i, float x, float other)
{
    const uint32_t w = i < 32 ? (uint32_t)bits : (uint32_t)(bits >> 32);
    const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)w, i & 31, 1);
    return __uint_as_float((__float_as_uint(x) & m) | (__float_as_uint(other) & ~m));
}

/* Whether a softmax moves to another base (to base two; -inf: none yet): the weights may grow to
 * 2^kSlack before it does, as moving costs a product for every sum. */
constexpr float kSlack = 8.0f;
__device__ __forceinline__ bool rebase(float base, float above)
{
    return base == -inf32() ? above > -inf32() : above > kSlack;
}

/* Eight bf16 of a matrix operand. */
union Frag {
    uint32_t w[4];
    bf16x8 v;
    i16x4 half; /* its first four */
};

/* Two codes of a word and their scale (a power of two) as bf16, which holds every product. */
template <bool HI>
__device__ __forceinline__ uint32_t widen2(uint32_t w, float scale)
{
    const bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI);
    return __builtin_bit_cast(uint32_t, r);
}

/* Low and high halves of two words. */
__device__ __forceinline__ uint32_t lows(uint32_t a, uint32_t b)
{
    return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
__device__ __forceinline__ uint32_t highs(uint32_t a, uint32_t b)
{
    return __builtin_amdgcn_perm(b, a, 0x07060302u);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b)
{
    bf16x2 r;
    r[0] = (__bf16)a;
    r[1] = (__bf16)b;
    return __builtin_bit_cast(uint32_t, r);
}

/* 1 in each byte of a word that is a NaN code. */
__device__ __forceinline__ uint32_t nan_codes(uint32_t w)
{
    return (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;
}
/* x, or NaN where the count n (0, 1, ..) is not 0.  (Arithmetic: comparisons for every register
 * of a tile would each hold a mask.) */
__device__ __forceinline__ float nan_where(float x, float n)
{
    const int32_t some = -(int32_t)__float_as_uint(n) >> 31;
    return __uint_as_float(__float_as_uint(x) | ((uint32_t)some & 0x7FC00000u));
}
/* The word with +0 in the place of NaN codes. */
__device__ __forceinline__ uint32_t without_nan(uint32_t w) { return w & ~(nan_codes(w) * 0xFFu); }

/* Words of four dims of eight (or four) tokens, as operands of these tokens for each of the dims. */
template <int NJ>
__device__ __forceinline__ void value_frags(const uint32_t (&w)[NJ], const float (&scale)[NJ],
                                            Frag (&f)[4])
{
#pragma unroll
    for (int j = 0; j < NJ; j += 2) {
        const uint32_t a0 = widen2<false>(w[j], scale[j]);
        const uint32_t b0 = widen2<true>(w[j], scale[j]);
        const uint32_t a1 = widen2<false>(w[j + 1], scale[j + 1]);
        const uint32_t b1 = widen2<true>(w[j + 1], scale[j + 1]);
        f[0].w[j >> 1] = lows(a0, a1);
        f[1].w[j >> 1] = highs(a0, a1);
        f[2].w[j >> 1] = lows(b0, b1);
        f[3].w[j >> 1] = highs(b0, b1);
    }
}
/* The product over these tokens. */
template <int NJ>
__device__ __forceinline__ f32x4 multiply(const Frag& a, const Frag& b, f32x4 c)
{
    if constexpr (NJ == 8)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a.half, b.half, c, 0, 0, 0);
}

/* Eight consecutive elements of a query as a matrix operand: bf16 as they are, binary32 cut
 * into three bf16 pieces of eight bits, which together are the value (their
 * products with bf16 are exact).  An infinity becomes NaN (in binary32 the second piece does by
 * itself).  `in` false gives zeros, p is read all the same: a branch for each load costs more. */
template <int DT>
__device__ __forceinline__ void load_query(const char* p, bool in, bool negate,
                                           Frag (&f)[DT == G4S_DTYPE_F32 ? 3 : 1])
{
    const uint32_t keep = in ? ~0u : 0u, sign = negate ? 0x80008000u : 0u;
    if constexpr (DT == G4S_DTYPE_F32) {
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const u32x4 x = reinterpret_cast<const u32x4*>(p)[v];
            uint32_t part[3][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t u = x[i] & keep;
                const float r = __uint_as_float(u) - __uint_as_float(u & 0xFFFF0000u);
                const uint32_t w = __float_as_uint(r);
                part[0][i] = u;
                part[1][i] = w;
                part[2][i] = __float_as_uint(r - __uint_as_float(w & 0xFFFF0000u));
            }
#pragma unroll
            for (int s = 0; s < 3; ++s) {
                f[s].w[v * 2] = highs(part[s][0], part[s][1]) ^ sign;
                f[s].w[v * 2 + 1] = highs(part[s][2], part[s][3]) ^ sign;
            }
        }
    } else {
        const u32x4 x = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = x[i] & keep;
            /* (an exponent of ones carries into the sign's bit, which then sets the first of the fraction) */
            f[0].w[i] = (w | (((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u) >> 9) ^ sign;
        }
    }
}

template <int DT>
__device__ __forceinline__ void store4(char* p, f32x4 x)
{
    if constexpr (DT == G4S_DTYPE_F32) {
        *reinterpret_cast<f32x4*>(p) = x;
    } else {
        uint2 w;
        w.x = pack_bf16(x[0], x[1]);
        w.y = pack_bf16(x[2], x[3]);
        *reinterpret_cast<uint2*>(p) = w;
    }
}

/* 16 bytes at byte `at` of the workspace that another workgroup of this launch reads or wrote:
 * past the caches that are not common to all (st_dev and ld_dev, four times as wide). */
constexpr int kDeviceScope = 16;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t shared_space(float* p, uint32_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(p, 0, (int)bytes, 0x00027000);
}
__device__ __forceinline__ void st_dev4(__amdgpu_buffer_rsrc_t space, uint32_t at, f32x4 v)
{
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), space, (int)at, 0, kDeviceScope);
}
__device__ __forceinline__ f32x4 ld_dev4(__amdgpu_buffer_rsrc_t space, uint32_t at)
{
    return __builtin_bit_cast(
        f32x4, __builtin_amdgcn_raw_buffer_load_b128(space, (int)at, 0, kDeviceScope));
}

/* The joining of parts of a column, `n` of them at once: their maximum so far, sum and sums. */
struct Joined {
    float top = -inf32(), sum = 0.0f;
    f32x4 v = f32x4{0, 0, 0, 0};
};
template <int N>
__device__ __forceinline__ void join(Joined& j, int n, const float2 (&stats)[N], const f32x4 (&part)[N])
{
    float now = j.top;
#pragma unroll
    for (int w = 0; w < N; ++w) now = fmaxf(now, w < n ? stats[w].x : now);
    const float keep = j.top == -inf32() ? 0.0f : __builtin_amdgcn_exp2f(j.top - now);
    j.sum *= keep;
    j.v *= keep;
    j.top = now;
#pragma unroll
    for (int w = 0; w < N; ++w) {
        if (w >= n) break;
        const float f = stats[w].x == -inf32() ? 0.0f : __builtin_amdgcn_exp2f(stats[w].x - now);
        j.sum += stats[w].y * f;
        j.v += part[w] * f;
    }
}

/* A barrier for what is in LDS: loads and stores of memory stay in flight (the full one waits for a
 * workgroup's partial sums to reach the memory, 2 to 3 us). */
__device__ __forceinline__ void lds_barrier()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

/* Writes to LDS of this wave are read by its other lanes from here on. */
__device__ __forceinline__ void wave_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

}  // namespace g4s

#endif
