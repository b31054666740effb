/*
 * g4s_append.hip -- new keys and values into the pages of a cache in 8 bits,
 * rotated by their positions on the way, and the queries rotated beside
 * them, on gfx950.
 *
 * A workgroup takes up to TILE places of one row, whole blocks of tokens that share a
 * scale, so that a scale and the codes under it have one writer.  It goes
 * over their keys and values twice: for the largest magnitude of each block and
 * head, and to store them (the second time they come from the caches).
 * Rotations are computed in binary64 and rounded once: next to a border between two codes
 * a rounding in between would choose the other one.  Cosines and sines are computed once per
 * token and pair, in LDS for all heads.
 */
#include "g4s_cache.h"
#include "g4s_device.h"
#include "g4s_launch.h"

namespace g4s {

namespace {

constexpr int kB = 256;
constexpr int kTile = 16;    /* places of a workgroup, or one block where that is longer */
constexpr int kChunk = 8;    /* dims of a thread */
constexpr int kStep = 8;     /* tokens whose angles are in LDS at once */

typedef float f32x2 __attribute__((ext_vector_type(2)));

/* sin and cos of x (|x| < 2^40) to some 2^-52: x - n pi/2 with pi/2 in three
 * parts, then the Taylor series of both up to x^17 and x^18, whose next terms are below 2^-62 at
 * pi/4. */
__device__ __forceinline__ void sincos64(double x, double& s, double& c)
{
    const double n = __builtin_rint(x * 0x1.45f306dc9c883p-1);
    double r = __builtin_fma(-n, 0x1.921fb54442d18p+0, x);
    r = __builtin_fma(-n, 0x1.1a62633145c07p-54, r);
    r = __builtin_fma(-n, -0x1.f1976b7ed8fbcp-110, r);
    const double z = r * r;
    double p = 1.0 / 355687428096000.0;                       /* 1/17! */
    p = __builtin_fma(p, z, -1.0 / 1307674368000.0);          /* 1/15! */
    p = __builtin_fma(p, z, 1.0 / 6227020800.0);              /* 1/13! */
    p = __builtin_fma(p, z, -1.0 / 39916800.0);               /* 1/11! */
    p = __builtin_fma(p, z, 1.0 / 362880.0);                  /* 1/9! */
    p = __builtin_fma(p, z, -1.0 / 5040.0);                   /* 1/7! */
    p = __builtin_fma(p, z, 1.0 / 120.0);                     /* 1/5! */
    p = __builtin_fma(p, z, -1.0 / 6.0);                      /* 1/3! */
    const double sr = __builtin_fma(p * z, r, r);
    double q = -1.0 / 6402373705728000.0;                     /* 1/18! */
    q = __builtin_fma(q, z, 1.0 / 20922789888000.0);          /* 1/16! */
    q = __builtin_fma(q, z, -1.0 / 87178291200.0);            /* 1/14! */
    q = __builtin_fma(q, z, 1.0 / 479001600.0);               /* 1/12! */
    q = __builtin_fma(q, z, -1.0 / 3628800.0);                /* 1/10! */
    q = __builtin_fma(q, z, 1.0 / 40320.0);                   /* 1/8! */
    q = __builtin_fma(q, z, -1.0 / 720.0);                    /* 1/6! */
    q = __builtin_fma(q, z, 1.0 / 24.0);                      /* 1/4! */
    q = __builtin_fma(q, z, -0.5);
    const double cr = __builtin_fma(q, z, 1.0);
    const int k = (int)(int64_t)n & 3;
    const double a = k & 1 ? cr : sr, b = k & 1 ? sr : cr;
    s = k & 2 ? -a : a;
    c = (k + 1) & 2 ? -b : b;
}

template <int DT>
__device__ __forceinline__ const char* element(const CacheView& v, int64_t token, int head, int dim)
{
    return v.data + (token * v.token_stride + head * v.head_stride + dim) * Elem<DT>::SIZE;
}

/* kChunk elements, 16-byte aligned. */
template <int DT>
__device__ __forceinline__ void load_chunk(const char* p, float (&x)[kChunk])
{
    if constexpr (DT == G4S_DTYPE_F32) {
        const float4 a = reinterpret_cast<const float4*>(p)[0];
        const float4 b = reinterpret_cast<const float4*>(p)[1];
        const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = v[i];
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
}

template <int DT>
__device__ __forceinline__ float load_one(const char* p)
{
    if constexpr (DT == G4S_DTYPE_F32)
        return *reinterpret_cast<const float*>(p);
    else
        return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16);
}

/* A binary64 as the binary32 next to it whose last bit is odd, unless it is one: what is
 * then rounded to a type with two bits less or fewer is rounded as if at once (a second
 * rounding to nearest would take what the first moved onto a tie for one). */
__device__ __forceinline__ float to_odd(double x)
{
    const float f = (float)x;
    const uint32_t u = __float_as_uint(f);
    const double d = (double)f;
    if ((u & 1u) || d == x || x != x) return f;
    return __uint_as_float(__builtin_fabs(x) > __builtin_fabs(d) ? u + 1 : u - 1);
}

__device__ __forceinline__ uint16_t bf16_of(double x)
{
    const uint32_t u = __float_as_uint(to_odd(x));
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)(u >> 16 | 0x40u);
    return (uint16_t)((u + 0x7FFFu + (u >> 16 & 1u)) >> 16);
}

template <int DT>
__device__ __forceinline__ void store_chunk(char* p, const double (&y)[kChunk])
{
    if constexpr (DT == G4S_DTYPE_F32) {
        float4 a, b;
        a.x = (float)y[0], a.y = (float)y[1], a.z = (float)y[2], a.w = (float)y[3];
        b.x = (float)y[4], b.y = (float)y[5], b.z = (float)y[6], b.w = (float)y[7];
        reinterpret_cast<float4*>(p)[0] = a;
        reinterpret_cast<float4*>(p)[1] = b;
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = (uint32_t)bf16_of(y[2 * i]) | (uint32_t)bf16_of(y[2 * i + 1]) << 16;
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

/* x / scale as an e4m3 code: within the type's range first, as the conversion gives NaN
 * for what lies outside. */
__device__ __forceinline__ uint32_t codes4(const double* y, double inv)
{
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double v = y[i] * inv;
        f[i] = to_odd(v > 448.0 ? 448.0 : v < -448.0 ? -448.0 : v);
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], w, true);
}

struct Tile {
    int row, first, end; /* places first .. end - 1 of the row */
    int64_t token;       /* the view's token at `first` */
    int before;          /* earlier tokens in the first block */
};

/* Chunk `c` of a head of one token, rotated where ROTATE. */
template <int DT, bool ROTATE>
__device__ __forceinline__ void rotated(const AppendArgs& a, const CacheView& view, int64_t token,
                                        int head, int c, const double2* turn, double (&y)[kChunk])
{
    const int d0 = c * kChunk;
    float x[kChunk];
    load_chunk<DT>(element<DT>(view, token, head, d0), x);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) y[i] = (double)x[i];
    if (!ROTATE || d0 >= a.rotary_dims) return;
    if (a.rotary_pairs == G4S_ROTARY_NEIGHBOURS) {
#pragma unroll
        for (int i = 0; i < kChunk; i += 2) {
            if (d0 + i >= a.rotary_dims) break;
            const double2 t = turn[(d0 + i) >> 1];
            const double u = y[i], w = y[i + 1];
            y[i] = __builtin_fma(u, t.x, -(w * t.y));
            y[i + 1] = __builtin_fma(w, t.x, u * t.y);
        }
        return;
    }
    const int half = a.rotary_dims >> 1;
    float o[kChunk];
    if ((half & (kChunk - 1)) == 0) {
        load_chunk<DT>(element<DT>(view, token, head, d0 < half ? d0 + half : d0 - half), o);
    } else {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            const int d = d0 + i;
            o[i] = d < a.rotary_dims
                       ? load_one<DT>(element<DT>(view, token, head, d < half ? d + half : d - half))
                       : 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
        const int d = d0 + i;
        if (d >= a.rotary_dims) break;
        const bool low = d < half;
        const double2 t = turn[low ? d : d - half];
        /* (the order of the two products is the same for both dims of a pair) */
        y[i] = low ? __builtin_fma(y[i], t.x, -((double)o[i] * t.y))
                   : __builtin_fma(y[i], t.x, (double)o[i] * t.y);
    }
}

/* Offset of a place in a plane, or -1 where its page is outside the pool. */
__device__ __forceinline__ int64_t place_offset(const AppendArgs& a, int row, int place, int head)
{
    const int slot = divide(place, a.pool.page_tokens);
    const int page = a.table[(int64_t)row * a.pool.max_slots + slot];
    if (page < 0 || page >= a.pool.n_pages) return -1;
    return cache_offset(a.pool, page, place - slot * a.pool.page_tokens.d, head);
}

/* The row and places of slot x of the grid; false where it has none. */
__device__ __forceinline__ bool find_tile(const AppendArgs& a, int64_t x, int tile, Tile& t)
{
    int row = (int)x;
    if (a.starts) {
        row = find_share(a.starts, a.rows, x, 1, tile, 2);
    }
    const RowTokens r = row_tokens(a.starts, a.lengths, row, a.tokens, cache_room(a.pool));
    int64_t nth = a.starts ? x - share_begin(a.starts, row, 1, tile, 2) : 0;
    if (r.count == 0 || r.length == 0 || nth < 0) return false;
    const int from = r.length > r.count ? r.length - r.count : 0; /* the first place */
    const int64_t begin = (from / tile + nth) * tile;
    if (begin >= r.length) return false;
    t.row = row;
    t.first = (int)(begin > from ? begin : from);
    t.end = (int)(begin + tile < r.length ? begin + tile : r.length);
    t.token = (int64_t)r.start + (t.first - (r.length - r.count));
    t.before = begin < t.first ? (t.first - (int)begin) % a.pool.scale_tokens.d : 0;
    return true;
}

/* The largest finite magnitude of a chunk, as the bits of a binary64 (which are in order). */
__device__ __forceinline__ uint64_t top_of(const double (&y)[kChunk])
{
    double m = 0.0;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
        const double v = __builtin_fabs(y[i]);
        m = v > m && v < __builtin_inf() ? v : m;
    }
    return (uint64_t)__double_as_longlong(m);
}

template <int DT>
__global__ __launch_bounds__(kB) void append_kernel(AppendArgs a, int tile)
{
    extern __shared__ char lds[];
    Tile t;
    if (!find_tile(a, blockIdx.x, tile, t)) return;
    const int tid = threadIdx.x;
    const int half = a.rotary_dims >> 1;
    const int chunks = a.pool.head_dim / kChunk;
    const int B = a.pool.scale_tokens.d;
    const int first_block = t.first / B;
    const int blocks = (t.end - 1) / B - first_block + 1;
    /* the heads of this slice: of queries, and of keys followed by values */
    const int slice = blockIdx.y, slices = gridDim.y;
    const int nq = a.q.data ? (a.heads - slice + slices - 1) / slices : 0;
    const int items = a.k.data ? 2 * a.kv_heads : 0;
    const int nkv = items > slice ? (items - slice + slices - 1) / slices : 0;
    double2* turn = reinterpret_cast<double2*>(lds);                    /* [kStep][half] */
    uint64_t* top = reinterpret_cast<uint64_t*>(turn + kStep * half);   /* [blocks][nkv] */
    for (int i = tid; i < blocks * nkv; i += kB) top[i] = 0;

    for (int pass = 0; pass < (nkv > 0 ? 2 : 1); ++pass) {
        for (int s0 = t.first; s0 < t.end; s0 += kStep) {
            const int n = t.end - s0 < kStep ? t.end - s0 : kStep;
            __syncthreads();
            for (int i = tid; i < n * half; i += kB) {
                const int j = i / half, f = i - j * half;
                const int64_t token = t.token + (s0 - t.first) + j;
                const int p = a.positions ? a.positions[token] : s0 + j;
                double s, c;
                sincos64((double)p * (double)a.freqs[f], s, c);
                turn[i] = make_double2(c, s);
            }
            __syncthreads();
            if (pass == 0 && nq > 0) {
                /* the threads of a head's chunks lie in one wave: it has read the head
                 * before it writes it, so that q_out may be q */
                const int per_wave = 64 / chunks;
                const int lane = tid & 63, c = lane % chunks, g = lane / chunks;
                const int heads = nq * n;
                for (int i0 = (tid >> 6) * per_wave; i0 < heads; i0 += kB / 64 * per_wave) {
                    const int i = i0 + g;
                    if (g >= per_wave || i >= heads) continue;
                    const int j = i / nq, head = slice + (i - j * nq) * slices;
                    const int64_t token = t.token + (s0 - t.first) + j;
                    double y[kChunk];
                    rotated<DT, true>(a, a.q, token, head, c, turn + j * half, y);
                    store_chunk<DT>(const_cast<char*>(element<DT>(a.q_out, token, head, c * kChunk)),
                                    y);
                }
            }
            for (int i = tid; i < n * nkv * chunks; i += kB) {
                const int c = i % chunks, u = i / chunks;
                const int j = u / nkv, nth = u - j * nkv;
                const int item = slice + nth * slices;
                const bool value = item >= a.kv_heads;
                const int head = value ? item - a.kv_heads : item;
                const int place = s0 + j;
                const int64_t token = t.token + (place - t.first);
                double y[kChunk];
                if (value)
                    rotated<DT, false>(a, a.v, token, head, c, nullptr, y);
                else
                    rotated<DT, true>(a, a.k, token, head, c, turn + j * half, y);
                uint64_t* at = &top[(place / B - first_block) * nkv + nth];
                if (pass == 0) {
                    atomicMax((unsigned long long*)at, (unsigned long long)top_of(y));
                    continue;
                }
                const int64_t off = place_offset(a, t.row, place, head);
                if (off < 0) continue;
                const double inv = 1.0 / __longlong_as_double((long long)*at);
                char* p = (value ? a.v_plane : a.k_plane) + off;
                uint32_t* w = reinterpret_cast<uint32_t*>(p + c * kChunk);
                w[0] = codes4(y, inv);
                w[1] = codes4(y + 4, inv);
            }
        }
        if (pass == 1 || nkv == 0) break;
        __syncthreads();
        /* scales, in the place of the magnitudes; what a block holds already brought to its new one */
        for (int i = tid; i < blocks * nkv; i += kB) {
            const int b = i / nkv, item = slice + (i - b * nkv) * slices;
            const bool value = item >= a.kv_heads;
            const int head = value ? item - a.kv_heads : item;
            const int place = (first_block + b) * B;
            const int64_t off = place_offset(a, t.row, place, head);
            float scale = __builtin_ldexpf(1.0f, scale_exponent(__longlong_as_double((long long)top[i])));
            if (off >= 0) {
                char* p = (value ? a.v_plane : a.k_plane) + off;
                float* at = reinterpret_cast<float*>(p + a.pool.head_dim);
                if (b == 0 && t.before > 0) {
                    const float old = *at;
                    if (old >= scale && old < __builtin_inff()) {
                        scale = old;
                    } else if (old > 0.0f) {
                        const float ratio = old / scale;
                        for (int j = 0; j < t.before; ++j) {
                            uint32_t* w = reinterpret_cast<uint32_t*>(p + (int64_t)j * a.pool.token_bytes);
                            for (int c = 0; c < a.pool.head_dim / 4; ++c) {
                                const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[c], false);
                                const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[c], true);
                                int v = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * ratio, lo[1] * ratio, 0, false);
                                w[c] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * ratio, hi[1] * ratio, v, true);
                            }
                        }
                    }
                }
                *at = scale;
            }
            top[i] = (uint64_t)__double_as_longlong((double)scale);
        }
    }
}

}  // namespace

hipError_t append_launch(const AppendArgs& a, int32_t dtype, hipStream_t stream)
{
    const int B = a.pool.scale_tokens.d;
    const int tile = B > kTile ? B : kTile / B * B;
    const int64_t tiles = a.starts ? (int64_t)a.tokens / tile + 2 * (int64_t)a.rows : a.rows;
    const int slices = 1;
    const int items = a.k.data ? 2 * a.kv_heads : 0;
    const size_t lds = (size_t)kStep * (a.rotary_dims / 2) * sizeof(double2) +
                       (size_t)((tile + B - 1) / B + 1) * ((items + slices - 1) / slices) *
                           sizeof(uint64_t);
    const dim3 grid((unsigned)tiles, (unsigned)slices);
    return dtype == G4S_DTYPE_F32 ? launch(append_kernel<G4S_DTYPE_F32>, grid, kB, lds, stream, a, tile)
                                  : launch(append_kernel<G4S_DTYPE_BF16>, grid, kB, lds, stream, a, tile);
}

}  // namespace g4s
