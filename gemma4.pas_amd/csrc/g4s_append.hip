/*
 * g4s_append.hip -- new keys and values into the pages of a cache in 8 bits,
 * rotated by their positions on the way, and the queries rotated beside
 * them, on gfx950.
 *
 * A code is x / scale with a scale that depends on all of a block's new values, so the vectors are looked
 * at twice: for the largest magnitude of each block and head, and to store them.  A
 * workgroup takes up to `tile` places of one row, whole blocks of tokens that share a scale, so that
 * a scale and the codes under it have one writer, and some of the heads: of queries, or of keys
 * and values.  A thread keeps its vectors in registers between the looks where a tile has no more than
 * four tokens for it (read twice, from the caches, they took 174 instead of 115 us for seven prompts of
 * 2,000 tokens, 32 and 8 heads of 128 dims).  Keys are rotated in binary64 and rounded once: next to a
 * border between two codes a rounding in between would choose the other one.  Cosines and sines
 * are computed once per token and pair, in LDS for all heads of the workgroup.
 *
 * One token a row: 4.0 us for a row and 4.4 for 192, the latency of a launch and of lengths, page, scale
 * and vectors one after the other.  The seven prompts: 115 us for 361 MB (3.1 TB/s, a copy 4.9): queries alone
 * 66, keys and values alone 57, of which the angles are 16.  Vector instructions (binary64 most of
 * them) are issued in 54% of the cycles, and two to three workgroups a CU do not have the memory's latency behind
 * them.
 */
#include "g4s_cache.h"
#include "g4s_device.h"
#include "g4s_launch.h"

namespace g4s {

namespace {

constexpr int kB = 256;
constexpr int kTile = 16;  /* places of a workgroup, or one block where that is longer */
constexpr int kChunk = 8;  /* dims of a thread */
constexpr int kPairs = 2048; /* angles in LDS at once */
constexpr int kQueryHeads = 8; /* of a workgroup at least, where there are several tokens */
constexpr int kFill = 768;     /* workgroups, three a CU */

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

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

/* kChunk elements as they are stored, 16-byte aligned. */
template <int DT>
struct Words {
    uint4 x[DT == G4S_DTYPE_F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ Words<DT> load_words(const char* p)
{
    Words<DT> w;
    w.x[0] = reinterpret_cast<const uint4*>(p)[0];
    if constexpr (DT == G4S_DTYPE_F32) w.x[1] = reinterpret_cast<const uint4*>(p)[1];
    return w;
}
template <int DT>
__device__ __forceinline__ void widen(const Words<DT>& v, float (&x)[kChunk])
{
    if constexpr (DT == G4S_DTYPE_F32) {
        const uint32_t w[8] = {v.x[0].x, v.x[0].y, v.x[0].z, v.x[0].w, v.x[1].x, v.x[1].y, v.x[1].z, v.x[1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
    } else {
        const uint32_t w[4] = {v.x[0].x, v.x[0].y, v.x[0].z, v.x[0].w};
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

/* bf16 by way of binary32: off by 2^-16 of a bf16 step more than in one rounding. */
template <int DT>
__device__ __forceinline__ void store_chunk(char* p, const double (&y)[kChunk])
{
    float x[kChunk];
#pragma unroll
    for (int i = 0; i < kChunk; ++i) x[i] = (float)y[i];
    if constexpr (DT == G4S_DTYPE_F32) {
        reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        bf16x8 w;
#pragma unroll
        for (int i = 0; i < kChunk; ++i) w[i] = (__bf16)x[i];
        *reinterpret_cast<bf16x8*>(p) = w;
    }
}

/* Codes of four quotients (binary32, not between two codes where the exact ones are not): within
 * the type's range first, as the conversion gives NaN for what lies outside. */
__device__ __forceinline__ uint32_t codes4(const float* x)
{
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = x[i] > 448.0f ? 448.0f : x[i] < -448.0f ? -448.0f : x[i];
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], w, true);
}

struct Tile {
    int row, first, end; /* places first .. end - 1 of the row */
    int64_t token;       /* the view's token at `first` */
    int before;          /* earlier tokens in the first block */
};

/* How dims are paired: halves or neighbours where no chunk of dims lies across a border, or
 * whatever else, dim by dim. */
enum Mode { kHalves, kNeighbours, kAny };

/* Chunk `c` of a head of one token: what is in it, and what is paired with it. */
template <int DT, int MODE>
struct Chunk {
    Words<DT> x, o;
};
template <int DT>
struct Chunk<DT, kNeighbours> {
    Words<DT> x;
};
template <int DT>
struct Chunk<DT, kAny> {
    Words<DT> x;
    float o[kChunk];
};
template <int DT, int MODE>
__device__ __forceinline__ void read_chunk(const AppendArgs& a, const CacheView& view, int64_t token,
                                           int head, int c, bool rotate, Chunk<DT, MODE>& w)
{
    const int d0 = c * kChunk, half = a.rotary_dims >> 1;
    w.x = load_words<DT>(element<DT>(view, token, head, d0));
    if (!rotate || d0 >= a.rotary_dims) return;
    if constexpr (MODE == kHalves)
        w.o = load_words<DT>(element<DT>(view, token, head, d0 < half ? d0 + half : d0 - half));
    if constexpr (MODE == kAny) {
        for (int i = 0; i < kChunk; ++i) {
            const int d = d0 + i;
            const int pair = a.rotary_pairs == G4S_ROTARY_NEIGHBOURS ? d ^ 1 : d < half ? d + half : d - half;
            const float v = d < a.rotary_dims ? load_one<DT>(element<DT>(view, token, head, pair)) : 0.0f;
#pragma unroll
            for (int k = 0; k < kChunk; ++k) w.o[k] = k == i ? v : w.o[k];
        }
    }
}
/* Cosines and sines for the dims of a chunk (1 and 0 behind the last dim that is rotated). */
struct Turn {
    double2 t[kChunk];
};
template <int MODE>
__device__ __forceinline__ void read_turn(const AppendArgs& a, int c, const double2* turn, Turn& r)
{
    const int d0 = c * kChunk, half = a.rotary_dims >> 1;
    if (d0 >= a.rotary_dims) return;
    if (MODE == kHalves) {
        const double2* at = turn + (d0 < half ? d0 : d0 - half);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) r.t[i] = at[i];
    } else if (MODE == kNeighbours) {
#pragma unroll
        for (int i = 0; i < kChunk; i += 2) r.t[i] = turn[(d0 + i) >> 1];
    } else {
        for (int i = 0; i < kChunk; ++i) {
            const int d = d0 + i;
            const int f = a.rotary_pairs == G4S_ROTARY_NEIGHBOURS ? d >> 1 : d < half ? d : d - half;
            const double2 t = d < a.rotary_dims ? turn[f] : make_double2(1.0, 0.0);
#pragma unroll
            for (int k = 0; k < kChunk; ++k) {
                r.t[k].x = k == i ? t.x : r.t[k].x;
                r.t[k].y = k == i ? t.y : r.t[k].y;
            }
        }
    }
}
template <int DT, int MODE>
__device__ __forceinline__ void rotate(const AppendArgs& a, const Chunk<DT, MODE>& w, int c,
                                       const Turn& r, double (&y)[kChunk])
{
    const int d0 = c * kChunk, half = a.rotary_dims >> 1;
    float x[kChunk];
    widen(w.x, x);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) y[i] = (double)x[i];
    if (d0 >= a.rotary_dims) return;
    if constexpr (MODE == kNeighbours) {
#pragma unroll
        for (int i = 0; i < kChunk; i += 2) {
            const double u = y[i], v = y[i + 1];
            y[i] = __builtin_fma(u, r.t[i].x, -(v * r.t[i].y));
            y[i + 1] = __builtin_fma(v, r.t[i].x, u * r.t[i].y);
        }
    } else {
        float o[kChunk];
        if constexpr (MODE == kHalves) widen(w.o, o);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            if constexpr (MODE == kAny) o[i] = w.o[i];
            const bool low = MODE == kHalves ? d0 < half
                             : a.rotary_pairs == G4S_ROTARY_NEIGHBOURS ? (i & 1) == 0
                                                                      : d0 + i < half;
            const double v = (double)o[i] * r.t[i].y;
            y[i] = __builtin_fma(y[i], r.t[i].x, low ? -v : v);
        }
    }
}

/* Where a row's places are.  The page of the first one is read ahead of its use. */
struct Places {
    const int32_t* pages; /* of the row */
    int slot, page;
};
__device__ __forceinline__ Places places_of(const AppendArgs& a, int row, int first)
{
    Places p;
    p.pages = a.table + (int64_t)row * a.pool.max_slots;
    p.slot = divide(first, a.pool.page_tokens);
    p.page = p.pages[p.slot];
    return p;
}
/* Offset of a place in a plane, or -1 where its page is outside the pool. */
__device__ __forceinline__ int64_t place_offset(const AppendArgs& a, const Places& p, int place,
                                                int head)
{
    const int slot = divide(place, a.pool.page_tokens);
    const int page = slot == p.slot ? p.page : p.pages[slot];
    if (page < 0 || page >= a.pool.n_pages) return -1;
    return cache_offset(a.pool, page, place - slot * a.pool.page_tokens.d, head);
}

/* A block's scale for new values of magnitude `top`, and in `grown` what codes that it
 * holds under `old` are multiplied by (1: nothing). */
__device__ __forceinline__ float block_scale(uint32_t top, bool earlier, float old, float& grown)
{
    const float scale = __builtin_ldexpf(1.0f, scale_exponent((double)__uint_as_float(top)));
    grown = 1.0f;
    if (!earlier) return scale;
    if (old >= scale && old < __builtin_inff()) return old;
    if (old > 0.0f) grown = old / scale;
    return scale;
}
/* The row and places of slot x of the grid; false where it has none. */
__device__ __forceinline__ bool find_tile(const AppendArgs& a, int64_t x, int tile, Tile& t)
{
    t.row = find_share(a.starts, a.rows, x, 1, tile, 2);
    const RowTokens r = row_tokens(a.starts, a.lengths, t.row, a.tokens, cache_room(a.pool));
    const int64_t nth = x - share_begin(a.starts, t.row, 1, tile, 2);
    if (r.count == 0 || r.length == 0 || nth < 0) return false;
    const int from = r.length > r.count ? r.length - r.count : 0; /* the first place */
    const int64_t begin = (from / tile + nth) * tile;
    if (begin >= r.length) return false;
    t.first = (int)(begin > from ? begin : from);
    t.end = (int)(begin + tile < r.length ? begin + tile : r.length);
    t.token = (int64_t)r.start + (t.first - (r.length - r.count));
    t.before = t.first - divide(t.first, a.pool.scale_tokens) * a.pool.scale_tokens.d;
    return true;
}

/* The largest finite magnitude of a chunk, as the bits of a binary32, which are in order.
 * (to_odd keeps a value on its side of 448 * 2^e, whose last bit is even.) */
__device__ __forceinline__ uint32_t top_of(const float (&x)[kChunk])
{
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
        const float v = __builtin_fabsf(x[i]);
        m = v > m && v < __builtin_inff() ? v : m;
    }
    return __float_as_uint(m);
}

/* Four codes under a scale that grew. */
__device__ __forceinline__ uint32_t regrown(uint32_t w, float ratio)
{
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
    const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    const float x[4] = {lo[0] * ratio, lo[1] * ratio, hi[0] * ratio, hi[1] * ratio};
    return codes4(x);
}

/* The largest of a vector's lanes (a power of two of them). */
__device__ __forceinline__ uint32_t lanes_max(uint32_t m, int chunks)
{
    for (int d = 1; d < chunks; d <<= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)m, d);
        m = o > m ? o : m;
    }
    return m;
}

/* What of a chunk is stored: a value as it is, a rotated key as the odd binary32 next to it,
 * whose product with a scale's inverse (a power of two) is exact and rounds to the code that the key
 * itself has. */
template <int DT, int MODE>
__device__ __forceinline__ void stored(const AppendArgs& a, const Chunk<DT, MODE>& w, int c, bool value,
                                       const Turn& r, float (&x)[kChunk])
{
    widen(w.x, x);
    if (value || c * kChunk >= a.rotary_dims) return;
    double y[kChunk];
    rotate(a, w, c, r, y);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) x[i] = to_odd(y[i]);
}
__device__ __forceinline__ void store_codes(char* at, const float (&x)[kChunk], float scale)
{
    const float inv = 1.0f / scale;
    float q[kChunk];
#pragma unroll
    for (int i = 0; i < kChunk; ++i) q[i] = x[i] * inv;
    uint32_t* to = reinterpret_cast<uint32_t*>(at);
    to[0] = codes4(q);
    to[1] = codes4(q + 4);
}

/* ------------------------------------------------------- a token for each row */

/* A workgroup has the row's vectors (queries, keys, values) from first_vector on, one for each
 * kChunk-dim lane group; a block's new values are those of one vector. */
template <int DT, int MODE>
__global__ __launch_bounds__(kB) void append_step_kernel(AppendArgs a, int queries, int vectors)
{
    __shared__ double2 turn[G4S_CACHE_MAX_HEAD_DIM / 2];
    __shared__ uint32_t s_top[kB];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = blockIdx.x, half = a.rotary_dims >> 1;
    const int chunks = a.pool.head_dim / kChunk, each = 64 / chunks;
    const int g = lane / chunks, c = lane - g * chunks;
    const int nth = wave * each + g, vector = (int)blockIdx.y * (kB / 64 * each) + nth;
    const bool in = g < each && vector < vectors;
    /* queries, keys, values */
    const bool query = vector < queries;
    const int item = vector - queries;
    const bool value = !query && item >= a.kv_heads;
    const int head = query ? vector : value ? item - a.kv_heads : item;
    Chunk<DT, MODE> w;
    if (in) read_chunk(a, query ? a.q : value ? a.v : a.k, row, head, c, !value, w);
    const float freq = tid < half ? a.freqs[tid] : 0.0f;
    const int position = a.positions ? a.positions[row] : 0;
    const int length = a.lengths[row];
    s_top[tid] = 0;
    if (length <= 0 || length > cache_room(a.pool)) return;
    const int place = length - 1;
    const int before = place - divide(place, a.pool.scale_tokens) * a.pool.scale_tokens.d;
    int64_t off = -1;
    float old = 0.0f;
    if (in && !query) {
        const Places p = places_of(a, row, place);
        off = place_offset(a, p, place - before, head);
    }
    char* const block = (value ? a.v_plane : a.k_plane) + off; /* its first token */
    float* const scale_at = reinterpret_cast<float*>(block + a.pool.head_dim);
    if (off >= 0 && before > 0) old = *scale_at;
    for (int i = tid; i < half; i += kB) {
        double s, t;
        sincos64((double)(a.positions ? position : place) * (double)freq, s, t);
        turn[i] = make_double2(t, s);
    }
    __syncthreads();
    float x[kChunk];
    uint32_t top = 0;
    if (in) {
        Turn t;
        if (!value) read_turn<MODE>(a, c, turn, t);
        if (query) {
            double y[kChunk];
            rotate(a, w, c, t, y);
            store_chunk<DT>(const_cast<char*>(element<DT>(a.q_out, row, head, c * kChunk)), y);
        } else {
            stored(a, w, c, value, t, x);
            top = top_of(x);
        }
    }
    if ((chunks & (chunks - 1)) == 0) {
        top = lanes_max(top, chunks);
    } else {
        if (in) atomicMax(&s_top[nth], top);
        __syncthreads();
        if (in) top = s_top[nth];
    }
    if (off < 0) return;
    float grown;
    const float scale = block_scale(top, before > 0, old, grown);
    store_codes(block + (int64_t)before * a.pool.token_bytes + c * kChunk, x, scale);
    if (c == 0) *scale_at = scale;
    if (grown == 1.0f) return;
    for (int j = 0; j < before; ++j) {
        uint32_t* at = reinterpret_cast<uint32_t*>(block + (int64_t)j * a.pool.token_bytes + c * kChunk);
        const uint32_t w0 = at[0], w1 = at[1];
        at[0] = regrown(w0, grown);
        at[1] = regrown(w1, grown);
    }
}

/* ------------------------------------------------------------- ragged tokens */

/* How a workgroup's threads lie over tokens and chunks: `tokens` vectors at once. */
struct Lanes {
    int chunks, tokens;
    int c, token; /* this thread's; token = tokens: none */
};
__device__ __forceinline__ Lanes lanes_of(int chunks)
{
    Lanes l;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, each = 64 / chunks;
    const int g = lane / chunks;
    l.chunks = chunks;
    l.tokens = kB / 64 * each;
    l.c = lane - g * chunks;
    l.token = g < each ? wave * each + g : l.tokens;
    return l;
}

/* Cosines and sines of n tokens from place s0 on. */
__device__ __forceinline__ void fill_turns(const AppendArgs& a, const Tile& t, int s0, int n,
                                           double2* turn)
{
    const int half = a.rotary_dims >> 1;
    for (int i = threadIdx.x; i < n * half; i += kB) {
        const int j = i / half, f = i - j * half;
        const float freq = a.freqs[f];
        const int p = a.positions ? a.positions[t.token + (s0 - t.first) + j] : s0 + j;
        double s, c;
        sincos64((double)p * (double)freq, s, c);
        turn[i] = make_double2(c, s);
    }
}

/* Queries: each vector in one wave, which has read it before it writes it, so that q_out may
 * be q. */
template <int DT, int MODE>
__device__ __forceinline__ void append_queries(const AppendArgs& a, const Tile& t, int head0,
                                               int heads, int step, double2* turn)
{
    const int half = a.rotary_dims >> 1;
    const Lanes l = lanes_of(a.pool.head_dim / kChunk);
    const int end = head0 + heads < a.heads ? head0 + heads : a.heads;
    for (int s0 = t.first; s0 < t.end; s0 += step) {
        const int n = t.end - s0 < step ? t.end - s0 : step;
        const int64_t token0 = t.token + (s0 - t.first);
        __syncthreads();
        fill_turns(a, t, s0, n, turn);
        __syncthreads();
        if (l.token == l.tokens) continue;
        for (int j = l.token; j < n; j += l.tokens) {
            Turn r;
            read_turn<MODE>(a, l.c, turn + j * half, r);
            constexpr int HELD = DT == G4S_DTYPE_F32 ? 2 : 4;
            for (int h = head0; h < end; h += HELD) {
                Chunk<DT, MODE> w[HELD];
#pragma unroll
                for (int k = 0; k < HELD; ++k)
                    if (h + k < end) read_chunk(a, a.q, token0 + j, h + k, l.c, true, w[k]);
#pragma unroll
                for (int k = 0; k < HELD; ++k) {
                    if (h + k >= end) break;
                    double y[kChunk];
                    rotate(a, w[k], l.c, r, y);
                    store_chunk<DT>(const_cast<char*>(element<DT>(a.q_out, token0 + j, h + k, l.c * kChunk)), y);
                }
            }
        }
    }
}

/* What a workgroup does between the two looks at a group of heads' vectors: scales of its blocks in the
 * place of their magnitudes, and the codes of earlier tokens under scales that grew. */
__device__ __forceinline__ void settle_scales(const AppendArgs& a, const Tile& t, const Places& places,
                                              char* plane, int head0, int heads, uint32_t* top,
                                              float* ratio)
{
    const int B = a.pool.scale_tokens.d, tid = threadIdx.x;
    const int first_block = divide(t.first, a.pool.scale_tokens);
    const int blocks = divide(t.end - 1, a.pool.scale_tokens) - first_block + 1;
    __syncthreads();
    for (int i = tid; i < blocks * heads; i += kB) {
        const int b = i / heads, k = i - b * heads;
        const int64_t off = place_offset(a, places, (first_block + b) * B, head0 + k);
        const bool earlier = b == 0 && t.before > 0 && off >= 0;
        float* at = reinterpret_cast<float*>(plane + off + a.pool.head_dim);
        float grown;
        const float scale = block_scale(top[i], earlier, earlier ? *at : 0.0f, grown);
        if (off >= 0) *at = scale;
        top[i] = __float_as_uint(scale);
        if (b == 0) ratio[k] = grown;
    }
    __syncthreads();
    if (t.before == 0) return;
    const int words = a.pool.head_dim / 4;
    for (int i = tid; i < heads * t.before * words; i += kB) {
        const int v = i / words, k = v / t.before, j = v - k * t.before;
        if (ratio[k] == 1.0f) continue;
        const int64_t off = place_offset(a, places, first_block * B + j, head0 + k);
        if (off < 0) continue;
        uint32_t* at = reinterpret_cast<uint32_t*>(plane + off) + (i - v * words);
        *at = regrown(*at, ratio[k]);
    }
}

/* Keys, or values, of `heads` heads.  HELD: a thread keeps its vectors of a group of heads, HELD
 * tokens' of each, in registers from the first look to the second; 0: of tiles with more tokens,
 * whose vectors are read twice. */
constexpr int kHeld = 4;
/* Keeps what follows behind what came before: the angles of one vector, in binary64, are as many
 * registers as there is room for. */
__device__ __forceinline__ void one_by_one()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
/* Heads at once: as many vectors as a thread holds (one head each where it holds two tokens: 133 us for the
 * prompts instead of 123). */
constexpr int group_heads(int held) { return held > 0 ? kHeld / held : kHeld; }
template <int DT, int MODE, bool VALUE, int HELD>
__device__ __forceinline__ void append_heads(const AppendArgs& a, const Tile& t, int head0, int heads,
                                             int step, double2* turn, uint32_t* top, float* ratio)
{
    constexpr int GROUP = group_heads(HELD);
    const int half = a.rotary_dims >> 1, tid = threadIdx.x;
    const CacheView& view = VALUE ? a.v : a.k;
    char* const plane = VALUE ? a.v_plane : a.k_plane;
    const Places places = places_of(a, t.row, t.first);
    const int first_block = divide(t.first, a.pool.scale_tokens);
    const int blocks = divide(t.end - 1, a.pool.scale_tokens) - first_block + 1;
    const int end = head0 + heads < a.kv_heads ? head0 + heads : a.kv_heads;
    const Lanes l = lanes_of(a.pool.head_dim / kChunk);
    const bool pow2 = (l.chunks & (l.chunks - 1)) == 0;
    auto raise = [&](int at, bool in, uint32_t m) {
        if (pow2) m = lanes_max(m, l.chunks);
        if (in && (!pow2 || l.c == 0)) atomicMax(&top[at], m);
    };
    for (int h0 = head0; h0 < end; h0 += GROUP) {
        const int n_heads = end - h0 < GROUP ? end - h0 : GROUP;
        if constexpr (HELD > 0) {
            /* (lanes without a token take the first one, and keep nothing) */
            Chunk<DT, MODE> w[HELD][GROUP];
            float x[HELD][GROUP][kChunk];
            bool in[HELD];
            int at[HELD], turn_at[HELD];
            int64_t off[HELD];
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                int j = i * l.tokens + l.token;
                in[i] = l.token < l.tokens && t.first + j < t.end;
                j = in[i] ? j : 0;
                turn_at[i] = j * half;
                at[i] = (divide(t.first + j, a.pool.scale_tokens) - first_block) * n_heads;
#pragma unroll
                for (int k = 0; k < GROUP; ++k)
                    read_chunk(a, view, t.token + j, h0 + (k < n_heads ? k : 0), l.c, !VALUE, w[i][k]);
                off[i] = place_offset(a, places, t.first + j, h0);
            }
            __syncthreads(); /* (the group before has read its scales) */
            for (int i = tid; i < blocks * n_heads; i += kB) top[i] = 0;
            if (!VALUE && h0 == head0) fill_turns(a, t, t.first, t.end - t.first, turn);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                Turn r;
                if (!VALUE) read_turn<MODE>(a, l.c, turn + turn_at[i], r);
#pragma unroll
                for (int k = 0; k < GROUP; ++k) {
                    stored(a, w[i][k], l.c, VALUE, r, x[i][k]);
                    if (k < n_heads) raise(at[i] + k, in[i], in[i] ? top_of(x[i][k]) : 0);
                }
                one_by_one();
            }
            settle_scales(a, t, places, plane, h0, n_heads, top, ratio);
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                if (!in[i] || off[i] < 0) continue;
#pragma unroll
                for (int k = 0; k < GROUP; ++k)
                    if (k < n_heads)
                        store_codes(plane + off[i] + (int64_t)k * a.pool.part_bytes + l.c * kChunk, x[i][k],
                                    __uint_as_float(top[at[i] + k]));
            }
        } else {
            __syncthreads();
            for (int i = tid; i < blocks * n_heads; i += kB) top[i] = 0;
            for (int pass = 0; pass < 2; ++pass) {
                for (int s0 = t.first; s0 < t.end; s0 += step) {
                    const int n = t.end - s0 < step ? t.end - s0 : step;
                    __syncthreads();
                    if (!VALUE) fill_turns(a, t, s0, n, turn);
                    __syncthreads();
                    for (int j0 = 0; j0 < n; j0 += l.tokens) {
                        const int j = j0 + l.token, place = s0 + j;
                        const bool in = l.token < l.tokens && j < n;
                        Turn r;
                        if (!VALUE && in) read_turn<MODE>(a, l.c, turn + j * half, r);
                        const int64_t off = pass == 1 && in ? place_offset(a, places, place, h0) : -1;
                        const int at = in ? (divide(place, a.pool.scale_tokens) - first_block) * n_heads : 0;
                        for (int k = 0; k < n_heads; ++k) {
                            Chunk<DT, MODE> w;
                            float x[kChunk];
                            if (in) {
                                read_chunk(a, view, t.token + (place - t.first), h0 + k, l.c, !VALUE, w);
                                stored(a, w, l.c, VALUE, r, x);
                            }
                            if (pass == 0)
                                raise(at + k, in, in ? top_of(x) : 0);
                            else if (off >= 0)
                                store_codes(plane + off + (int64_t)k * a.pool.part_bytes + l.c * kChunk, x,
                                            __uint_as_float(top[at + k]));
                        }
                    }
                }
                if (pass == 0) settle_scales(a, t, places, plane, h0, n_heads, top, ratio);
            }
        }
    }
}

/* Workgroups of queries, of keys and of values, one behind the other in y. */
template <int DT, int MODE, int HELD>
__global__ __launch_bounds__(kB, 3) /* (123 us for the prompts; 2: 144, 4: 143, which spills) */
void append_tiles_kernel(AppendArgs a, int tile, int step,
                                                             int q_heads, int q_slices, int kv_heads,
                                                             int kv_slices)
{
    extern __shared__ char lds[];
    Tile t;
    if (!find_tile(a, blockIdx.x, tile, t)) return;
    double2* turn = reinterpret_cast<double2*>(lds); /* [step][rotary_dims / 2] */
    const int blocks = (tile + a.pool.scale_tokens.d - 1) / a.pool.scale_tokens.d;
    uint32_t* top = reinterpret_cast<uint32_t*>(turn + step * (a.rotary_dims >> 1)); /* [blocks][kHeld] */
    float* ratio = reinterpret_cast<float*>(top + blocks * kHeld);                   /* [kHeld] */
    const int y = blockIdx.y;
    if (y < q_slices)
        append_queries<DT, MODE>(a, t, y * q_heads, q_heads, step, turn);
    else if (y < q_slices + kv_slices)
        append_heads<DT, MODE, false, HELD>(a, t, (y - q_slices) * kv_heads, kv_heads, step, turn, top, ratio);
    else
        append_heads<DT, MODE, true, HELD>(a, t, (y - q_slices - kv_slices) * kv_heads, kv_heads, step, turn,
                                           top, ratio);
}

/* Heads of a workgroup: the more, the fewer angles are computed again; but as few as `unit` where
 * there would not be kFill workgroups otherwise (the prompts' queries: 67 us with 768, 66 with 400, 83
 * with 1,500; keys without angles 80, 69 and 98). */
int32_t heads_each(int32_t heads, int32_t unit, int64_t tiles)
{
    int32_t each = unit;
    while (each < heads && tiles * ((heads + 2 * each - 1) / (2 * each)) >= kFill) each *= 2;
    return each < heads ? each : heads;
}

template <int DT, int MODE>
hipError_t launch_mode(const AppendArgs& a, hipStream_t stream)
{
    const int at_once = kB / 64 * (64 / (a.pool.head_dim / kChunk)); /* vectors of a workgroup */
    if (!a.starts) {
        const int queries = a.q.data ? a.heads : 0;
        const int vectors = queries + (a.k.data ? 2 * a.kv_heads : 0);
        const dim3 grid((unsigned)a.rows, (unsigned)((vectors + at_once - 1) / at_once));
        return launch(append_step_kernel<DT, MODE>, grid, kB, 0, stream, a, queries, vectors);
    }
    const int B = a.pool.scale_tokens.d, half = a.rotary_dims / 2;
    const int tile = B > kTile ? B : kTile / B * B;
    int step = half > 0 ? kPairs / half : tile;
    step = step > tile ? tile : step;
    /* tokens of a thread that it can keep, if it has the angles of all of a tile's */
    const int tokens = (tile + at_once - 1) / at_once;
    const int held = step < tile || tokens > kHeld ? 0 : tokens == 3 ? 4 : tokens;
    const int64_t tiles = (int64_t)a.tokens / tile + 2 * (int64_t)a.rows;
    const int q_heads = heads_each(a.heads, kQueryHeads, tiles);
    const int kv_heads = heads_each(a.kv_heads, group_heads(held), tiles);
    const int q_slices = a.q.data ? (a.heads + q_heads - 1) / q_heads : 0;
    const int kv_slices = a.k.data ? (a.kv_heads + kv_heads - 1) / kv_heads : 0;
    const size_t lds = (size_t)step * half * sizeof(double2) +
                       ((size_t)(tile + B - 1) / B + 1) * kHeld * sizeof(uint32_t);
    const dim3 grid((unsigned)tiles, (unsigned)(q_slices + 2 * kv_slices));
    auto kernel = held == 1   ? append_tiles_kernel<DT, MODE, 1>
                  : held == 2 ? append_tiles_kernel<DT, MODE, 2>
                  : held == 4 ? append_tiles_kernel<DT, MODE, 4>
                              : append_tiles_kernel<DT, MODE, 0>;
    return launch(kernel, grid, kB, lds, stream, a, tile, step, q_heads, q_slices, kv_heads, kv_slices);
}

template <int DT>
hipError_t by_mode(const AppendArgs& a, hipStream_t stream)
{
    if (a.rotary_pairs == G4S_ROTARY_HALVES && a.rotary_dims / 2 % kChunk == 0)
        return launch_mode<DT, kHalves>(a, stream);
    if (a.rotary_pairs == G4S_ROTARY_NEIGHBOURS && a.rotary_dims % kChunk == 0)
        return launch_mode<DT, kNeighbours>(a, stream);
    return launch_mode<DT, kAny>(a, stream);
}

}  // namespace

hipError_t append_launch(const AppendArgs& a, int32_t dtype, hipStream_t stream)
{
    return dtype == G4S_DTYPE_F32 ? by_mode<G4S_DTYPE_F32>(a, stream)
                                  : by_mode<G4S_DTYPE_BF16>(a, stream);
}

}  // namespace g4s
