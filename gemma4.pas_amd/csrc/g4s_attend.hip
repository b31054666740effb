/*
 * g4s_attend.hip -- attention over the pages of an 8-bit cache, on gfx950.
 *
 * A workgroup per query and head: each wave takes every fourth token, with the running
 * maximum and sum of its softmax, and the waves join at the end.
 */
#include "g4s_cache.h"
#include "g4s_device.h"
#include "g4s_launch.h"

namespace g4s {

namespace {

constexpr int kB = 256;
constexpr int kDims = G4S_CACHE_MAX_HEAD_DIM / 64;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

template <int DT>
__device__ __forceinline__ float load_one(const char* p, int64_t i)
{
    if constexpr (DT == G4S_DTYPE_F32)
        return reinterpret_cast<const float*>(p)[i];
    else
        return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
}
template <int DT>
__device__ __forceinline__ void store_one(char* p, int64_t i, float x)
{
    if constexpr (DT == G4S_DTYPE_F32)
        reinterpret_cast<float*>(p)[i] = x;
    else
        reinterpret_cast<__bf16*>(p)[i] = (__bf16)x;
}

__device__ __forceinline__ float code(const char* p)
{
    return __builtin_amdgcn_cvt_f32_fp8(*reinterpret_cast<const uint8_t*>(p), 0);
}

template <int DT>
__global__ __launch_bounds__(kB) void attend_kernel(AttendArgs a)
{
    __shared__ float s_m[4], s_l[4], s_o[4][G4S_CACHE_MAX_HEAD_DIM];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int head = blockIdx.y, d = a.pool.head_dim;
    int row = blockIdx.x;
    if (a.starts) {
        int lo = 0, hi = a.rows - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (a.starts[mid] <= (int)blockIdx.x)
                lo = mid;
            else
                hi = mid - 1;
        }
        row = lo;
    }
    const RowTokens r = row_tokens(a.starts, a.lengths, row, a.tokens, cache_room(a.pool));
    const int64_t token = blockIdx.x, nth = token - r.start;
    if (nth < 0 || nth >= r.count) return;
    const int64_t place = (int64_t)r.length - r.count + nth;
    int64_t from = a.window > 0 ? place - a.window + 1 : 0;
    if (from < 0) from = 0;
    const int kv = divide(head, a.group);
    float q[kDims], o[kDims];
    bool finite = true;
#pragma unroll
    for (int i = 0; i < kDims; ++i) {
        const int x = i * 64 + lane;
        q[i] = x < d ? load_one<DT>(a.q.data, token * a.q.token_stride + head * a.q.head_stride + x)
                     : 0.0f;
        finite = finite && __builtin_fabsf(q[i]) < __builtin_inff();
        o[i] = 0.0f;
    }
    finite = __all(finite);
    float m = -__builtin_inff(), l = 0.0f;
    for (int64_t t = from + wave; t <= place; t += 4) {
        const int slot = divide((int)t, a.pool.page_tokens);
        const int in = (int)t - slot * a.pool.page_tokens.d;
        const int first = in - (in - divide(in, a.pool.scale_tokens) * a.pool.scale_tokens.d);
        int page = a.table[(int64_t)row * a.pool.max_slots + slot];
        const bool ok = page >= 0 && page < a.pool.n_pages;
        if (!ok) page = 0;
        const int64_t at = cache_offset(a.pool, page, in, kv);
        const int64_t sc = cache_offset(a.pool, page, first, kv) + d;
        const float ks = *reinterpret_cast<const float*>(a.k_plane + sc);
        const float vs = *reinterpret_cast<const float*>(a.v_plane + sc);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kDims; ++i) {
            const int x = i * 64 + lane;
            if (x < d) s += q[i] * (code(a.k_plane + at + x) * ks);
        }
        for (int w = 32; w; w >>= 1) s += __shfl_xor(s, w);
        s = ok && finite ? s * a.scale * kLog2e : __builtin_nanf("");
        const float now = s > m ? s : m;
        const float keep = __builtin_exp2f(m - now), p = __builtin_exp2f(s - now);
        m = now;
        l = m == -__builtin_inff() ? __builtin_nanf("") : l * keep + p;
#pragma unroll
        for (int i = 0; i < kDims; ++i) {
            const int x = i * 64 + lane;
            if (x < d) o[i] = (l == l || 1 ? o[i] * keep : 0.0f) + p * (code(a.v_plane + at + x) * vs);
        }
    }
    if (lane == 0) {
        s_m[wave] = m;
        s_l[wave] = l;
    }
#pragma unroll
    for (int i = 0; i < kDims; ++i)
        if (i * 64 + lane < d) s_o[wave][i * 64 + lane] = o[i];
    __syncthreads();
    const float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    float sum = 0.0f, f[4];
    for (int w = 0; w < 4; ++w) {
        f[w] = s_m[w] == -__builtin_inff() ? 0.0f : __builtin_exp2f(s_m[w] - top);
        sum += s_l[w] != s_l[w] ? s_l[w] : s_l[w] * f[w];
    }
    const bool empty = !r.bad && place < 0;
    const float inv = empty ? 0.0f : r.bad ? __builtin_nanf("") : 1.0f / sum;
    for (int x = threadIdx.x; x < d; x += kB) {
        float v = 0.0f;
        for (int w = 0; w < 4; ++w) v += s_o[w][x] * f[w];
        store_one<DT>(a.out.data, token * a.out.token_stride + head * a.out.head_stride + x,
                      empty ? 0.0f : v * inv);
    }
    if (a.lse && threadIdx.x == 0)
        a.lse[token * a.heads + head] = empty ? -__builtin_inff()
                                        : r.bad ? __builtin_nanf("")
                                                : (top + __builtin_log2f(sum)) * kLn2;
}

}  // namespace

hipError_t attend_launch(const AttendArgs& a, int32_t dtype, hipStream_t stream)
{
    const dim3 grid((unsigned)a.tokens, (unsigned)a.heads);
    return dtype == G4S_DTYPE_F32 ? launch(attend_kernel<G4S_DTYPE_F32>, grid, kB, 0, stream, a)
                                  : launch(attend_kernel<G4S_DTYPE_BF16>, grid, kB, 0, stream, a);
}

}  // namespace g4s
