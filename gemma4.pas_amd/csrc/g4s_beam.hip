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

__device__ __forceinline__ double softcap64(float x, double cap)
{
    return cap > 0.0 ? cap * tanh((double)x / cap) : (double)x;
}

/* exp(y - top) for y <= top; an infinite top (no softcap, x = +inf) counts 1
 * for itself and leaves nothing for the rest. */
__device__ __forceinline__ double term64(double y, double top)
{
    return y == top ? 1.0 : exp(y - top);
}

struct TopShared {
    uint32_t tmax[kB];
    uint32_t hist[256];
    int misc[8];
    int scan[kB / 64];
    double red[kB / 64];
    int count;
    alignas(16) uint64_t list[kListCap]; /* every element at or above `bound`, any order */
    uint64_t sorted[kNMax];              /* the n best of them, best first */
};

template <int BLOCK>
__device__ double block_sum_f64(double v, double* s_wave)
{
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
    if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x >> 6] = v;
    __syncthreads();
    double r = 0.0;
#pragma unroll
    for (int w = 0; w < BLOCK / 64; ++w) r += s_wave[w];
    __syncthreads();
    return r;
}

/* The n best (n <= kNMax) of the workgroup's candidates into sh.sorted; returns
 * how many there are (fewer than n where there are no more).  x: this thread's E logits,
 * token(e) their tokens.  On return `listed` entries of sh.list hold every
 * candidate at or above `bound`, except `more` further copies of `bound` itself.
 *
 * The n-th largest of the threads' largest keys bounds the n-th largest key
 * from below, and for n well below the threads few elements beside the n best
 * reach it: those are listed and ranked by counting.  Where more are at or above
 * the bound than the list holds (equal logits in masses), the n-th largest
 * key is selected exactly and of its copies the lowest tokens are taken, in
 * the order of (vector j, thread, element i) that `token` rises in. */
template <int E, int VW, typename TokenF>
__device__ int top_list(const float (&x)[E], TokenF token, int n, TopShared& sh, float& bound,
                        int& listed, int& more)
{
    const int tid = threadIdx.x, lane = tid & 63;
    float m = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) m = fmaxf(m, x[e]);
    const uint32_t mkey = cand_key(m);
    sh.tmax[tid] = mkey;
    if (tid == 0) sh.count = 0;
    __syncthreads();
    uint32_t v[kB / 64];
    int nz = 0;
#pragma unroll
    for (int q = 0; q < kB / 64; ++q) {
        v[q] = sh.tmax[lane + 64 * q];
        nz += __popcll(__ballot(v[q] != 0u));
    }
    const uint32_t t = nz >= n ? wave_kth_bound<kB / 64>(v, n, 32) : 1u;
    bound = t == 1u ? -__builtin_inff() : key2f(t);
    if (mkey >= t) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (x[e] > kMasked && x[e] >= bound) {
                const int p = atomicAdd(&sh.count, 1);
                if (p < kListCap) sh.list[p] = entry_of(f2key(x[e]), token(e));
            }
    }
    __syncthreads();
    int cnt = sh.count;
    more = 0;
    if (cnt > kListCap) {
        uint32_t keys[E];
#pragma unroll
        for (int e = 0; e < E; ++e) keys[e] = cand_key(x[e]);
        int gt, eq;
        const uint32_t kth = regs_radix_kth<kB, E>(keys, n, sh.hist, sh.misc, &gt, &eq);
        bound = key2f(kth);
        if (tid == 0) sh.count = 0;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (keys[e] > kth) sh.list[atomicAdd(&sh.count, 1)] = entry_of(keys[e], token(e));
        __syncthreads();
        int taken = gt;
#pragma unroll
        for (int j = 0; j < E / VW; ++j) {
            int c = 0, total;
#pragma unroll
            for (int i = 0; i < VW; ++i) c += keys[j * VW + i] == kth;
            int p = taken + block_exclusive_scan<kB>(c, sh.scan, total);
#pragma unroll
            for (int i = 0; i < VW; ++i)
                if (keys[j * VW + i] == kth) {
                    if (p < n) sh.list[p] = entry_of(kth, token(j * VW + i));
                    ++p;
                }
            taken += total;
        }
        cnt = n;
        more = gt + eq - n;
        __syncthreads();
    }
    listed = cnt;
    for (int i = tid; i < cnt; i += kB) {
        const uint64_t mine = sh.list[i];
        int rank = 0;
        for (int j = 0; j < cnt; ++j) rank += sh.list[j] > mine;
        if (rank < n) sh.sorted[rank] = mine;
    }
    __syncthreads();
    return cnt < n ? cnt : n;
}

/* ------------------------------------------------------------------ chunks */

template <int DT>
__global__ __launch_bounds__(kB) void beam_chunk_kernel(BeamSelectArgs a)
{
    constexpr int VW = Elem<DT>::VW;
    constexpr int NV = kE / VW;
    __shared__ TopShared sh;
    const int row = blockIdx.y, ch = blockIdx.x, tid = threadIdx.x;
    if (!(a.scores[row] > kMasked)) return;
    const char* base = static_cast<const char*>(a.logits) + (int64_t)row * a.row_stride * Elem<DT>::SIZE;
    const int64_t first = (int64_t)ch * kBeamChunk;
    float x[kE];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        float v[VW];
        load_vec<DT>(base, first + (int64_t)(j * kB + tid) * VW, a.vocab, v);
#pragma unroll
        for (int i = 0; i < VW; ++i) x[j * VW + i] = v[i];
    }
    auto token = [&](int e) {
        return (uint32_t)first + (uint32_t)(((e / VW) * kB + tid) * VW + e % VW);
    };
    float bound;
    int listed, more;
    const int cnt = top_list<kE, VW>(x, token, a.n, sh, bound, listed, more);
    const int64_t at = (int64_t)row * a.chunks + ch;
    uint64_t* cand = a.ws.cand + at * a.n;
    for (int i = tid; i < a.n; i += kB) cand[i] = i < cnt ? sh.sorted[i] : 0ull;

    /* the listed candidates, the heaviest terms, and their further copies
     * in binary64; the rest of the chunk */
    const double cap = (double)a.softcap;
    const double top = cnt ? softcap64(key2f(entry_key(sh.sorted[0])), cap) : -__builtin_inf();
    double s = 0.0;
    if (cnt) {
        for (int i = tid; i < listed; i += kB)
            s += term64(softcap64(key2f(entry_key(sh.list[i])), cap), top);
        if (tid == 0 && more) s += (double)more * term64(softcap64(bound, cap), top);
#pragma unroll
        for (int e = 0; e < kE; ++e)
            if (x[e] > kMasked && x[e] < bound) s += term64(softcap64(x[e], cap), top);
    }
    s = block_sum_f64<kB>(s, sh.red);
    if (tid == 0) a.ws.parts[at] = BeamPart{top, s};
}

/* -------------------------------------------------------------------- rows */

/* A row's n best and its normaliser from its chunks'. */
__global__ __launch_bounds__(kB) void beam_row_kernel(BeamSelectArgs a)
{
    constexpr int E = 16;
    __shared__ TopShared sh;
    const int row = blockIdx.x, tid = threadIdx.x;
    const bool live = a.scores[row] > kMasked;
    uint64_t* best = a.ws.best + (int64_t)row * a.n;
    const uint64_t* cand = a.ws.cand + (int64_t)row * a.chunks * a.n;
    const int64_t total = live ? (int64_t)a.chunks * a.n : 0;
    int cnt = 0;
    /* tiles of candidates beside the best of those before; the chunks' lists
     * lie in token order, so copies of one key do too */
    for (int64_t base = 0; base < total;) {
        float x[E];
        uint32_t tok[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = e * kB + tid;
            uint64_t c = 0ull;
            if (i < cnt)
                c = sh.sorted[i];
            else if (base + i - cnt < total)
                c = cand[base + i - cnt];
            x[e] = c ? key2f(entry_key(c)) : -__builtin_inff();
            tok[e] = entry_token(c);
        }
        base += E * kB - cnt;
        __syncthreads();
        float bound;
        int listed, more;
        cnt = top_list<E, 1>(x, [&](int e) { return tok[e]; }, a.n, sh, bound, listed, more);
    }
    __syncthreads();
    const BeamPart* parts = a.ws.parts + (int64_t)row * a.chunks;
    const double cap = (double)a.softcap;
    const double top = cnt ? softcap64(key2f(entry_key(sh.sorted[0])), cap) : -__builtin_inf();
    double s = 0.0;
    if (cnt)
        for (int c = tid; c < a.chunks; c += kB) {
            const BeamPart p = parts[c];
            if (p.sum > 0.0) s += p.sum * term64(p.top, top);
        }
    s = block_sum_f64<kB>(s, sh.red);
    const double ls = log(s);
    double* ys = a.ws.y + (int64_t)row * a.n;
    for (int i = tid; i < a.n; i += kB) {
        uint64_t e = i < cnt ? sh.sorted[i] : 0ull;
        double y = -__builtin_inf();
        if (e) {
            /* where tanh saturates its last bit may waver: the list may not rise */
            y = top;
            for (int j = 1; j <= i; ++j)
                y = fmin(y, softcap64(key2f(entry_key(sh.sorted[j])), cap));
            /* beside an infinite largest logit the rest have probability 0 */
            if (top == __builtin_inf() && y != top) e = 0ull;
        }
        best[i] = e;
        ys[i] = y;
    }
    if (tid == 0) {
        a.ws.norm[2 * row] = top;
        a.ws.norm[2 * row + 1] = ls;
        if (a.lse) a.lse[row] = cnt ? (float)(top + ls) : -__builtin_inff();
    }
}

/* --------------------------------------------------------------- sequences */

/* The n best of the sequence's W sorted lists: a candidate's rank is the
 * number of better ones, found in each list by bisection. */
__global__ __launch_bounds__(kB) void beam_sequence_kernel(BeamSelectArgs a)
{
    extern __shared__ double sc[]; /* [W][n] scores, -inf = none */
    __shared__ int s_wave[kB / 64];
    const int b = blockIdx.x, tid = threadIdx.x;
    const int W = a.beams, n = a.n, total = W * n;
    const uint64_t* best = a.ws.best + (int64_t)b * total;
    const double* ys = a.ws.y + (int64_t)b * total;
    int found = 0;
    for (int i = tid; i < total; i += kB) {
        const int w = i / n;
        double s = -__builtin_inf();
        if (best[i]) {
            const double* norm = a.ws.norm + 2 * ((int64_t)b * W + w);
            s = (double)a.scores[b * W + w] + ((ys[i] == norm[0] ? 0.0 : ys[i] - norm[0]) - norm[1]);
            ++found;
        }
        sc[i] = s;
    }
    found = block_sum_i32<kB>(found, s_wave);
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
            tokens[rank] = (int32_t)entry_token(best[i]);
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

hipError_t beam_select_launch(const BeamSelectArgs& a, int32_t dtype, hipStream_t stream)
{
    const dim3 grid((unsigned)a.chunks, (unsigned)(a.batch * a.beams));
    if (dtype == G4S_DTYPE_F32)
        beam_chunk_kernel<0><<<grid, kB, 0, stream>>>(a);
    else
        beam_chunk_kernel<1><<<grid, kB, 0, stream>>>(a);
    beam_row_kernel<<<(unsigned)(a.batch * a.beams), kB, 0, stream>>>(a);
    beam_sequence_kernel<<<(unsigned)a.batch, kB, sizeof(double) * a.beams * a.n, stream>>>(a);
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
