/*
 * g4s_kv.hip -- C ABI of the 8-bit cache (include/gemma4_cache.h): handles and
 * checks of arguments.  Errors follow the library's convention, a negative
 * g4s_status and a message kept in the handle.
 */
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <new>

#include "g4s_cache.h"
#include "g4s_host.h"

using g4s::CacheView;
using g4s::DeviceGuard;
using g4s::overlap;
using g4s::Span;

namespace {

thread_local char t_cache_error[512] = "";

}  // namespace

struct g4s_cache : g4s::Handle {
    g4s_page_geometry geo{};
    g4s_cache_config config{};
    g4s::CachePool pool{};
    void* memory = nullptr;
    g4s::AttendSpace ws{};
};

namespace {

int fail(g4s_cache* h, int code, const char* fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    const int rc = g4s::fail_in(h ? h->err : t_cache_error, code, fmt, ap);
    va_end(ap);
    return rc;
}

constexpr int64_t kMaxElements = (int64_t)1 << 50;

int64_t dtype_size(int32_t dtype) { return dtype == G4S_DTYPE_F32 ? 4 : 2; }

/* A view as checked: as the kernels take it, and its bytes. */
struct Checked {
    const char* name;
    CacheView view;
    g4s::Vectors vectors;
};

int check_view(g4s_cache* h, const char* name, const g4s_cache_view* v, int32_t heads,
               int32_t tokens, int64_t esize, Checked* out)
{
    *out = Checked{name, CacheView{}, g4s::Vectors{}};
    if (!v) return G4S_OK;
    if (!v->data) return fail(h, G4S_ERR_INVALID_ARGUMENT, "%s->data is NULL", name);
    const int64_t d = h->config.head_dim;
    const int64_t ts = tokens > 1 ? v->token_stride : 0, hs = heads > 1 ? v->head_stride : 0;
    if (ts < 0 || hs < 0 || ts > kMaxElements / tokens || hs > kMaxElements / heads)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "%s: a stride is negative or too large", name);
    if (((uintptr_t)v->data & 15) || ((ts * esize) & 15) || ((hs * esize) & 15))
        return fail(h, G4S_ERR_INVALID_ARGUMENT,
                    "%s: data and strides must be multiples of 16 bytes", name);
    const int64_t head_end = (heads - 1) * hs + d, token_end = (tokens - 1) * ts + d;
    /* heads within a token, or tokens within a head, none on another */
    const bool a = (heads == 1 || hs >= d) && (tokens == 1 || ts >= head_end);
    const bool b = (tokens == 1 || ts >= d) && (heads == 1 || hs >= token_end);
    if (!a && !b)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "%s: vectors of head_dim %d overlap", name,
                    h->config.head_dim);
    out->view = CacheView{static_cast<char*>(v->data), ts, hs};
    out->vectors = g4s::Vectors{(uint64_t)(uintptr_t)v->data, tokens, heads, ts * esize, hs * esize, d * esize};
    return G4S_OK;
}

Span span(const Checked& c) { return Span{c.name, c.view.data, c.view.data ? c.vectors.end() : 0}; }
bool overlap(const Checked& a, const Checked& b) { return vectors_meet(a.vectors, b.vectors); }

int check_call(g4s_cache* h, const g4s_page_state* state, int32_t rows, const int32_t* d_starts,
               int32_t tokens, int32_t dtype)
{
    if (!state || !state->table || !state->lengths)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "the state, its table and lengths must be non-NULL");
    if (rows < 1 || rows > h->geo.max_rows)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "rows %d outside [1, %d]", rows, h->geo.max_rows);
    if (tokens < 1 || tokens > G4S_CACHE_MAX_TOKENS)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "tokens %d outside [1, %d]", tokens,
                    G4S_CACHE_MAX_TOKENS);
    if (!d_starts && tokens != rows)
        return fail(h, G4S_ERR_INVALID_ARGUMENT,
                    "without d_starts every row has one token: tokens %d, rows %d", tokens, rows);
    if (dtype != G4S_DTYPE_F32 && dtype != G4S_DTYPE_BF16)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "dtype %d is neither F32 nor BF16", dtype);
    return G4S_OK;
}

int check_planes(g4s_cache* h, const void* d_pool, int32_t k_plane, int32_t v_plane)
{
    if (!d_pool) return fail(h, G4S_ERR_INVALID_ARGUMENT, "d_pool is NULL");
    if ((uintptr_t)d_pool & 3)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "d_pool must be 4-byte aligned");
    if (k_plane < 0 || k_plane >= h->geo.planes || v_plane < 0 || v_plane >= h->geo.planes ||
        k_plane == v_plane)
        return fail(h, G4S_ERR_INVALID_ARGUMENT,
                    "k_plane %d and v_plane %d must be two planes of %d", k_plane, v_plane,
                    h->geo.planes);
    return G4S_OK;
}

/* Arrays that every call reads. */
struct Inputs {
    Span at[6];
    int n = 0;
    void add(const char* name, const void* p, int64_t bytes)
    {
        if (p) at[n++] = Span{name, p, bytes};
    }
};
Inputs inputs(const g4s_cache* h, const g4s_page_state* state, int32_t rows,
              const int32_t* d_starts)
{
    Inputs in;
    in.add("state->table", state->table, (int64_t)h->geo.max_rows * h->geo.max_slots * 4);
    in.add("state->lengths", state->lengths, (int64_t)h->geo.max_rows * 4);
    in.add("d_starts", d_starts, (int64_t)(rows + 1) * 4);
    return in;
}

/* Integers and floats: scalar loads take no notice of an address' last two bits. */
int check_alignment(g4s_cache* h, const Inputs& in)
{
    for (int i = 0; i < in.n; ++i)
        if ((uintptr_t)in.at[i].at & 3)
            return fail(h, G4S_ERR_INVALID_ARGUMENT, "%s must be 4-byte aligned", in.at[i].name);
    return G4S_OK;
}

int refuse_overlap(g4s_cache* h, const char* a, const char* b)
{
    return fail(h, G4S_ERR_INVALID_ARGUMENT, "%s overlaps %s", a, b);
}

}  // namespace

G4S_API const char* g4s_cache_last_error(const g4s_cache* h)
{
    return h ? h->err : t_cache_error;
}

G4S_API int g4s_cache_create(g4s_cache** out, const g4s_page_geometry* geometry,
                             const g4s_cache_config* config, void* hip_stream)
{
    g4s_cache* none = nullptr;
    t_cache_error[0] = 0;
    if (!out) return fail(none, G4S_ERR_INVALID_ARGUMENT, "out is NULL");
    *out = nullptr;
    if (!geometry || !config)
        return fail(none, G4S_ERR_INVALID_ARGUMENT, "geometry and config must be non-NULL");
    const g4s_page_geometry& g = *geometry;
    const g4s_cache_config& c = *config;
    if (!g4s::geometry_ok(g))
        return fail(none, G4S_ERR_INVALID_ARGUMENT,
                    "geometry: outside the limits of g4s_pages_create, or pages overlap");
    if (c.kv_heads < 1 || c.kv_heads > G4S_CACHE_MAX_KV_HEADS || c.heads < 1 ||
        c.heads > G4S_CACHE_MAX_HEADS || c.heads % c.kv_heads != 0 ||
        c.heads / c.kv_heads > G4S_CACHE_MAX_GROUP)
        return fail(none, G4S_ERR_INVALID_ARGUMENT,
                    "heads %d (at most %d, %d for each kv head) / kv_heads %d (at most %d)",
                    c.heads, G4S_CACHE_MAX_HEADS, G4S_CACHE_MAX_GROUP, c.kv_heads,
                    G4S_CACHE_MAX_KV_HEADS);
    if (c.head_dim < 16 || c.head_dim > G4S_CACHE_MAX_HEAD_DIM || c.head_dim % 16 != 0)
        return fail(none, G4S_ERR_INVALID_ARGUMENT, "head_dim %d is no multiple of 16 up to %d",
                    c.head_dim, G4S_CACHE_MAX_HEAD_DIM);
    if (c.scale_tokens < 1 || c.scale_tokens > G4S_CACHE_MAX_SCALE_TOKENS ||
        g.page_tokens % c.scale_tokens != 0)
        return fail(none, G4S_ERR_INVALID_ARGUMENT,
                    "scale_tokens %d outside [1, %d], or no divisor of page_tokens %d",
                    c.scale_tokens, G4S_CACHE_MAX_SCALE_TOKENS, g.page_tokens);
    if (c.rotary_dims < 0 || c.rotary_dims > c.head_dim || c.rotary_dims % 2 != 0 ||
        (c.rotary_pairs != G4S_ROTARY_HALVES && c.rotary_pairs != G4S_ROTARY_NEIGHBOURS))
        return fail(none, G4S_ERR_INVALID_ARGUMENT,
                    "rotary_dims %d (even, 0 .. head_dim) / rotary_pairs %d", c.rotary_dims,
                    c.rotary_pairs);
    if (g.planes < 2 || g.parts != c.kv_heads || g.token_bytes != c.head_dim + 4 ||
        g.plane_stride % 4 != 0 || g.page_stride % 4 != 0)
        return fail(none, G4S_ERR_INVALID_ARGUMENT,
                    "geometry: planes %d (2 at least), parts %d (kv_heads %d), token_bytes %lld "
                    "(head_dim + 4 = %d), strides %lld and %lld (multiples of 4)",
                    g.planes, g.parts, c.kv_heads, (long long)g.token_bytes, c.head_dim + 4,
                    (long long)g.plane_stride, (long long)g.page_stride);
    if ((int64_t)g.max_slots * g.page_tokens > G4S_CACHE_MAX_CONTEXT)
        return fail(none, G4S_ERR_INVALID_ARGUMENT, "geometry: max_slots %d of %d tokens, a row holds at most %d",
                    g.max_slots, g.page_tokens, G4S_CACHE_MAX_CONTEXT);
    int device = 0;
    auto refuse = [&](int code, auto... a) { return fail(none, code, a...); };
    int ncu = 0;
    const int rc = g4s::pick_device(refuse, &device, &ncu);
    if (rc) return rc;
    g4s_cache* h = new (std::nothrow) g4s_cache();
    if (!h) return fail(none, G4S_ERR_OUT_OF_MEMORY, "host memory");
    h->device = device;
    h->stream = (hipStream_t)hip_stream;
    h->geo = g;
    h->config = c;
    h->pool.plane_stride = g.plane_stride;
    h->pool.page_stride = g.page_stride;
    h->pool.part_bytes = (int32_t)(g.page_tokens * g.token_bytes);
    h->pool.token_bytes = (int32_t)g.token_bytes;
    h->pool.n_pages = g.n_pages;
    h->pool.max_slots = g.max_slots;
    h->pool.page_tokens = g4s::divisor(g.page_tokens);
    h->pool.scale_tokens = g4s::divisor(c.scale_tokens);
    h->pool.head_dim = c.head_dim;
    h->ws.groups = g4s::attend_groups(ncu);
    const size_t groups = (size_t)h->ws.groups;
    g4s::Carver w;
    auto lay = [&] {
        w.add(&h->ws.sums, groups * g4s::kAttendSums);
        w.add(&h->ws.stats, groups * g4s::kAttendStats);
        w.add(&h->ws.tickets, groups);
        w.add(&h->ws.records, groups);
    };
    lay();
    const size_t bytes = w.used();
    if (hipMalloc(&h->memory, bytes) != hipSuccess) {
        (void)hipGetLastError();
        delete h;
        return fail(none, G4S_ERR_OUT_OF_MEMORY, "workspace of %zu bytes", bytes);
    }
    w.start(h->memory);
    lay();
    hipError_t e = g4s::attend_init_launch(h->ws, h->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(h->stream);
    if (e != hipSuccess) {
        (void)hipFree(h->memory);
        delete h;
        return fail(none, G4S_ERR_HIP, "workspace initialisation: %s", hipGetErrorString(e));
    }
    *out = h;
    return G4S_OK;
}

G4S_API int g4s_cache_destroy(g4s_cache* h)
{
    if (!h) return G4S_OK;
    DeviceGuard guard(h->device);
    (void)hipStreamSynchronize(h->stream);
    (void)hipFree(h->memory);
    delete h;
    return G4S_OK;
}

G4S_API int g4s_cache_append(g4s_cache* h, const g4s_page_state* state, int32_t rows,
                             const int32_t* d_starts, int32_t tokens, int32_t dtype,
                             const g4s_cache_view* q, const g4s_cache_view* k,
                             const g4s_cache_view* v, const g4s_cache_view* q_out,
                             const int32_t* d_positions, const float* d_freqs, void* d_pool,
                             int32_t k_plane, int32_t v_plane)
{
    if (!h) return fail(h, G4S_ERR_INVALID_ARGUMENT, "cache is NULL");
    h->err[0] = 0;
    int rc = check_call(h, state, rows, d_starts, tokens, dtype);
    if (rc) return rc;
    const g4s_cache_config& c = h->config;
    if (!q != !q_out || !k != !v || (!q && !k))
        return fail(h, G4S_ERR_INVALID_ARGUMENT,
                    "q and q_out, and k and v, come together, and one pair at least");
    if (!d_freqs && c.rotary_dims > 0)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "d_freqs is NULL");
    const int64_t esize = dtype_size(dtype);
    Checked cq, ck, cv, co;
    rc = check_view(h, "q", q, c.heads, tokens, esize, &cq);
    if (!rc) rc = check_view(h, "k", k, c.kv_heads, tokens, esize, &ck);
    if (!rc) rc = check_view(h, "v", v, c.kv_heads, tokens, esize, &cv);
    if (!rc) rc = check_view(h, "q_out", q_out, c.heads, tokens, esize, &co);
    if (!rc && k) rc = check_planes(h, d_pool, k_plane, v_plane);
    if (rc) return rc;
    Inputs in = inputs(h, state, rows, d_starts);
    in.add("d_positions", d_positions, (int64_t)tokens * 4);
    in.add("d_freqs", d_freqs, (int64_t)c.rotary_dims / 2 * 4);
    rc = check_alignment(h, in);
    if (rc) return rc;
    const Span pool{"d_pool", k ? d_pool : nullptr, g4s::pool_extent(h->geo)};
    for (int i = 0; i < in.n; ++i) {
        if (overlap(span(co), in.at[i])) return refuse_overlap(h, "q_out", in.at[i].name);
        if (overlap(pool, in.at[i])) return refuse_overlap(h, "d_pool", in.at[i].name);
    }
    for (const Checked* x : {&cq, &ck, &cv, &co})
        if (overlap(pool, span(*x))) return refuse_overlap(h, "d_pool", x->name);
    const bool same = cq.view.data == co.view.data &&
                      cq.view.token_stride == co.view.token_stride &&
                      cq.view.head_stride == co.view.head_stride;
    if (!same && overlap(co, cq))
        return fail(h, G4S_ERR_INVALID_ARGUMENT,
                    "q_out overlaps q (it may be q, with the same strides)");
    for (const Checked* x : {&ck, &cv})
        if (overlap(co, *x)) return refuse_overlap(h, "q_out", x->name);
    DeviceGuard guard(h->device);
    if (!guard.ok()) return fail(h, G4S_ERR_HIP, "device %d cannot be made current", h->device);
    g4s::AppendArgs a{};
    a.pool = h->pool;
    a.table = state->table;
    a.lengths = state->lengths;
    a.starts = d_starts;
    a.rows = rows;
    a.tokens = tokens;
    a.q = cq.view;
    a.k = ck.view;
    a.v = cv.view;
    a.q_out = co.view;
    a.positions = d_positions;
    a.freqs = d_freqs;
    if (k) {
        a.k_plane = static_cast<char*>(d_pool) + k_plane * h->pool.plane_stride;
        a.v_plane = static_cast<char*>(d_pool) + v_plane * h->pool.plane_stride;
    }
    a.heads = c.heads;
    a.kv_heads = c.kv_heads;
    a.rotary_dims = c.rotary_dims;
    a.rotary_pairs = c.rotary_pairs;
    const hipError_t e = g4s::append_launch(a, dtype, h->stream);
    if (e != hipSuccess) return fail(h, G4S_ERR_HIP, "append launch: %s", hipGetErrorString(e));
    return G4S_OK;
}

G4S_API int g4s_cache_attend(g4s_cache* h, const g4s_page_state* state, int32_t rows,
                             const int32_t* d_starts, int32_t tokens, int32_t dtype,
                             const g4s_cache_view* q, const void* d_pool, int32_t k_plane,
                             int32_t v_plane, float scale, int32_t window,
                             const g4s_cache_view* out, float* d_lse)
{
    if (!h) return fail(h, G4S_ERR_INVALID_ARGUMENT, "cache is NULL");
    h->err[0] = 0;
    int rc = check_call(h, state, rows, d_starts, tokens, dtype);
    if (rc) return rc;
    const g4s_cache_config& c = h->config;
    if (!q || !out) return fail(h, G4S_ERR_INVALID_ARGUMENT, "q and out must be non-NULL");
    if (!(std::fabs(scale) <= 0x1p127f)) /* (times log2(e) it is a number) */
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "scale %g is not within +-2^127", scale);
    if (window < 0) return fail(h, G4S_ERR_INVALID_ARGUMENT, "window %d is negative", window);
    const int64_t esize = dtype_size(dtype);
    Checked cq, co;
    rc = check_view(h, "q", q, c.heads, tokens, esize, &cq);
    if (!rc) rc = check_view(h, "out", out, c.heads, tokens, esize, &co);
    if (!rc) rc = check_planes(h, d_pool, k_plane, v_plane);
    if (rc) return rc;
    if ((uintptr_t)d_lse & 3)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "d_lse must be 4-byte aligned");
    Inputs in = inputs(h, state, rows, d_starts);
    in.add("d_pool", d_pool, g4s::pool_extent(h->geo));
    rc = check_alignment(h, in);
    if (rc) return rc;
    const Span lse{"d_lse", d_lse, (int64_t)tokens * c.heads * 4};
    for (int i = 0; i < in.n; ++i) {
        if (overlap(span(co), in.at[i])) return refuse_overlap(h, "out", in.at[i].name);
        if (overlap(lse, in.at[i])) return refuse_overlap(h, "d_lse", in.at[i].name);
    }
    if (overlap(co, cq)) return refuse_overlap(h, "out", "q");
    if (overlap(lse, span(cq))) return refuse_overlap(h, "d_lse", "q");
    if (overlap(lse, span(co))) return refuse_overlap(h, "d_lse", "out");
    DeviceGuard guard(h->device);
    if (!guard.ok()) return fail(h, G4S_ERR_HIP, "device %d cannot be made current", h->device);
    g4s::AttendArgs a{};
    a.pool = h->pool;
    a.table = state->table;
    a.lengths = state->lengths;
    a.starts = d_starts;
    a.rows = rows;
    a.tokens = tokens;
    a.q = cq.view;
    a.out = co.view;
    a.k_plane = static_cast<const char*>(d_pool) + k_plane * h->pool.plane_stride;
    a.v_plane = static_cast<const char*>(d_pool) + v_plane * h->pool.plane_stride;
    a.lse = d_lse;
    a.scale = scale;
    a.window = window;
    a.heads = c.heads;
    a.kv_heads = c.kv_heads;
    a.group = g4s::divisor(c.heads / c.kv_heads);
    a.ws = h->ws;
    /* Which rows have how many tokens is known on the device alone, so a call of ragged ones
     * enqueues both kernels, but for those that cannot have prompts and the one row that is one. */
    const bool prompts = d_starts && (int64_t)tokens * a.group.d > g4s::kFewCols;
    a.few = prompts && rows == 1 ? 0 : g4s::kFewCols;
    hipError_t e = hipSuccess;
    if (a.few > 0) e = g4s::attend_rows_launch(a, dtype, h->stream);
    if (e == hipSuccess && prompts) e = g4s::attend_prompts_launch(a, dtype, h->stream);
    if (e != hipSuccess) return fail(h, G4S_ERR_HIP, "attention launch: %s", hipGetErrorString(e));
    return G4S_OK;
}
