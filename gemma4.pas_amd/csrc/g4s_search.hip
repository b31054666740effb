/*
 * g4s_search.hip -- C ABI of the beam search, the page cache and the search
 * loop (include/gemma4_beam.h): handles, checks of arguments, and the host
 * side of g4s_beam_generate.  Errors follow the library's convention, a
 * negative g4s_status and a message kept in the handle.
 */
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <limits>
#include <new>
#include <vector>

#include "g4s_beam.h"
#include "g4s_pages.h"

#define G4S_API extern "C" __attribute__((visibility("default")))

namespace {

struct Handle {
    int device = 0;
    hipStream_t stream = nullptr;
    char err[512] = "";
};

thread_local char t_beam_error[512] = "";
thread_local char t_pages_error[512] = "";

int fail_in(char (&buf)[512], int code, const char* fmt, va_list ap)
{
    vsnprintf(buf, sizeof(buf), fmt, ap);
    return code;
}

}  // namespace

struct g4s_beam : Handle {
    int32_t vocab = 0, max_batch = 0, max_beams = 0, ncu = 0;
    g4s::BeamSoftcap cap{};
    int32_t plan_rows = 0, plan_dtype = 0; /* the last call's */
    g4s::BeamPlan plan{};
    void* memory = nullptr;
    g4s::BeamWorkspace ws{};
};

struct g4s_pages : Handle {
    g4s_page_geometry geo{};
    int32_t words = 0;
    void* memory = nullptr;
    g4s::PageWorkspace ws{};
};

namespace {

int fail(g4s_beam* h, int code, const char* fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    const int rc = fail_in(h ? h->err : t_beam_error, code, fmt, ap);
    va_end(ap);
    return rc;
}

int fail(g4s_pages* h, int code, const char* fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    const int rc = fail_in(h ? h->err : t_pages_error, code, fmt, ap);
    va_end(ap);
    return rc;
}

template <typename H>
int hip_fail(H* h, hipError_t e, const char* what)
{
    return fail(h, G4S_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

/* The handle's device is current while a call works with it. */
class DeviceGuard {
public:
    explicit DeviceGuard(int device)
    {
        if (hipGetDevice(&old_) != hipSuccess) old_ = device;
        if (old_ != device)
            ok_ = hipSetDevice(device) == hipSuccess;
        else
            old_ = -1;
    }
    ~DeviceGuard()
    {
        if (old_ >= 0) (void)hipSetDevice(old_);
    }
    bool ok() const { return ok_; }

private:
    int old_ = -1;
    bool ok_ = true;
};

/* The current device, if the library runs on it. */
template <typename H>
int pick_device(H* none, int* device, int* ncu = nullptr)
{
    int n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess || n < 1)
        return fail(none, G4S_ERR_NO_DEVICE, "no HIP device visible");
    hipDeviceProp_t prop;
    if (hipGetDevice(device) != hipSuccess ||
        hipGetDeviceProperties(&prop, *device) != hipSuccess)
        return fail(none, G4S_ERR_NO_DEVICE, "the current HIP device is not usable");
    if (std::strncmp(prop.gcnArchName, "gfx950", 6) != 0)
        return fail(none, G4S_ERR_NO_DEVICE, "device %d is %s; this library targets gfx950",
                    *device, prop.gcnArchName);
    if (ncu) *ncu = prop.multiProcessorCount;
    return G4S_OK;
}

bool overlap(const void* a, int64_t na, const void* b, int64_t nb)
{
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return na > 0 && nb > 0 && x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

/* An array of a call; NULL ones overlap nothing. */
struct Span {
    const char* name;
    const void* at;
    int64_t bytes;
};
bool overlap(const Span& a, const Span& b)
{
    return a.at && b.at && overlap(a.at, a.bytes, b.at, b.bytes);
}

/* Parts of one allocation, each on a 256-byte boundary. */
class Carver {
public:
    template <typename T>
    void add(T** p, size_t count)
    {
        if (base_) *p = reinterpret_cast<T*>(base_ + used_);
        used_ += (count * sizeof(T) + 255) & ~(size_t)255;
    }
    size_t used() const { return used_; }
    void start(void* base)
    {
        base_ = static_cast<char*>(base);
        used_ = 0;
    }

private:
    char* base_ = nullptr;
    size_t used_ = 0;
};

constexpr int64_t kMaxExtent = (int64_t)1 << 56;

/* `outer` blocks of `inner` pieces of `bytes`, neither overlapping the other. */
bool strides_ok(int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t bytes)
{
    if (s1 < 0 || s2 < 0 || s1 > kMaxExtent / n1 || s2 > kMaxExtent / n2) return false;
    const bool a = (n2 == 1 || s2 >= bytes) && (n1 == 1 || s1 >= (n2 - 1) * s2 + bytes);
    const bool b = (n1 == 1 || s1 >= bytes) && (n2 == 1 || s2 >= (n1 - 1) * s1 + bytes);
    return a || b;
}

}  // namespace

/* ------------------------------------------------------------------ search */

G4S_API const char* g4s_beam_last_error(const g4s_beam* h) { return h ? h->err : t_beam_error; }

G4S_API int g4s_beam_create(g4s_beam** out, int32_t vocab, int32_t max_batch, int32_t max_beams,
                            float softcap, void* hip_stream)
{
    g4s_beam* none = nullptr;
    t_beam_error[0] = 0;
    if (!out) return fail(none, G4S_ERR_INVALID_ARGUMENT, "out is NULL");
    *out = nullptr;
    if (vocab < 2) return fail(none, G4S_ERR_INVALID_ARGUMENT, "vocab %d below 2", vocab);
    if (vocab > g4s::kBeamMaxVocab)
        return fail(none, G4S_ERR_UNSUPPORTED, "vocab %d above %d", vocab, g4s::kBeamMaxVocab);
    if (max_beams < 1 || max_beams > G4S_BEAM_MAX_BEAMS)
        return fail(none, G4S_ERR_INVALID_ARGUMENT, "max_beams %d outside [1, %d]", max_beams,
                    G4S_BEAM_MAX_BEAMS);
    if (max_batch < 1 || (int64_t)max_batch * max_beams > G4S_BEAM_MAX_ROWS)
        return fail(none, G4S_ERR_INVALID_ARGUMENT, "max_batch %d x max_beams %d outside [1, %d]",
                    max_batch, max_beams, G4S_BEAM_MAX_ROWS);
    if (!std::isfinite(softcap))
        return fail(none, G4S_ERR_INVALID_ARGUMENT, "softcap %g is not finite", softcap);
    int device = 0, ncu = 0;
    const int rc = pick_device(none, &device, &ncu);
    if (rc) return rc;
    g4s_beam* h = new (std::nothrow) g4s_beam();
    if (!h) return fail(none, G4S_ERR_OUT_OF_MEMORY, "host memory");
    h->device = device;
    h->stream = (hipStream_t)hip_stream;
    h->ncu = ncu;
    h->vocab = vocab;
    h->max_batch = max_batch;
    h->max_beams = max_beams;
    h->cap = g4s::beam_softcap(softcap);
    const size_t rows = (size_t)max_batch * max_beams, n = 2 * (size_t)max_beams;
    const size_t chunks = (size_t)g4s::beam_max_chunks(vocab, (int32_t)rows, ncu);
    Carver c;
    auto lay = [&] {
        c.add(&h->ws.cand, chunks * n);
        c.add(&h->ws.sums, chunks * 2);
        c.add(&h->ws.best, rows * n);
        c.add(&h->ws.y, rows * n);
        c.add(&h->ws.norm, rows * 2);
        c.add(&h->ws.tickets, rows + max_batch);
        c.add(&h->ws.table, (size_t)2 * g4s::kBeamTableHalf);
    };
    lay();
    const size_t bytes = c.used();
    if (hipMalloc(&h->memory, bytes) != hipSuccess) {
        (void)hipGetLastError();
        delete h;
        return fail(none, G4S_ERR_OUT_OF_MEMORY, "workspace of %zu bytes", bytes);
    }
    c.start(h->memory);
    lay();
    hipError_t e =
        g4s::beam_init_launch(h->ws, h->cap, (int32_t)(rows + max_batch), h->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(h->stream);
    if (e != hipSuccess) {
        (void)hipFree(h->memory);
        delete h;
        return hip_fail(none, e, "workspace initialisation");
    }
    *out = h;
    return G4S_OK;
}

G4S_API int g4s_beam_destroy(g4s_beam* h)
{
    if (!h) return G4S_OK;
    DeviceGuard guard(h->device);
    (void)hipStreamSynchronize(h->stream);
    (void)hipFree(h->memory);
    delete h;
    return G4S_OK;
}

namespace {

int check_shape(g4s_beam* h, int32_t batch, int32_t beams)
{
    if (batch < 1 || batch > h->max_batch)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "batch %d outside [1, %d]", batch, h->max_batch);
    if (beams < 1 || beams > h->max_beams)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "beams %d outside [1, %d]", beams, h->max_beams);
    return G4S_OK;
}

int check_logits(g4s_beam* h, const void* d_logits, int32_t dtype, int64_t row_stride, int64_t rows)
{
    if (!d_logits) return fail(h, G4S_ERR_INVALID_ARGUMENT, "d_logits is NULL");
    if (dtype != G4S_DTYPE_F32 && dtype != G4S_DTYPE_BF16)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "dtype %d is neither F32 nor BF16", dtype);
    const int64_t esize = dtype == G4S_DTYPE_F32 ? 4 : 2;
    if (((uintptr_t)d_logits & 15u) != 0)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "d_logits must be 16-byte aligned");
    if (rows > 1 && (row_stride < h->vocab || row_stride > kMaxExtent / (rows * esize)))
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "row_stride %lld < vocab %d, or too large",
                    (long long)row_stride, h->vocab);
    if (rows > 1 && ((row_stride * esize) & 15) != 0)
        return fail(h, G4S_ERR_INVALID_ARGUMENT,
                    "row_stride * sizeof(dtype) must be a multiple of 16 bytes");
    return G4S_OK;
}

int select(g4s_beam* h, const void* d_logits, int32_t dtype, int64_t row_stride, int32_t batch,
           int32_t beams, const float* d_scores, int32_t n, int32_t* d_parents, int32_t* d_tokens,
           float* d_out, float* d_lse)
{
    g4s::BeamSelectArgs a{};
    a.logits = d_logits;
    a.row_stride = batch * beams > 1 ? row_stride : 0;
    a.vocab = h->vocab;
    a.batch = batch;
    a.beams = beams;
    a.n = n;
    if (h->plan_rows != batch * beams || h->plan_dtype != dtype) {
        h->plan_rows = batch * beams;
        h->plan_dtype = dtype;
        h->plan = g4s::beam_plan(h->vocab, batch * beams, dtype, h->cap.mode, h->ncu);
    }
    a.chunks = h->plan.chunks;
    a.tiles = h->plan.tiles;
    a.cap = h->cap;
    a.scores = d_scores;
    a.parents = d_parents;
    a.tokens = d_tokens;
    a.out = d_out;
    a.lse = d_lse;
    a.ws = h->ws;
    const hipError_t e = g4s::beam_select_launch(a, h->plan, dtype, h->stream);
    return e == hipSuccess ? G4S_OK : hip_fail(h, e, "beam selection launch");
}

int reorder(g4s_beam* h, const void* d_src, void* d_dst, int64_t planes, int64_t plane_stride,
            int32_t batch, int32_t beams, int64_t row_stride, int64_t row_bytes,
            const int32_t* d_parents)
{
    if (!d_src || !d_dst || !d_parents)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "d_src, d_dst and d_parents must be non-NULL");
    const int64_t rows = (int64_t)batch * beams;
    if (planes < 1 || planes > ((int64_t)1 << 31) || row_bytes < 0 ||
        row_bytes > ((int64_t)1 << 38) ||
        !strides_ok(planes, plane_stride, rows, row_stride, row_bytes))
        return fail(h, G4S_ERR_INVALID_ARGUMENT,
                    "planes %lld / plane_stride %lld / row_stride %lld / row_bytes %lld: "
                    "negative, too large or overlapping",
                    (long long)planes, (long long)plane_stride, (long long)row_stride,
                    (long long)row_bytes);
    const int64_t extent = (planes - 1) * plane_stride + (rows - 1) * row_stride + row_bytes;
    if (d_src != d_dst && overlap(d_src, extent, d_dst, extent))
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "d_src and d_dst overlap");
    if (overlap(d_parents, rows * 4, d_dst, extent))
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "d_parents overlaps d_dst");
    if (row_bytes == 0) return G4S_OK;
    g4s::BeamReorderArgs a{};
    a.src = (const char*)d_src;
    a.dst = (char*)d_dst;
    a.planes = planes;
    a.plane_stride = planes > 1 ? plane_stride : 0;
    a.batch = batch;
    a.beams = beams;
    a.row_stride = rows > 1 ? row_stride : 0;
    a.row_bytes = row_bytes;
    a.parents = d_parents;
    const hipError_t e = g4s::beam_reorder_launch(a, h->stream);
    return e == hipSuccess ? G4S_OK : hip_fail(h, e, "state reordering launch");
}

}  // namespace

G4S_API int g4s_beam_select(g4s_beam* h, const void* d_logits, int32_t dtype, int64_t row_stride,
                            int32_t batch, int32_t beams, const float* d_scores, int32_t n_select,
                            int32_t* d_parents, int32_t* d_tokens, float* d_out, float* d_lse)
{
    if (!h) return fail(h, G4S_ERR_INVALID_ARGUMENT, "beam is NULL");
    h->err[0] = 0;
    int rc = check_shape(h, batch, beams);
    if (!rc) rc = check_logits(h, d_logits, dtype, row_stride, (int64_t)batch * beams);
    if (rc) return rc;
    if (!d_scores || !d_parents || !d_tokens || !d_out)
        return fail(h, G4S_ERR_INVALID_ARGUMENT,
                    "d_scores, d_parents, d_tokens and d_out must be non-NULL");
    if (n_select < 1 || n_select > 2 * h->max_beams)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "n_select %d outside [1, %d]", n_select,
                    2 * h->max_beams);
    /* a sequence's results are written while others' logits and scores, or its own lse, are
     * still to be read or written */
    const int64_t rows = (int64_t)batch * beams, found = (int64_t)batch * n_select * 4;
    const int64_t esize = dtype == G4S_DTYPE_F32 ? 4 : 2;
    const Span out[4] = {{"d_parents", d_parents, found},
                         {"d_tokens", d_tokens, found},
                         {"d_out", d_out, found},
                         {"d_lse", d_lse, rows * 4}};
    const Span in[2] = {{"d_scores", d_scores, rows * 4},
                        {"d_logits", d_logits, ((rows - 1) * row_stride + h->vocab) * esize}};
    for (int i = 0; i < 4; ++i) {
        for (int j = 0; j < i; ++j)
            if (overlap(out[i], out[j]))
                return fail(h, G4S_ERR_INVALID_ARGUMENT, "%s overlaps %s", out[i].name,
                            out[j].name);
        for (const Span& x : in)
            if (overlap(out[i], x) &&
                !(i == 2 && &x == &in[0] && d_out == d_scores && n_select == beams))
                return fail(h, G4S_ERR_INVALID_ARGUMENT,
                            "%s overlaps %s (d_out may be d_scores where n_select == beams)",
                            out[i].name, x.name);
    }
    DeviceGuard guard(h->device);
    if (!guard.ok()) return fail(h, G4S_ERR_HIP, "device %d cannot be made current", h->device);
    return select(h, d_logits, dtype, row_stride, batch, beams, d_scores, n_select, d_parents,
                  d_tokens, d_out, d_lse);
}

G4S_API int g4s_beam_reorder(g4s_beam* h, const void* d_src, void* d_dst, int64_t planes,
                             int64_t plane_stride, int32_t batch, int32_t beams,
                             int64_t row_stride, int64_t row_bytes, const int32_t* d_parents)
{
    if (!h) return fail(h, G4S_ERR_INVALID_ARGUMENT, "beam is NULL");
    h->err[0] = 0;
    const int rc = check_shape(h, batch, beams);
    if (rc) return rc;
    DeviceGuard guard(h->device);
    if (!guard.ok()) return fail(h, G4S_ERR_HIP, "device %d cannot be made current", h->device);
    return reorder(h, d_src, d_dst, planes, plane_stride, batch, beams, row_stride, row_bytes,
                   d_parents);
}

/* ------------------------------------------------------------------- pages */

G4S_API const char* g4s_pages_last_error(const g4s_pages* h)
{
    return h ? h->err : t_pages_error;
}

G4S_API int g4s_pages_create(g4s_pages** out, const g4s_page_geometry* geometry, void* hip_stream)
{
    g4s_pages* none = nullptr;
    t_pages_error[0] = 0;
    if (!out) return fail(none, G4S_ERR_INVALID_ARGUMENT, "out is NULL");
    *out = nullptr;
    if (!geometry) return fail(none, G4S_ERR_INVALID_ARGUMENT, "geometry is NULL");
    const g4s_page_geometry& g = *geometry;
    if (!g4s::geometry_ok(g))
        return fail(none, G4S_ERR_INVALID_ARGUMENT,
                    "page_tokens %d, n_pages %d, max_rows %d, max_slots %d, planes %d, parts %d, "
                    "token_bytes %lld, plane_stride %lld, page_stride %lld: outside the limits, "
                    "or pages overlap",
                    g.page_tokens, g.n_pages, g.max_rows, g.max_slots, g.planes, g.parts,
                    (long long)g.token_bytes, (long long)g.plane_stride, (long long)g.page_stride);
    int device = 0;
    const int rc = pick_device(none, &device);
    if (rc) return rc;
    g4s_pages* h = new (std::nothrow) g4s_pages();
    if (!h) return fail(none, G4S_ERR_OUT_OF_MEMORY, "host memory");
    h->device = device;
    h->stream = (hipStream_t)hip_stream;
    h->geo = g;
    h->words = (g.n_pages + 63) / 64;
    Carver c;
    auto lay = [&] {
        c.add(&h->ws.count, (size_t)g.n_pages);
        c.add(&h->ws.free, (size_t)h->words);
        c.add(&h->ws.before, (size_t)h->words + 1);
        c.add(&h->ws.jobs, (size_t)g.max_rows);
        c.add(&h->ws.steps, (size_t)g.max_rows * 3);
        c.add(&h->ws.plan, 1);
    };
    lay();
    const size_t bytes = c.used();
    if (hipMalloc(&h->memory, bytes) != hipSuccess) {
        (void)hipGetLastError();
        delete h;
        return fail(none, G4S_ERR_OUT_OF_MEMORY, "workspace of %zu bytes", bytes);
    }
    c.start(h->memory);
    lay();
    hipError_t e = g4s::pages_init_launch(h->ws, g.n_pages, h->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(h->stream);
    if (e != hipSuccess) {
        (void)hipFree(h->memory);
        delete h;
        return hip_fail(none, e, "workspace initialisation");
    }
    *out = h;
    return G4S_OK;
}

G4S_API int g4s_pages_destroy(g4s_pages* h)
{
    if (!h) return G4S_OK;
    DeviceGuard guard(h->device);
    (void)hipStreamSynchronize(h->stream);
    (void)hipFree(h->memory);
    delete h;
    return G4S_OK;
}

namespace {

/* Bytes from a pool's start to the end of its last page. */
int64_t pool_extent(const g4s_page_geometry& g)
{
    if (g.planes == 0) return 0;
    return (g.planes - 1) * g.plane_stride + (g.n_pages - 1) * g.page_stride +
           (int64_t)g.parts * g.page_tokens * g.token_bytes;
}

int check_states(g4s_pages* h, const g4s_page_state* from, const g4s_page_state* to, int32_t rows,
                 const int32_t* d_parents, const int32_t* d_grow, const void* d_pool,
                 const int32_t* d_status)
{
    if (!from || !to || !from->table || !from->lengths || !from->refs || !to->table ||
        !to->lengths || !to->refs || !d_status || (!d_pool && h->geo.planes > 0))
        return fail(h, G4S_ERR_INVALID_ARGUMENT,
                    "the states, their arrays, d_pool and d_status must be non-NULL");
    if (rows < 1 || rows > h->geo.max_rows)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "rows %d outside [1, %d]", rows,
                    h->geo.max_rows);
    const int64_t cells = (int64_t)h->geo.max_rows * h->geo.max_slots * 4;
    const int64_t lens = (int64_t)h->geo.max_rows * 4, refs = (int64_t)h->geo.n_pages * 4;
    const void* f[3] = {from->table, from->lengths, from->refs};
    const void* t[3] = {to->table, to->lengths, to->refs};
    const int64_t n[3] = {cells, lens, refs};
    for (int i = 0; i < 3; ++i)
        for (int j = 0; j < 3; ++j)
            if (overlap(f[i], n[i], t[j], n[j]))
                return fail(h, G4S_ERR_INVALID_ARGUMENT, "the two states share memory");
    /* what the call writes lies apart from all that it reads or writes besides */
    const Span out[5] = {{"to->table", to->table, cells},
                         {"to->lengths", to->lengths, lens},
                         {"to->refs", to->refs, refs},
                         {"d_status", d_status, 16},
                         {"d_pool", d_pool, pool_extent(h->geo)}};
    const Span in[5] = {{"from->table", from->table, cells},
                        {"from->lengths", from->lengths, lens},
                        {"from->refs", from->refs, refs},
                        {"d_parents", d_parents, (int64_t)rows * 4},
                        {"d_grow", d_grow, (int64_t)rows * 4}};
    for (int i = 0; i < 5; ++i) {
        for (int j = 0; j < i; ++j)
            if (overlap(out[i], out[j]))
                return fail(h, G4S_ERR_INVALID_ARGUMENT, "%s overlaps %s", out[i].name,
                            out[j].name);
        for (const Span& x : in)
            if (overlap(out[i], x))
                return fail(h, G4S_ERR_INVALID_ARGUMENT, "%s overlaps %s", out[i].name, x.name);
    }
    return G4S_OK;
}

g4s::PagesArgs pages_args(g4s_pages* h, const g4s_page_state* from, const g4s_page_state* to,
                          int32_t rows, void* d_pool, int32_t* d_status)
{
    g4s::PagesArgs a{};
    a.geo = h->geo;
    a.from = *from;
    a.to = *to;
    a.from_rows = rows;
    a.rows = rows;
    a.pool = (char*)d_pool;
    a.status = d_status;
    a.words = h->words;
    a.ws = h->ws;
    return a;
}

}  // namespace

G4S_API int g4s_pages_advance(g4s_pages* h, const g4s_page_state* from, int32_t from_rows,
                              const g4s_page_state* to, int32_t rows, const int32_t* d_parents,
                              const int32_t* d_grow, void* d_pool, int32_t* d_status)
{
    if (!h) return fail(h, G4S_ERR_INVALID_ARGUMENT, "pages is NULL");
    h->err[0] = 0;
    const int rc = check_states(h, from, to, rows, d_parents, d_grow, d_pool, d_status);
    if (rc) return rc;
    if (!d_parents) return fail(h, G4S_ERR_INVALID_ARGUMENT, "d_parents is NULL");
    if (from_rows < 1 || from_rows > h->geo.max_rows)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "from_rows %d outside [1, %d]", from_rows,
                    h->geo.max_rows);
    DeviceGuard guard(h->device);
    if (!guard.ok()) return fail(h, G4S_ERR_HIP, "device %d cannot be made current", h->device);
    g4s::PagesArgs a = pages_args(h, from, to, rows, d_pool, d_status);
    a.from_rows = from_rows;
    a.parents = d_parents;
    a.grow = d_grow;
    const hipError_t e = g4s::pages_advance_launch(a, h->stream);
    return e == hipSuccess ? G4S_OK : hip_fail(h, e, "page step launch");
}

G4S_API int g4s_pages_compact(g4s_pages* h, const g4s_page_state* from, const g4s_page_state* to,
                              int32_t rows, void* d_pool, int32_t* d_status)
{
    if (!h) return fail(h, G4S_ERR_INVALID_ARGUMENT, "pages is NULL");
    h->err[0] = 0;
    const int rc = check_states(h, from, to, rows, nullptr, nullptr, d_pool, d_status);
    if (rc) return rc;
    DeviceGuard guard(h->device);
    if (!guard.ok()) return fail(h, G4S_ERR_HIP, "device %d cannot be made current", h->device);
    const hipError_t e =
        g4s::pages_compact_launch(pages_args(h, from, to, rows, d_pool, d_status), h->stream);
    return e == hipSuccess ? G4S_OK : hip_fail(h, e, "page compaction launch");
}

G4S_API int g4s_pages_copy(g4s_pages* h, const void* d_src_pool, void* d_dst_pool, int32_t n,
                           const int32_t* d_src_pages, const int32_t* d_dst_pages,
                           const int32_t* d_tokens)
{
    if (!h) return fail(h, G4S_ERR_INVALID_ARGUMENT, "pages is NULL");
    h->err[0] = 0;
    if (n < 0) return fail(h, G4S_ERR_INVALID_ARGUMENT, "n %d below 0", n);
    if (n == 0 || h->geo.planes == 0) return G4S_OK;
    if (!d_src_pool || !d_dst_pool || !d_src_pages || !d_dst_pages)
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "pools and page lists must be non-NULL");
    const g4s_page_geometry& g = h->geo;
    const int64_t extent = pool_extent(g);
    if (d_src_pool != d_dst_pool && overlap(d_src_pool, extent, d_dst_pool, extent))
        return fail(h, G4S_ERR_INVALID_ARGUMENT, "the two pools overlap");
    for (const int32_t* list : {d_src_pages, d_dst_pages, d_tokens})
        if (list && overlap(list, (int64_t)n * 4, d_dst_pool, extent))
            return fail(h, G4S_ERR_INVALID_ARGUMENT, "a page list overlaps d_dst_pool");
    DeviceGuard guard(h->device);
    if (!guard.ok()) return fail(h, G4S_ERR_HIP, "device %d cannot be made current", h->device);
    const hipError_t e =
        g4s::pages_copy_launch(g, (const char*)d_src_pool, (char*)d_dst_pool, n, d_src_pages,
                               d_dst_pages, d_tokens, h->stream);
    return e == hipSuccess ? G4S_OK : hip_fail(h, e, "page copy launch");
}

/* -------------------------------------------------------------------- loop */

namespace {

bool is_end(int32_t t)
{
    return t == G4S_EOS_TOKEN_1 || t == G4S_EOS_TOKEN_2 || t == G4S_EOS_TOKEN_3;
}

/* Device and pinned memory of one g4s_beam_generate call; nothing of the call
 * is under way any more when they go. */
struct LoopMemory {
    hipStream_t stream;
    void* device = nullptr;
    void* host = nullptr;
    explicit LoopMemory(hipStream_t s) : stream(s) {}
    ~LoopMemory()
    {
        (void)hipStreamSynchronize(stream);
        if (device) (void)hipFree(device);
        if (host) (void)hipHostFree(host);
    }
};

struct LoopArrays {
    /* selected candidates [batch * 2 * beams] */
    int32_t *parents, *tokens;
    float* scores;
    /* the step taken [batch * beams] */
    int32_t *step_parents, *step_tokens, *grow;
    float* running;
    int32_t* status; /* [4] */
    void lay(Carver& c, size_t rows)
    {
        c.add(&parents, 2 * rows);
        c.add(&tokens, 2 * rows);
        c.add(&scores, 2 * rows);
        c.add(&status, 4);
        c.add(&step_parents, rows);
        c.add(&step_tokens, rows);
        c.add(&grow, rows);
        c.add(&running, rows);
    }
};

/* One generated token and the one before it.  Indices in 64 bits: 65,535 rows
 * make 2^31 nodes in 32,768 steps. */
struct Node {
    int32_t token;
    int64_t before; /* -1 = the prompt */
};

struct Result {
    float score; /* with the length penalty */
    int64_t last;
    int32_t length;
};

float penalised(float score, int32_t length, float penalty)
{
    return (float)((double)score / std::pow((double)length, (double)penalty));
}

int generate(g4s_beam* h, int32_t batch, const g4s_beam_config& cfg, const void* d_logits,
             int32_t dtype, int64_t row_stride, const g4s_beam_states* states,
             const g4s_beam_cache* cache, g4s_beam_forward_fn forward, void* user,
             int32_t* tokens, int32_t* lengths, float* scores)
{
    const int32_t W = cfg.beams, rows = batch * W, n = 2 * W;
    const float none = -std::numeric_limits<float>::infinity();
    LoopMemory mem(h->stream);
    LoopArrays d{}, p{};
    Carver c;
    d.lay(c, (size_t)rows);
    const size_t bytes = c.used();
    if (hipMalloc(&mem.device, bytes) != hipSuccess ||
        hipHostMalloc(&mem.host, bytes, hipHostMallocDefault) != hipSuccess) {
        (void)hipGetLastError();
        return fail(h, G4S_ERR_OUT_OF_MEMORY, "loop buffers of %zu bytes", bytes);
    }
    c.start(mem.device);
    d.lay(c, (size_t)rows);
    c.start(mem.host);
    p.lay(c, (size_t)rows);
    const size_t found_bytes = (char*)p.status - (char*)p.parents;
    const size_t step_bytes = bytes - ((char*)p.step_parents - (char*)p.parents);

    std::vector<Node> nodes;
    std::vector<int64_t> at((size_t)rows, -1), next((size_t)rows, -1); /* rows' last nodes */
    std::vector<std::vector<Result>> results((size_t)batch);
    std::vector<uint8_t> done((size_t)batch, 0);
    for (int32_t r = 0; r < rows; ++r) {
        p.running[r] = r % W == 0 ? 0.0f : none;
        p.step_parents[r] = p.step_tokens[r] = -1;
        p.grow[r] = 0;
    }
    hipError_t e = hipMemcpyAsync(d.step_parents, p.step_parents, step_bytes,
                                  hipMemcpyHostToDevice, h->stream);
    if (e != hipSuccess) return hip_fail(h, e, "upload of the first scores");
    int32_t current = 0;
    auto add = [&](int32_t b, float score, int64_t last, int32_t length) {
        auto& rs = results[(size_t)b];
        const Result r{penalised(score, length, cfg.length_penalty), last, length};
        auto it = std::find_if(rs.begin(), rs.end(),
                               [&](const Result& o) { return r.score > o.score; });
        rs.insert(it, r);
        if ((int32_t)rs.size() > W) rs.pop_back();
    };
    for (int32_t length = 1;; ++length) {
        int rc = select(h, d_logits, dtype, row_stride, batch, W, d.running, n, d.parents,
                        d.tokens, d.scores, nullptr);
        if (rc) return rc;
        e = hipMemcpyAsync(p.parents, d.parents, found_bytes, hipMemcpyDeviceToHost, h->stream);
        if (e == hipSuccess) e = hipStreamSynchronize(h->stream);
        if (e != hipSuccess) return hip_fail(h, e, "selected candidates");
        bool any = false;
        for (int32_t b = 0; b < batch; ++b) {
            int32_t go = 0;
            for (int32_t w = 0; w < W; ++w) {
                const int32_t r = b * W + w;
                p.step_parents[r] = p.step_tokens[r] = -1;
                p.grow[r] = 0;
                p.running[r] = none;
                next[(size_t)r] = -1;
            }
            if (done[(size_t)b]) continue;
            for (int32_t i = 0; i < n && go < W; ++i) {
                const int32_t parent = p.parents[b * n + i], token = p.tokens[b * n + i];
                if (parent < 0) break;
                const float score = p.scores[b * n + i];
                if (is_end(token)) {
                    if (i >= W) continue;
                    nodes.push_back({token, at[(size_t)parent]});
                    add(b, score, (int64_t)nodes.size() - 1, length);
                    continue;
                }
                const int32_t r = b * W + go++;
                nodes.push_back({token, at[(size_t)parent]});
                next[(size_t)r] = (int64_t)nodes.size() - 1;
                p.step_parents[r] = parent;
                p.step_tokens[r] = token;
                p.grow[r] = 1;
                p.running[r] = score;
            }
            const auto& rs = results[(size_t)b];
            bool end = go == 0 || length == cfg.max_tokens;
            if (!end && (int32_t)rs.size() >= W)
                end = cfg.early_stop != 0 ||
                      rs.back().score >= penalised(p.running[b * W], length, cfg.length_penalty);
            if (end) {
                for (int32_t w = 0; w < go; ++w) {
                    const int32_t r = b * W + w;
                    if (length == cfg.max_tokens) add(b, p.running[r], next[(size_t)r], length);
                    p.step_parents[r] = p.step_tokens[r] = -1;
                    p.grow[r] = 0;
                    p.running[r] = none;
                }
                done[(size_t)b] = 1;
            } else {
                any = true;
            }
        }
        if (!any) break;
        at.swap(next);
        e = hipMemcpyAsync(d.step_parents, p.step_parents, step_bytes, hipMemcpyHostToDevice,
                           h->stream);
        if (e != hipSuccess) return hip_fail(h, e, "upload of the step");
        if (states) {
            rc = reorder(h, states->d_state, states->d_state, states->planes,
                         states->plane_stride, batch, W, states->row_stride, states->row_bytes,
                         d.step_parents);
            if (rc) return rc;
        }
        if (cache) {
            rc = g4s_pages_advance(cache->pages, &cache->states[current], rows,
                                   &cache->states[1 - current], rows, d.step_parents, d.grow,
                                   cache->d_pool, d.status);
            if (rc) return fail(h, rc, "pages: %s", cache->pages->err);
            e = hipMemcpyAsync(p.status, d.status, 4 * sizeof(int32_t), hipMemcpyDeviceToHost,
                               h->stream);
            if (e == hipSuccess) e = hipStreamSynchronize(h->stream);
            if (e != hipSuccess) return hip_fail(h, e, "page step");
            if (p.status[0] != G4S_OK)
                return fail(h, p.status[0], "page step of token %d: %s", length,
                            p.status[0] == G4S_ERR_OUT_OF_MEMORY ? "too few free pages"
                            : p.status[0] == G4S_ERR_FORMAT      ? "a page outside the pool"
                                                                 : "a length beyond max_slots");
            current = 1 - current;
        }
        const g4s_beam_step step{p.step_tokens, p.step_parents, d.step_tokens,
                                 d.step_parents, rows,          current};
        const int refused = forward(user, &step);
        /* it may have left another device current, whose null stream is not ours */
        e = hipSetDevice(h->device);
        if (e != hipSuccess) return hip_fail(h, e, "the search's device behind the forward call");
        if (refused != 0)
            return fail(h, G4S_ERR_ABORTED, "the forward callback failed");
    }
    for (int32_t b = 0; b < batch; ++b)
        for (int32_t k = 0; k < cfg.n_best; ++k) {
            const size_t o = (size_t)b * cfg.n_best + k;
            const bool have = k < (int32_t)results[(size_t)b].size();
            lengths[o] = have ? results[(size_t)b][(size_t)k].length : 0;
            scores[o] = have ? results[(size_t)b][(size_t)k].score : none;
            int32_t i = lengths[o];
            for (int64_t node = have ? results[(size_t)b][(size_t)k].last : -1; node >= 0;
                 node = nodes[(size_t)node].before)
                tokens[o * (size_t)cfg.max_tokens + (size_t)--i] = nodes[(size_t)node].token;
        }
    return G4S_OK;
}

}  // namespace

G4S_API int g4s_beam_generate(g4s_beam* h, int32_t batch, const g4s_beam_config* config,
                              const void* d_logits, int32_t dtype, int64_t row_stride,
                              const g4s_beam_states* states, const g4s_beam_cache* cache,
                              g4s_beam_forward_fn forward, void* user, int32_t* tokens,
                              int32_t* lengths, float* scores)
{
    if (!h) return fail(h, G4S_ERR_INVALID_ARGUMENT, "beam is NULL");
    h->err[0] = 0;
    if (!config || !forward || !tokens || !lengths || !scores)
        return fail(h, G4S_ERR_INVALID_ARGUMENT,
                    "config, forward, tokens, lengths and scores must be non-NULL");
    int rc = check_shape(h, batch, config->beams);
    if (!rc) rc = check_logits(h, d_logits, dtype, row_stride, (int64_t)batch * config->beams);
    if (rc) return rc;
    if (config->max_tokens < 1 || config->n_best < 1 || config->n_best > config->beams ||
        !std::isfinite(config->length_penalty))
        return fail(h, G4S_ERR_INVALID_ARGUMENT,
                    "max_tokens %d / n_best %d / length_penalty %g", config->max_tokens,
                    config->n_best, config->length_penalty);
    if (cache) {
        if (!cache->pages) return fail(h, G4S_ERR_INVALID_ARGUMENT, "cache->pages is NULL");
        if (cache->pages->stream != h->stream || cache->pages->device != h->device)
            return fail(h, G4S_ERR_INVALID_ARGUMENT,
                        "the page cache is on another stream or device than the search");
    }
    DeviceGuard guard(h->device);
    if (!guard.ok()) return fail(h, G4S_ERR_HIP, "device %d cannot be made current", h->device);
    try {
        rc = generate(h, batch, *config, d_logits, dtype, row_stride, states, cache, forward, user,
                      tokens, lengths, scores);
    } catch (const std::bad_alloc&) {
        rc = fail(h, G4S_ERR_OUT_OF_MEMORY, "host memory");
    }
    return rc;
}
