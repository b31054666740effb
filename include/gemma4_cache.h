/*
 * gemma4_cache.h -- keys and values in 8 bits in the pages of a cache that
 * rows share (gemma4_beam.h), on MI355X gfx950 (libgemma4_sampler.so): the
 * append, with the position rotation on the way, and the attention that reads
 * them, for single tokens and for prompts.
 *
 * g4s_pages_advance makes room for a step's tokens; g4s_cache_append writes
 * their keys and values there, layer by layer, and g4s_cache_attend attends
 * over what the rows then hold.  In the engine's decoder layer they stand for its
 * rotation, its append to the cache and its attention (the rope, kv_append
 * and attn_* kernels of shaders/src).
 *
 * Conventions are those of gemma4_beam.h: 0 or a negative g4s_status, the
 * message of the last failure kept per handle (with a NULL handle that of the
 * thread's last failed call without one), one handle = one HIP stream, a
 * handle is not thread-safe, device pointers are memory of the handle's device
 * (which need not be the current one), those of integers and floats 4-byte aligned.  Only g4s_cache_create allocates;
 * append and attend are kernel launches alone and may be captured into a
 * hipGraph.  A graph that attends uses its handle's workspace: it is
 * replayed on one stream at a time with the handle's other calls.
 */
#ifndef GEMMA4_CACHE_H
#define GEMMA4_CACHE_H

#include "gemma4_beam.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Most heads of queries and of keys, query heads of one key head, dims of a head, tokens that
 * share a scale, tokens of a call, and tokens that a row has slots for. */
#define G4S_CACHE_MAX_HEADS 512
#define G4S_CACHE_MAX_KV_HEADS 64
#define G4S_CACHE_MAX_GROUP 64
#define G4S_CACHE_MAX_HEAD_DIM 512
#define G4S_CACHE_MAX_SCALE_TOKENS 256
#define G4S_CACHE_MAX_TOKENS 1048576
#define G4S_CACHE_MAX_CONTEXT 1073741824

/* Which dims of a head the rotation pairs, j = 0 .. rotary_dims / 2 - 1. */
#define G4S_ROTARY_HALVES 0     /* j and j + rotary_dims / 2 */
#define G4S_ROTARY_NEIGHBOURS 1 /* 2 j and 2 j + 1 */

typedef struct g4s_cache g4s_cache;

/* What a token of one kv head holds in a plane: head_dim e4m3 codes (OCP, no
 * infinities, 0x7F and 0xFF NaN) and a binary32 scale behind them.  scale_tokens
 * tokens of a page, from its first on, share a scale: the one that stands behind
 * the first of them.  Those of the others have no meaning.  A scale is a
 * power of two, and a code stands for its value times the scale.  So the
 * geometry has parts = kv_heads, token_bytes = head_dim + 4, page_tokens a
 * multiple of scale_tokens, strides that are multiples of 4, and the keys and
 * the values of a layer in a plane each; page copies of any count of tokens
 * (g4s_pages_advance, _copy) carry their scales along. */
typedef struct g4s_cache_config {
    int32_t heads;        /* of queries, a multiple of kv_heads */
    int32_t kv_heads;
    int32_t head_dim;     /* 16 .. 512, a multiple of 16 */
    int32_t scale_tokens;
    int32_t rotary_dims;  /* 0 .. head_dim, even: the leading dims that are rotated */
    int32_t rotary_pairs; /* G4S_ROTARY_* */
} g4s_cache_config;

/* Vectors of head_dim consecutive elements for tokens and heads: head h of
 * token i at data + i * token_stride + h * head_stride elements.  Data and
 * strides (in bytes) are multiples of 16. */
typedef struct g4s_cache_view {
    void* data;
    int64_t token_stride;
    int64_t head_stride;
} g4s_cache_view;

/* A cache of this geometry (max_rows, max_slots, n_pages as in its
 * g4s_pages).  Allocates the workspace. */
int g4s_cache_create(g4s_cache** out, const g4s_page_geometry* geometry,
                     const g4s_cache_config* config, void* hip_stream);

/* Release the handle and its workspace.  NULL is accepted. */
int g4s_cache_destroy(g4s_cache* cache);

const char* g4s_cache_last_error(const g4s_cache* cache);

/* The new tokens of each row into its pages, and their queries rotated.
 * The tokens are the last that the rows hold: `state` has room for them already.
 *   rows       rows of the state, 1 .. max_rows
 *   d_starts   device [rows + 1]: tokens d_starts[r] .. d_starts[r+1] - 1 are row
 *              r's, ascending within 0 .. tokens; NULL: token r is row r's
 *              (tokens == rows)
 *   tokens     tokens of the views; those that no row has are left alone
 *   dtype      of q, k, v and q_out (G4S_DTYPE_F32 or G4S_DTYPE_BF16)
 *   q, q_out   queries and where they go rotated, both or neither; q_out may
 *              be q, with the same strides
 *   k, v       keys and values, both or neither (a layer that reads another's cache)
 *   d_positions  device [tokens], or NULL: a token's place in its row (0, 1, ..)
 *   d_freqs    device [rotary_dims / 2] radians per position (NULL if rotary_dims == 0)
 *   d_pool, k_plane, v_plane   the pool and the layer's planes, which differ
 * Token i of a row with n new tokens and `length` tokens has place length - n + i; one
 * whose place is negative (a row that has ended) is left out, its query too, and
 * so is every token of a row whose length is outside the table.
 *   angle(j) = position * d_freqs[j]
 *   (a, b) -> (a cos - b sin, b cos + a sin)     for each pair (a, b) of q and k
 * in 64 bits, rounded to q_out's type (to bf16 by way of binary32).  Keys and values: with top the
 * largest finite magnitude that is new in a block of scale_tokens tokens of one head, the
 * scale is the least power of two with top <= 448 * scale, from 2^-100 to
 * 2^119, or the one that the block has if it holds earlier tokens and theirs is
 * larger.  A code is the e4m3 value nearest to x / scale (ties to even;
 * infinities and what is larger give +-448, NaN gives NaN), and earlier tokens' codes in
 * the block are brought to a scale that grew.  Angles are below 2^40.
 * Tokens whose page lies outside the pool are not stored.  A page that a row's new
 * tokens lie in is held by no other row (g4s_pages_advance sees to that).
 * Outputs that overlap another array of the call are refused.  Stream-ordered. */
int g4s_cache_append(g4s_cache* cache, const g4s_page_state* state, int32_t rows,
                     const int32_t* d_starts, int32_t tokens, int32_t dtype,
                     const g4s_cache_view* q, const g4s_cache_view* k, const g4s_cache_view* v,
                     const g4s_cache_view* q_out, const int32_t* d_positions,
                     const float* d_freqs, void* d_pool, int32_t k_plane, int32_t v_plane);

/* Each row's queries over the tokens that it holds.  Query i of a row with n
 * queries and `length` tokens stands at place t = length - n + i and sees the
 * places 0 .. t, with window > 0 those above t - window alone; head h reads kv
 * head h / (heads / kv_heads):
 *   s(j) = scale * dot(q, key(j))
 *   lse = log(sum of exp(s(j)))      out = sum of exp(s(j) - lse) * value(j)
 * Sums and exponentials in 32 bits.  For bf16 outputs the weights exp(s) are off by
 * 2^-16 at most where they meet the values; those of fp32 outputs, keys, values and queries
 * are not rounded.
 *   rows, d_starts, tokens, dtype   as for g4s_cache_append (q and out)
 *   scale      within +-2^127
 *   d_lse      device [tokens * heads], or NULL
 * A query that sees nothing (a row that has ended) gets zeros and -inf.  A
 * query that is not finite, one that sees a NaN among the keys, a page outside the
 * pool, or a scale that is no number from 0 to 2^119, gets NaN, and so does every query of a row whose
 * length is outside the table; a NaN among the values gives one in its dim.  What a query does not see does not count, whatever it is.  Queries that no
 * row has are left alone.  An output that overlaps another array of the call is
 * refused.  Stream-ordered; the same call gives the same bits. */
int g4s_cache_attend(g4s_cache* cache, const g4s_page_state* state, int32_t rows,
                     const int32_t* d_starts, int32_t tokens, int32_t dtype,
                     const g4s_cache_view* q, const void* d_pool, int32_t k_plane,
                     int32_t v_plane, float scale, int32_t window, const g4s_cache_view* out,
                     float* d_lse);

#ifdef __cplusplus
}
#endif
#endif
