/*
 * gemma4_beam.h -- beam search over device-resident logits, and the cache
 * pages its beams live in (libgemma4_sampler.so, MI355X gfx950).
 *
 * Beside the samplers of gemma4_sampler.h: where TModel.Generate draws one
 * token (src/Gemma4.Model.pas:2829-2938), a search keeps `beams` token strings
 * per sequence, takes the best continuations of all of them in each step, and
 * makes every beam's state follow the beam it goes on from.  The reference
 * has no search; the softcap, the rule of which logits count and the end
 * tokens are its samplers'.
 *
 * Conventions are those of gemma4_sampler.h: 0 or a negative g4s_status, the
 * message of the last failure kept per handle, one handle = one HIP stream, a
 * handle is not thread-safe, device pointers are memory of the handle's device
 * (which need not be the current one).  A NULL handle gives the message of the
 * thread's last failed call without one.  No call but the two creates and
 * g4s_beam_generate allocates; the stream-ordered calls consist of kernel
 * launches alone and may be captured into a hipGraph.  Such a graph uses its
 * handle's workspace: it is replayed on one stream at a time with the
 * handle's other calls.
 */
#ifndef GEMMA4_BEAM_H
#define GEMMA4_BEAM_H

#include "gemma4_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Most beams of a sequence, rows (beams of all sequences) of a call, and
 * rows and pages of a page cache. */
#define G4S_BEAM_MAX_BEAMS 64
#define G4S_BEAM_MAX_ROWS 65535
#define G4S_PAGES_MAX_ROWS 2048
#define G4S_PAGES_MAX_PAGES 1048576

/* ------------------------------------------------------------------ search */

typedef struct g4s_beam g4s_beam;

/* A search over `vocab` (2 .. 2^22) logits per row, up to max_batch sequences
 * of up to max_beams beams (their product at most G4S_BEAM_MAX_ROWS).
 * `softcap` as for g4s_create.  Allocates the whole workspace. */
int g4s_beam_create(g4s_beam** out, int32_t vocab, int32_t max_batch, int32_t max_beams,
                    float softcap, void* hip_stream);

/* Release the handle and its workspace.  NULL is accepted. */
int g4s_beam_destroy(g4s_beam* beam);

const char* g4s_beam_last_error(const g4s_beam* beam);

/* The best n_select continuations of each sequence's beams.  Row
 * r = sequence * beams + beam has logits x and a running score s; with
 *   y = softcap * tanh(x / softcap)   (x where softcap <= 0)
 *   lse(r) = log(sum over the row's tokens of exp(y))
 *   score(r, token) = s(r) + (y - lse(r))
 * they are taken by score, the largest first: y and the score in 64 bits, the
 * terms of lse in 32, added by fours in 32 and from there on in 64.  Equal
 * scores go to the lower beam, then to the larger logit, then to the lower
 * token.  A logit that is not above -1e30 (-inf, NaN, the type's lowest value:
 * the samplers' rule) is no candidate and counts nothing in the sum; a row
 * whose score is not above -1e30 is dead: it has no candidates and is not
 * read.
 *   d_logits, dtype, row_stride  as for g4s_sample, batch * beams rows
 *   d_scores   device [batch*beams]
 *   n_select   1 .. 2 * max_beams
 *   d_parents  device [batch*n_select]  row that is continued
 *   d_tokens   device [batch*n_select]  its next token
 *   d_out      device [batch*n_select]  score, rounded once to binary32;
 *              may be d_scores where n_select == beams
 *   d_lse      device [batch*beams] lse of each row, or NULL; -inf for a dead
 *              row and for one without candidates
 * Where a sequence has fewer candidates the rest is -1, -1, -inf.
 * An output that overlaps another array of the call, or the span of the
 * logits, is refused but for d_out == d_scores.
 * Stream-ordered.  The lse that scores are made from is off by less than
 * 2.6e-7 + 2^-49 |lse|, and d_lse is that value rounded once to binary32: scores of
 * different beams that lie closer than 5.2e-7 may come in either order. */
int g4s_beam_select(g4s_beam* beam, const void* d_logits, int32_t dtype, int64_t row_stride,
                    int32_t batch, int32_t beams, const float* d_scores, int32_t n_select,
                    int32_t* d_parents, int32_t* d_tokens, float* d_out, float* d_lse);

/* Contiguous states follow their parents: with row r of plane p at
 * p * plane_stride + r * row_stride bytes, each of the batch * beams rows of
 * d_dst becomes what row d_parents[r] of d_src holds (row_bytes of it).
 * d_dst == d_src moves the rows in place, whatever the parents' order.  A
 * parent of another sequence, or -1, leaves row r of d_dst as it is in place
 * and copies row r of d_src otherwise.  Bytes between rows are left alone.
 * d_src and d_dst are the same pointer or do not overlap, and d_parents lies
 * outside d_dst.  Any alignment; multiples of 16 bytes throughout and at most 16
 * beams are fastest.  Stream-ordered. */
int g4s_beam_reorder(g4s_beam* beam, const void* d_src, void* d_dst, int64_t planes,
                     int64_t plane_stride, int32_t batch, int32_t beams, int64_t row_stride,
                     int64_t row_bytes, const int32_t* d_parents);

/* ------------------------------------------------------------------- pages */

/* A paged cache: every row (a beam of a sequence) holds `length` tokens in
 * pages of page_tokens tokens, named by its row of a table; rows share pages.
 * The handle knows the geometry; the tables (states) and the pool of pages
 * are the caller's. */
typedef struct g4s_pages g4s_pages;

/* A page is `parts` blocks of page_tokens * token_bytes bytes behind each
 * other (one part: [token][...]; a part per head: [head][token][...]), once in
 * each plane (a layer's keys or values): page g of plane p starts at
 * p * plane_stride + g * page_stride bytes of the pool.  Planes may lie
 * outside the pages or the other way round, without overlap. */
typedef struct g4s_page_geometry {
    int32_t page_tokens; /* 1 .. 65536 */
    int32_t n_pages;     /* 1 .. G4S_PAGES_MAX_PAGES */
    int32_t max_rows;    /* 1 .. G4S_PAGES_MAX_ROWS */
    int32_t max_slots;   /* 1 .. G4S_PAGES_MAX_PAGES, pages of a row at most (at most 2^31 - 1
                            tokens); row stride of the tables */
    int32_t planes;
    int32_t parts;
    int64_t token_bytes; /* of a token in one part of one plane */
    int64_t plane_stride;
    int64_t page_stride;
} g4s_page_geometry;

/* The state of all rows, in device memory.
 *   table   [max_rows * max_slots]  page of each slot; a row of n tokens uses
 *           its first ceil(n / page_tokens) slots, what stands behind them
 *           has no meaning and is not written
 *   lengths [max_rows]              tokens
 *   refs    [n_pages]               rows that hold the page; 0 = free */
typedef struct g4s_page_state {
    int32_t* table;
    int32_t* lengths;
    int32_t* refs;
} g4s_page_state;

int g4s_pages_create(g4s_pages** out, const g4s_page_geometry* geometry, void* hip_stream);

/* Release the handle and its workspace.  NULL is accepted. */
int g4s_pages_destroy(g4s_pages* pages);

const char* g4s_pages_last_error(const g4s_pages* pages);

/* One step of the rows from state `from` (from_rows rows) to state `to`
 * (`rows` rows): row r of `to` is row d_parents[r] of `from`, d_grow[r] tokens
 * longer (shorter where negative, not below 0; d_grow NULL = 0).  Parent -1 is
 * a row without tokens; a row of `from` that is nobody's parent ends, and its
 * pages are free in `to` if no other row holds them.  So one call forks rows,
 * reorders beams, admits, truncates and ends sequences.  A row that grows goes on
 * writing its last page if that page is partly filled; where another row
 * holds the page too, its tokens are first copied into a free page (of rows
 * that all go on writing one page the first keeps it).  Pages come from those
 * that are free in `from`, the lowest first: rows in order, a row's copy
 * before its new slots.
 *   d_pool    the pool, for the copies; NULL if planes == 0
 *   d_status  device int32 [4]: G4S_OK or what went wrong, free pages of
 *             `to`, pages taken, pages copied
 * All or nothing: with too few free pages (G4S_ERR_OUT_OF_MEMORY), a length
 * beyond max_slots pages or a parent outside [-1, from_rows)
 * (G4S_ERR_INVALID_ARGUMENT), or a page outside the pool in a table
 * (G4S_ERR_FORMAT) `to` is left with empty rows and no page held, status
 * words 2 and 3 are 0, and the pool is not written.  `from` stays valid in any case
 * (its live pages are not written, so the call can be repeated from it); the
 * two states share no memory, and the arrays of `to`, the pool and d_status none
 * with each other or with any other array of the call.  Rows of `to` from `rows`
 * on are left alone.  Stream-ordered. */
int g4s_pages_advance(g4s_pages* pages, const g4s_page_state* from, int32_t from_rows,
                      const g4s_page_state* to, int32_t rows, const int32_t* d_parents,
                      const int32_t* d_grow, void* d_pool, int32_t* d_status);

/* The live pages moved together: with n pages held in `from`, the i-th live
 * page at n or above moves into the i-th free page below n, in the pool and
 * in the tables of `to`, which holds pages 0 .. n-1 alone.  Arguments, status
 * (word 2 is 0, word 3 the pages moved) and errors as for g4s_pages_advance;
 * `from` stays valid.  `rows` covers every row that holds pages: the tables of
 * rows behind them are left as they are, but the pages move. */
int g4s_pages_compact(g4s_pages* pages, const g4s_page_state* from, const g4s_page_state* to,
                      int32_t rows, void* d_pool, int32_t* d_status);

/* Page d_src_pages[i] of d_src_pool copied to page d_dst_pages[i] of d_dst_pool
 * (pools of this geometry, or the same pool), the first d_tokens[i] tokens of
 * each part (d_tokens NULL = whole pages; clamped to 0 .. page_tokens).  A
 * pair with a page outside [0, n_pages) is left out.  The destination pages differ
 * from each other, and within one pool from the source pages; the lists lie
 * outside the destination pool.  Stream-ordered. */
int g4s_pages_copy(g4s_pages* pages, const void* d_src_pool, void* d_dst_pool, int32_t n,
                   const int32_t* d_src_pages, const int32_t* d_dst_pages,
                   const int32_t* d_tokens);

/* -------------------------------------------------------------------- loop */

typedef struct g4s_beam_config {
    int32_t beams;        /* 1 .. max_beams */
    int32_t max_tokens;   /* of a result, its end token included */
    int32_t n_best;       /* 1 .. beams results per sequence */
    int32_t early_stop;   /* != 0: a sequence is done with its `beams`-th result;
                             0: when its best beam, at its present length, does
                             not beat the worst of `beams` results */
    float length_penalty; /* results compare by score / length^length_penalty */
} g4s_beam_config;

/* Contiguous states to be reordered in place (arguments of g4s_beam_reorder). */
typedef struct g4s_beam_states {
    void* d_state;
    int64_t planes;
    int64_t plane_stride;
    int64_t row_stride;
    int64_t row_bytes;
} g4s_beam_states;

/* A paged cache that follows the beams: before the first forward call
 * states[0] holds each sequence's prompt in row sequence * beams (its other
 * rows are empty), afterwards the two states take turns. */
typedef struct g4s_beam_cache {
    g4s_pages* pages; /* on the search's stream and device */
    g4s_page_state states[2];
    void* d_pool;
} g4s_beam_cache;

/* What the caller's model step gets: rows = batch * beams, tokens[r] the token
 * row r feeds next or -1 (no step), parents[r] the row of the last step it
 * goes on from or -1; on the host and on the device.  `state` is the page state
 * that is current: it has room for the new token. */
typedef struct g4s_beam_step {
    const int32_t* tokens;
    const int32_t* parents;
    const int32_t* d_tokens;
    const int32_t* d_parents;
    int32_t rows;
    int32_t state;
} g4s_beam_step;

/* The caller's model step: on return the raw logits of each row with a token
 * are in that row of the loop's logits buffer, written by work on the search's
 * stream or already complete.  It may leave another device current.  0 to go
 * on; anything else ends the loop with G4S_ERR_ABORTED. */
typedef int (*g4s_beam_forward_fn)(void* user, const g4s_beam_step* step);

/* Beam search for `batch` sequences at once.  Row sequence * beams of d_logits
 * holds the logits after the sequence's prompt.  In each step 2 * beams
 * candidates are selected; in their order, an end token (g4s_generate's) makes
 * a result if it is among the first `beams` and is passed over otherwise, any
 * other token goes on, until `beams` do.  Results are kept by
 * score / length^length_penalty, the best `beams`, the earlier before its
 * equals.  A sequence that reaches max_tokens adds its beams to its results.
 * `states` and `cache` (each may be NULL) follow the beams before `forward` is
 * called.
 * Outputs (host): tokens [batch*n_best*max_tokens], lengths [batch*n_best]
 * and scores [batch*n_best] (score / length^length_penalty), the best result
 * first; a missing result has length 0 and score -inf.  Synchronous. */
int g4s_beam_generate(g4s_beam* beam, int32_t batch, const g4s_beam_config* config,
                      const void* d_logits, int32_t dtype, int64_t row_stride,
                      const g4s_beam_states* states, const g4s_beam_cache* cache,
                      g4s_beam_forward_fn forward, void* user, int32_t* tokens, int32_t* lengths,
                      float* scores);

#ifdef __cplusplus
}
#endif
#endif
