/*
 * g4s_beam.h -- launch interface of the beam search kernels (g4s_beam.hip).
 */
#ifndef G4S_BEAM_H
#define G4S_BEAM_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gemma4_beam.h"

namespace g4s {

constexpr int kBeamBlock = 256;
constexpr int kBeamItems = 32;                        /* logits per thread of a chunk */
constexpr int kBeamChunk = kBeamBlock * kBeamItems;   /* logits per workgroup */
constexpr int kBeamMaxVocab = 1 << 22;

/* The softcap in the form that the kernels evaluate, in units of log2:
 *   v(x) = log2(e) * cap * tanh(x / cap)
 * as x * (q[0] + q[1] x^2 + ... + q[9] x^18) where |x| <= limit. */
struct BeamSoftcap {
    float cap;
    int32_t mode;
    float limit;
    double q[10];
};
constexpr int kCapNone = 0;  /* v(x) = log2(e) * x */
constexpr int kCapPoly = 1;
constexpr int kCapExact = 2; /* a cap beyond the polynomial's accuracy */

/* Workspace of a search: the chunks' best candidates, then the rows'.
 * An entry is a candidate's key (cand_key) over the complement of its token,
 * so that the larger entry is the better candidate; 0 = none. */
struct BeamWorkspace {
    uint64_t* cand;    /* [rows][chunks][n]  each chunk's, best first */
    uint64_t* sums;    /* [rows][chunks]  binary64: sum of 2^(v(x) - v(largest x)) */
    uint64_t* best;    /* [rows][n] */
    uint64_t* y;       /* [rows][n]  binary64: their softcapped logits */
    uint64_t* norm;    /* [rows][2]  binary64: largest y, log of the sum relative to it */
    uint32_t* tickets; /* [rows + batch]  0 between calls */
};

struct BeamSelectArgs {
    const void* logits;
    int64_t row_stride;
    int32_t vocab;
    int32_t batch;
    int32_t beams;
    int32_t n;
    int32_t chunks;
    BeamSoftcap cap;
    const float* scores;
    int32_t* parents;
    int32_t* tokens;
    float* out;
    float* lse;
    BeamWorkspace ws;
};

struct BeamReorderArgs {
    const char* src;
    char* dst;
    int64_t planes;
    int64_t plane_stride;
    int32_t batch;
    int32_t beams;
    int64_t row_stride;
    int64_t row_bytes;
    const int32_t* parents;
};

inline int32_t beam_chunks(int32_t vocab) { return (vocab + kBeamChunk - 1) / kBeamChunk; }

BeamSoftcap beam_softcap(float cap);

hipError_t beam_select_launch(const BeamSelectArgs& a, int32_t dtype, hipStream_t stream);
hipError_t beam_reorder_launch(const BeamReorderArgs& a, hipStream_t stream);

}  // namespace g4s

#endif
