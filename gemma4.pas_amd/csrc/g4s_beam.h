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

/* A chunk's part of the softmax denominator: sum of exp(y - top). */
struct BeamPart {
    double top; /* largest y of the chunk (-inf: no candidate) */
    double sum;
};

/* Workspace of a search: the chunks' best candidates, then the rows'.
 * An entry is a candidate's key (cand_key) over the complement of its token,
 * so that the larger entry is the better candidate; 0 = none. */
struct BeamWorkspace {
    uint64_t* cand;     /* [rows][chunks][n_max] */
    BeamPart* parts;    /* [rows][chunks] */
    uint64_t* best;     /* [rows][n_max] */
    double* y;          /* [rows][n_max]  their softcapped logits */
    double* norm;       /* [rows][2]  largest y, log of the sum relative to it */
};

struct BeamSelectArgs {
    const void* logits;
    int64_t row_stride;
    int32_t vocab;
    int32_t batch;
    int32_t beams;
    int32_t n;
    int32_t chunks;
    float softcap;
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

hipError_t beam_select_launch(const BeamSelectArgs& a, int32_t dtype, hipStream_t stream);
hipError_t beam_reorder_launch(const BeamReorderArgs& a, hipStream_t stream);

}  // namespace g4s

#endif
