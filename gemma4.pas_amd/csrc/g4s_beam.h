/*
 * g4s_beam.h -- launch interface of the beam search kernels (g4s_beam.hip).
 */
#ifndef G4S_BEAM_H
#define G4S_BEAM_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gemma4_beam.h"

namespace g4s {

constexpr int kBeamTile = 4096;       /* logits that a workgroup takes at once */
constexpr int kBeamTableTile = 16384; /* and one that looks its terms up */
constexpr int kBeamMaxVocab = 1 << 22;
constexpr int kBeamMaxTiles = kBeamMaxVocab / kBeamTile; /* of a row */

/* The softcap in the form that the kernels evaluate, in units of log2:
 *   v(x) = log2(e) * cap * tanh(x / cap)
 * as x * (q[0] + q[1] x^2 + ... + q[9] x^18) where |x| <= limit. */
struct BeamSoftcap {
    float cap;
    int32_t mode;
    float limit; /* of the way without a reference: 2^v is a normal binary32 there */
    double q[10];
};
constexpr int kCapNone = 0;  /* v(x) = log2(e) * x */
constexpr int kCapPoly = 1;
constexpr int kCapExact = 2; /* a cap beyond the polynomial's accuracy or binary32's range */

/* 2^v(x) of the bf16 values with 2^-24 <= |x| < 64 (first entry: below), by magnitude bits, the
 * negative ones behind the others. */
constexpr int kBeamTableLow = 0x3380;
constexpr int kBeamTableHigh = 0x4280;
constexpr int kBeamTableHalf = kBeamTableHigh - kBeamTableLow;

/* Workspace of a search: the chunks' best candidates, then the rows'.
 * An entry is a candidate's key (cand_key) over the complement of its token,
 * so that the larger entry is the better candidate; 0 = none. */
struct BeamWorkspace {
    uint64_t* cand;    /* [rows][chunks][n]  each chunk's, best first */
    uint64_t* sums;    /* [rows][chunks][2]  binary64: sum of 2^(v(x) - ref), and ref */
    uint64_t* best;    /* [rows][n] */
    uint64_t* y;       /* [rows][n]  binary64: their softcapped logits */
    uint64_t* norm;    /* [rows][2]  binary64: largest y, log of the sum relative to it */
    uint32_t* tickets; /* [rows + batch]  0 between calls */
    float* table;      /* [2 * kBeamTableHalf] */
};

struct BeamSelectArgs {
    const void* logits;
    int64_t row_stride;
    int32_t vocab;
    int32_t batch;
    int32_t beams;
    int32_t n;
    int32_t chunks; /* workgroups of a row, */
    int32_t tiles;  /* each with so many tiles */
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

/* How a row is split: how many workgroups, each with how many tiles. */
struct BeamPlan {
    int32_t chunks;
    int32_t tiles;
    bool table;
};
BeamPlan beam_plan(int32_t vocab, int32_t rows, int32_t dtype, int32_t mode, int32_t ncu);
/* Most chunks of a call with at most `rows` rows, times its rows. */
int64_t beam_max_chunks(int32_t vocab, int32_t rows, int32_t ncu);

BeamSoftcap beam_softcap(float cap);

hipError_t beam_init_launch(const BeamWorkspace& ws, const BeamSoftcap& cap, int32_t tickets,
                            hipStream_t stream);
hipError_t beam_select_launch(const BeamSelectArgs& a, const BeamPlan& plan, int32_t dtype,
                              hipStream_t stream);
hipError_t beam_reorder_launch(const BeamReorderArgs& a, hipStream_t stream);

}  // namespace g4s

#endif
