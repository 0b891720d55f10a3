// Launch descriptors of the beam search's kernels: the selection over beams and vocabulary, and the reordering of what the beams keep.
#pragma once
#include "gq_kernels.h"

namespace gq {

constexpr int BEAM_MAX = 32;            // beams of a group
constexpr int BEAM_MAX_VOCAB = 1 << 20;

// Group g's beams are rows g * n_beam + b. Beam b's candidate v has the value score + x[v] - log sum e^x in 64 bits; the n_beam best of
// the group, in descending order, equal ones by lower b * n_vocab + v. A beam whose last token is eos has the one candidate eos, at
// its score. NaN logits and scores count as -inf, +inf logits as FP32's largest number.
struct BeamSelectArgs {
    const float * x;  // row r at x + r * stride
    long long stride;
    int n_vocab, n_group, n_beam, eos;
    const float * score;   // [rows]
    const int32_t * last;  // [rows] or NULL: no beam has ended
    float * score_out;     // [rows], may be score
    int32_t * token;       // [rows], may be last
    int32_t * parent;      // [rows], beams of the group
    void * work;
    int per;               // set at launch: logits a thread takes in the first kernel
    int chunks;            // set at launch: workgroups a row there
};
size_t beam_work(int n_group, int n_beam, int n_vocab);
hipError_t launch_beam_select(const BeamSelectArgs & a, hipStream_t s);

// What each beam keeps, moved along with it: row i of a group becomes a copy of row parent[i], in place. Of every part p of a row (at
// data + row * row_stride + p * part_stride) the bytes lo .. hi - 1 move; with used, hi is also at most the source row's
// ceil(used / unit_len) units.
struct BeamMove {
    uint8_t * data;
    unsigned long long row_stride, part_stride, lo, hi;
    const int32_t * used;
    uint32_t unit_bytes, unit_len;
    int used_stride;
    uint32_t tiles;  // workgroups of a part
    uint32_t end;    // workgroups of this array and those before it
    uint32_t wide;   // every address is a multiple of 16
};
constexpr int BEAM_MOVES = 24;      // arrays of one launch
constexpr uint32_t BEAM_TILE = 4096;  // bytes of a part that a workgroup moves
struct BeamReorderArgs {
    BeamMove m[BEAM_MOVES];
    const int32_t * parent;  // [n_group * n_beam], values outside 0 .. n_beam - 1: the row stays
    int n, n_group, n_beam;
};
hipError_t launch_beam_reorder(const BeamReorderArgs & a, hipStream_t s);

}  // namespace gq
