// Launch descriptors of the beam search's kernels: the selection over beams and vocabulary, and the reordering of what the beams keep.
#pragma once
#include "gq_kernels.h"

namespace gq {

constexpr int BEAM_MAX = 32;            // beams of a group
constexpr int BEAM_MAX_VOCAB = 1 << 20;

// Group g's beams are rows g * n_beam + b. Beam b's candidate v has the value score + x[v] - log sum e^x in 64 bits (the logarithm to
// within 6e-10: a polynomial's 1.1e-10 in each term, in each of three joins of sums, and in the logarithm itself); the n_beam best of
// the group, in descending order, equal ones by lower b * n_vocab + v. A beam whose last token is eos has the one candidate eos, at
// its score. NaN logits and scores count as -inf, +inf logits as FP32's largest number.
struct BeamSelectArgs {
    const float * x;  // row r at x + r * stride
    long long stride;
    int n_vocab, n_group, n_beam, eos;
    const float * score;   // row r's at score[r * slot], and so the others
    const int32_t * last;  // or NULL: no beam has ended
    float * score_out;     // may be score
    int32_t * token;       // may be last
    int32_t * parent;      // beams of the group
    int slot;
    // With pos: row r is at position pos[r * slot] of its prompt (n_prompt[r * slot] ids, at most cap, at prompt + r * cap). While the
    // group's first row's prompt has a next id, the group reads prompts: each row's next id is its token (none left: the token stays), the
    // row its own parent, the score stays; a beam has ended only behind its prompt.
    const int32_t * pos;
    const int32_t * n_prompt;
    const int32_t * prompt;
    int cap;
    void * work;
    int per;               // set at launch: logits a thread takes in the first kernel
    int chunks;            // set at launch: workgroups a row there
    unsigned chunk_mul;    // set at launch: list / chunks = the high word of list * chunk_mul (lists below 2^13); 0: one chunk
};

// Logits as words that order as their values do, > 0 for every number. Both zeros are one word: a wave counts its candidates by the
// words and takes them by the values, and equal logits go by their index.
__host__ __device__ inline uint32_t beam_order(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);  // (-0 + 0 is +0)
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__host__ __device__ inline float beam_number(uint32_t o) { return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o); }

constexpr int BEAM_SLACK = 4;  // lanes beyond n_beam that a bound may let pass (25.1, 25.2 and 25.6 us with 4, 8 and 16 at 8 groups of 8 of 151936)

// A bound on a wave's words, of which at_least(w) lanes' are w or more (0: none; low: the smallest, high: the largest): at least k of
// them are >= it, and no more than k + BEAM_SLACK if equal ones do not forbid that; with fewer than k words: 1. n: how many pass.
template <typename F>
__host__ __device__ inline uint32_t beam_bound(F at_least, int k, uint32_t low, uint32_t high, int & n) {
    uint32_t lo = 1, hi = high + 1;  // at least k (or all) are >= lo, fewer than k are >= hi
    n = at_least(1u);
    if (n <= k + BEAM_SLACK) return lo;
    if (low) lo = low;
    while (hi - lo > 1 && n > k + BEAM_SLACK) {
        const uint32_t mid = lo + (hi - lo) / 2;
        const int c = at_least(mid);
        if (c >= k) {
            lo = mid;
            n = c;
        } else {
            hi = mid;
        }
    }
    return lo;
}

// Entries of a wave's list of candidates, `per` logits a lane.
constexpr int beam_list(int n_beam, int per) { return (n_beam + BEAM_SLACK) * per; }

size_t beam_work(int n_group, int n_beam, int n_vocab);
hipError_t launch_beam_select(const BeamSelectArgs & a, hipStream_t s);

// What each beam keeps, moved along with it: row i of a group becomes a copy of row parent[i], in place. Of every part p of a row (at
// data + row * row_stride + p * part_stride) the bytes lo .. hi - 1 move; with used, hi is also at most the source row's
// ceil(used / unit_len) units.
struct BeamMove {  // hi: used[...] + used_more units of the source row
    uint8_t * data;
    unsigned long long row_stride, part_stride, lo, hi;
    const int32_t * used;
    uint32_t unit_bytes, unit_len;
    int used_stride, used_more;
    uint32_t tiles;  // workgroups of a part
    uint32_t end;    // workgroups of this array and those before it
    uint32_t wide;   // every address is a multiple of 16
};
constexpr int BEAM_MOVES = 24;      // arrays of one launch
constexpr uint32_t BEAM_TILE = 4096;  // bytes of a part that a workgroup moves
constexpr uint32_t BEAM_GRID = (1u << 24) - 1;  // workgroups of a launch: fewer than 2^32 threads
struct BeamReorderArgs {
    BeamMove m[BEAM_MOVES];
    const int32_t * parent;  // row r's at parent[r * parent_stride], values outside 0 .. n_beam - 1: the row stays
    int n, n_group, n_beam, parent_stride;
};
// Rows apart, and parts apart: all rows of a part before the next part, or all parts of a row before the next row (the sizes in any
// unit, below 2^46).
inline bool beam_rows_apart(uint64_t rows, uint64_t size, uint64_t row_stride, uint64_t part_stride, uint64_t n_part) {
    if (rows > 1 && row_stride < size) return false;
    if (n_part <= 1) return true;
    return part_stride >= (rows - 1) * row_stride + size ||
           (part_stride >= size && (rows == 1 || row_stride >= (n_part - 1) * part_stride + size));
}
// The workgroups of an array.
inline uint64_t beam_move_groups(uint64_t lo, uint64_t hi, uint64_t n_part) { return (hi - lo + BEAM_TILE - 1) / BEAM_TILE * n_part; }
// The workgroups of an array whose addresses are set, behind those of `end`, and whether it moves in pieces of 16 bytes.
inline void beam_move_shape(BeamMove & m, uint32_t n_part, uint32_t & end) {
    m.wide = (reinterpret_cast<uintptr_t>(m.data) | m.row_stride | (n_part > 1 ? m.part_stride : 0) | m.lo | m.unit_bytes) % 16 == 0;
    m.tiles = uint32_t((m.hi - m.lo + BEAM_TILE - 1) / BEAM_TILE);
    m.end = end += m.tiles * n_part;
}

// The beams' new tokens into their id lists, and on to the next position: out[s * cap + pos + 1] = tok, pos += 1, for slots 16 apart.
struct BeamNextArgs {
    const int32_t * tok;
    int32_t * pos;
    int32_t * out;
    int cap, n_seq;
};
hipError_t launch_beam_next(const BeamNextArgs & a, hipStream_t s);
hipError_t launch_beam_reorder(const BeamReorderArgs & a, hipStream_t s);

}  // namespace gq
