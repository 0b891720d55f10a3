// Launch descriptor of the rotary positions on caller-owned memory.
#pragma once
#include "gq_kernels.h"

namespace gq {

constexpr int ROPE_ARRAYS = 4;      // arrays of a call
constexpr int ROPE_MAX_DIM = 1024;  // elements of a head

// Row (s * n_tok + t) of x starts at x_row floats a row, head h of it at x_head floats a head; y likewise; y == x: in place.
struct RotaryArray {
    const float * x;
    float * y;
    long long x_row, x_head, y_row, y_head;
    int n_head;
    int end;  // set at launch: heads of this array and those before it
};

// Pair i of a head (elements i and i + n_rot / 2, or 2 i and 2 i + 1) turns by (pos[s] + t) * freqs[i] full turns and grows by
// freqs[n_rot / 2]; elements from n_rot on stay. Tokens t < num[s] (num NULL: n_tok) with positions of 0 and above.
struct RotaryArgs {
    RotaryArray a[ROPE_ARRAYS];
    const double * freqs;
    const int32_t * pos;
    const int32_t * num;
    int n, n_seq, n_tok, head_dim, n_rot;
    int pairs;       // 0: halves, 1: neighbours
    int tokens;      // set at launch: token rows of a workgroup
    int heads;       // set at launch: heads of a workgroup
    unsigned per_mul, heads_mul;  // set at launch: i / d = the high word of i * mul, for the pieces of a head and for heads; 0: d is 1
};
hipError_t launch_rotary(const RotaryArgs & a, hipStream_t s);

// The table: turns per position of every pair, then the magnitude. factors: NULL or a divisor a pair. yarn_ctx 0: every angle over
// `factor`; else pairs that turn more than beta_fast times over yarn_ctx positions keep theirs, those that turn less than beta_slow
// times have it over `factor`, the ones between a share of both, and the magnitude is 0.1 ln(factor) + 1 (YaRN).
void rope_table(int n_rot, double base, double factor, int yarn_ctx, double beta_fast, double beta_slow, const double * factors,
                double * out);

}  // namespace gq
