// Launch descriptor of the verification of drafted tokens.
#pragma once
#include "gq_kernels.h"

namespace gq {

constexpr int DRAFT_MAX = 32;             // drafted tokens of a sequence
constexpr int DRAFT_MAX_VOCAB = 1 << 20;

struct DraftScale {  // c = log2(e) / temperature, in FP32 its two parts, 1000 / c; whether FP32 has room for both
    double c, reach;
    float ch, cl;
    bool fast;
};
// Sequence s has tokens d_0 .. d_{k-1} drafted (k = num[s], at most n_draft; below 0: not in use), the target's rows s * (n_draft + 1) + t
// for t = 0 .. k (row k follows the last token) and the draft's rows s * n_draft + t. p_t and q_t are the rows' distributions,
// e^((x - max x) / temperature) over their sum (below 2^-1000 of the largest: 0); without draft rows q_t is 1 at d_t. Token t is accepted if u_t q_t(d_t) <
// p_t(d_t) and all before it are. At the first that is not, a new token comes from max(p_t - q_t, 0) (from p_t where nothing is left),
// behind the last from p_k: the first whose weights' sum up to it is above u_{n_draft} times the sum of all. Temperature 0: the
// target's largest logit, the lowest index of equal ones, is what a token is compared with and what is new; log-probabilities are
// then those of temperature 1. NaN logits count as -inf, +inf as FP32's largest number; a row of nothing but -inf has no token (-1).
struct DraftArgs {
    const float * target;
    const float * draft;     // or NULL
    long long target_stride, draft_stride;
    const int32_t * token;   // s * n_draft + t
    const int32_t * num;     // or NULL: n_draft each
    const float * uniform;   // s * (n_draft + 1) + t
    int32_t * n_accept;
    int32_t * out;           // s * (n_draft + 1) + t: the accepted tokens, the new one, then -1
    float * logp;            // or NULL; log p_t of each, 0 behind them
    DraftScale scale, draft_scale;  // (of temperature 1 where greedy)
    bool greedy;                    // temperature 0
    int n_vocab, n_seq, n_draft;
    void * work;
    int chunks;  // set at launch: the first kernel's workgroups a row
    int parts;   // set at launch: the second one's workgroups a sequence
};

DraftScale draft_scale(double temperature);
size_t draft_work(int n_seq, int n_draft, int n_vocab);
hipError_t launch_draft(const DraftArgs & a, hipStream_t s);

}  // namespace gq
