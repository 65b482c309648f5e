// What the losses on chosen log-probabilities leave of a row of logits for its gradient
// (token_loss.hip), also where the logits are GroupSum's scores (groupsum.hip).
#pragma once

#include "common.h"

namespace cl {

// What the backward needs of a row.
template <typename A>
struct alignas(4 * sizeof(A)) RowState {
    A m;      // largest logit
    A inv_s;  // 1 / sum exp(x - m)
    A rest;   // 1 - p of the action
    A slope;  // d loss term / d lp, 0 for a row that does not count
};

// exp of a difference d = x - m <= 0.  fp32: the hardware's 2^t of t = d log2 e, log2 e in two
// terms, so that t is rounded once and without a drift: over d in [-16, 0] the mean relative error
// measures 3e-9 (1e-7 with log2 e as one fp32 number, which a sum over a vocabulary, and then over
// a sequence, does not average out), the largest 7e-7, at the far end.
__device__ __forceinline__ float exp_diff(float d) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(d, 1.44269502162933349609f,
                                                 d * 1.92596299112661746887e-8f));
}
__device__ __forceinline__ double exp_diff(double d) { return exp(d); }

// ---- the upstream gradient of a row's slope
template <typename A>
struct Upstream {
    const A* rows;           // a gradient per row, or null
    const A* scalar;         // the gradient of a scalar loss, or null
    const A* count;          // what a mean divides by, or null
    const int32_t* row_seq;  // preference: the row's sequence (-1: none), else null
    const A* seq_slope;      // per sequence; sequence q belongs to pair q % pairs
    const A* pair_grad;      // a gradient per pair, or null
    int64_t pairs;
    __device__ __forceinline__ A operator()(int64_t n, A slope) const {
        if (slope == A(0)) return A(0);
        A g = slope;
        if (row_seq) {
            const int64_t q = row_seq[n];
            if (q < 0) return A(0);
            g *= seq_slope[q];
            if (pair_grad) g *= pair_grad[q < pairs ? q : q - pairs];
        }
        if (rows) g *= rows[n];
        if (scalar) g *= count ? scalar[0] / count[0] : scalar[0];  // (1: as GradOut has it)
        return g;
    }
};

}  // namespace cl
