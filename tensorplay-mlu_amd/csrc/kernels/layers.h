// Argument blocks and launch entries of what stands between a language
// model's matrix products: dropout whose mask is never stored
// (seeded_dropout.hip), the join of a block to its residual stream with the
// norms on both sides of it (residual_norm.hip), and the log probabilities of
// given tokens (token_log_probs.hip).  Strides are in elements.
#pragma once

#include <cstdint>

#include "philox.h"

namespace tp_amd {

void launch_seeded_dropout(int dtype, int64_t n, const void* x, const DropArgs& drop, void* out, int device);

constexpr int64_t kMaxRows = int64_t{1} << 30;  // fewer than that, of all that follow

// Rows of one tensor, the last axis dense.
struct Rows {
    const void* data;  // null: not there
    int64_t step;
};

// z = a x + b g drop(n), n = y r1 w1 (or y); h = z r2 w2.
struct ResidualNormArgs {
    Rows x, y;
    Rows gate;              // a row of `dim`, or (gate_one) one element, for every rows_per_gate rows
    int64_t rows_per_gate;
    bool gate_one;
    const void *w1, *w2;  // [dim], or null for 1
    bool norm1, norm2;
    bool drops;
    DropArgs drop;
    float a, b, eps1, eps2;
    int64_t rows;
    int dim;
    float *r1, *r2;  // [rows]: written by the forward, read by the backward
    void *z, *h;     // forward; z is not written where there is no y
    Rows dz, dh;     // backward
    void *dx, *dy, *dgate, *dw1, *dw2;  // backward; null: not wanted
};

constexpr int kResidualNormMaxDim = 16384;

void launch_residual_norm(int dtype, const ResidualNormArgs& p, int device);
void launch_residual_norm_backward(int dtype, const ResidualNormArgs& p, int device);

struct TokenProbsArgs {
    Rows logits;
    int64_t rows, vocab;
    const void* target;  // [rows] or null
    bool wide_target;    // int64, else int32
    int64_t ignore;      // rows with this target are skipped
    float scale;
    int top;
    float* logprob;     // [rows] or null
    float* entropy;     // [rows] or null
    float* stats;       // [rows][2]: largest logit, log of the sum over it
    float* top_values;  // [rows][top]
    int64_t* top_index;
    const float *da, *db;  // backward: gradients of logprob and entropy, or null
    void* dlogits;
};

constexpr int kTokenProbsMaxTop = 64;

void launch_token_log_probs(int dtype, const TokenProbsArgs& p, int device);
void launch_token_log_probs_backward(int dtype, const TokenProbsArgs& p, int device);

}  // namespace tp_amd
