// Argument blocks and launch entries of the attention layer's kernels: the
// norm and rotation of each head's query and key (head_norm.hip), and causal
// attention with a sliding window and first tokens that stay visible
// (attention.hip, attention_backward.hip).  Strides are in elements.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../common.h"

namespace tp_amd {

// Blocks of a launch, whose threads are counted in 32 bits.
inline unsigned grid_of(int64_t blocks, int threads, const char* op) {
    TP_AMD_CHECK(blocks * threads < (int64_t{1} << 32), op, ": too many rows for one launch");
    return static_cast<unsigned>(blocks);
}

// Rows [outer][inner][head][D] of one tensor, the last axis dense.
struct HeadRows {
    const void* data;
    int64_t outer, inner, head;
};

struct HeadNormSide {
    HeadRows x;
    HeadRows dy;         // backward only
    const void* weight;  // [D], or null for 1
    void* out;           // y, or dx: dense; null (backward): not wanted
    float* rstd;         // [tokens][heads]
    void* dweight;       // backward: [D], or null
    int heads;
};

struct HeadNormArgs {
    HeadNormSide side[2];  // queries, keys
    int64_t outer, inner;  // tokens = outer x inner
    int dim, rotary;
    bool interleaved;
    const float* table;  // [table_rows][rotary]: cosines, then sines
    int64_t table_rows;
    const void* positions;
    bool wide_positions;  // int64, else int32
    int64_t pos_outer, pos_inner;
    float eps;
};

constexpr int kHeadNormMaxDim = 1024;

void launch_head_norm(int dtype, const HeadNormArgs& p, int device);
void launch_head_norm_backward(int dtype, const HeadNormArgs& p, int device);

// Tokens of one tensor: element (b, t, h, d) at data[b batch + t token + h head + d].
struct TokenRows {
    const void* data;
    int64_t batch, token, head;
};

struct AttentionArgs {
    TokenRows q, k, v;
    TokenRows o, dout;  // backward only
    int batch, queries, keys, heads, kv_heads, dim;
    int64_t window;  // < 0: none
    int64_t sinks;
    float scale;
    const void* lengths;  // [batch] or null: keys
    const void* starts;   // [batch] or null: length - queries
    bool wide_lengths, wide_starts;
    int64_t lengths_step, starts_step;
    void* out;   // [batch][queries][heads][dim]
    float* lse;  // [batch][heads][queries]: written by the forward, read by the backward
    void *dq, *dk, *dv;
};

constexpr int kAttentionMaxDim = 128;

void launch_attention(int dtype, const AttentionArgs& p, int device);
void launch_attention_backward(int dtype, const AttentionArgs& p, int device);

}  // namespace tp_amd
