// Attention: what the entry points hand to the kernels.
#pragma once
#include "op_util.cuh"

constexpr int TENMO_ATTN_MAX_DIM = 128;

struct TenmoHeadsView {  // element (b, h, row, d) at ptr[b*sb + h*sh + row*sr + d]
    float* ptr;
    int64_t sb, sh, sr;
};

struct TenmoAttnParams {
    TenmoHeadsView q, k, v, o, go, dq, dk, dv;  // go: gradient of the output
    float* stats;       // (B, H, Sq, 2): row maximum of the scores in units of log 2, and the row sum
    float* delta;       // (B, H, Sq): sum_d go * o, written by the dq pass and read by the dk / dv pass
    const int32_t* q_lengths;
    const int32_t* k_lengths;
    int B, H, Hkv, Sq, Sk, D;
    float scale, scale_log2;  // scale * log2(e)
    int causal;
    float beta;  // 1: the gradients are added to what dq, dk, dv hold
};

// Valid rows / keys of batch entry b (out-of-range lengths are clamped).
__device__ __forceinline__ int tenmo_attn_rows(const int32_t* lengths, int b, int full) {
    return lengths ? max(0, min(lengths[b], full)) : full;
}
