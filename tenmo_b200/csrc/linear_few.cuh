// Products of a few rows (at most TENMO_FEW_ROWS at a time) with a large matrix, fp32, each reading the matrix once (linear_few.cu).
#pragma once
#include "op_util.cuh"

constexpr int TENMO_FEW_ROWS = 32;

// out[n, c] = sum_k a[n, k] B[k, c] (+ bias[c]): B row-major (K, C), its rows ldb apart.
// out[n, r] = sum_c a[n, c] B[r, c] (+ bias[r]): B row-major (R, C).
// a: (N, .) rows lda apart; out rows ldo apart; partial: scratch of tenmo_few_bytes(ctx, N, outputs, contraction).
size_t tenmo_few_bytes(const tenmo_ctx* ctx, int64_t N, int64_t outputs, int64_t contraction);
int tenmo_few_cols(tenmo_ctx* ctx, const float* a, int64_t lda, int64_t N, int64_t K, const float* B, int64_t ldb, int64_t C, const float* bias,
                   float* out, int64_t ldo, float* partial);
int tenmo_few_dot(tenmo_ctx* ctx, const float* a, int64_t lda, int64_t N, int64_t C, const float* B, int64_t ldb, int64_t R, const float* bias,
                  float* out, int64_t ldo, float* partial);
// out[r, c] = sum_n a[n, r] b[n, c]: (R, C) contiguous, any N
int tenmo_few_outer(tenmo_ctx* ctx, const float* a, int64_t lda, const float* b, int64_t ldb, int64_t N, int64_t R, int64_t C, float* out);
