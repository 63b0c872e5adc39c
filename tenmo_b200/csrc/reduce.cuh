// Column-sum kernels shared between entry points (see reduce.cu).
#pragma once
#include "common.cuh"

// Up to this many rows the column sum runs one thread per column in ascending row order
// (bit-identical to the reference's sequential CPU reduction).
#define TENMO_COLSUM_SEQ_ROWS 512

void tenmo_colsum_plan(int sm_count, int64_t M, int64_t N, bool vec, int* strips, int* slabs, int* rows_per_slab);
int tenmo_colsum_launch(tenmo_ctx* ctx, const float* x, int64_t M, int64_t N, int64_t ldx, float* out, float beta,
                        float* partials, unsigned int* tickets, int strips, int slabs, int rows_per_slab, bool vec);
int tenmo_colsum_scratch(tenmo_ctx* ctx, int slabs, int64_t N, int strips, float** partials, unsigned int** tickets);

// The same column sums (and bits) with scratch that the caller owns, tenmo_colsum_own_bytes of it, 16-byte aligned: for operators whose captured
// graphs must not hold the shared workspace, which moves when it grows.
size_t tenmo_colsum_own_bytes(const tenmo_ctx* ctx, int64_t M, int64_t N);
int tenmo_colsum_own(tenmo_ctx* ctx, const float* x, int64_t M, int64_t N, int64_t ldx, float* out, float beta, void* scratch);
