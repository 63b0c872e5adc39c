// Tensor-core attention: the host-side interface, and the device pieces that the forward and backward kernels share.
#pragma once
#include "attention.cuh"

// Rule that chooses between the row kernels and the tensor-core kernels (see attention_tc.cu).
bool tenmo_attn_tc_profitable(const TenmoAttnParams& p, bool backward);
int tenmo_attn_tc_fwd(tenmo_ctx* ctx, const TenmoAttnParams& p);
int tenmo_attn_tc_bwd(tenmo_ctx* ctx, const TenmoAttnParams& p);

// ---- tile images of (batch, heads, rows, dim) views (see tcgen05.cuh) ----
constexpr int ATTN_TILE = 64;  // rows of an image
struct TenmoTileJob {
    TenmoHeadsView src;
    const int32_t* lengths;  // rows from here on become zeros
    uint8_t* img;            // tile t of head (b, h): ((b * heads + h) * tiles + t) * ATTN_TILE * DP * 4 bytes
    float* inverse;          // 2^-e of every tile
    int heads, rows, tiles, vec;
};
struct TenmoTileJobs {
    TenmoTileJob job[4];
    int B, D;
};
int tenmo_attn_make_tiles(tenmo_ctx* ctx, const TenmoTileJobs& jobs, int count, int dp);
bool tenmo_attn_row_vec(const TenmoHeadsView& v, int D);
static inline int tenmo_attn_padded(int D) { return D <= 64 ? 64 : 128; }
