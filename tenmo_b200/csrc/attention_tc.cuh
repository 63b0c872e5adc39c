// Tensor-core attention: the host-side interface, and the device pieces that the forward and backward kernels share.
#pragma once
#include "attention.cuh"
#include "tcgen05.cuh"

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
    // With o.ptr set (src is the gradient of o): the per-row numbers of the backward pass as well.  Per tile 256 floats:
    // [0, 64) m_i (+inf for rows that take no part), [64, 128) 1 / l_i times the tile's power of two PS that brings the largest
    // to at most 2^15 (0 for those rows), [128, 192) delta_i, 192: PS, 193: the largest |delta|, 194: 1 / PS; the rest is unused.
    TenmoHeadsView o;
    const float* stats;
    float* info;
    int o_vec;
};
constexpr int ATTN_INFO = 256;  // floats of a tile's row numbers
struct TenmoTileJobs {
    TenmoTileJob job[4];
    int B, D;
};
int tenmo_attn_make_tiles(tenmo_ctx* ctx, const TenmoTileJobs& jobs, int count, int dp);
bool tenmo_attn_row_vec(const TenmoHeadsView& v, int D);
static inline int tenmo_attn_padded(int D) { return D <= 64 ? 64 : 128; }

// A row of an operand, split into fp16 pairs scaled by the row's power of two, into tensor memory (hi from `addr` on, lo DP / 2
// columns further) or, with `plane` set, into a 128-row tile image in shared memory.  Called by the threads of WGS warpgroups, which
// share the columns of a row; `exchange` holds 256 floats.  Returns the inverse scale.
template <int DP, bool SMEM, int WGS>
__device__ __forceinline__ float tenmo_attn_stationary(const float* src, bool in, bool vec, int D, bool negate, int wg, int row,
                                                       uint32_t addr, uint8_t* plane, float* exchange) {
    constexpr int W = DP / WGS;
    float x[W];
    float mx = 0.f;
#pragma unroll
    for (int e = 0; e < W; e += 4) {
        const int d = wg * W + e;
        if (in && vec && d + 4 <= D) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(src + d));
            x[e] = f.x; x[e + 1] = f.y; x[e + 2] = f.z; x[e + 3] = f.w;
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) x[e + u] = in && d + u < D ? __ldg(src + d + u) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) mx = fmaxf(mx, tc::finite_abs(x[e + u]));
    }
    if (WGS == 2) {
        asm volatile("bar.sync 1, 256;" ::: "memory");  // an earlier use of `exchange` is over
        exchange[wg * 128 + row] = mx;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        mx = fmaxf(mx, exchange[(wg ^ 1) * 128 + row]);
    }
    float inverse;
    float scale = tc::block_scale(mx, &inverse);
    if (negate) scale = -scale;
#pragma unroll
    for (int g = 0; g < W / 32; ++g) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) tc::split_pair(x[32 * g + 2 * e] * scale, x[32 * g + 2 * e + 1] * scale, hi[e], lo[e]);
        if (SMEM) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int c = (wg * W + 32 * g) / 8 + q;
                const int at = (c >> 3) * (128 * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
                *reinterpret_cast<uint4*>(plane + at) = make_uint4(hi[4 * q], hi[4 * q + 1], hi[4 * q + 2], hi[4 * q + 3]);
                *reinterpret_cast<uint4*>(plane + 128 * DP * 2 + at) = make_uint4(lo[4 * q], lo[4 * q + 1], lo[4 * q + 2], lo[4 * q + 3]);
            }
        } else {
            const uint32_t col = (uint32_t)(wg * (W / 2) + 16 * g);
            tc::st16(addr + col, hi);
            tc::st16(addr + DP / 2 + col, lo);
        }
    }
    if (SMEM) tc::fence_proxy_async();
    else tc::st_wait();
    return inverse;
}
