// Tensor-core attention: the host-side interface, and the device pieces that the forward and backward kernels share.
#pragma once
#include "attention.cuh"
#include "tcgen05.cuh"

// Rule that chooses between the row kernels and the tensor-core kernels (see attention_tc.cu).
bool tenmo_attn_tc_profitable(const TenmoAttnParams& p, bool backward);
int tenmo_attn_tc_fwd(tenmo_ctx* ctx, const TenmoAttnParams& p);
int tenmo_attn_tc_bwd(tenmo_ctx* ctx, const TenmoAttnParams& p);

// ---- tile images of (batch, heads, rows, dim) views (see tcgen05.cuh) ----
constexpr int ATTN_TILE = 64;  // rows of an image in the backward pass
struct TenmoTileJob {
    TenmoHeadsView src;
    const int32_t* lengths;  // rows from here on become zeros
    uint8_t* img;            // tile t of head (b, h): ((b * heads + h) * tiles + t) * (rows of a tile) * DP * 4 bytes
    float* inverse;          // 2^-e of every tile
    int heads, rows, tiles, vec;
    int first;               // rows before this one become zeros too: they see no key
    // causal keys (seen_by > 0): what the last row that takes part does not see becomes zeros
    const int32_t* q_lengths;
    int seen_by, offset;     // rows of q, k_len - q_len
    // With o.ptr set (src is the gradient of o): the per-row numbers of the backward pass as well.  Per tile 256 floats:
    // for rows 2 r, 2 r + 1 the four at 4 r: their -m (-inf for rows that take no part) and their 1 / l times the tile's power of two
    // PS that brings the largest to at most 2^15 (0 for those rows); [128, 192) delta; 192: PS, 193: the largest |delta|, 194: 1 / PS.
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
int tenmo_attn_make_tiles(tenmo_ctx* ctx, const TenmoTileJobs& jobs, int count, int dp, int tile_rows);  // 64 or 128 (without row numbers)
void tenmo_attn_causal_keys(const TenmoAttnParams& a, TenmoTileJob* j);  // fills seen_by and so on of a job of k or v
bool tenmo_attn_row_vec(const TenmoHeadsView& v, int D);

// Order of the blocks: heads in groups whose images fit into half of L2, so that a head's tiles are read again while L2 holds them (one
// group over 384 heads of 512x64, 100 MB, read 437 MB from HBM, two read 192 MB and took 125 us for 131); within a group tile by tile, so
// that the long ones of a causal head start first.  Smaller groups than that end unevenly: 16 heads of 4001x128 causal, 64 MB, took 191 us
// in one group and 204 in two.
struct TenmoAttnOrder { unsigned heads, group; int tiles; };
constexpr int64_t TENMO_ATTN_GROUP_BYTES = (int64_t)64 << 20;
static inline TenmoAttnOrder tenmo_attn_order(const TenmoAttnParams& a, int tiles, size_t image_bytes) {
    const int64_t heads = (int64_t)a.B * a.H, most = ((int64_t)image_bytes + TENMO_ATTN_GROUP_BYTES - 1) / TENMO_ATTN_GROUP_BYTES;
    const int64_t groups = most < 1 ? 1 : most < heads ? most : heads;
    return TenmoAttnOrder{(unsigned)heads, (unsigned)((heads + groups - 1) / groups), tiles};
}
__device__ __forceinline__ void tenmo_attn_block(const TenmoAttnOrder& o, unsigned block, int* tile, int* head) {
    const unsigned first = block / (o.group * o.tiles) * o.group, in = block - first * o.tiles, heads = min(o.group, o.heads - first);
    *tile = (int)(in / heads);
    *head = (int)(first + in % heads);
}
static inline int tenmo_attn_padded(int D) { return D <= 64 ? 64 : 128; }

// A warp's 32 rows x W columns between memory and one row per thread, through `scratch` (32 * W floats of the warp's own): the 16-byte
// chunks of a row are permuted so that neither the row-wise nor the thread-wise accesses conflict, and memory sees whole
// rows (a thread that walks its own row touches 32 rows per instruction).
template <int W>
__device__ __forceinline__ float4* tenmo_attn_chunk(float* scratch, int r, int q) {
    return reinterpret_cast<float4*>(scratch + r * W + ((q ^ (W >= 32 ? r & 7 : (r >> 1) & 3)) << 2));
}
// x: columns [0, cols) of this lane's row; rows from `rows` on and columns from `cols` on are zeros
template <int W>
__device__ __forceinline__ void tenmo_attn_read_rows(float (&x)[W], const float* src, int64_t stride, int rows, int cols, bool vec, float* scratch) {
    constexpr int LPR = W / 4, RPI = 32 / LPR;
    const int lane = threadIdx.x & 31, q = lane % LPR;
    const float* p = src + (lane / LPR) * stride + 4 * q;
    float4 v[LPR];  // all loads are in flight before the first is used
    if (vec) {
#pragma unroll
        for (int it = 0; it < LPR; ++it)
            v[it] = it * RPI + lane / LPR < rows && 4 * q < cols ? __ldg(reinterpret_cast<const float4*>(p + it * RPI * stride)) : make_float4(0.f, 0.f, 0.f, 0.f);
    } else {
#pragma unroll
        for (int it = 0; it < LPR; ++it) {
            const bool in = it * RPI + lane / LPR < rows;
            const float* r = p + it * RPI * stride;
            v[it].x = in && 4 * q < cols ? __ldg(r) : 0.f;
            v[it].y = in && 4 * q + 1 < cols ? __ldg(r + 1) : 0.f;
            v[it].z = in && 4 * q + 2 < cols ? __ldg(r + 2) : 0.f;
            v[it].w = in && 4 * q + 3 < cols ? __ldg(r + 3) : 0.f;
        }
    }
#pragma unroll
    for (int it = 0; it < LPR; ++it) *tenmo_attn_chunk<W>(scratch, it * RPI + lane / LPR, q) = v[it];
    __syncwarp();
#pragma unroll
    for (int c = 0; c < LPR; ++c) {
        const float4 v = *tenmo_attn_chunk<W>(scratch, lane, c);
        x[4 * c] = v.x; x[4 * c + 1] = v.y; x[4 * c + 2] = v.z; x[4 * c + 3] = v.w;
    }
    __syncwarp();
}
template <int W>
__device__ __forceinline__ void tenmo_attn_write_rows(const float (&x)[W], float* dst, int64_t stride, int rows, int cols, bool vec, bool add, float* scratch) {
    constexpr int LPR = W / 4, RPI = 32 / LPR;
    const int lane = threadIdx.x & 31, q = lane % LPR;
    __syncwarp();
#pragma unroll
    for (int c = 0; c < LPR; ++c) *tenmo_attn_chunk<W>(scratch, lane, c) = make_float4(x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
    __syncwarp();
#pragma unroll 8
    for (int it = 0; it < LPR; ++it) {
        const int r = it * RPI + lane / LPR;
        float4 v = *tenmo_attn_chunk<W>(scratch, r, q);
        if (r >= rows || 4 * q >= cols) continue;
        float* p = dst + r * stride + 4 * q;
        if (vec) {
            if (add) {
                const float4 o = *reinterpret_cast<const float4*>(p);
                v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
            }
            *reinterpret_cast<float4*>(p) = v;
        } else {
            const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (4 * q + u < cols) p[u] = add ? p[u] + f[u] : f[u];
        }
    }
}

// A block whose rows take no part: zeros in rows [row0, row0 + 128) of `rows`, by the whole block.
template <int DP>
__device__ __forceinline__ void tenmo_attn_zero_rows(float* head, int64_t stride, int row0, int rows, int D, bool vec) {
    constexpr int Q = DP / 4;
    const int n = min(128, rows - row0) * Q;
    float* const first = head + row0 * stride;
#pragma unroll 4
    for (int e = threadIdx.x; e < n; e += blockDim.x) {
        const int d = 4 * (e % Q);
        float* p = first + (e / Q) * stride + d;
        if (vec) {
            if (d < D) *reinterpret_cast<float4*>(p) = make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (d + u < D) p[u] = 0.f;
        }
    }
}

// This thread's columns of its row of an operand; `scratch` holds 128 * DP floats.  Asked for before anything else of a block: the way to memory
// takes as long as the barriers and the tensor memory.
template <int DP, int WGS>
__device__ __forceinline__ void tenmo_attn_fetch(float (&x)[DP / WGS], const float* src, int64_t stride, int rows, bool vec, int D, float* scratch) {
    constexpr int W = DP / WGS;
    const int warp = threadIdx.x >> 5, wg = warp >> 2, row0 = 32 * (warp & 3);
    tenmo_attn_read_rows<W>(x, src + row0 * stride + wg * W, stride, rows - row0, D - wg * W, vec, scratch + warp * (32 * W));
}
// The rows of an operand (128 of them; x: this thread's columns of its row), split into fp16 pairs scaled by a power of two per row, into
// tensor memory (hi from `addr` on, lo DP / 2 columns further) or, with SMEM, into a 128-row tile image in shared memory.  Called by the
// threads of WGS warpgroups, which share the columns of a row; `exchange` holds WGS * 128 floats.  Returns the row's inverse scale.
template <int DP, bool SMEM, int WGS>
__device__ __forceinline__ float tenmo_attn_stationary(const float (&x)[DP / WGS], bool negate, uint32_t addr, uint8_t* plane, float* exchange) {
    constexpr int W = DP / WGS;
    const int wg = threadIdx.x >> 7, row = threadIdx.x & 127;
    float mx = 0.f;
#pragma unroll
    for (int e = 0; e < W; ++e) mx = fmaxf(mx, tc::finite_abs(x[e]));
    asm volatile("bar.sync 1, %0;" ::"n"(128 * WGS) : "memory");  // an earlier use of `exchange` is over
    exchange[wg * 128 + row] = mx;
    asm volatile("bar.sync 1, %0;" ::"n"(128 * WGS) : "memory");
#pragma unroll
    for (int w = 0; w < WGS; ++w) mx = fmaxf(mx, exchange[w * 128 + row]);
    float inverse;
    float scale = tc::block_scale(mx, &inverse);
    if (negate) scale = -scale;
#pragma unroll
    for (int g = 0; g < W / 16; ++g) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) tc::split_rounded(x[16 * g + 2 * e] * scale, x[16 * g + 2 * e + 1] * scale, hi[e], lo[e]);
        if (SMEM) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int c = (wg * W + 16 * g) / 8 + q;
                const int at = (c >> 3) * (128 * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
                *reinterpret_cast<uint4*>(plane + at) = make_uint4(hi[4 * q], hi[4 * q + 1], hi[4 * q + 2], hi[4 * q + 3]);
                *reinterpret_cast<uint4*>(plane + 128 * DP * 2 + at) = make_uint4(lo[4 * q], lo[4 * q + 1], lo[4 * q + 2], lo[4 * q + 3]);
            }
        } else {
            const uint32_t col = (uint32_t)((wg * W + 16 * g) / 2);
            tc::st8(addr + col, hi);
            tc::st8(addr + DP / 2 + col, lo);
        }
    }
    tc::fence_proxy_async();  // the rows came through a stage that a copy fills next (and with SMEM the tensor core reads the image)
    if (!SMEM) tc::st_wait();
    return inverse;
}
