// fp32 matrix products on fp16 tensor cores with block-scaled operands (see gemm_h3.cu).
#pragma once
#include "tcgen05.cuh"

// An operand of rows x cols as 128 x 128 blocks, row-major over the blocks.  A block is 64 KB: the hi plane, then the lo plane, each
// as two panels (64 columns) of 128 rows x 128 bytes in the 128-byte swizzle (tcgen05.cuh).  `inverse` holds a block's 2^-e.
constexpr int H3_BLOCK = 128;
constexpr int64_t H3_BLOCK_BYTES = 128 * 128 * 4;
constexpr int H3_PLANE = 128 * 64 * 2;  // a panel: 128 rows x 64 columns
struct TenmoH3Operand {
    uint8_t* img;
    float* inverse;
    int64_t rows, cols;
    int64_t block_rows() const { return (rows + H3_BLOCK - 1) / H3_BLOCK; }
    int64_t block_cols() const { return (cols + H3_BLOCK - 1) / H3_BLOCK; }
    int64_t blocks() const { return block_rows() * block_cols(); }
    size_t img_bytes() const { return (size_t)blocks() * H3_BLOCK_BYTES; }
    size_t inverse_bytes() const { return ((size_t)blocks() * sizeof(float) + 255) & ~(size_t)255; }
};

// Makes the blocks of a strided matrix.  With `labels`, rows whose label equals `ignore` become zeros.
int tenmo_h3_make(tenmo_ctx* ctx, const float* src, int64_t rs, int64_t cs, const TenmoH3Operand& o, const void* labels, int is_i64, int64_t ignore);

// What happens to the M x N product.
struct TenmoH3Epilogue {
    float* C;            // result, leading dimension ldc, or NULL (statistics only)
    int64_t ldc;
    // C is stored as 128 x 128 blocks (ldc unused), row-major over the blocks, each as tenmo_h3_patch says: an operand image can replace it.
    // Blocks are written whole; what lies past M or N in them is unspecified.
    int blocked;
    int add;             // C += product
    const float* bias;   // N floats added to every row, or NULL
    // softmax statistics of the rows (stats != NULL): for every row and 64-column group g, at [g * M + row]: the maximum and the
    // sum of exp(z - maximum); sums: the plain sums (or NULL).  at_label[row] receives the entry in the row's label column.
    float2* stats;
    float* sums;
    float* at_label;
    const void* labels;
    int label_is_i64;
};
// product = A . B over K.  a_rows_are_k: A is stored (K, M), else (M, K); b_rows_are_k: B is stored (K, N), else (N, K).
// (A stored (K, M) with B stored (N, K) is not built.)  `partial`: scratch for the slices of a contraction; tenmo_h3_partial_bytes says how
// much lets the product choose freely, and with less it takes fewer slices.
size_t tenmo_h3_partial_bytes(const tenmo_ctx* ctx, int64_t M, int64_t N, int64_t K);
int tenmo_h3_gemm(tenmo_ctx* ctx, int64_t M, int64_t N, int64_t K, const TenmoH3Operand& A, bool a_rows_are_k, const TenmoH3Operand& B,
                  bool b_rows_are_k, const TenmoH3Epilogue& e, void* partial, size_t partial_bytes);

// Place (in floats) of columns [4 q, 4 q + 4) of row r in a block of logits: 32 rows x 64 columns are contiguous, and of those the 32 rows of four
// columns, which is how a warp of the epilogue (a row per lane) holds them: its stores need no staging.
__device__ __forceinline__ int tenmo_h3_patch(int r, int q) { return ((((r >> 5) * 2 + (q >> 4)) * 16 + (q & 15)) * 32 + (r & 31)) * 4; }

__device__ __forceinline__ int64_t tenmo_h3_label(const void* labels, int is_i64, int64_t n) {
    return is_i64 ? __ldg((const long long*)labels + n) : (int64_t)__ldg((const int*)labels + n);
}

// Splits the 128 x 128 values that the block's 512 threads hold (a thread: rows row + 32 s, columns 8 c ..) into img.
__device__ __forceinline__ void tenmo_h3_write_block(const float (&x)[4][8], int row, int c, uint8_t* img, float* inverse) {
    __shared__ float largest[16];
    float mx = 0.f;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[s][e]));  // a NaN does not count
    if (!(mx <= 3.402823466e38f)) {  // an infinity does not either
        mx = 0.f;
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, tc::finite_abs(x[s][e]));
    }
    mx = tenmo_warp_max(mx);
    if ((threadIdx.x & 31) == 0) largest[threadIdx.x >> 5] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; ++w) mx = fmaxf(mx, largest[w]);
    float inv;
    const float scale = tc::block_scale(mx, &inv);
    if (threadIdx.x == 0) *inverse = inv;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int r = row + 32 * s;
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) tc::split_rounded(x[s][2 * e] * scale, x[s][2 * e + 1] * scale, hi[e], lo[e]);
        const int at = (c >> 3) * H3_PLANE + r * 128 + (((c & 7) ^ (r & 7)) << 4);
        *reinterpret_cast<uint4*>(img + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(img + 2 * H3_PLANE + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
}
