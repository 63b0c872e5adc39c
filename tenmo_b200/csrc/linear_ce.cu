// Softmax cross-entropy of a linear layer's logits without keeping the logits, forward and gradient, fp32.
//
//   z = x W + b (N, V);  lse_n = log sum_v exp z_nv;  loss_n = (1 - ls)(lse_n - z_n,y) + ls (lse_n - mean_v z_nv)
//   dz_nv = u_n (softmax(z)_nv - (1 - ls)[v = y_n] - ls / V),  u_n = upstream (/ valid rows for the mean), 0 for ignored rows
//   dx = dz W^T;  dW = x^T dz;  db = column sums of dz
//
// The rows are taken in pieces whose logits fit a bounded part of the workspace.  A piece's logits are computed, turned into
// the gradient in place, multiplied into dx and added to dW and db, and then forgotten: three products per piece, where a
// loss that forgets the logits between forward and backward needs a fourth to recompute them.
// Ignored rows: their x is replaced by zeros, so that whatever padding holds (NaN included) reaches no gradient.
#include <cfloat>

#include "op_util.cuh"

namespace {

constexpr size_t LCE_PIECE_BYTES = (size_t)512 << 20;  // logits of one piece
constexpr int LCE_THREADS = 256;

__device__ __forceinline__ int64_t lce_label(const void* labels, int is_i64, int64_t n) {
    return is_i64 ? __ldg((const long long*)labels + n) : (int64_t)__ldg((const int*)labels + n);
}

// block-wide reductions; `slots` holds a value per warp and may be reused after the next barrier
template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float* slots) {
    v = MAX ? tenmo_warp_max(v) : tenmo_warp_sum(v);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    __syncthreads();
    if (lane == 0) slots[warp] = v;
    __syncthreads();
    v = lane < warps ? slots[lane] : (MAX ? -INFINITY : 0.f);
    return MAX ? tenmo_warp_max(v) : tenmo_warp_sum(v);
}

// valid rows and the factor of the mean
__global__ void __launch_bounds__(1024) lce_count_kernel(const void* labels, int is_i64, int64_t N, int64_t ignore, int reduction,
                                                         int32_t* valid, float* factor) {
    __shared__ int slots[32];
    tenmo_grid_dependency_sync();
    int c = 0;
    for (int64_t n = threadIdx.x; n < N; n += blockDim.x) c += lce_label(labels, is_i64, n) != ignore;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = c;
    __syncthreads();
    if (threadIdx.x == 0) {
        c = 0;
        for (int w = 0; w < 32; ++w) c += slots[w];
        *valid = c;
        *factor = reduction == 0 && c > 0 ? 1.f / (float)c : 1.f;
    }
}

// rows of x, contiguous; ignored rows become zeros
__global__ void lce_rows_kernel(const float* x, int64_t rs, int64_t cs, const void* labels, int is_i64, int64_t ignore,
                                int64_t row0, int64_t rows, int64_t D, float* out) {
    tenmo_grid_dependency_sync();
    for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < rows * D; e += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = e / D, d = e % D;
        out[e] = lce_label(labels, is_i64, row0 + r) == ignore ? 0.f : __ldg(x + (row0 + r) * rs + d * cs);
    }
}

struct LceRow {
    float* z;  // (rows, V) logits; overwritten with the gradient when `grad`
    const void* labels;
    float* row_loss;
    const float* upstream; const float* factor;
    uint32_t* status;
    int64_t row0, V, ignore;
    float ls;
    int is_i64, reduction, grad;
};

// a block is a row
__global__ void __launch_bounds__(LCE_THREADS) lce_row_kernel(const LceRow p) {
    __shared__ float slots[32];
    tenmo_grid_dependency_sync();
    const int64_t n = p.row0 + blockIdx.x;
    float* z = p.z + (int64_t)blockIdx.x * p.V;
    const int64_t y = lce_label(p.labels, p.is_i64, n);
    const bool counted = y != p.ignore, good = counted && y >= 0 && y < p.V;
    if (!good) {
        if (counted && threadIdx.x == 0) atomicOr(p.status, TENMO_DEV_BAD_LABEL);
        if (threadIdx.x == 0) p.row_loss[n] = 0.f;
        if (p.grad)
            for (int64_t v = threadIdx.x; v < p.V; v += LCE_THREADS) z[v] = 0.f;
        return;
    }
    float m = -INFINITY;
    for (int64_t v = threadIdx.x; v < p.V; v += LCE_THREADS) m = fmaxf(m, z[v]);
    m = block_reduce<true>(m, slots);
    float l = 0.f, s = 0.f;
    for (int64_t v = threadIdx.x; v < p.V; v += LCE_THREADS) {
        const float t = z[v] - m;
        l += expf(t);
        s += t;
    }
    l = block_reduce<false>(l, slots);
    if (p.ls > 0.f) s = block_reduce<false>(s, slots);
    if (threadIdx.x == 0) {
        const float lse = logf(l);  // relative to the maximum
        float loss = (1.f - p.ls) * (lse - (z[y] - m));
        if (p.ls > 0.f) loss += p.ls * (lse - s / (float)p.V);
        p.row_loss[n] = loss;
    }
    if (!p.grad) return;
    __syncthreads();  // z[y] has been read
    float u = *p.factor;
    if (p.upstream) u *= p.upstream[p.reduction == 2 ? n : 0];
    const float inv = 1.f / l, smooth = p.ls / (float)p.V;
    for (int64_t v = threadIdx.x; v < p.V; v += LCE_THREADS) {
        const float g = expf(z[v] - m) * inv - smooth - (v == y ? 1.f - p.ls : 0.f);
        z[v] = g * u;
    }
}

// loss from the row losses, added in a fixed order (double: the mean of many rows keeps the bits of each)
__global__ void __launch_bounds__(1024) lce_loss_kernel(const float* row_loss, int64_t N, int reduction, const int32_t* valid, float* loss) {
    __shared__ double slots[32];
    tenmo_grid_dependency_sync();
    if (reduction == 2) {
        for (int64_t n = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; n < N; n += (int64_t)gridDim.x * blockDim.x) loss[n] = row_loss[n];
        return;
    }
    double s = 0.0;
    for (int64_t n = threadIdx.x; n < N; n += blockDim.x) s += row_loss[n];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int w = 0; w < 32; ++w) s += slots[w];
        if (reduction == 0 && *valid > 0) s /= *valid;
        *loss = (float)s;
    }
}

struct LceCall {
    const tenmo_mat* x; const tenmo_mat* w; const float* bias; const void* labels; int is_i64;
    int64_t N, D, V, ignore; float ls; int reduction; float* loss; int32_t* valid;
    const float* upstream; float* dx; float* dw; float* db; bool grad;
};

tenmo_mat plain(const float* p, int64_t rs, int64_t cs) {
    tenmo_mat m;
    memset(&m, 0, sizeof(m));
    m.ptr = p;
    m.row_stride = rs;
    m.col_stride = cs;
    return m;
}
tenmo_mat transposed(tenmo_mat m) {
    const int64_t t = m.row_stride;
    m.row_stride = m.col_stride;
    m.col_stride = t;
    return m;
}

int check(tenmo_ctx* ctx, const char* who, const LceCall& c) {
    if (c.N < 0 || c.D < 1 || c.V < 1 || c.V > INT32_MAX || c.D > INT32_MAX)
        return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: N=%lld D=%lld V=%lld", who, (long long)c.N, (long long)c.D, (long long)c.V);
    if (!c.x || !c.w || !c.w->ptr || !c.loss || !c.valid || (c.N && (!c.x->ptr || !c.labels)))
        return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: null pointer", who);
    if (c.grad && (!c.dw || (c.N && !c.dx)))
        return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: dx or dw is NULL", who);
    if (c.grad && c.db && !c.bias) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: db without a bias", who);
    if (c.x->batch_rank || c.w->batch_rank) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: x and w are plain matrices", who);
    if (c.x->row_stride < 0 || c.x->col_stride < 0) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: x has a negative stride", who);
    if (c.w->row_stride != 1 && c.w->col_stride != 1)
        return tenmo_set_error(ctx, TENMO_ERR_UNSUPPORTED, "%s: w needs a unit stride on one axis", who);
    if (c.reduction < 0 || c.reduction > 2) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: reduction %d", who, c.reduction);
    if (!(c.ls >= 0.f && c.ls <= 1.f)) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: label_smoothing outside [0,1]", who);
    return TENMO_OK;
}

int lce_run(tenmo_ctx* ctx, const char* who, const LceCall& c) {
    int st = check(ctx, who, c);
    if (st != TENMO_OK) return st;
    TenmoDeviceGuard guard(ctx);
    int64_t piece = (int64_t)(LCE_PIECE_BYTES / ((size_t)c.V * sizeof(float))) / 128 * 128;
    if (piece < 128) piece = 128;
    if (piece > c.N) piece = c.N;
    const size_t z_bytes = ((size_t)piece * c.V * sizeof(float) + 255) & ~(size_t)255;
    const size_t x_bytes = ((size_t)piece * c.D * sizeof(float) + 255) & ~(size_t)255;
    const size_t l_bytes = ((size_t)c.N * sizeof(float) + 255) & ~(size_t)255;
    void* ws = nullptr;
    if ((st = tenmo_op_workspace(ctx, z_bytes + x_bytes + l_bytes + 256, &ws)) != TENMO_OK) return st;
    float* z = (float*)ws;
    float* xr = (float*)((char*)ws + z_bytes);
    float* row_loss = (float*)((char*)ws + z_bytes + x_bytes);
    float* factor = (float*)((char*)ws + z_bytes + x_bytes + l_bytes);
    TENMO_CUDA_TRY(ctx, tenmo_launch(lce_count_kernel, 1, 1024, 0, ctx->stream, ctx->pdl, c.labels, c.is_i64, c.N, c.ignore, c.reduction,
                                     c.valid, factor));
    TENMO_LAUNCH_CHECK(ctx, "lce_count_kernel");
    const tenmo_mat wt = transposed(*c.w);
    const bool tied = c.w->row_stride == 1 && c.w->col_stride != 1;  // storage is (V, D)
    for (int64_t r0 = 0; r0 < c.N; r0 += piece) {
        const int64_t rows = r0 + piece < c.N ? piece : c.N - r0;
        lce_rows_kernel<<<tenmo_stream_grid(ctx, rows * c.D, 256 * 4, 8), 256, 0, ctx->stream>>>(
            c.x->ptr + c.x->offset, c.x->row_stride, c.x->col_stride, c.labels, c.is_i64, c.ignore, r0, rows, c.D, xr);
        TENMO_LAUNCH_CHECK(ctx, "lce_rows_kernel");
        const tenmo_mat mx = plain(xr, c.D, 1), mz = plain(z, c.V, 1);
        st = tenmo_gemm_f32(ctx, TENMO_ALGO_SIMT_FP32, rows, c.V, c.D, &mx, c.w, z, 0.f, c.bias, TENMO_ACT_NONE, nullptr, nullptr);
        if (st != TENMO_OK) return st;
        const LceRow p{z, c.labels, row_loss, c.upstream, factor, ctx->dev_status, r0, c.V, c.ignore, c.ls, c.is_i64, c.reduction, c.grad};
        lce_row_kernel<<<(unsigned)rows, LCE_THREADS, 0, ctx->stream>>>(p);
        TENMO_LAUNCH_CHECK(ctx, "lce_row_kernel");
        if (!c.grad) continue;
        const float beta = r0 ? 1.f : 0.f;
        st = tenmo_gemm_f32(ctx, TENMO_ALGO_SIMT_FP32, rows, c.D, c.V, &mz, &wt, c.dx + r0 * c.D, 0.f, nullptr, TENMO_ACT_NONE, nullptr, nullptr);
        if (st != TENMO_OK) return st;
        const tenmo_mat zt = transposed(mz), xt = transposed(mx);
        if (tied)
            st = tenmo_gemm_f32(ctx, TENMO_ALGO_SIMT_FP32, c.V, c.D, rows, &zt, &mx, c.dw, beta, nullptr, TENMO_ACT_NONE, nullptr, nullptr);
        else
            st = tenmo_gemm_f32(ctx, TENMO_ALGO_SIMT_FP32, c.D, c.V, rows, &xt, &mz, c.dw, beta, nullptr, TENMO_ACT_NONE, nullptr, nullptr);
        if (st != TENMO_OK) return st;
        if (c.db && (st = tenmo_colsum_f32(ctx, z, rows, c.V, c.V, c.db, beta)) != TENMO_OK) return st;
    }
    if (c.N == 0 && c.grad) {
        TENMO_CUDA_TRY(ctx, cudaMemsetAsync(c.dw, 0, (size_t)c.D * c.V * sizeof(float), ctx->stream));
        if (c.db) TENMO_CUDA_TRY(ctx, cudaMemsetAsync(c.db, 0, (size_t)c.V * sizeof(float), ctx->stream));
    }
    const int grid = c.reduction == 2 ? tenmo_stream_grid(ctx, c.N, 1024, 1) : 1;
    TENMO_CUDA_TRY(ctx, tenmo_launch(lce_loss_kernel, grid, 1024, 0, ctx->stream, ctx->pdl, (const float*)row_loss, c.N, c.reduction,
                                     (const int32_t*)c.valid, c.loss));
    TENMO_LAUNCH_CHECK(ctx, "lce_loss_kernel");
    return TENMO_OK;
}

}  // namespace

extern "C" {

int tenmo_linear_ce_fwd_f32(tenmo_ctx* ctx, const tenmo_mat* x, const tenmo_mat* w, const float* bias, const void* labels,
                            int label_is_i64, int64_t N, int64_t D, int64_t V, int64_t ignore_index, float label_smoothing,
                            int reduction, float* loss, int32_t* valid_count) {
    TENMO_CHECK_CTX(ctx);
    LceCall c = {};
    c.x = x; c.w = w; c.bias = bias; c.labels = labels; c.is_i64 = label_is_i64; c.N = N; c.D = D; c.V = V;
    c.ignore = ignore_index; c.ls = label_smoothing; c.reduction = reduction; c.loss = loss; c.valid = valid_count;
    return lce_run(ctx, "linear_ce_fwd", c);
}

int tenmo_linear_ce_fwd_bwd_f32(tenmo_ctx* ctx, const tenmo_mat* x, const tenmo_mat* w, const float* bias, const void* labels,
                                int label_is_i64, int64_t N, int64_t D, int64_t V, int64_t ignore_index, float label_smoothing,
                                int reduction, float* loss, int32_t* valid_count, const float* upstream, float* dx, float* dw,
                                float* db) {
    TENMO_CHECK_CTX(ctx);
    LceCall c = {};
    c.x = x; c.w = w; c.bias = bias; c.labels = labels; c.is_i64 = label_is_i64; c.N = N; c.D = D; c.V = V;
    c.ignore = ignore_index; c.ls = label_smoothing; c.reduction = reduction; c.loss = loss; c.valid = valid_count;
    c.upstream = upstream; c.dx = dx; c.dw = dw; c.db = db; c.grad = true;
    return lce_run(ctx, "linear_ce_fwd_bwd", c);
}

}  // extern "C"
