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
// Bound: the three products (gemm_h3.cu); turning a piece's logits into the gradient is a pass over HBM, 8 bytes an element: 2048 x 65536 in
// 0.24 ms (4.5 TB/s) beside 3.6 ms of products.
#include <cfloat>

#include "gemm_h3.cuh"
#include "linear_few.cuh"
#include "reduce.cuh"

namespace {

constexpr size_t LCE_PIECE_BYTES = (size_t)512 << 20;  // logits (or statistics) of one piece, and as much for its rows of x
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
__global__ void __launch_bounds__(1024) lce_row_kernel(const LceRow p) {
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
            for (int64_t v = threadIdx.x; v < p.V; v += blockDim.x) z[v] = 0.f;
        return;
    }
    float m = -INFINITY;
#pragma unroll 8
    for (int64_t v = threadIdx.x; v < p.V; v += blockDim.x) m = fmaxf(m, z[v]);
    m = block_reduce<true>(m, slots);
    float l = 0.f, s = 0.f;
#pragma unroll 8
    for (int64_t v = threadIdx.x; v < p.V; v += blockDim.x) {
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
#pragma unroll 8
    for (int64_t v = threadIdx.x; v < p.V; v += blockDim.x) {
        const float g = expf(z[v] - m) * inv - smooth - (v == y ? 1.f - p.ls : 0.f);
        z[v] = g * u;
    }
}

// ---- tensor-core path: the softmax statistics come out of the product's epilogue ----
struct LceStats {
    const float2* stats; const float* sums; const float* at_label;  // per 64-column group and row, see gemm_h3.cuh
    int64_t groups, rows, row0, V, ignore;
    const void* labels;
    const float* upstream; const float* factor;
    float* row_loss;
    float4* numbers;  // per row of the piece: maximum, 1 / sum of exponentials, u_n, unused
    uint32_t* status;
    float ls;
    int is_i64, reduction;
};
// 32 rows per block; the warps take the column groups in turn, four loads in flight, and are joined in order
constexpr int LCE_STAT_WARPS = 32;
__global__ void __launch_bounds__(32 * LCE_STAT_WARPS) lce_stats_kernel(const LceStats p) {
    __shared__ float sm[LCE_STAT_WARPS][32], sl[LCE_STAT_WARPS][32], sa[LCE_STAT_WARPS][32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t r = (int64_t)blockIdx.x * 32 + lane;
    float m = -INFINITY, l = 0.f, all = 0.f;
    if (r < p.rows) {
        for (int64_t g0 = w; g0 < p.groups; g0 += 4 * LCE_STAT_WARPS) {
            float2 v[4];
            float top = m;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t g = g0 + k * LCE_STAT_WARPS;
                v[k] = g < p.groups ? __ldg(p.stats + g * p.rows + r) : make_float2(-INFINITY, 0.f);
                if (p.sums && g < p.groups) all += __ldg(p.sums + g * p.rows + r);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) top = fmaxf(top, v[k].x);
            const float base = top == -INFINITY ? 0.f : top;  // nothing but -inf or NaN so far: sums of 0 or NaN
            l *= expf(m - base);
#pragma unroll
            for (int k = 0; k < 4; ++k) l += v[k].x == -INFINITY ? v[k].y : v[k].y * expf(v[k].x - base);
            m = top;
        }
    }
    sm[w][lane] = m;
    sl[w][lane] = l;
    sa[w][lane] = all;
    __syncthreads();
    if (w || r >= p.rows) return;
    for (int k = 1; k < LCE_STAT_WARPS; ++k) m = fmaxf(m, sm[k][lane]);
    const float base = m == -INFINITY ? 0.f : m;
    l = 0.f;
    all = 0.f;
    for (int k = 0; k < LCE_STAT_WARPS; ++k) {
        l += sm[k][lane] == -INFINITY ? sl[k][lane] : sl[k][lane] * expf(sm[k][lane] - base);
        all += sa[k][lane];
    }
    const int64_t n = p.row0 + r, y = lce_label(p.labels, p.is_i64, n);
    const bool counted = y != p.ignore, good = counted && y >= 0 && y < p.V;
    if (counted && !good) atomicOr(p.status, TENMO_DEV_BAD_LABEL);
    float loss = 0.f, u = 0.f;
    if (good) {
        const float lse = logf(l);
        loss = (1.f - p.ls) * (lse - (p.at_label[r] - base));
        if (p.ls > 0.f) loss += p.ls * (lse - (all / (float)p.V - base));
        u = *p.factor;
        if (p.upstream) u *= p.upstream[p.reduction == 2 ? n : 0];
    }
    p.row_loss[n] = loss;
    if (p.numbers) p.numbers[r] = make_float4(base, 1.f / l, u, good ? 1.f : 0.f);
}

// The logits of a 128 x 128 block become the gradient, as an operand image in their place, and its column sums per block row.
// Two blocks on an SM (64 registers): one's loads run beside the other's stores.
__global__ void __launch_bounds__(512, 2) lce_grad_kernel(uint8_t* z, float* inverse, const float4* numbers, const void* labels, int is_i64,
                                                       int64_t row0, int64_t rows, int64_t V, int block_cols, float ls, float* db_part) {
    __shared__ float sums[32][H3_BLOCK + 1];  // + 1: the eight rows of a warp in different banks
    const int64_t block = blockIdx.x;
    const int64_t r0 = block / block_cols * H3_BLOCK, c0 = block % block_cols * H3_BLOCK;
    // a warp takes 8 rows x 32 columns: 128 contiguous bytes of each four columns (tenmo_h3_patch)
    const int row = (threadIdx.x & 7) + 8 * (threadIdx.x >> 7), c = 8 * ((threadIdx.x >> 3) & 15);
    const float* src = reinterpret_cast<const float*>(z + block * H3_BLOCK_BYTES);
    const float smooth = ls / (float)V;
    const int cols = (int)min((int64_t)8, V - c0 - c);  // of this thread that exist
    float x[4][8], col[8];
    float4 num[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {  // all loads first; a row that takes no part has u = 0 and its logits are not looked at
        const int lr = row + 32 * s;
        num[s] = r0 + lr < rows ? __ldg(numbers + r0 + lr) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 a = *reinterpret_cast<const float4*>(src + tenmo_h3_patch(lr, c >> 2)), b = *reinterpret_cast<const float4*>(src + tenmo_h3_patch(lr, (c >> 2) + 1));
        x[s][0] = a.x; x[s][1] = a.y; x[s][2] = a.z; x[s][3] = a.w;
        x[s][4] = b.x; x[s][5] = b.y; x[s][6] = b.z; x[s][7] = b.w;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) col[e] = 0.f;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int64_t r = r0 + row + 32 * s;
        if (num[s].w == 0.f) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[s][e] = 0.f;
            continue;
        }
        const int64_t y = lce_label(labels, is_i64, row0 + r) - c0 - c;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[s][e] = tc::ex2((x[s][e] - num[s].x) * 1.44269504088896341f) * num[s].y - smooth;
        if (y >= 0 && y < 8) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[s][e] -= e == (int)y ? 1.f - ls : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) x[s][e] *= num[s].z;
        if (cols < 8) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[s][e] = e < cols ? x[s][e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) col[e] += x[s][e];
    }
    if (db_part) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[row][c + e] = col[e];
        __syncthreads();
        if (threadIdx.x < H3_BLOCK && c0 + threadIdx.x < V) {
            float t = 0.f;
#pragma unroll
            for (int k = 0; k < 32; ++k) t += sums[k][threadIdx.x];
            db_part[block / block_cols * V + c0 + threadIdx.x] = t;
        }
    }
    // every thread's logits are in registers (the barrier inside) before the image is written over them
    tenmo_h3_write_block(x, row, c >> 3, z + block * H3_BLOCK_BYTES, inverse + block);
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
    if (c.w->row_stride < 0 || c.w->col_stride < 0) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: w has a negative stride", who);
    if (c.w->row_stride != 1 && c.w->col_stride != 1)
        return tenmo_set_error(ctx, TENMO_ERR_UNSUPPORTED, "%s: w needs a unit stride on one axis", who);
    if (c.reduction < 0 || c.reduction > 2) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: reduction %d", who, c.reduction);
    if (!(c.ls >= 0.f && c.ls <= 1.f)) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: label_smoothing outside [0,1]", who);
    return TENMO_OK;
}

// Of one product: against the few-row kernels, which up to 256 rows otherwise run (200x300x1200, 1.4e8: 100 us for 97; 100x768x1000, 1.5e8:
// 97 us for 83), and against the strict-fp32 GEMM (594x40x2465, 1.2e8: 112 us for 120; 980x207x450, 1.8e8: 104 for 114; 512x512x300,
// 1.6e8: 94 for 86; 790x39x1249, 0.8e8: 107 for 123, 1442x72x249, 0.5e8: 100 for 82).
constexpr double TC_FLOP_FEW = 2e8, TC_FLOP = 1e8;
// Rows: with 17 to 32 the weight's split into blocks costs less than the few-row kernels' arithmetic on large weights (24x1318x44771 476 us
// for 607, its loss alone 206 for 263; 24x1024x8000 128 for 122); with up to 16 those read the weight as fast (16x1318x44771 451 us for 475).
constexpr int TC_ROWS = 16;
constexpr int LCE_FEW_MOST = 8 * TENMO_FEW_ROWS;  // rows of the few-row kernels
// Large problems: the products on tensor cores (gemm_h3.cu).  Without a gradient no logit is ever stored: the product's epilogue
// reduces them to two numbers per row and 64 columns.
bool tc_profitable(const LceCall& c) { return c.N > TC_ROWS && 2.0 * c.N * c.D * c.V >= (c.N <= LCE_FEW_MOST ? TC_FLOP_FEW : TC_FLOP); }

// rows of a piece, a multiple of `whole`: what takes z_row bytes a row and what takes x_row bytes each within the budget
int64_t piece_rows(const LceCall& c, size_t z_row, size_t x_row, int64_t whole) {
    const int64_t rows = (int64_t)(LCE_PIECE_BYTES / max(z_row, x_row)) / whole * whole;
    return min(max(rows, whole), c.N);
}

int lce_run_tc(tenmo_ctx* ctx, const LceCall& c) {
    const int64_t vb = (c.V + H3_BLOCK - 1) / H3_BLOCK;
    const bool tied = c.w->row_stride == 1 && c.w->col_stride != 1;  // storage is (V, D)
    // whole tiles of 256 rows
    const size_t x_row = (size_t)((c.D + H3_BLOCK - 1) / H3_BLOCK) * H3_BLOCK * sizeof(float);
    const int64_t piece = piece_rows(c, c.grad ? (size_t)vb * H3_BLOCK * sizeof(float) : (size_t)vb * 2 * sizeof(float2), x_row, 256);
    TenmoH3Operand W = {nullptr, nullptr, tied ? c.V : c.D, tied ? c.D : c.V}, X = {nullptr, nullptr, piece, c.D}, Z = {nullptr, nullptr, piece, c.V};
    const int64_t groups = (c.V + 63) / 64;
    size_t need = 0;
    auto take = [&](size_t bytes) { const size_t at = need; need += (bytes + 1023) & ~(size_t)1023; return at; };
    const size_t w_img = take(W.img_bytes()), w_inv = take(W.inverse_bytes()), x_img = take(X.img_bytes()), x_inv = take(X.inverse_bytes());
    const size_t z_img = c.grad ? take(Z.img_bytes()) : 0, z_inv = c.grad ? take(Z.inverse_bytes()) : 0;
    const size_t stats = take((size_t)groups * piece * sizeof(float2)), sums = c.ls > 0.f ? take((size_t)groups * piece * sizeof(float)) : 0;
    const size_t at_label = take(piece * sizeof(float)), numbers = c.grad ? take(piece * sizeof(float4)) : 0;
    const size_t row_loss = take(c.N * sizeof(float)), factor = take(sizeof(float));
    const size_t db_part = c.db ? take((size_t)((piece + H3_BLOCK - 1) / H3_BLOCK) * c.V * sizeof(float)) : 0;
    size_t part = 0, db_sums = 0;  // for dx, dw and db of a whole piece and of the last one
    for (int64_t rows : {piece, c.N % piece}) {
        if (!c.grad || !rows) continue;
        if (c.db) db_sums = max(db_sums, tenmo_colsum_own_bytes(ctx, (rows + H3_BLOCK - 1) / H3_BLOCK, c.V));
        const size_t dx = tenmo_h3_partial_bytes(ctx, rows, c.D, c.V);
        const size_t dw = tied ? tenmo_h3_partial_bytes(ctx, c.V, c.D, rows) : tenmo_h3_partial_bytes(ctx, c.D, c.V, rows);
        if (dx > part) part = dx;
        if (dw > part) part = dw;
    }
    const size_t partial = take(part), db_scratch = take(db_sums);
    void* ws = nullptr;
    int st = tenmo_op_workspace(ctx, need, &ws);
    if (st != TENMO_OK) return st;
    uint8_t* at = (uint8_t*)ws;
    W.img = at + w_img; W.inverse = (float*)(at + w_inv);
    X.img = at + x_img; X.inverse = (float*)(at + x_inv);
    Z.img = at + z_img; Z.inverse = (float*)(at + z_inv);
    TENMO_CUDA_TRY(ctx, tenmo_launch(lce_count_kernel, 1, 1024, 0, ctx->stream, ctx->pdl, c.labels, c.is_i64, c.N, c.ignore, c.reduction,
                                     c.valid, (float*)(at + factor)));
    TENMO_LAUNCH_CHECK(ctx, "lce_count_kernel");
    const float* wp = c.w->ptr + c.w->offset;
    if ((st = tenmo_h3_make(ctx, wp, tied ? c.w->col_stride : c.w->row_stride, 1, W, nullptr, 0, 0)) != TENMO_OK) return st;
    const size_t label_bytes = c.is_i64 ? 8 : 4;
    for (int64_t r0 = 0; r0 < c.N; r0 += piece) {
        const int64_t rows = r0 + piece < c.N ? piece : c.N - r0;
        X.rows = Z.rows = rows;
        const void* labels = (const char*)c.labels + r0 * label_bytes;
        if ((st = tenmo_h3_make(ctx, c.x->ptr + c.x->offset + r0 * c.x->row_stride, c.x->row_stride, c.x->col_stride, X, labels, c.is_i64, c.ignore)) != TENMO_OK)
            return st;
        TenmoH3Epilogue e = {};
        e.C = c.grad ? (float*)Z.img : nullptr;
        e.blocked = 1;
        e.bias = c.bias;
        e.stats = (float2*)(at + stats);
        e.sums = c.ls > 0.f ? (float*)(at + sums) : nullptr;
        e.at_label = (float*)(at + at_label);
        e.labels = labels;
        e.label_is_i64 = c.is_i64;
        if ((st = tenmo_h3_gemm(ctx, rows, c.V, c.D, X, false, W, !tied, e, nullptr, 0)) != TENMO_OK) return st;
        const LceStats ps{e.stats, e.sums, e.at_label, groups, rows, r0, c.V, c.ignore, c.labels, c.upstream, (const float*)(at + factor),
                          (float*)(at + row_loss), c.grad ? (float4*)(at + numbers) : nullptr, ctx->dev_status, c.ls, c.is_i64, c.reduction};
        lce_stats_kernel<<<(unsigned)((rows + 31) / 32), 32 * LCE_STAT_WARPS, 0, ctx->stream>>>(ps);
        TENMO_LAUNCH_CHECK(ctx, "lce_stats_kernel");
        if (!c.grad) continue;
        lce_grad_kernel<<<(unsigned)Z.blocks(), 512, 0, ctx->stream>>>(Z.img, Z.inverse, ps.numbers, c.labels, c.is_i64, r0, rows, c.V, (int)vb, c.ls,
                                                                       c.db ? (float*)(at + db_part) : nullptr);
        TENMO_LAUNCH_CHECK(ctx, "lce_grad_kernel");
        TenmoH3Epilogue ex = {};
        ex.C = c.dx + r0 * c.D;
        ex.ldc = c.D;
        if ((st = tenmo_h3_gemm(ctx, rows, c.D, c.V, Z, false, W, tied, ex, at + partial, part)) != TENMO_OK) return st;
        TenmoH3Epilogue ew = {};
        ew.C = c.dw;
        ew.ldc = tied ? c.D : c.V;
        ew.add = r0 > 0;
        st = tied ? tenmo_h3_gemm(ctx, c.V, c.D, rows, Z, true, X, true, ew, at + partial, part) : tenmo_h3_gemm(ctx, c.D, c.V, rows, X, true, Z, true, ew, at + partial, part);
        if (st != TENMO_OK) return st;
        if (c.db && (st = tenmo_colsum_own(ctx, (const float*)(at + db_part), Z.block_rows(), c.V, c.V, c.db, r0 ? 1.f : 0.f, at + db_scratch)) != TENMO_OK) return st;
    }
    const int grid = c.reduction == 2 ? tenmo_stream_grid(ctx, c.N, 1024, 1) : 1;
    TENMO_CUDA_TRY(ctx, tenmo_launch(lce_loss_kernel, grid, 1024, 0, ctx->stream, ctx->pdl, (const float*)(at + row_loss), c.N, c.reduction,
                                     (const int32_t*)c.valid, c.loss));
    TENMO_LAUNCH_CHECK(ctx, "lce_loss_kernel");
    return TENMO_OK;
}

// A handful of rows: the products of linear_few.cu, which read the weight once each and write its gradient once.
int lce_run_few(tenmo_ctx* ctx, const LceCall& c) {
    const bool tied = c.w->row_stride == 1 && c.w->col_stride != 1;
    const int64_t ldw = tied ? c.w->col_stride : c.w->row_stride;
    const float* w = c.w->ptr + c.w->offset;
    size_t need = 0;
    auto take = [&](size_t bytes) { const size_t at = need; need += (bytes + 255) & ~(size_t)255; return at; };
    const size_t z_at = take((size_t)c.N * c.V * sizeof(float)), x_at = take((size_t)c.N * c.D * sizeof(float)), l_at = take(c.N * sizeof(float)), f_at = take(sizeof(float));
    size_t part = tenmo_few_bytes(ctx, c.N, c.V, c.D);
    if (c.grad && tenmo_few_bytes(ctx, c.N, c.D, c.V) > part) part = tenmo_few_bytes(ctx, c.N, c.D, c.V);
    const size_t p_at = take(part);
    void* ws = nullptr;
    int st = tenmo_op_workspace(ctx, need, &ws);
    if (st != TENMO_OK) return st;
    float *z = (float*)((char*)ws + z_at), *x = (float*)((char*)ws + x_at), *row_loss = (float*)((char*)ws + l_at), *factor = (float*)((char*)ws + f_at);
    float* partial = (float*)((char*)ws + p_at);
    TENMO_CUDA_TRY(ctx, tenmo_launch(lce_count_kernel, 1, 1024, 0, ctx->stream, ctx->pdl, c.labels, c.is_i64, c.N, c.ignore, c.reduction, c.valid, factor));
    TENMO_LAUNCH_CHECK(ctx, "lce_count_kernel");
    const int rows_grid = tenmo_stream_grid(ctx, c.N * c.D, 256, 8);
    TENMO_CUDA_TRY(ctx, tenmo_launch(lce_rows_kernel, rows_grid, 256, 0, ctx->stream, tenmo_pdl_ok(ctx, rows_grid), c.x->ptr + c.x->offset, c.x->row_stride,
                                     c.x->col_stride, c.labels, c.is_i64, c.ignore, (int64_t)0, c.N, c.D, x));
    TENMO_LAUNCH_CHECK(ctx, "lce_rows_kernel");
    st = tied ? tenmo_few_dot(ctx, x, c.D, c.N, c.D, w, ldw, c.V, c.bias, z, c.V, partial) : tenmo_few_cols(ctx, x, c.D, c.N, c.D, w, ldw, c.V, c.bias, z, c.V, partial);
    if (st != TENMO_OK) return st;
    const LceRow p{z, c.labels, row_loss, c.upstream, factor, ctx->dev_status, 0, c.V, c.ignore, c.ls, c.is_i64, c.reduction, c.grad};
    TENMO_CUDA_TRY(ctx, tenmo_launch(lce_row_kernel, (unsigned)c.N, c.V > 4096 ? 1024 : LCE_THREADS, 0, ctx->stream, tenmo_pdl_ok(ctx, c.N), p));
    TENMO_LAUNCH_CHECK(ctx, "lce_row_kernel");
    if (c.grad) {
        st = tied ? tenmo_few_cols(ctx, z, c.V, c.N, c.V, w, ldw, c.D, nullptr, c.dx, c.D, partial) : tenmo_few_dot(ctx, z, c.V, c.N, c.V, w, ldw, c.D, nullptr, c.dx, c.D, partial);
        if (st != TENMO_OK) return st;
        st = tied ? tenmo_few_outer(ctx, z, c.V, x, c.D, c.N, c.V, c.D, c.dw) : tenmo_few_outer(ctx, x, c.D, z, c.V, c.N, c.D, c.V, c.dw);
        if (st != TENMO_OK) return st;
        if (c.db && (st = tenmo_colsum_own(ctx, z, c.N, c.V, c.V, c.db, 0.f, nullptr)) != TENMO_OK) return st;
    }
    const int grid = c.reduction == 2 ? tenmo_stream_grid(ctx, c.N, 1024, 1) : 1;
    TENMO_CUDA_TRY(ctx, tenmo_launch(lce_loss_kernel, grid, 1024, 0, ctx->stream, ctx->pdl, (const float*)row_loss, c.N, c.reduction, (const int32_t*)c.valid, c.loss));
    TENMO_LAUNCH_CHECK(ctx, "lce_loss_kernel");
    return TENMO_OK;
}

// The strict-fp32 GEMM adds up the whole contraction in one chain, whose rounding grows with its length: 385,494 rows of dim 1 cost the weight's
// gradient 1.5e-4 of its norm, 160,000 classes dx 1.2e-4 (as below: 2.6e-7 and 3.6e-7).  Above 2048 the contraction is therefore cut into slices of
// 512 (longer ones where 512 slices, or the budget, do not suffice), all but the last in one batched product, and the partial results are
// added in order.  From 1024 on it would take 83 us for 79 at 1030x200x200 and 81 for 87 at 1442x72x249; 20000x50x49 takes 138 for 540.
struct LceSlices { int64_t length, count; };
LceSlices lce_slices(int64_t results, int64_t K) {
    const int64_t most = min((int64_t)TENMO_COLSUM_SEQ_ROWS, (int64_t)(LCE_PIECE_BYTES / sizeof(float)) / results);
    if (K <= 2048 || most < 2) return LceSlices{K, 1};
    const int64_t length = max((int64_t)512, (K + most - 1) / most);
    return LceSlices{length, (K + length - 1) / length};
}
size_t lce_slice_bytes(int64_t results, int64_t K) {
    const LceSlices s = lce_slices(results, K);
    return s.count > 1 ? (size_t)s.count * (size_t)results * sizeof(float) : 0;
}
// C (M, N) (+)= A . B + bias; partial: lce_slice_bytes(M * N, K)
int lce_product(tenmo_ctx* ctx, int64_t M, int64_t N, int64_t K, tenmo_mat A, tenmo_mat B, float* C, float beta, const float* bias, float* partial) {
    const LceSlices s = lce_slices(M * N, K);
    if (s.count == 1) return tenmo_gemm_f32(ctx, TENMO_ALGO_SIMT_FP32, M, N, K, &A, &B, C, beta, bias, TENMO_ACT_NONE, nullptr, nullptr);
    const int64_t before = s.count - 1;
    A.batch_rank = B.batch_rank = 1;
    A.batch_shape[0] = B.batch_shape[0] = before;
    A.batch_stride[0] = s.length * A.col_stride;
    B.batch_stride[0] = s.length * B.row_stride;
    int st = tenmo_gemm_f32(ctx, TENMO_ALGO_SIMT_FP32, M, N, s.length, &A, &B, partial, 0.f, nullptr, TENMO_ACT_NONE, nullptr, nullptr);
    if (st != TENMO_OK) return st;
    A.batch_rank = B.batch_rank = 0;
    A.offset += before * A.batch_stride[0];
    B.offset += before * B.batch_stride[0];
    st = tenmo_gemm_f32(ctx, TENMO_ALGO_SIMT_FP32, M, N, K - before * s.length, &A, &B, partial + before * M * N, 0.f, bias, TENMO_ACT_NONE, nullptr, nullptr);
    if (st != TENMO_OK) return st;
    return tenmo_colsum_own(ctx, partial, s.count, M * N, M * N, C, beta, nullptr);
}

int lce_run(tenmo_ctx* ctx, const char* who, const LceCall& c) {
    int st = check(ctx, who, c);
    if (st != TENMO_OK) return st;
    TenmoOpCall call(ctx);
    if (!ctx->op_fp32 && tc_profitable(c)) return lce_run_tc(ctx, c);
    // Up to 256 rows the kernels for a handful of rows, taken in groups of 32, keep more of the GPU busy than the strict-fp32 GEMM's tiles:
    // 204x1884x28 forward 34 us for 81, 180x855x112 training 54 for 87, 100x768x1000 training 83 for 116; level at 300x128x1000,
    // behind at 512x512x300 (155 for 89).
    if (c.N > 0 && c.N <= LCE_FEW_MOST) return lce_run_few(ctx, c);
    const int64_t piece = piece_rows(c, (size_t)c.V * sizeof(float), (size_t)c.D * sizeof(float), 128);
    const size_t z_bytes = ((size_t)piece * c.V * sizeof(float) + 255) & ~(size_t)255;
    const size_t x_bytes = ((size_t)piece * c.D * sizeof(float) + 255) & ~(size_t)255;
    const size_t l_bytes = ((size_t)c.N * sizeof(float) + 255) & ~(size_t)255, db_at = z_bytes + x_bytes + l_bytes + 256;
    const size_t db_sums = c.db && piece ? max(tenmo_colsum_own_bytes(ctx, piece, c.V), tenmo_colsum_own_bytes(ctx, c.N % piece, c.V)) : 0;
    const size_t part_at = db_at + ((db_sums + 255) & ~(size_t)255);
    size_t part = 0;
    for (int64_t rows : {piece, piece ? c.N % piece : 0}) {
        if (!rows) continue;
        part = max(part, lce_slice_bytes(rows * c.V, c.D));
        if (c.grad) part = max(part, max(lce_slice_bytes(rows * c.D, c.V), lce_slice_bytes(c.D * c.V, rows)));
    }
    void* ws = nullptr;
    if ((st = tenmo_op_workspace(ctx, part_at + part, &ws)) != TENMO_OK) return st;
    float* partial = (float*)((char*)ws + part_at);
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
        st = lce_product(ctx, rows, c.V, c.D, mx, *c.w, z, 0.f, c.bias, partial);
        if (st != TENMO_OK) return st;
        const LceRow p{z, c.labels, row_loss, c.upstream, factor, ctx->dev_status, r0, c.V, c.ignore, c.ls, c.is_i64, c.reduction, c.grad};
        lce_row_kernel<<<(unsigned)rows, c.V > 4096 ? 1024 : LCE_THREADS, 0, ctx->stream>>>(p);
        TENMO_LAUNCH_CHECK(ctx, "lce_row_kernel");
        if (!c.grad) continue;
        const float beta = r0 ? 1.f : 0.f;
        st = lce_product(ctx, rows, c.D, c.V, mz, wt, c.dx + r0 * c.D, 0.f, nullptr, partial);
        if (st != TENMO_OK) return st;
        const tenmo_mat zt = transposed(mz), xt = transposed(mx);
        st = tied ? lce_product(ctx, c.V, c.D, rows, zt, mx, c.dw, beta, nullptr, partial) : lce_product(ctx, c.D, c.V, rows, xt, mz, c.dw, beta, nullptr, partial);
        if (st != TENMO_OK) return st;
        if (c.db && (st = tenmo_colsum_own(ctx, z, rows, c.V, c.V, c.db, beta, (char*)ws + db_at)) != TENMO_OK) return st;
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
