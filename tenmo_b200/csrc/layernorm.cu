// Layer normalisation over the last axis, forward and backward, fp32.
//
//   y = (x - mean) * rstd * gamma + bias,  rstd = 1 / sqrt(var + eps),  var = mean((x - mean)^2)
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat)),  g = dy * gamma,  xhat = (x - mean) * rstd
//   dgamma[c] = sum_m dy * xhat,  dbias[c] = sum_m dy
//
// Bound: HBM.  Forward reads x and writes y (8 bytes an element), backward reads x and dy and writes dx (12 bytes); a row
// stays in registers between the loads and the stores, so each is moved once.  The variance is the mean of the squared
// differences from the mean (two sums over the registers), not E[x^2] - mean^2, which cancels.
// Split: a row belongs to as many threads as it has groups of eight columns (a warp for 256 columns, a block of up to 1024
// threads for 8192), each holding two float4.  Few registers per thread keep several rows in flight per SM, which is what
// hides the two block-wide sums; the next row is fetched before this row's.  Wider rows are walked in pieces and re-read from L2.
// Measured: forward 8192 x 4096 44 us (6.1 TB/s), 16384 x 768 18.5 us; backward 16384 x 768 33 us (4.6 TB/s) and 7 us for the column sums'
// last step; 64 x 128 (launches) 15 us for both passes.
// The column sums of the backward pass: a block keeps them in registers for the rows it takes (rows are dealt round-robin to
// a resident grid), writes one partial row, and a second kernel adds the partials in a fixed order, so that the gradients of
// gamma and bias repeat bit for bit.
#include "common.cuh"
#include "op_util.cuh"

namespace {

constexpr int LN_EPT = 8;          // elements per thread of the register-resident kernels
constexpr int LN_MAX_THREADS = 1024;

struct LnFwd {
    const float* x; const float* gamma; const float* bias; float* y; float* mean; float* rstd;
    int64_t ldx, M; int C; float eps, inv_c;
};

// Sum over the `threads` threads that share a row (a warp, or the whole block).  `slots` holds one value per warp; calls
// alternate between two sets so that one barrier per sum is enough.
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float* slots) {
    v = tenmo_warp_sum(v);
    if (WARP) return v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) slots[warp] = v;
    __syncthreads();
    return tenmo_warp_sum(lane < warps ? slots[lane] : 0.f);
}
template <bool WARP>
__device__ __forceinline__ float2 row_sum2(float a, float b, float2* slots) {
    a = tenmo_warp_sum(a);
    b = tenmo_warp_sum(b);
    if (WARP) return make_float2(a, b);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) slots[warp] = make_float2(a, b);
    __syncthreads();
    const float2 s = lane < warps ? slots[lane] : make_float2(0.f, 0.f);
    return make_float2(tenmo_warp_sum(s.x), tenmo_warp_sum(s.y));
}

// column of element e of thread t in a row shared by `threads` threads
template <bool VEC>
__device__ __forceinline__ int ln_col(int e, int t, int threads) {
    return VEC ? 4 * (t + (e >> 2) * threads) + (e & 3) : t + e * threads;
}
template <bool VEC>
__device__ __forceinline__ void ln_load(float (&v)[LN_EPT], const float* row, int C, int t, int threads) {
    if (VEC) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = 4 * (t + h * threads);
            const float4 f = c < C ? __ldg(reinterpret_cast<const float4*>(row + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
            v[4 * h] = f.x; v[4 * h + 1] = f.y; v[4 * h + 2] = f.z; v[4 * h + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < LN_EPT; ++e) {
            const int c = t + e * threads;
            v[e] = c < C ? __ldg(row + c) : 0.f;
        }
    }
}
template <bool VEC>
__device__ __forceinline__ void ln_store(const float (&v)[LN_EPT], float* row, int C, int t, int threads, bool add) {
    if (VEC) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = 4 * (t + h * threads);
            if (c < C) {
                float4 f = make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
                if (add) {
                    const float4 o = *reinterpret_cast<const float4*>(row + c);
                    f.x += o.x; f.y += o.y; f.z += o.z; f.w += o.w;
                }
                *reinterpret_cast<float4*>(row + c) = f;
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < LN_EPT; ++e) {
            const int c = t + e * threads;
            if (c < C) row[c] = add ? row[c] + v[e] : v[e];
        }
    }
}

// WARP: a block is several warps with a row each; else the block is one row.
template <bool VEC, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : LN_MAX_THREADS) ln_fwd_kernel(const LnFwd p) {
    __shared__ float slots[2][32];
    tenmo_grid_dependency_sync();
    const int t = WARP ? (threadIdx.x & 31) : threadIdx.x, threads = WARP ? 32 : blockDim.x;
    const int64_t first = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    const int64_t step = WARP ? (int64_t)gridDim.x * (blockDim.x >> 5) : gridDim.x;
    float gam[LN_EPT], bia[LN_EPT];
    ln_load<VEC>(gam, p.gamma, p.C, t, threads);
    ln_load<VEC>(bia, p.bias, p.C, t, threads);
    float next[LN_EPT];
    if (first < p.M) ln_load<VEC>(next, p.x + first * p.ldx, p.C, t, threads);
    for (int64_t m = first; m < p.M; m += step) {
        float v[LN_EPT];
#pragma unroll
        for (int e = 0; e < LN_EPT; ++e) v[e] = next[e];
        if (m + step < p.M) ln_load<VEC>(next, p.x + (m + step) * p.ldx, p.C, t, threads);  // in flight during the two sums
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < LN_EPT; ++e) s += v[e];
        const float mean = row_sum<WARP>(s, slots[0]) * p.inv_c;
        s = 0.f;
#pragma unroll
        for (int e = 0; e < LN_EPT; ++e) {
            v[e] -= mean;
            if (ln_col<VEC>(e, t, threads) < p.C) s += v[e] * v[e];
        }
        const float rstd = 1.f / sqrtf(row_sum<WARP>(s, slots[1]) * p.inv_c + p.eps);
#pragma unroll
        for (int e = 0; e < LN_EPT; ++e) v[e] = v[e] * rstd * gam[e] + bia[e];
        ln_store<VEC>(v, p.y + m * p.C, p.C, t, threads, false);
        if (t == 0) {
            if (p.mean) p.mean[m] = mean;
            if (p.rstd) p.rstd[m] = rstd;
        }
    }
}

// Rows wider than the register kernels hold: three walks over the row (the later two hit L2).
__global__ void __launch_bounds__(LN_MAX_THREADS) ln_fwd_wide_kernel(const LnFwd p) {
    __shared__ float slots[2][32];
    for (int64_t m = blockIdx.x; m < p.M; m += gridDim.x) {
        const float* x = p.x + m * p.ldx;
        float s = 0.f;
        for (int c = threadIdx.x; c < p.C; c += blockDim.x) s += __ldg(x + c);
        const float mean = row_sum<false>(s, slots[0]) * p.inv_c;
        s = 0.f;
        for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
            const float d = __ldg(x + c) - mean;
            s += d * d;
        }
        const float rstd = 1.f / sqrtf(row_sum<false>(s, slots[1]) * p.inv_c + p.eps);
        for (int c = threadIdx.x; c < p.C; c += blockDim.x)
            p.y[m * p.C + c] = (__ldg(x + c) - mean) * rstd * __ldg(p.gamma + c) + __ldg(p.bias + c);
        if (threadIdx.x == 0) {
            if (p.mean) p.mean[m] = mean;
            if (p.rstd) p.rstd[m] = rstd;
        }
    }
}

struct LnBwd {
    const float* x; const float* dy; const float* gamma; const float* mean; const float* rstd; float* dx;
    float* partial;  // [grid][2][C]: column sums of dy * xhat and of dy over the rows of a block
    int64_t ldx, M; int C; float inv_c; int add;
};

// MOST: threads of a block.  Scalar loads need more registers than 1024 threads leave (their addresses), so rows of up to 4096 have a
// kernel for 512 threads.
template <bool VEC, int MOST>
__global__ void __launch_bounds__(MOST, 1) ln_bwd_kernel(const LnBwd p) {
    constexpr bool WARP = MOST == 128;
    __shared__ float2 slots[2][32];
    extern __shared__ float fold[];  // WARP: one row pair of partials per block
    tenmo_grid_dependency_sync();
    const int t = WARP ? (threadIdx.x & 31) : threadIdx.x, threads = WARP ? 32 : blockDim.x;
    const int64_t first = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    const int64_t step = WARP ? (int64_t)gridDim.x * (blockDim.x >> 5) : gridDim.x;
    float gam[LN_EPT], dg[LN_EPT], db[LN_EPT];
    ln_load<VEC>(gam, p.gamma, p.C, t, threads);
#pragma unroll
    for (int e = 0; e < LN_EPT; ++e) dg[e] = db[e] = 0.f;
    float next_x[LN_EPT], next_g[LN_EPT], next_mean = 0.f, next_rstd = 0.f;
    auto fetch = [&](int64_t m) {
        ln_load<VEC>(next_x, p.x + m * p.ldx, p.C, t, threads);
        ln_load<VEC>(next_g, p.dy + m * p.C, p.C, t, threads);
        next_mean = __ldg(p.mean + m);
        next_rstd = __ldg(p.rstd + m);
    };
    constexpr bool AHEAD = VEC || MOST < LN_MAX_THREADS;  // a row ahead, where the registers allow it
    if (AHEAD && first < p.M) fetch(first);
    int flip = 0;
    for (int64_t m = first; m < p.M; m += step) {
        float v[LN_EPT], g[LN_EPT];
        if (!AHEAD) fetch(m);
#pragma unroll
        for (int e = 0; e < LN_EPT; ++e) {
            v[e] = next_x[e];
            g[e] = next_g[e];
        }
        const float mean = next_mean, rstd = next_rstd;
        if (AHEAD && m + step < p.M) fetch(m + step);
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int e = 0; e < LN_EPT; ++e) {
            v[e] = (v[e] - mean) * rstd;  // columns past C: dy and gamma are zero there, so nothing is added
            dg[e] += g[e] * v[e];
            db[e] += g[e];
            g[e] *= gam[e];
            a += g[e];
            b += g[e] * v[e];
        }
        const float2 s = row_sum2<WARP>(a, b, slots[flip]);
        flip ^= 1;
        const float ma = s.x * p.inv_c, mb = s.y * p.inv_c;
#pragma unroll
        for (int e = 0; e < LN_EPT; ++e) v[e] = rstd * (g[e] - ma - v[e] * mb);
        ln_store<VEC>(v, p.dx + m * p.C, p.C, t, threads, p.add != 0);
    }
    if (WARP) {  // the block's warps hold the same columns: add them in warp order
        for (int w = 0; w < (int)(blockDim.x >> 5); ++w) {
            if ((int)(threadIdx.x >> 5) == w) {
#pragma unroll
                for (int e = 0; e < LN_EPT; ++e) {
                    const int c = ln_col<VEC>(e, t, threads);
                    if (c < p.C) {
                        fold[c] = w ? fold[c] + dg[e] : dg[e];
                        fold[p.C + c] = w ? fold[p.C + c] + db[e] : db[e];
                    }
                }
            }
            __syncthreads();
        }
        float* out = p.partial + (int64_t)blockIdx.x * 2 * p.C;
        for (int c = threadIdx.x; c < 2 * p.C; c += blockDim.x) out[c] = fold[c];
    } else {
        float* out = p.partial + (int64_t)blockIdx.x * 2 * p.C;
        if (VEC) {
            ln_store<VEC>(dg, out, p.C, t, threads, false);
            ln_store<VEC>(db, out + p.C, p.C, t, threads, false);
        } else {
            ln_store<false>(dg, out, p.C, t, threads, false);
            ln_store<false>(db, out + p.C, p.C, t, threads, false);
        }
    }
}

__global__ void __launch_bounds__(LN_MAX_THREADS) ln_bwd_wide_kernel(const LnBwd p) {
    __shared__ float2 slots[2][32];
    float* out = p.partial + (int64_t)blockIdx.x * 2 * p.C;
    for (int64_t c = threadIdx.x; c < 2 * (int64_t)p.C; c += blockDim.x) out[c] = 0.f;  // (2 C + 1023 can pass 2^31)
    __syncthreads();
    int flip = 0;
    for (int64_t m = blockIdx.x; m < p.M; m += gridDim.x) {
        const float *x = p.x + m * p.ldx, *dy = p.dy + m * p.C;
        const float mean = __ldg(p.mean + m), rstd = __ldg(p.rstd + m);
        float a = 0.f, b = 0.f;
        for (int c = threadIdx.x; c < p.C; c += blockDim.x) {  // a column is always the same thread's: no race on `out`
            const float xh = (__ldg(x + c) - mean) * rstd, d = __ldg(dy + c), g = d * __ldg(p.gamma + c);
            out[c] += d * xh;
            out[p.C + c] += d;
            a += g;
            b += g * xh;
        }
        const float2 s = row_sum2<false>(a, b, slots[flip]);
        flip ^= 1;
        const float ma = s.x * p.inv_c, mb = s.y * p.inv_c;
        for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
            const float xh = (__ldg(x + c) - mean) * rstd, g = __ldg(dy + c) * __ldg(p.gamma + c);
            const float d = rstd * (g - ma - xh * mb);
            float* o = p.dx + m * p.C + c;
            *o = p.add ? *o + d : d;
        }
    }
}

// out[c] (+)= sum over the partial rows, 32 columns x 32 row groups per block, groups added in order.
__global__ void __launch_bounds__(1024) ln_fold_kernel(const float* partial, int rows, int C, float* dgamma, float* dbias, int add) {
    __shared__ float s[32][33];
    tenmo_grid_dependency_sync();
    const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;  // over 2 C columns
    float a = 0.f;
    if (c < 2 * (int64_t)C) {
        int r = grp;
        for (; r + 96 < rows; r += 128) {  // four loads in flight
            const float v0 = partial[(int64_t)r * 2 * C + c], v1 = partial[(int64_t)(r + 32) * 2 * C + c];
            const float v2 = partial[(int64_t)(r + 64) * 2 * C + c], v3 = partial[(int64_t)(r + 96) * 2 * C + c];
            a += (v0 + v1) + (v2 + v3);
        }
        for (; r < rows; r += 32) a += partial[(int64_t)r * 2 * C + c];
    }
    s[grp][lane] = a;
    __syncthreads();
    if (grp == 0 && c < 2 * (int64_t)C) {
        float v = 0.f;
#pragma unroll
        for (int g = 0; g < 32; ++g) v += s[g][lane];
        float* o = c < C ? (dgamma ? dgamma + c : nullptr) : (dbias ? dbias + (c - C) : nullptr);
        if (o) *o = add ? *o + v : v;
    }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// threads that share a row: one for every eight columns, whole warps
int row_threads(int64_t C) { return (int)(((C + LN_EPT - 1) / LN_EPT + 31) / 32 * 32); }

}  // namespace

extern "C" {

int tenmo_layernorm_fwd_f32(tenmo_ctx* ctx, const float* x, int64_t ldx, const float* gamma, const float* bias, float eps,
                            float* y, float* mean, float* rstd, int64_t M, int64_t C) {
    TENMO_CHECK_CTX(ctx);
    if (M < 0 || C < 1 || C > INT32_MAX / 2 || ldx < C)
        return tenmo_set_error(ctx, TENMO_ERR_INVALID, "layernorm_fwd: M=%lld C=%lld ldx=%lld", (long long)M, (long long)C, (long long)ldx);
    if (!(eps >= 0.f)) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "layernorm_fwd: eps must be >= 0");
    if (M == 0) return TENMO_OK;
    if (!x || !gamma || !bias || !y) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "layernorm_fwd: null pointer");
    TenmoOpCall call(ctx);
    const LnFwd p{x, gamma, bias, y, mean, rstd, ldx, M, (int)C, eps, 1.f / (float)C};
    const bool vec = C % 4 == 0 && ldx % 4 == 0 && aligned16(x) && aligned16(gamma) && aligned16(bias) && aligned16(y);
    const int threads = row_threads(C);
    if (threads > LN_MAX_THREADS) {
        ln_fwd_wide_kernel<<<tenmo_stream_grid(ctx, M, 1, 2), LN_MAX_THREADS, 0, ctx->stream>>>(p);
        TENMO_LAUNCH_CHECK(ctx, "ln_fwd_wide_kernel");
        return TENMO_OK;
    }
    const bool warp = threads == 32;
    const int block = warp ? 128 : threads;
    const int grid = tenmo_stream_grid(ctx, M, warp ? 4 : 1, 2048 / block);
    auto kernel = vec ? (warp ? ln_fwd_kernel<true, true> : ln_fwd_kernel<true, false>)
                      : (warp ? ln_fwd_kernel<false, true> : ln_fwd_kernel<false, false>);
    TENMO_CUDA_TRY(ctx, tenmo_launch(kernel, grid, block, 0, ctx->stream, tenmo_pdl_ok(ctx, grid), p));
    TENMO_LAUNCH_CHECK(ctx, "ln_fwd_kernel");
    return TENMO_OK;
}

int tenmo_layernorm_bwd_f32(tenmo_ctx* ctx, const float* x, int64_t ldx, const float* dy, const float* gamma,
                            const float* mean, const float* rstd, float* dx, float* dgamma, float* dbias, float beta, int64_t M,
                            int64_t C) {
    TENMO_CHECK_CTX(ctx);
    if (M < 0 || C < 1 || C > INT32_MAX / 2 || ldx < C)
        return tenmo_set_error(ctx, TENMO_ERR_INVALID, "layernorm_bwd: M=%lld C=%lld ldx=%lld", (long long)M, (long long)C, (long long)ldx);
    if (beta != 0.f && beta != 1.f) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "layernorm_bwd: beta must be 0 or 1");
    TenmoOpCall call(ctx);
    if (M == 0) {  // sums over no rows
        if (beta == 0.f && dgamma) TENMO_CUDA_TRY(ctx, cudaMemsetAsync(dgamma, 0, C * sizeof(float), ctx->stream));
        if (beta == 0.f && dbias) TENMO_CUDA_TRY(ctx, cudaMemsetAsync(dbias, 0, C * sizeof(float), ctx->stream));
        return TENMO_OK;
    }
    if (!x || !dy || !gamma || !mean || !rstd || !dx) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "layernorm_bwd: null pointer");
    LnBwd p{x, dy, gamma, mean, rstd, dx, nullptr, ldx, M, (int)C, 1.f / (float)C, beta != 0.f};
    const bool vec = C % 4 == 0 && ldx % 4 == 0 && aligned16(x) && aligned16(dy) && aligned16(gamma) && aligned16(dx);
    const int threads = row_threads(C);
    const bool wide = threads > LN_MAX_THREADS, warp = threads == 32;
    const int block = wide ? LN_MAX_THREADS : warp ? 128 : threads;
    const int grid = tenmo_stream_grid(ctx, M, warp ? 4 : 1, block >= 768 ? 1 : 768 / block);
    void* ws = nullptr;
    const int st = tenmo_op_workspace(ctx, (size_t)grid * 2 * (size_t)C * sizeof(float), &ws);
    if (st != TENMO_OK) return st;
    p.partial = (float*)ws;
    if (wide) {
        ln_bwd_wide_kernel<<<grid, block, 0, ctx->stream>>>(p);
    } else {
        auto kernel = vec ? (warp ? ln_bwd_kernel<true, 128> : ln_bwd_kernel<true, LN_MAX_THREADS>)
                          : (warp ? ln_bwd_kernel<false, 128> : block <= 512 ? ln_bwd_kernel<false, 512> : ln_bwd_kernel<false, LN_MAX_THREADS>);
        const size_t smem = warp ? 2 * (size_t)C * sizeof(float) : 0;
        TENMO_CUDA_TRY(ctx, tenmo_launch(kernel, grid, block, smem, ctx->stream, tenmo_pdl_ok(ctx, grid), p));
    }
    TENMO_LAUNCH_CHECK(ctx, "ln_bwd_kernel");
    if (!dgamma && !dbias) return TENMO_OK;
    const int64_t fold_grid = (2 * C + 31) / 32;
    TENMO_CUDA_TRY(ctx, tenmo_launch(ln_fold_kernel, (unsigned)fold_grid, 1024, 0, ctx->stream, tenmo_pdl_ok(ctx, fold_grid),
                                     (const float*)p.partial, grid, (int)C, dgamma, dbias, p.add));
    TENMO_LAUNCH_CHECK(ctx, "ln_fold_kernel");
    return TENMO_OK;
}

}  // extern "C"
