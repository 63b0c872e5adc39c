// Few rows against a large matrix: the head's products for a handful of tokens, where a tile of a matrix product would be mostly empty
// and the time is that of reading (or, for the weight's gradient, writing) the matrix once.
//
// Up to 32 rows ride along with every element of the matrix that is loaded (32 multiply-adds per 4 bytes is about where the
// FP32 pipe and HBM take the same time); more rows are further blocks that find the matrix in L2.  Two forms for the two axes:
//   cols  the output axis is contiguous: a lane owns four columns, the contraction goes by rows of the matrix, the few rows'
//         numbers are broadcast from shared memory; eight warps take the rows in turn and are added in order
//   dot   the contraction is contiguous: a warp owns four rows of the matrix, lanes run along them, and the 4 x 32 sums are
//         exchanged by halving at the end (a lane passes on the half it does not keep)
// Where the output axis gives too few blocks, the contraction is cut into slices that a second kernel adds in order.
// Bound: HBM, 4 bytes per element of the matrix.
// Measured (kernels of a call, cold): 64 rows of 128 x 1000, 12 us for the logits, 8 + 4 for dx, 8 for dW; 16 rows of 1318 x 44771 (236 MB), 132 us for
// the logits, 164 for dx, 100 for dW; 7 rows of 1039 x 33938 (141 MB) 47, 62 and 44.
#include "linear_few.cuh"

namespace {

constexpr int WARPS = 8;
constexpr int KC = 64;    // contraction staged at a time (cols)
constexpr int CC = 128;   // contraction staged at a time (dot)

struct FewArgs {
    const float* a; int64_t lda;
    const float* B; int64_t ldb;
    const float* bias;
    float* out; int64_t ldo;
    float* partial;  // slices > 1: (slices, N, outputs)
    int64_t N, outputs, len;  // len: contraction
    int slices, vec;
};

__device__ __forceinline__ void few_store(const FewArgs& p, int slice, int64_t n, int64_t c, float v) {
    if (p.slices > 1) p.partial[((int64_t)slice * p.N + n) * p.outputs + c] = v;
    else p.out[n * p.ldo + c] = p.bias ? v + __ldg(p.bias + c) : v;
}

// Two blocks on an SM up to 16 rows: the loads in flight are what reads the matrix fast.
template <int NR>
__global__ void __launch_bounds__(32 * WARPS, NR <= 16 ? 2 : 1) few_cols_kernel(const FewArgs p) {
    __shared__ __align__(16) float as[KC][NR + 4];  // + 4: rows stay aligned and the staging stores spread over the banks
    __shared__ __align__(16) float sum[NR][128];
    tenmo_grid_dependency_sync();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slice = blockIdx.y;
    const int64_t n0 = (int64_t)blockIdx.z * NR, c0 = (int64_t)blockIdx.x * 128;
    const int rows = (int)min((int64_t)NR, p.N - n0);
    const int64_t per = (p.len + p.slices - 1) / p.slices, begin = min(p.len, slice * per), end = min(p.len, begin + per);
    float acc[NR][4];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[n][u] = 0.f;
    // vec: this lane's columns are 4 lane ..; else lane + 32 u, which keeps scalar loads coalesced
    const float* base = p.B + c0 + (p.vec ? 4 * lane : lane);
    const bool in = c0 + 4 * lane < p.outputs;
    for (int64_t k0 = begin; k0 < end; k0 += KC) {
        const int kn = (int)min((int64_t)KC, end - k0);
        float av[NR * KC / (32 * WARPS)];
#pragma unroll
        for (int i = 0; i < NR * KC / (32 * WARPS); ++i) {
            const int e = threadIdx.x + i * 32 * WARPS, n = e / KC, k = e % KC;
            av[i] = n < rows && k < kn ? __ldg(p.a + (n0 + n) * p.lda + k0 + k) : 0.f;
        }
        float4 x[KC / WARPS];  // all of this warp's rows of the chunk are in flight
#pragma unroll
        for (int i = 0; i < KC / WARPS; ++i) {
            const int k = warp + WARPS * i;
            const float* src = base + (k0 + k) * p.ldb;
            x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k < kn) {
                if (p.vec) {
                    if (in) x[i] = __ldg(reinterpret_cast<const float4*>(src));
                } else {
                    if (c0 + lane < p.outputs) x[i].x = __ldg(src);
                    if (c0 + lane + 32 < p.outputs) x[i].y = __ldg(src + 32);
                    if (c0 + lane + 64 < p.outputs) x[i].z = __ldg(src + 64);
                    if (c0 + lane + 96 < p.outputs) x[i].w = __ldg(src + 96);
                }
            }
        }
        __syncthreads();  // the chunk before has been read
#pragma unroll
        for (int i = 0; i < NR * KC / (32 * WARPS); ++i) {
            const int e = threadIdx.x + i * 32 * WARPS;
            as[e % KC][e / KC] = av[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < KC / WARPS; ++i) {
            const float4* w4 = reinterpret_cast<const float4*>(as[warp + WARPS * i]);
            float w[NR];
#pragma unroll
            for (int n = 0; n < NR; n += 4) {
                const float4 f = w4[n / 4];
                w[n] = f.x; w[n + 1] = f.y; w[n + 2] = f.z; w[n + 3] = f.w;
            }
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                const float s = w[n];
                acc[n][0] = fmaf(s, x[i].x, acc[n][0]);
                acc[n][1] = fmaf(s, x[i].y, acc[n][1]);
                acc[n][2] = fmaf(s, x[i].z, acc[n][2]);
                acc[n][3] = fmaf(s, x[i].w, acc[n][3]);
            }
        }
    }
    for (int w = 0; w < WARPS; ++w) {  // the warps in order
        if (warp == w) {
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                if (p.vec) {
                    float4* d = reinterpret_cast<float4*>(&sum[n][4 * lane]);
                    const float4 o = w ? *d : make_float4(0.f, 0.f, 0.f, 0.f);
                    *d = make_float4(o.x + acc[n][0], o.y + acc[n][1], o.z + acc[n][2], o.w + acc[n][3]);
                } else {
#pragma unroll
                    for (int u = 0; u < 4; ++u) sum[n][lane + 32 * u] = w ? sum[n][lane + 32 * u] + acc[n][u] : acc[n][u];
                }
            }
        }
        __syncthreads();
    }
    for (int e = threadIdx.x; e < NR * 128; e += 32 * WARPS) {
        const int n = e >> 7, c = e & 127;
        if (n < rows && c0 + c < p.outputs) few_store(p, slice, n0 + n, c0 + c, sum[n][c]);
    }
}

// Two blocks on an SM up to 16 rows: the loads in flight are what reads the matrix fast.
template <int NR>
__global__ void __launch_bounds__(32 * WARPS, NR <= 16 ? 2 : 1) few_dot_kernel(const FewArgs p) {
    __shared__ __align__(16) float as[NR][CC];
    tenmo_grid_dependency_sync();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slice = blockIdx.y;
    const int64_t n0 = (int64_t)blockIdx.z * NR, r0 = ((int64_t)blockIdx.x * WARPS + warp) * 4;
    const int rows = (int)min((int64_t)NR, p.N - n0);
    // slices begin at multiples of CC, so that vectors stay aligned
    const int64_t chunks = (p.len + CC - 1) / CC, per = (chunks + p.slices - 1) / p.slices * CC;
    const int64_t begin = min(p.len, slice * per), end = min(p.len, begin + per);
    float acc[4 * NR];
#pragma unroll
    for (int e = 0; e < 4 * NR; ++e) acc[e] = 0.f;
    auto fetch = [&](int64_t c0, float4 (&x)[4]) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            x[r] = make_float4(0.f, 0.f, 0.f, 0.f);
            const int64_t c = c0 + 4 * lane;
            if (r0 + r >= p.outputs) continue;
            const float* src = p.B + (r0 + r) * p.ldb;
            if (p.vec) {
                if (c < end) x[r] = __ldg(reinterpret_cast<const float4*>(src + c));
            } else {
                if (c < end) x[r].x = __ldg(src + c);
                if (c + 1 < end) x[r].y = __ldg(src + c + 1);
                if (c + 2 < end) x[r].z = __ldg(src + c + 2);
                if (c + 3 < end) x[r].w = __ldg(src + c + 3);
            }
        }
    };
    float4 next[4];
    fetch(begin, next);
    for (int64_t c0 = begin; c0 < end; c0 += CC) {
        const int cn = (int)min((int64_t)CC, end - c0);
        float4 x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = next[r];
        float av[NR * CC / (32 * WARPS)];
#pragma unroll
        for (int i = 0; i < NR * CC / (32 * WARPS); ++i) {
            const int e = threadIdx.x + i * 32 * WARPS, n = e / CC, c = e % CC;
            av[i] = n < rows && c < cn ? __ldg(p.a + (n0 + n) * p.lda + c0 + c) : 0.f;
        }
        if (c0 + CC < end) fetch(c0 + CC, next);
        __syncthreads();  // the chunk before has been read
#pragma unroll
        for (int i = 0; i < NR * CC / (32 * WARPS); ++i) {
            const int e = threadIdx.x + i * 32 * WARPS;
            as[e / CC][e % CC] = av[i];
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const float4 s = *reinterpret_cast<const float4*>(&as[n][4 * lane]);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                acc[r * NR + n] = fmaf(s.x, x[r].x, fmaf(s.y, x[r].y, fmaf(s.z, x[r].z, fmaf(s.w, x[r].w, acc[r * NR + n]))));
        }
    }
    int n = 4 * NR, at = 0;
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) {
        if (n > 1) {
            n >>= 1;
            const bool up = (lane & w) != 0;
#pragma unroll
            for (int e = 0; e < 2 * NR; ++e)
                if (e < n) {
                    const float give = up ? acc[e] : acc[e + n], keep = up ? acc[e + n] : acc[e];
                    acc[e] = keep + __shfl_xor_sync(0xffffffffu, give, w);
                }
            at += up ? n : 0;
        } else {
            acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], w);
        }
    }
#pragma unroll
    for (int e = 0; e < 4 * NR; ++e)
        if (e < n) {
            const int r = (at + e) / NR, k = (at + e) % NR;
            if (k < rows && r0 + r < p.outputs) few_store(p, slice, n0 + k, r0 + r, acc[e]);
        }
}

__global__ void __launch_bounds__(256) few_fold_kernel(const FewArgs p) {
    tenmo_grid_dependency_sync();
    const int64_t total = p.N * p.outputs;
    for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < total; e += (int64_t)gridDim.x * blockDim.x) {
        float s = 0.f;
        for (int k = 0; k < p.slices; ++k) s += p.partial[k * total + e];
        const int64_t n = e / p.outputs, c = e % p.outputs;
        p.out[n * p.ldo + c] = p.bias ? s + __ldg(p.bias + c) : s;
    }
}

// 128 columns of the result per block, 32 of its rows at a time (`tiles` times), 4 x 4 per thread.  Up to 32 of the contraction stay for all the block's row
// tiles (b's part in shared memory; a's next part is fetched while this one is multiplied); more are taken in turn per row tile.
// Columns of a thread: 4 in a row where the result's rows are aligned, else 32 apart, so that scalar stores cover whole sectors too.
template <bool VEC>
__global__ void __launch_bounds__(256) few_outer_kernel(const float* a, int64_t lda, const float* b, int64_t ldb, int64_t N, int64_t R, int64_t C, float* out, int tiles) {
    __shared__ __align__(16) float sa[TENMO_FEW_ROWS][32], sb[TENMO_FEW_ROWS][128];
    tenmo_grid_dependency_sync();
    const int64_t first = (int64_t)blockIdx.y * (32 * tiles), c0 = (int64_t)blockIdx.x * 128;
    const int tr = (threadIdx.x >> 5) * 4, lane = threadIdx.x & 31;
    const int64_t parts = (N + TENMO_FEW_ROWS - 1) / TENMO_FEW_ROWS;
    const int64_t end = min(R, first + 32 * tiles);
    float av[4];
    auto fetch_a = [&](int64_t r0, int64_t n0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t n = n0 + (threadIdx.x >> 5) + 8 * i, r = r0 + lane;
            av[i] = n < N && r < R ? __ldg(a + n * lda + r) : 0.f;
        }
    };
    fetch_a(first, 0);
    for (int64_t r0 = first; r0 < end; r0 += 32) {
        float acc[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
        for (int64_t part = 0; part < parts; ++part) {
            const int64_t n0 = part * TENMO_FEW_ROWS;
            const int rows = (int)min((int64_t)TENMO_FEW_ROWS, N - n0);
            const bool load_b = parts > 1 || r0 == first;
            float bv[16];
            if (load_b) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {  // all loads first
                    const int n = (threadIdx.x >> 7) + 2 * i, c = threadIdx.x & 127;
                    bv[i] = n < rows && c0 + c < C ? __ldg(b + (n0 + n) * ldb + c0 + c) : 0.f;
                }
            }
            __syncthreads();  // the part before has been read
#pragma unroll
            for (int i = 0; i < 4; ++i) sa[(threadIdx.x >> 5) + 8 * i][lane] = av[i];
            if (load_b) {
#pragma unroll
                for (int i = 0; i < 16; ++i) sb[(threadIdx.x >> 7) + 2 * i][threadIdx.x & 127] = bv[i];
            }
            if (part + 1 < parts) fetch_a(r0, n0 + TENMO_FEW_ROWS);
            else if (r0 + 32 < end) fetch_a(r0 + 32, 0);
            __syncthreads();
#pragma unroll 4
            for (int n = 0; n < rows; ++n) {
                const float4 x = *reinterpret_cast<const float4*>(&sa[n][tr]);
                float4 y;
                if (VEC) y = *reinterpret_cast<const float4*>(&sb[n][4 * lane]);
                else y = make_float4(sb[n][lane], sb[n][lane + 32], sb[n][lane + 64], sb[n][lane + 96]);
                const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[i], ys[j], acc[i][j]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = r0 + tr + i;
            if (r >= R) continue;
            float* dst = out + r * C + c0;
            if (VEC) {
                if (c0 + 4 * lane < C) *reinterpret_cast<float4*>(dst + 4 * lane) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c0 + lane + 32 * j < C) dst[lane + 32 * j] = acc[i][j];
            }
        }
    }
}

int rows_per_block(int64_t N) { return N > 16 ? 32 : N > 8 ? 16 : N > 4 ? 8 : 4; }
// slices of the contraction, at least 128 long, that give every SM about three blocks
int pick_slices(const tenmo_ctx* ctx, int64_t blocks, int64_t len) {
    int64_t s = (3 * (int64_t)ctx->sm_count + blocks - 1) / blocks;
    if (s > len / 128) s = len / 128;
    if (s > 64) s = 64;
    return s < 1 ? 1 : (int)s;
}
// the larger count of the two forms, so that one size of scratch serves both
int slices_bound(const tenmo_ctx* ctx, int64_t N, int64_t outputs, int64_t len) {
    const int64_t groups = (N + rows_per_block(N) - 1) / rows_per_block(N);
    const int a = pick_slices(ctx, (outputs + 127) / 128 * groups, len), b = pick_slices(ctx, (outputs + 4 * WARPS - 1) / (4 * WARPS) * groups, len);
    return a > b ? a : b;
}

int fold(tenmo_ctx* ctx, const FewArgs& p) {
    if (p.slices == 1) return TENMO_OK;
    const int grid = tenmo_stream_grid(ctx, p.N * p.outputs, 256, 8);
    TENMO_CUDA_TRY(ctx, tenmo_launch(few_fold_kernel, (unsigned)grid, 256, 0, ctx->stream, tenmo_pdl_ok(ctx, grid), p));
    TENMO_LAUNCH_CHECK(ctx, "few_fold_kernel");
    return TENMO_OK;
}

template <typename K>
int launch(tenmo_ctx* ctx, K kernel, dim3 grid, const FewArgs& p, const char* name) {
    TENMO_CUDA_TRY(ctx, tenmo_launch(kernel, grid, 32 * WARPS, 0, ctx->stream, tenmo_pdl_ok(ctx, (int64_t)grid.x * grid.y * grid.z), p));
    TENMO_LAUNCH_CHECK(ctx, name);
    return fold(ctx, p);
}

}  // namespace

size_t tenmo_few_bytes(const tenmo_ctx* ctx, int64_t N, int64_t outputs, int64_t contraction) {
    const int s = slices_bound(ctx, N, outputs, contraction);
    return s > 1 ? (size_t)s * (size_t)N * (size_t)outputs * sizeof(float) : 0;
}

int tenmo_few_cols(tenmo_ctx* ctx, const float* a, int64_t lda, int64_t N, int64_t K, const float* B, int64_t ldb, int64_t C, const float* bias,
                   float* out, int64_t ldo, float* partial) {
    const int nr = rows_per_block(N);
    const int64_t groups = (N + nr - 1) / nr, blocks = (C + 127) / 128;
    FewArgs p{a, lda, B, ldb, bias, out, ldo, partial, N, C, K, pick_slices(ctx, blocks * groups, K), 0};
    p.vec = ldb % 4 == 0 && C % 4 == 0 && ((uintptr_t)B & 15u) == 0;
    const dim3 grid((unsigned)blocks, (unsigned)p.slices, (unsigned)groups);
    return nr == 32 ? launch(ctx, few_cols_kernel<32>, grid, p, "few_cols_kernel") : nr == 16 ? launch(ctx, few_cols_kernel<16>, grid, p, "few_cols_kernel")
         : nr == 8  ? launch(ctx, few_cols_kernel<8>, grid, p, "few_cols_kernel") : launch(ctx, few_cols_kernel<4>, grid, p, "few_cols_kernel");
}

int tenmo_few_dot(tenmo_ctx* ctx, const float* a, int64_t lda, int64_t N, int64_t C, const float* B, int64_t ldb, int64_t R, const float* bias,
                  float* out, int64_t ldo, float* partial) {
    const int nr = rows_per_block(N);
    const int64_t groups = (N + nr - 1) / nr, blocks = (R + 4 * WARPS - 1) / (4 * WARPS);
    FewArgs p{a, lda, B, ldb, bias, out, ldo, partial, N, R, C, pick_slices(ctx, blocks * groups, C), 0};
    p.vec = ldb % 4 == 0 && C % 4 == 0 && ((uintptr_t)B & 15u) == 0;
    const dim3 grid((unsigned)blocks, (unsigned)p.slices, (unsigned)groups);
    return nr == 32 ? launch(ctx, few_dot_kernel<32>, grid, p, "few_dot_kernel") : nr == 16 ? launch(ctx, few_dot_kernel<16>, grid, p, "few_dot_kernel")
         : nr == 8  ? launch(ctx, few_dot_kernel<8>, grid, p, "few_dot_kernel") : launch(ctx, few_dot_kernel<4>, grid, p, "few_dot_kernel");
}

int tenmo_few_outer(tenmo_ctx* ctx, const float* a, int64_t lda, const float* b, int64_t ldb, int64_t N, int64_t R, int64_t C, float* out) {
    // as many row tiles per block, up to eight, as leave every SM four blocks: 44771 x 1318 of 16 rows 100 us with eight
    const int64_t gx = (C + 127) / 128, fit = gx * ((R + 31) / 32) / (4 * (int64_t)ctx->sm_count);
    const int tiles = fit > 8 ? 8 : fit < 1 ? 1 : (int)fit;
    const int64_t TILE = 32 * tiles, gy = (R + TILE - 1) / TILE;
    if (gy > 65535) {  // the grid's second axis: in parts
        for (int64_t r = 0; r < R; r += 65535 * TILE) {
            const int st = tenmo_few_outer(ctx, a + r, lda, b, ldb, N, R - r < 65535 * TILE ? R - r : 65535 * TILE, C, out + r * C);
            if (st != TENMO_OK) return st;
        }
        return TENMO_OK;
    }
    const bool vec = C % 4 == 0 && ((uintptr_t)out & 15u) == 0;
    TENMO_CUDA_TRY(ctx, tenmo_launch(vec ? few_outer_kernel<true> : few_outer_kernel<false>, dim3((unsigned)gx, (unsigned)gy), 256, 0, ctx->stream,
                                     tenmo_pdl_ok(ctx, gx * gy), a, lda, b, ldb, N, R, C, out, tiles));
    TENMO_LAUNCH_CHECK(ctx, "few_outer_kernel");
    return TENMO_OK;
}
