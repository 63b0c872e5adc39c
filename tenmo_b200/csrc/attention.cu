// Attention without a score matrix in memory, fp32: entry points and the kernels for small problems.
//
//   s_ij = scale * q_i . k_j  over the visible keys j of row i;  m_i = max_j s_ij;  l_i = sum_j exp(s_ij - m_i)
//   o_i  = sum_j exp(s_ij - m_i) v_j / l_i
//   p_ij = exp(s_ij - m_i) / l_i;  dv_j = sum_i p_ij go_i;  delta_i = go_i . o_i
//   ds_ij = scale * p_ij (go_i . v_j - delta_i);  dq_i = sum_j ds_ij k_j;  dk_j = sum_i ds_ij q_i
// A key / value head serves H / Hkv query heads; its gradients sum over them.  Key j is visible to row i when
// j < k_lengths[b], i < q_lengths[b] and, if causal, j <= i + Sk - Sq.  A row that sees nothing gives o = 0 and no gradient.
//
// The backward pass recomputes the probabilities from q, k and the two saved numbers per row, m_i and l_i (kept apart: with
// their sum, the log-sum-exp, a large m would cost p its last bits).
//
// Kernels here, without tensor cores: the forward pass for few rows (one new token against a long cache, small problems), and
// the backward pass of small problems with one warp per row, scores 32 keys at a time (a lane is a key) and the weighted sum
// with a lane per column.  No large tile is filled, so small problems finish in one launch latency per pass.
#include "attention_tc.cuh"

#include <cfloat>

namespace {

constexpr int ROW_WARPS = 4;
constexpr int DSLOTS = TENMO_ATTN_MAX_DIM / 32;

// dot product of a row in shared memory (broadcast) and a row in global memory (this lane's)
__device__ __forceinline__ float dot_row(const float* sh, const float* g, int D, bool vec) {
    float a = 0.f, b = 0.f;
    if (vec) {
        for (int d = 0; d < D; d += 4) {
            const float4 x = *reinterpret_cast<const float4*>(sh + d);
            const float4 y = __ldg(reinterpret_cast<const float4*>(g + d));
            a = fmaf(x.x, y.x, a);
            b = fmaf(x.y, y.y, b);
            a = fmaf(x.z, y.z, a);
            b = fmaf(x.w, y.w, b);
        }
    } else {
        for (int d = 0; d < D; ++d) a = fmaf(sh[d], __ldg(g + d), a);
    }
    return a + b;
}
__device__ __forceinline__ bool row_vec(const TenmoHeadsView& v, int D) {
    return D % 4 == 0 && v.sb % 4 == 0 && v.sh % 4 == 0 && v.sr % 4 == 0 && ((uintptr_t)v.ptr & 15u) == 0;
}
// keys that row i of batch entry b sees: the first n
__device__ __forceinline__ int visible_keys(const TenmoAttnParams& p, int b, int i) {
    if (i >= tenmo_attn_rows(p.q_lengths, b, p.Sq)) return 0;
    int n = tenmo_attn_rows(p.k_lengths, b, p.Sk);
    if (p.causal) n = min(n, max(0, i + p.Sk - p.Sq + 1));
    return n;
}

// (b, h, i) of a warp's row; false past the end
__device__ __forceinline__ bool warp_row(int64_t rows_per_head, int heads, int64_t total, int* b, int* h, int* i) {
    const int64_t r = (int64_t)blockIdx.x * ROW_WARPS + (threadIdx.x >> 5);
    if (r >= total) return false;
    *i = (int)(r % rows_per_head);
    const int64_t bh = r / rows_per_head;
    *h = (int)(bh % heads);
    *b = (int)(bh / heads);
    return true;
}

// ---------------------------------------------------------------------------------------------------------------------
// Forward with few rows: R rows of a key/value head (its query heads' rows, flattened) against a slice of the keys.
// A lane holds four columns; LPK lanes are a row of k or v, so a warp's load covers 32 / LPK whole rows.  Scores: partial dot products of
// eight loads, summed over the lanes by halving (a lane passes on the half it does not keep: V shuffles for V sums instead of
// log2(LPK) V).  The exponentials of 32 keys are taken with a lane per key, and go through shared memory to be multiplied with v.
// Four warps take 32 keys (16 above 32 columns) in turn and are joined at the end; with few rows and many keys the keys are cut into slices, one block
// each, which attn_join_kernel adds in order.
// Bound: HBM for one token (k and v are read once, 16 bytes a lane), launch latency for the smallest calls.
// Measured: 16 requests of one token, 16 heads on 4, dim 64, up to 4099 keys (97 MB): 34 us and 8 us to join, 2.8 TB/s: the chain of a step (dot
// products, sums over the lanes, maximum, exponentials, weighted sum, some 2000 cycles) with 12 warps on an SM.  Loading a step ahead did
// not help.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int FEW_WARPS = 4;
struct FewParams {
    TenmoAttnParams a;
    int groups, slices;   // row groups of a key/value head, slices of the keys
    int k_vec, v_vec;
    float* partial;       // slices > 1: per (b, h, i, slice): D sums, then m, l
    int ldp;
};

// row rr of a key/value head: query head and position
__device__ __forceinline__ void few_row(const TenmoAttnParams& p, int kvh, int rr, int* h, int* i) {
    *h = kvh * (p.H / p.Hkv) + rr / p.Sq;
    *i = rr % p.Sq;
}

template <int LPK, int R>
__global__ void __launch_bounds__(FEW_WARPS * 32) attn_fwd_few_kernel(const FewParams f) {
    constexpr int KPL = 32 / LPK, V = 8 * R;           // rows per load; partial sums of eight loads
    constexpr int LOADS = LPK == 32 ? 16 : 8, KEYS = LOADS * KPL;  // of a warp at a time: 32 keys, 16 above 32 columns
    __shared__ __align__(16) float pk[FEW_WARPS][32 * R];
    __shared__ __align__(16) float so[FEW_WARPS][R][4 * LPK];
    __shared__ float sm[FEW_WARPS][R], sl[FEW_WARPS][R];
    const TenmoAttnParams& p = f.a;
    tenmo_grid_dependency_sync();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l4 = 4 * (lane % LPK), sub = lane / LPK;
    const int slice = blockIdx.x % f.slices, gi = blockIdx.x / f.slices;
    const int group = gi % f.groups, kvh = gi / f.groups % p.Hkv, b = gi / f.groups / p.Hkv;
    const int total = p.H / p.Hkv * p.Sq, row0 = group * R;
    float4 q[R];
    int seen[R], most = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        seen[r] = 0;
        q[r] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row0 + r < total) {
            int h, i;
            few_row(p, kvh, row0 + r, &h, &i);
            seen[r] = visible_keys(p, b, i);
            most = max(most, seen[r]);
            const float* src = p.q.ptr + b * p.q.sb + h * p.q.sh + i * p.q.sr;
            if (seen[r]) {
                if (l4 < p.D) q[r].x = __ldg(src + l4);
                if (l4 + 1 < p.D) q[r].y = __ldg(src + l4 + 1);
                if (l4 + 2 < p.D) q[r].z = __ldg(src + l4 + 2);
                if (l4 + 3 < p.D) q[r].w = __ldg(src + l4 + 3);
            }
        }
    }
    // this block's keys: whole groups of what its warps take at a time
    constexpr int ALL = KEYS * FEW_WARPS;
    const int per = ((most + f.slices - 1) / f.slices + ALL - 1) / ALL * ALL;
    const int begin = min(most, slice * per), end = min(most, begin + per);
    const float* k = p.k.ptr + b * p.k.sb + kvh * p.k.sh;
    const float* v = p.v.ptr + b * p.v.sb + kvh * p.v.sh;
    auto load = [&](const float* base, int64_t stride, int j, bool vec) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (j < end) {
            const float* src = base + j * stride + l4;
            if (vec) {
                if (l4 < p.D) x = __ldg(reinterpret_cast<const float4*>(src));
            } else {
                if (l4 < p.D) x.x = __ldg(src);
                if (l4 + 1 < p.D) x.y = __ldg(src + 1);
                if (l4 + 2 < p.D) x.z = __ldg(src + 2);
                if (l4 + 3 < p.D) x.w = __ldg(src + 3);
            }
        }
        return x;
    };
    float m[R], l[R];
    float4 o[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
        o[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float* const mine = pk[warp];
    for (int j0 = begin + KEYS * warp; j0 < end; j0 += KEYS * FEW_WARPS) {
        float4 xk[LOADS], xv[LOADS];  // the rows of k and of v are all in flight before the first is used
#pragma unroll
        for (int t = 0; t < LOADS; ++t) xk[t] = load(k, p.k.sr, j0 + t * KPL + sub, f.k_vec);
#pragma unroll
        for (int t = 0; t < LOADS; ++t) xv[t] = load(v, p.v.sr, j0 + t * KPL + sub, f.v_vec);
#pragma unroll
        for (int t0 = 0; t0 < LOADS; t0 += 8) {
            float s[V];
#pragma unroll
            for (int t = 0; t < 8; ++t)
#pragma unroll
                for (int r = 0; r < R; ++r)
                    s[t * R + r] = fmaf(xk[t0 + t].x, q[r].x, xk[t0 + t].y * q[r].y) + fmaf(xk[t0 + t].z, q[r].z, xk[t0 + t].w * q[r].w);
            int n = V, at = 0;
#pragma unroll
            for (int w = LPK / 2; w > 0; w >>= 1) {
                if (n > 1) {
                    n >>= 1;
                    const bool up = (lane & w) != 0;
#pragma unroll
                    for (int e = 0; e < V / 2; ++e)
                        if (e < n) {
                            const float give = up ? s[e] : s[e + n], keep = up ? s[e + n] : s[e];
                            s[e] = keep + __shfl_xor_sync(0xffffffffu, give, w);
                        }
                    at += up ? n : 0;
                } else {
                    s[0] += __shfl_xor_sync(0xffffffffu, s[0], w);
                }
            }
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (e < n) {
                    const int t = (at + e) / R, r = (at + e) % R;
                    mine[((t0 + t) * KPL + sub) * R + r] = s[e];
                }
        }
        __syncwarp();
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float s = lane < KEYS && j0 + lane < min(end, seen[r]) ? mine[(lane % KEYS) * R + r] * p.scale_log2 : -INFINITY;
            const float top = fmaxf(m[r], tenmo_warp_max(s));
            const float base = top == -INFINITY ? 0.f : top;  // every score so far is -inf
            const float e = exp2f(s - base), shrink = exp2f(m[r] - base);
            m[r] = top;
            l[r] = l[r] * shrink + e;
            o[r].x *= shrink; o[r].y *= shrink; o[r].z *= shrink; o[r].w *= shrink;
            if (lane < KEYS) mine[lane * R + r] = e;
        }
        __syncwarp();
#pragma unroll
        for (int t = 0; t < LOADS; ++t) {
            const float* w = mine + (t * KPL + sub) * R;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                o[r].x = fmaf(w[r], xv[t].x, o[r].x);
                o[r].y = fmaf(w[r], xv[t].y, o[r].y);
                o[r].z = fmaf(w[r], xv[t].z, o[r].z);
                o[r].w = fmaf(w[r], xv[t].w, o[r].w);
            }
        }
        __syncwarp();
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        l[r] = tenmo_warp_sum(l[r]);
#pragma unroll
        for (int w = LPK; w < 32; w <<= 1) {
            o[r].x += __shfl_xor_sync(0xffffffffu, o[r].x, w);
            o[r].y += __shfl_xor_sync(0xffffffffu, o[r].y, w);
            o[r].z += __shfl_xor_sync(0xffffffffu, o[r].z, w);
            o[r].w += __shfl_xor_sync(0xffffffffu, o[r].w, w);
        }
        if (sub == 0) *reinterpret_cast<float4*>(&so[warp][r][l4]) = o[r];
        if (lane == 0) { sm[warp][r] = m[r]; sl[warp][r] = l[r]; }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < R * 4 * LPK; e += FEW_WARPS * 32) {
        const int r = e / (4 * LPK), d = e % (4 * LPK);
        if (row0 + r >= total) continue;
        float top = -INFINITY, sum = 0.f, x = 0.f;
#pragma unroll
        for (int w = 0; w < FEW_WARPS; ++w) top = fmaxf(top, sm[w][r]);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < FEW_WARPS; ++w) {
            const float s = exp2f(sm[w][r] - base);
            sum = fmaf(sl[w][r], s, sum);
            x = fmaf(so[w][r][d], s, x);
        }
        int h, i;
        few_row(p, kvh, row0 + r, &h, &i);
        const int64_t row = ((int64_t)b * p.H + h) * p.Sq + i;
        if (f.slices > 1) {
            float* dst = f.partial + (row * f.slices + slice) * f.ldp;
            if (d < p.D) dst[d] = x;
            if (d == 0) { dst[p.D] = top; dst[p.D + 1] = sum; }
        } else {
            // the sum is 0 for a row without visible keys (or with all scores -inf): its output is 0.  A NaN sum stays NaN.
            if (d < p.D) p.o.ptr[b * p.o.sb + h * p.o.sh + i * p.o.sr + d] = sum == 0.f ? 0.f : x / sum;
            if (d == 0 && p.stats) { p.stats[2 * row] = top; p.stats[2 * row + 1] = sum; }
        }
    }
}

// A warp joins the slices of a row, in order.
__global__ void __launch_bounds__(128) attn_join_kernel(const FewParams f) {
    tenmo_grid_dependency_sync();
    const TenmoAttnParams& p = f.a;
    int b, h, i;
    if (!warp_row(p.Sq, p.H, (int64_t)p.B * p.H * p.Sq, &b, &h, &i)) return;
    const int lane = threadIdx.x & 31;
    const int64_t row = ((int64_t)b * p.H + h) * p.Sq + i;
    const float* src = f.partial + row * f.slices * f.ldp;
    // a lane per slice (at most 64) for the weights, then a lane per column
    float ms[2], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        ms[u] = lane + 32 * u < f.slices ? src[(lane + 32 * u) * f.ldp + p.D] : -INFINITY;
        top = fmaxf(top, ms[u]);
    }
    top = tenmo_warp_max(top);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        ms[u] = exp2f(ms[u] - base);
        if (lane + 32 * u < f.slices) sum = fmaf(src[(lane + 32 * u) * f.ldp + p.D + 1], ms[u], sum);
    }
    sum = tenmo_warp_sum(sum);
    float x[DSLOTS];
#pragma unroll
    for (int t = 0; t < DSLOTS; ++t) x[t] = 0.f;
#pragma unroll 4
    for (int s = 0; s < f.slices; ++s) {
        const float w = __shfl_sync(0xffffffffu, s < 32 ? ms[0] : ms[1], s & 31);
#pragma unroll
        for (int t = 0; t < DSLOTS; ++t)
            if (lane + 32 * t < p.D) x[t] = fmaf(src[s * f.ldp + lane + 32 * t], w, x[t]);
    }
    float* o = p.o.ptr + b * p.o.sb + h * p.o.sh + i * p.o.sr;
#pragma unroll
    for (int t = 0; t < DSLOTS; ++t)
        if (lane + 32 * t < p.D) o[lane + 32 * t] = sum == 0.f ? 0.f : x[t] / sum;
    if (p.stats && lane == 0) { p.stats[2 * row] = top; p.stats[2 * row + 1] = sum; }
}

// probability from the recomputed score and the saved (maximum, sum); scores whose rounding exceeds 1 stay at the maximum's probability
__device__ __forceinline__ float prob(float s_log2, float m, float inv_l) {
    const float e = exp2f(s_log2 - m);
    return (e > 1.f ? 1.f : e) * inv_l;
}

__global__ void __launch_bounds__(ROW_WARPS * 32) attn_bwd_dq_row_kernel(const TenmoAttnParams p) {
    __shared__ __align__(16) float sq[ROW_WARPS][TENMO_ATTN_MAX_DIM], sg[ROW_WARPS][TENMO_ATTN_MAX_DIM];
    tenmo_grid_dependency_sync();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int b, h, i;
    if (!warp_row(p.Sq, p.H, (int64_t)p.B * p.H * p.Sq, &b, &h, &i)) return;
    const int kvh = h / (p.H / p.Hkv);
    const float* q = p.q.ptr + b * p.q.sb + h * p.q.sh + i * p.q.sr;
    const float* go = p.go.ptr + b * p.go.sb + h * p.go.sh + i * p.go.sr;
    const float* o = p.o.ptr + b * p.o.sb + h * p.o.sh + i * p.o.sr;
    const float* k = p.k.ptr + b * p.k.sb + kvh * p.k.sh;
    const float* v = p.v.ptr + b * p.v.sb + kvh * p.v.sh;
    const bool vk = row_vec(p.k, p.D), vv = row_vec(p.v, p.D);
    float delta = 0.f;
    for (int d = lane; d < p.D; d += 32) {
        sq[warp][d] = __ldg(q + d);
        const float g = __ldg(go + d);
        sg[warp][d] = g;
        delta = fmaf(g, __ldg(o + d), delta);
    }
    delta = tenmo_warp_sum(delta);
    __syncwarp();
    const int64_t r = ((int64_t)b * p.H + h) * p.Sq + i;
    const float m = __ldg(p.stats + 2 * r), l = __ldg(p.stats + 2 * r + 1);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int n = l == 0.f ? 0 : visible_keys(p, b, i);
    if (lane == 0) p.delta[r] = delta;
    float acc[DSLOTS];
#pragma unroll
    for (int t = 0; t < DSLOTS; ++t) acc[t] = 0.f;
    for (int j0 = 0; j0 < n; j0 += 32) {
        const int j = j0 + lane;
        float ds = 0.f;
        if (j < n) {
            const float pr = prob(dot_row(sq[warp], k + j * p.k.sr, p.D, vk) * p.scale_log2, m, inv);
            ds = pr * (dot_row(sg[warp], v + j * p.v.sr, p.D, vv) - delta) * p.scale;
        }
        const int cnt = min(32, n - j0);
#pragma unroll 8
        for (int jj = 0; jj < cnt; ++jj) {
            const float w = __shfl_sync(0xffffffffu, ds, jj);
            const float* row = k + (j0 + jj) * p.k.sr;
#pragma unroll
            for (int t = 0; t < DSLOTS; ++t) {
                const int d = lane + 32 * t;
                if (d < p.D) acc[t] = fmaf(w, __ldg(row + d), acc[t]);
            }
        }
    }
    float* dq = p.dq.ptr + b * p.dq.sb + h * p.dq.sh + i * p.dq.sr;
#pragma unroll
    for (int t = 0; t < DSLOTS; ++t) {
        const int d = lane + 32 * t;
        if (d < p.D) dq[d] = p.beta != 0.f ? dq[d] + acc[t] : acc[t];
    }
}

__global__ void __launch_bounds__(ROW_WARPS * 32) attn_bwd_dkv_row_kernel(const TenmoAttnParams p) {
    __shared__ __align__(16) float sk[ROW_WARPS][TENMO_ATTN_MAX_DIM], sv[ROW_WARPS][TENMO_ATTN_MAX_DIM];
    tenmo_grid_dependency_sync();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int b, kvh, j;
    if (!warp_row(p.Sk, p.Hkv, (int64_t)p.B * p.Hkv * p.Sk, &b, &kvh, &j)) return;
    const int group = p.H / p.Hkv;
    const float* k = p.k.ptr + b * p.k.sb + kvh * p.k.sh + j * p.k.sr;
    const float* v = p.v.ptr + b * p.v.sb + kvh * p.v.sh + j * p.v.sr;
    for (int d = lane; d < p.D; d += 32) {
        sk[warp][d] = __ldg(k + d);
        sv[warp][d] = __ldg(v + d);
    }
    __syncwarp();
    float ak[DSLOTS], av[DSLOTS];
#pragma unroll
    for (int t = 0; t < DSLOTS; ++t) ak[t] = av[t] = 0.f;
    const bool vq = row_vec(p.q, p.D), vg = row_vec(p.go, p.D);
    const int rows = tenmo_attn_rows(p.q_lengths, b, p.Sq);
    const bool seen = j < tenmo_attn_rows(p.k_lengths, b, p.Sk);
    const int first = p.causal ? max(0, j - (p.Sk - p.Sq)) : 0;
    for (int h = kvh * group; seen && h < (kvh + 1) * group; ++h) {
        const float* q = p.q.ptr + b * p.q.sb + h * p.q.sh;
        const float* go = p.go.ptr + b * p.go.sb + h * p.go.sh;
        const int64_t r0 = ((int64_t)b * p.H + h) * p.Sq;
        for (int i0 = first; i0 < rows; i0 += 32) {
            const int i = i0 + lane;
            float pr = 0.f, ds = 0.f;
            if (i < rows) {
                const float m = __ldg(p.stats + 2 * (r0 + i)), l = __ldg(p.stats + 2 * (r0 + i) + 1);
                if (l != 0.f) {
                    pr = prob(dot_row(sk[warp], q + i * p.q.sr, p.D, vq) * p.scale_log2, m, 1.f / l);
                    ds = pr * (dot_row(sv[warp], go + i * p.go.sr, p.D, vg) - __ldg(p.delta + r0 + i)) * p.scale;
                }
            }
            const int cnt = min(32, rows - i0);
#pragma unroll 8
            for (int ii = 0; ii < cnt; ++ii) {
                const float wp = __shfl_sync(0xffffffffu, pr, ii), wd = __shfl_sync(0xffffffffu, ds, ii);
                const float* rq = q + (i0 + ii) * p.q.sr;
                const float* rg = go + (i0 + ii) * p.go.sr;
#pragma unroll
                for (int t = 0; t < DSLOTS; ++t) {
                    const int d = lane + 32 * t;
                    if (d < p.D) {
                        ak[t] = fmaf(wd, __ldg(rq + d), ak[t]);
                        av[t] = fmaf(wp, __ldg(rg + d), av[t]);
                    }
                }
            }
        }
    }
    float* dk = p.dk.ptr + b * p.dk.sb + kvh * p.dk.sh + j * p.dk.sr;
    float* dv = p.dv.ptr + b * p.dv.sb + kvh * p.dv.sh + j * p.dv.sr;
#pragma unroll
    for (int t = 0; t < DSLOTS; ++t) {
        const int d = lane + 32 * t;
        if (d < p.D) {
            dk[d] = p.beta != 0.f ? dk[d] + ak[t] : ak[t];
            dv[d] = p.beta != 0.f ? dv[d] + av[t] : av[t];
        }
    }
}

template <int R>
int few_launch(tenmo_ctx* ctx, const FewParams& f, int64_t grid) {
    auto go = [&](auto kernel) -> int {
        TENMO_CUDA_TRY(ctx, tenmo_launch(kernel, (unsigned)grid, FEW_WARPS * 32, 0, ctx->stream, tenmo_pdl_ok(ctx, grid), f));
        TENMO_LAUNCH_CHECK(ctx, "attn_fwd_few_kernel");
        return TENMO_OK;
    };
    return f.a.D <= 32 ? go(attn_fwd_few_kernel<8, R>) : f.a.D <= 64 ? go(attn_fwd_few_kernel<16, R>) : go(attn_fwd_few_kernel<32, R>);
}

int few_fwd(tenmo_ctx* ctx, const TenmoAttnParams& p) {
    FewParams f = {};
    f.a = p;
    const int64_t total = (int64_t)(p.H / p.Hkv) * p.Sq;
    const int R = total >= 8 ? 8 : total >= 3 ? 4 : total == 2 ? 2 : 1;
    const int64_t groups = (total + R - 1) / R, blocks = groups * p.Hkv * p.B;
    if (groups > INT32_MAX || blocks > INT32_MAX / 64) return tenmo_set_error(ctx, TENMO_ERR_UNSUPPORTED, "attention_fwd: too many rows in one call");
    f.groups = (int)groups;
    // slices of at least 256 keys, as many as it takes to fill every SM once (by registers: two blocks of eight rows, three of four,
    // four of fewer), rounded up: the last few blocks may start in a second round (four of 448 in the following case).  16 requests of one token against 4099 keys, 16 heads on 4: 45 us for 49 with eight blocks per SM.
    int64_t slices = ((R == 8 ? 2 : R == 4 ? 3 : 4) * (int64_t)ctx->sm_count + blocks - 1) / blocks;
    if (slices > p.Sk / 256) slices = p.Sk / 256;
    if (slices > 64) slices = 64;
    if (slices < 1) slices = 1;
    f.slices = (int)slices;
    f.k_vec = tenmo_attn_row_vec(p.k, p.D);
    f.v_vec = tenmo_attn_row_vec(p.v, p.D);
    f.ldp = p.D + 2;
    int st;
    if (slices > 1) {
        void* ws = nullptr;
        if ((st = tenmo_op_workspace(ctx, (size_t)p.B * p.H * p.Sq * slices * f.ldp * sizeof(float), &ws)) != TENMO_OK) return st;
        f.partial = (float*)ws;
    }
    const int64_t grid = blocks * slices;
    st = R == 8 ? few_launch<8>(ctx, f, grid) : R == 4 ? few_launch<4>(ctx, f, grid) : R == 2 ? few_launch<2>(ctx, f, grid) : few_launch<1>(ctx, f, grid);
    if (st != TENMO_OK || slices == 1) return st;
    const int64_t join = ((int64_t)p.B * p.H * p.Sq + ROW_WARPS - 1) / ROW_WARPS;
    TENMO_CUDA_TRY(ctx, tenmo_launch(attn_join_kernel, (unsigned)join, ROW_WARPS * 32, 0, ctx->stream, tenmo_pdl_ok(ctx, join), f));
    TENMO_LAUNCH_CHECK(ctx, "attn_join_kernel");
    return TENMO_OK;
}

int check_shape(tenmo_ctx* ctx, const char* who, const tenmo_attn_shape* s, float scale, TenmoAttnParams* p) {
    if (!s) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: shape is NULL", who);
    if (s->batch < 0 || s->heads < 1 || s->kv_heads < 1 || s->q_len < 0 || s->k_len < 0 || s->dim < 1)
        return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: batch %lld, heads %lld / %lld, lengths %lld / %lld, dim %lld", who,
                               (long long)s->batch, (long long)s->heads, (long long)s->kv_heads, (long long)s->q_len,
                               (long long)s->k_len, (long long)s->dim);
    if (s->heads % s->kv_heads)
        return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: %lld query heads are not a multiple of %lld key/value heads", who,
                               (long long)s->heads, (long long)s->kv_heads);
    if (s->dim > TENMO_ATTN_MAX_DIM)
        return tenmo_set_error(ctx, TENMO_ERR_UNSUPPORTED, "%s: head dimension %lld is above %d", who, (long long)s->dim,
                               TENMO_ATTN_MAX_DIM);
    const int64_t lim = (int64_t)1 << 30;
    if (s->batch > lim || s->heads > 65535 || s->q_len > lim || s->k_len > lim || s->batch * s->heads > lim)
        return tenmo_set_error(ctx, TENMO_ERR_UNSUPPORTED, "%s: sizes beyond 2^30 rows", who);
    const int64_t longest = s->q_len > s->k_len ? s->q_len : s->k_len;
    if (s->batch * s->heads * longest >= ((int64_t)1 << 32))
        return tenmo_set_error(ctx, TENMO_ERR_UNSUPPORTED, "%s: more than 2^32 rows in one call", who);
    if (!(fabsf(scale) <= FLT_MAX / 2)) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: scale is not finite, or too large", who);
    p->B = (int)s->batch; p->H = (int)s->heads; p->Hkv = (int)s->kv_heads;
    p->Sq = (int)s->q_len; p->Sk = (int)s->k_len; p->D = (int)s->dim;
    p->scale = scale;
    p->scale_log2 = (float)((double)scale * 1.4426950408889634074);
    return TENMO_OK;
}

int take_view(tenmo_ctx* ctx, const char* who, const char* name, const tenmo_heads* t, bool needed, bool output, int64_t batch, int64_t heads,
              int64_t rows, int64_t dim, TenmoHeadsView* v) {
    if (!t || (!t->ptr && needed)) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: %s is NULL", who, name);
    if (t->batch_stride < 0 || t->head_stride < 0 || t->row_stride < 0)
        return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: %s has a negative stride", who, name);
    // an output's rows must not overlap: several blocks would write (or, with beta, add to) the same places.  From the smallest
    // stride up, each axis has to step over all that the axes before it cover.
    if (output && needed) {
        struct { int64_t n, stride; } axis[3] = {{batch, t->batch_stride}, {heads, t->head_stride}, {rows, t->row_stride}};
        for (int pass = 0; pass < 2; ++pass)
            for (int e = 0; e < 2; ++e)
                if (axis[e].stride > axis[e + 1].stride) {
                    const auto swap = axis[e];
                    axis[e] = axis[e + 1];
                    axis[e + 1] = swap;
                }
        int64_t covered = dim;
        for (int e = 0; e < 3; ++e) {
            if (axis[e].n <= 1) continue;
            if (axis[e].stride < covered)
                return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: rows of %s overlap (strides %lld, %lld, %lld)", who, name,
                                       (long long)t->batch_stride, (long long)t->head_stride, (long long)t->row_stride);
            if (axis[e].stride > (INT64_MAX - covered) / (axis[e].n - 1))
                return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: strides of %s are too large", who, name);
            covered += axis[e].stride * (axis[e].n - 1);
        }
    }
    *v = TenmoHeadsView{t->ptr, t->batch_stride, t->head_stride, t->row_stride};
    return TENMO_OK;
}

}  // namespace

extern "C" {

int tenmo_attention_fwd_f32(tenmo_ctx* ctx, const tenmo_attn_shape* shape, const tenmo_heads* q, const tenmo_heads* k,
                            const tenmo_heads* v, const tenmo_heads* o, float* stats, float scale, int causal,
                            const int32_t* q_lengths, const int32_t* k_lengths) {
    TENMO_CHECK_CTX(ctx);
    const char* who = "attention_fwd";
    TenmoAttnParams p = {};
    int st = check_shape(ctx, who, shape, scale, &p);
    if (st != TENMO_OK) return st;
    const bool any_q = p.B && p.Sq, any_k = p.B && p.Sk && p.Sq;
    if ((st = take_view(ctx, who, "q", q, any_k, false, p.B, p.H, p.Sq, p.D, &p.q)) != TENMO_OK) return st;
    if ((st = take_view(ctx, who, "k", k, any_k, false, p.B, p.Hkv, p.Sk, p.D, &p.k)) != TENMO_OK) return st;
    if ((st = take_view(ctx, who, "v", v, any_k, false, p.B, p.Hkv, p.Sk, p.D, &p.v)) != TENMO_OK) return st;
    if ((st = take_view(ctx, who, "o", o, any_q, true, p.B, p.H, p.Sq, p.D, &p.o)) != TENMO_OK) return st;
    if (!any_q) return TENMO_OK;
    if (any_k && (o->ptr == q->ptr || o->ptr == k->ptr || o->ptr == v->ptr))
        return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: o is one of the inputs", who);
    p.stats = stats;
    p.causal = causal != 0;
    p.q_lengths = q_lengths;
    p.k_lengths = k_lengths;
    TenmoOpCall call(ctx);
    if (!ctx->op_fp32 && tenmo_attn_tc_profitable(p, false)) return tenmo_attn_tc_fwd(ctx, p);
    return few_fwd(ctx, p);
}

int tenmo_attention_bwd_f32(tenmo_ctx* ctx, const tenmo_attn_shape* shape, const tenmo_heads* q, const tenmo_heads* k,
                            const tenmo_heads* v, const tenmo_heads* o, const float* stats, const tenmo_heads* go,
                            const tenmo_heads* dq, const tenmo_heads* dk, const tenmo_heads* dv, float beta, float scale,
                            int causal, const int32_t* q_lengths, const int32_t* k_lengths) {
    TENMO_CHECK_CTX(ctx);
    const char* who = "attention_bwd";
    TenmoAttnParams p = {};
    int st = check_shape(ctx, who, shape, scale, &p);
    if (st != TENMO_OK) return st;
    if (beta != 0.f && beta != 1.f) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "attention_bwd: beta must be 0 or 1");
    const bool any_q = p.B && p.Sq, any_k = p.B && p.Sk;
    if ((st = take_view(ctx, who, "q", q, any_q, false, p.B, p.H, p.Sq, p.D, &p.q)) != TENMO_OK) return st;
    if ((st = take_view(ctx, who, "k", k, any_k, false, p.B, p.Hkv, p.Sk, p.D, &p.k)) != TENMO_OK) return st;
    if ((st = take_view(ctx, who, "v", v, any_k, false, p.B, p.Hkv, p.Sk, p.D, &p.v)) != TENMO_OK) return st;
    if ((st = take_view(ctx, who, "o", o, any_q, false, p.B, p.H, p.Sq, p.D, &p.o)) != TENMO_OK) return st;
    if ((st = take_view(ctx, who, "go", go, any_q, false, p.B, p.H, p.Sq, p.D, &p.go)) != TENMO_OK) return st;
    if ((st = take_view(ctx, who, "dq", dq, any_q, true, p.B, p.H, p.Sq, p.D, &p.dq)) != TENMO_OK) return st;
    if ((st = take_view(ctx, who, "dk", dk, any_k, true, p.B, p.Hkv, p.Sk, p.D, &p.dk)) != TENMO_OK) return st;
    if ((st = take_view(ctx, who, "dv", dv, any_k, true, p.B, p.Hkv, p.Sk, p.D, &p.dv)) != TENMO_OK) return st;
    if (any_q && !stats) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "attention_bwd: stats is NULL");
    const float* in[5] = {p.q.ptr, p.k.ptr, p.v.ptr, p.o.ptr, p.go.ptr};
    const float* out[3] = {p.dq.ptr, p.dk.ptr, p.dv.ptr};
    for (int e = 0; e < 3 && any_q && any_k; ++e) {
        for (int u = 0; u < 5; ++u)
            if (out[e] == in[u]) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: a gradient is one of the inputs", who);
        if (out[e] == out[(e + 1) % 3]) return tenmo_set_error(ctx, TENMO_ERR_INVALID, "%s: two gradients are the same", who);
    }
    p.stats = const_cast<float*>(stats);
    p.causal = causal != 0;
    p.q_lengths = q_lengths;
    p.k_lengths = k_lengths;
    p.beta = beta;
    TenmoOpCall call(ctx);
    if (!ctx->op_fp32 && tenmo_attn_tc_profitable(p, true)) return tenmo_attn_tc_bwd(ctx, p);
    void* ws = nullptr;
    if ((st = tenmo_op_workspace(ctx, (size_t)p.B * p.H * p.Sq * sizeof(float) + 16, &ws)) != TENMO_OK) return st;
    p.delta = (float*)ws;
    if (any_q) {
        const int64_t grid = ((int64_t)p.B * p.H * p.Sq + ROW_WARPS - 1) / ROW_WARPS;
        TENMO_CUDA_TRY(ctx, tenmo_launch(attn_bwd_dq_row_kernel, (unsigned)grid, ROW_WARPS * 32, 0, ctx->stream, tenmo_pdl_ok(ctx, grid), p));
        TENMO_LAUNCH_CHECK(ctx, "attn_bwd_dq_row_kernel");
    }
    if (any_k) {
        const int64_t grid = ((int64_t)p.B * p.Hkv * p.Sk + ROW_WARPS - 1) / ROW_WARPS;
        TENMO_CUDA_TRY(ctx, tenmo_launch(attn_bwd_dkv_row_kernel, (unsigned)grid, ROW_WARPS * 32, 0, ctx->stream, tenmo_pdl_ok(ctx, grid), p));
        TENMO_LAUNCH_CHECK(ctx, "attn_bwd_dkv_row_kernel");
    }
    return TENMO_OK;
}

}  // extern "C"
