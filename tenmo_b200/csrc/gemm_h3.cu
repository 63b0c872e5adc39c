// fp32 matrix products on fp16 tensor cores (three fp16 products per fp32 product), block-scaled.
//
// Arithmetic: tcgen05.cuh.  The scale is per 128 x 128 block of an operand, so a block of small numbers (the gradient of rare
// classes) keeps its own precision, and one image of an operand serves the products over its columns and over its rows.
// The accumulator in tensor memory holds 128 of the contraction at a time; the epilogue warps add it to registers, scaled back
// and with rounding.  One chain over the whole contraction would lose to the tensor core's truncation what the second fp16 plane
// brings (measured on the TF32 kernel: 1e-4 at 8192), and block scales could not differ.
//
// Kernel: two CTAs on neighbouring SMs work on a 256 x 256 tile (tcgen05 cta_group::2): each stages its own 128 rows of A and
// half of the B tile, 64 KB per 64 of the contraction, three stages.  Persistent, 576 threads: warp 0 copies (plain tiled bulk copies
// without multicast, images are already swizzled), warp 1 of the leader issues the MMAs, warps 2-17 hold the 128 x 256 result of
// their CTA, 64 columns a thread: sixteen warps at 64 registers of sums instead of eight at 128, which would not leave room for
// the loads.  Two accumulators: while one is added up the tensor core fills the other, also across tiles.
// Tiles go round-robin to the pairs; with few tiles and a long contraction (the gradient of x) the contraction is cut into equal
// slices whose partial results a second kernel adds in order.
// Bound: tensor pipe, 3 * 2 M N K flop.
// Measured: 2048 x 65536 over 2048 (logits) 1.11 ms = 495 TFLOP/s of the product, 1490 of the pipe; over 65536 (gradient of x) 1.24 ms.  With a
// contraction of 768 the epilogue's statistics and 256 KB of results per tile of six chunks show: 2048 x 32011 logits 243 us (415 TFLOP/s; 206 us
// without storing them; 291 us when they went through shared memory and every element was asked for its column).
#include <cuda.h>

#include "gemm_h3.cuh"
#include "gemm_tc.cuh"
#include "tcgen05.cuh"

namespace {

constexpr int EPI_WARPS = 16;
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int STAGES = 3;
constexpr int PLANE = H3_PLANE;  // 128 of M (or N) x 64 of K
constexpr int STAGE = 4 * PLANE;
constexpr int ST_LD = 16;            // floats per row of a warp's staging block
constexpr int SMEM = STAGES * STAGE + EPI_WARPS * 32 * ST_LD * 4 + 256;
static_assert(SMEM <= 232448, "shared memory of a CTA");

// ---------------------------------------------------------------------------------------------------------------------
// operand blocks
// ---------------------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(512) h3_make_kernel(const float* src, int64_t rs, int64_t cs, int64_t rows, int64_t cols, int vec,
                                                      const void* labels, int is_i64, int64_t ignore, uint8_t* img, float* inverse,
                                                      int block_cols) {
    const int64_t block = blockIdx.x;
    const int64_t r0 = block / block_cols * H3_BLOCK, c0 = block % block_cols * H3_BLOCK + 8 * (threadIdx.x & 15);
    float x[4][8];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int64_t r = r0 + (threadIdx.x >> 4) + 32 * s;
        const bool in = r < rows && !(labels && tenmo_h3_label(labels, is_i64, r) == ignore);
        const float* p = src + r * rs + c0 * cs;
        if (in && vec && c0 + 8 <= cols) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
            x[s][0] = a.x; x[s][1] = a.y; x[s][2] = a.z; x[s][3] = a.w;
            x[s][4] = b.x; x[s][5] = b.y; x[s][6] = b.z; x[s][7] = b.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[s][e] = in && c0 + e < cols ? __ldg(p + e * cs) : 0.f;
        }
    }
    tenmo_h3_write_block(x, threadIdx.x >> 4, threadIdx.x & 15, img + block * H3_BLOCK_BYTES, inverse + block);
}

// ---------------------------------------------------------------------------------------------------------------------
// PTX for a CTA pair
// ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {  // the leader's shared-memory location of the same offset
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void expect_tx_cluster(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// lands in this CTA's shared memory, completes on the leader's barrier; no multicast
__device__ __forceinline__ void load_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int row) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(0), "r"(row)
        : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
__device__ __forceinline__ void commit_pair(uint32_t bar) {  // arrives in both CTAs
    const uint16_t both = 3;
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(both)
                 : "memory");
}

struct H3Params {
    TenmoH3Epilogue e;
    float* partial;  // slices > 1: (slices, M, N rounded up to 4)
    int64_t ldp;
    const float* a_inv; const float* b_inv;
    int64_t M, N;
    int vec;               // C can be written 16 bytes at a time
    int chunks;            // 128-blocks of the contraction
    int tiles_m, tiles_n, slices;
    int a_cb, b_cb;        // block columns of the operands' images
    int a_mb, b_nb;        // 128-blocks of M and of N
    uint32_t* status;
};

// tiles in groups of 8 tile rows, column by column: what runs at the same time shares panels in L2
__device__ __forceinline__ void h3_tile(int t, int tiles_m, int tiles_n, int* tm, int* tn) {
    constexpr int GROUP = 8;
    const int g = t / (GROUP * tiles_n), first = g * GROUP, rows = min(GROUP, tiles_m - first), in = t - g * GROUP * tiles_n;
    *tm = first + in % rows;
    *tn = in / rows;
}

// STATS: the product goes with the softmax statistics (and blocked results); in a kernel of its own, since their registers cost the other
// products 5 %.
template <bool A_MN, bool B_MN, bool STATS>
__global__ void __launch_bounds__(THREADS, 1) h3_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                             const __grid_constant__ H3Params p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    float* const staging = reinterpret_cast<float*>(smem + STAGES * STAGE);
    uint8_t* const tail = smem + STAGES * STAGE + EPI_WARPS * 32 * ST_LD * 4;
    const uint32_t bars = smem_u32(tail);
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (STAGES + s); };
    auto tfull = [&](int a) { return bars + 8u * (2 * STAGES + a); };
    auto tempty = [&](int a) { return bars + 8u * (2 * STAGES + 2 + a); };
    const uint32_t drain = bars + 8u * (2 * STAGES + 4);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(tail + 128);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cta_rank();
    const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;
    const int64_t units = (int64_t)p.tiles_m * p.tiles_n * p.slices;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full(s), 2); mbar_init(empty(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(tfull(a), 1); mbar_init(tempty(a), 2 * EPI_WARPS); }
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc::fence_before();
    __syncthreads();
    cluster_sync();
    tc::fence_after();
    const uint32_t tmem = *tmem_slot;

    // unit u: tile u / slices, slice u % slices of the contraction's chunks
    auto range = [&](int64_t u, int* tm, int* tn, int* c0, int* c1) {
        const int s = (int)(u % p.slices);
        h3_tile((int)(u / p.slices), p.tiles_m, p.tiles_n, tm, tn);
        *c0 = (int)((int64_t)p.chunks * s / p.slices);
        *c1 = (int)((int64_t)p.chunks * (s + 1) / p.slices);
    };

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0, count = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int64_t u = pair; ok && u < units; u += pairs) {
                int tm, tn, c0, c1;
                range(u, &tm, &tn, &c0, &c1);
                // blocks past the operand's edge are replaced by the last one: what they give lies outside the result
                const int mb = min(2 * tm + rank, p.a_mb - 1), nb = min(2 * tn + rank, p.b_nb - 1);
                for (int c = c0; ok && c < c1; ++c) {
                    const int64_t ab = A_MN ? (int64_t)c * p.a_cb + mb : (int64_t)mb * p.a_cb + c;
                    const int64_t bb = B_MN ? (int64_t)c * p.b_cb + nb : (int64_t)nb * p.b_cb + c;
                    for (int h = 0; h < 2; ++h) {  // 64 of the contraction
                        if (!mbar_wait(empty(stage), phase ^ 1u, abort_flag)) { ok = false; break; }
                        const uint32_t dst = smem_u32(smem) + stage * STAGE, bar = in_leader(full(stage));
                        expect_tx_cluster(bar, STAGE);
                        auto fetch = [&](uint32_t to, const CUtensorMap* map, int64_t block, bool mn) {
                            const int row = (int)(block * 512);
#pragma unroll
                            for (int plane = 0; plane < 2; ++plane) {
                                if (!mn) {
                                    load_pair(to + plane * PLANE, map, bar, row + 256 * plane + 128 * h);
                                } else {
#pragma unroll
                                    for (int q = 0; q < 2; ++q)
                                        load_pair(to + plane * PLANE + q * (PLANE / 2), map, bar, row + 256 * plane + 128 * q + 64 * h);
                                }
                            }
                        };
                        fetch(dst, &map_a, ab, A_MN);
                        fetch(dst + 2 * PLANE, &map_b, bb, B_MN);
                        ++count;
                        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                    }
                }
            }
            if (!ok && rank == 0) {  // the copies in flight of both CTAs end on the leader's barriers: wait for them (bounded)
                int never = 0;
                for (int t = max(0, count - STAGES); t < count; ++t) mbar_wait(full(t % STAGES), (uint32_t)(t / STAGES) & 1u, &never);
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t idesc = (1u << 4) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) | ((256u >> 3) << 17) | ((256u >> 4) << 24);
            auto operand = [&](uint32_t plane, int k, bool mn) {
                return mn ? tc::desc(plane + (uint32_t)k * 2048u, PLANE / 2, 1024u) : tc::desc(plane + (uint32_t)k * 32u, 16u, 1024u);
            };
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phases = 0;  // a bit per accumulator (an array would live in local memory)
            bool ok = true;
            for (int64_t u = pair; ok && u < units; u += pairs) {
                int tm, tn, c0, c1;
                range(u, &tm, &tn, &c0, &c1);
                for (int c = c0; ok && c < c1; ++c) {
                    if (!mbar_wait(tempty(acc), ((acc_phases >> acc) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
                    tc::fence_after();
                    const uint32_t d = tmem + (uint32_t)acc * 256u;
                    for (int h = 0; h < 2; ++h) {
                        if (!mbar_wait(full(stage), phase, abort_flag)) { ok = false; break; }
                        tc::fence_after();
                        const uint32_t a = smem_u32(smem) + stage * STAGE, b = a + 2 * PLANE;
#pragma unroll
                        for (int k = 0; k < 4; ++k) mma_pair(d, operand(a + PLANE, k, A_MN), operand(b, k, B_MN), idesc, h > 0 || k > 0);
#pragma unroll
                        for (int k = 0; k < 4; ++k) mma_pair(d, operand(a, k, A_MN), operand(b + PLANE, k, B_MN), idesc, true);
#pragma unroll
                        for (int k = 0; k < 4; ++k) mma_pair(d, operand(a, k, A_MN), operand(b, k, B_MN), idesc, true);
                        commit_pair(empty(stage));
                        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                    }
                    if (!ok) break;
                    commit_pair(tfull(acc));
                    acc_phases ^= 1u << acc;
                    acc ^= 1;
                }
            }
            if (!ok) {  // see the MMAs in flight to their end (bounded) before tensor memory is given back
                int never = 0;
                asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(drain) : "memory");
                mbar_wait(drain, 0, &never);
            }
        }
    } else {
        const int ew = warp - 2, quarter = warp & 3, group = ew >> 2;  // 32 rows, 64 columns
        float* const stage_buf = staging + ew * (32 * ST_LD);
        const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(group * 64);
        int acc = 0;
        uint32_t acc_phases = 0;  // a bit per accumulator
        bool ok = true;
        for (int64_t u = pair; ok && u < units; u += pairs) {
            int tm, tn, c0, c1;
            range(u, &tm, &tn, &c0, &c1);
            const int mb = min(2 * tm + rank, p.a_mb - 1), nb = min(2 * tn + (group >> 1), p.b_nb - 1);
            float s[64];
#pragma unroll
            for (int e = 0; e < 64; ++e) s[e] = 0.f;
            for (int c = c0; c < c1; ++c) {
                ok = __all_sync(0xffffffffu, mbar_wait(tfull(acc), (acc_phases >> acc) & 1u, abort_flag));
                if (!ok) break;
                tc::fence_after();
                const float f = __ldg(p.a_inv + (A_MN ? (int64_t)c * p.a_cb + mb : (int64_t)mb * p.a_cb + c)) *
                                __ldg(p.b_inv + (B_MN ? (int64_t)c * p.b_cb + nb : (int64_t)nb * p.b_cb + c));
                const uint64_t f2 = tc::pack2(f, f);
                // 16 columns at a time: 64 sums, 16 loaded values and the addresses, of which a thread's 112 registers leave out 32 to 80 bytes
                // (spilled, by form)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float t[16];
                    tc::ld16(lane_base + (uint32_t)acc * 256u + 16 * g, t);
#pragma unroll
                    for (int e = 0; e < 16; e += 2)
                        tc::unpack2(tc::fma2(tc::pack2(t[e], t[e + 1]), f2, tc::pack2(s[16 * g + e], s[16 * g + e + 1])), s[16 * g + e], s[16 * g + e + 1]);
                }
                tc::fence_before();
                __syncwarp();
                if (lane == 0) arrive_cluster(in_leader(tempty(acc)));
                acc_phases ^= 1u << acc;
                acc ^= 1;
            }
            if (!ok) break;
            const int64_t m0 = (int64_t)tm * 256 + rank * 128 + quarter * 32, n0 = (int64_t)tn * 256 + group * 64;
            if (m0 >= p.M || n0 >= p.N) continue;  // uniform over the warp
            // element (row, column) of this warp's part at C[row * ldc + column]
            float* C = p.e.C + m0 * p.e.ldc + n0;
            int64_t ldc = p.e.ldc;
            bool add = p.e.add != 0, vec = p.vec != 0;
            if (!STATS && p.slices > 1) {
                C = p.partial + ((u % p.slices) * p.M + m0) * p.ldp + n0;
                ldc = p.ldp;
                add = false;
                vec = true;
            }
            if (STATS) {
                if (p.e.bias) {
#pragma unroll
                    for (int e = 0; e < 64; ++e) s[e] += n0 + e < p.N ? __ldg(p.e.bias + n0 + e) : 0.f;
                }
                {
                    const int64_t m = m0 + lane;
                    const int cols = (int)min((int64_t)64, p.N - n0);
                    float mx = -INFINITY, sum = 0.f, all = 0.f;
                    if (cols == 64) {  // apart from the ragged edge, where every element is asked for
#pragma unroll
                        for (int e = 0; e < 64; e += 4) mx = fmaxf(mx, fmaxf(fmaxf(s[e], s[e + 1]), fmaxf(s[e + 2], s[e + 3])));
                    } else {
#pragma unroll
                        for (int e = 0; e < 64; ++e) mx = fmaxf(mx, e < cols ? s[e] : -INFINITY);
                    }
                    const float base = mx == -INFINITY ? 0.f : mx;
                    if (cols == 64) {
                        const uint64_t nb2 = tc::pack2(-base, -base), l2 = tc::pack2(1.44269504088896341f, 1.44269504088896341f);
                        uint64_t sum2 = 0;
#pragma unroll
                        for (int e = 0; e < 64; e += 2) {  // the difference first: it is exact where it matters
                            float x, y;
                            tc::unpack2(tc::mul2(tc::add2(tc::pack2(s[e], s[e + 1]), nb2), l2), x, y);
                            sum2 = tc::add2(sum2, tc::pack2(tc::ex2(x), tc::ex2(y)));
                        }
                        float x, y;
                        tc::unpack2(sum2, x, y);
                        sum = x + y;
                    } else {
#pragma unroll
                        for (int e = 0; e < 64; ++e) sum += e < cols ? tc::ex2((s[e] - base) * 1.44269504088896341f) : 0.f;
                    }
                    if (p.e.sums) {
#pragma unroll
                        for (int e = 0; e < 64; ++e) all += e < cols ? s[e] : 0.f;
                    }
                    if (m < p.M) {
                        const int64_t at = (n0 >> 6) * p.M + m;
                        p.e.stats[at] = make_float2(mx, sum);
                        if (p.e.sums) p.e.sums[at] = all;
                        const int64_t y = tenmo_h3_label(p.e.labels, p.e.label_is_i64, m) - n0;
                        if (y >= 0 && y < cols) {
                            float v = 0.f;
#pragma unroll
                            for (int e = 0; e < 64; ++e) v = e == (int)y ? s[e] : v;
                            p.e.at_label[m] = v;
                        }
                    }
                }
            }
            if (STATS) {  // blocks, or nothing
                if (p.e.C) {
                    float* out = p.e.C + ((int64_t)(2 * tm + rank) * p.b_nb + 2 * tn + (group >> 1)) * (H3_BLOCK * H3_BLOCK);
#pragma unroll
                    for (int q = 0; q < 16; ++q)
                        *reinterpret_cast<float4*>(out + tenmo_h3_patch(quarter * 32 + lane, (group & 1) * 16 + q)) =
                            make_float4(s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]);
                }
                continue;
            }
            // out through the warp's staging block, 16 columns at a time: 16-byte chunk q of row r at chunk q ^ ((r >> 1) & 3); a warp-wide
            // store then covers eight rows of 64 contiguous bytes
            const int q = lane & 3, sub = lane >> 2;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<float4*>(stage_buf + lane * ST_LD + (((e >> 2) ^ ((lane >> 1) & 3)) << 2)) =
                        make_float4(s[16 * g + e], s[16 * g + e + 1], s[16 * g + e + 2], s[16 * g + e + 3]);
                __syncwarp();
                if (vec && n0 + 16 * g + 16 <= p.N) {
                    const int at = 16 * g + 4 * q;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = 8 * i + sub;
                        float4 x = *reinterpret_cast<const float4*>(stage_buf + r * ST_LD + ((q ^ ((r >> 1) & 3)) << 2));
                        if (m0 + r >= p.M) continue;
                        float* dst = C + r * ldc + at;
                        if (add) {
                            const float4 o = *reinterpret_cast<const float4*>(dst);
                            x.x += o.x; x.y += o.y; x.z += o.z; x.w += o.w;
                        }
                        *reinterpret_cast<float4*>(dst) = x;
                    }
                } else {  // unaligned rows, and the ragged edge: a store covers two rows of 64 contiguous bytes
                    const int c = lane & 15, at = 16 * g + c;
#pragma unroll 4
                    for (int r = lane >> 4; r < 32; r += 2) {
                        const float x = stage_buf[r * ST_LD + (((c >> 2) ^ ((r >> 1) & 3)) << 2) + (c & 3)];
                        if (m0 + r >= p.M || n0 + at >= p.N) continue;
                        float* dst = C + r * ldc + at;
                        *dst = add ? *dst + x : x;
                    }
                }
            }
        }
    }
    tc::fence_before();
    __syncthreads();
    cluster_sync();  // neither CTA gives back memory that the other may still address
    if (threadIdx.x == 0 && *abort_flag) atomicOr(p.status, TENMO_DEV_TIMEOUT);
    if (warp == 1) {
        tc::fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// C (+)= the slices' partial results, in order
__global__ void __launch_bounds__(256) h3_fold_kernel(const float* partial, int slices, int64_t M, int64_t N, int64_t ldp, float* C, int64_t ldc, int add) {
    const int64_t per = ldp / 4, total = M * per;
    for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < total; e += (int64_t)gridDim.x * blockDim.x) {
        const int64_t m = e / per, n = e % per * 4;
        float4 s = *reinterpret_cast<const float4*>(partial + m * ldp + n);
        for (int k = 1; k < slices; ++k) {
            const float4 v = *reinterpret_cast<const float4*>(partial + (k * M + m) * ldp + n);
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        const float v[4] = {s.x, s.y, s.z, s.w};
        for (int u = 0; u < 4; ++u)
            if (n + u < N) {
                float* d = C + m * ldc + n + u;
                *d = add ? *d + v[u] : v[u];
            }
    }
}

int encode(tenmo_ctx* ctx, CUtensorMap* map, const TenmoH3Operand& o, bool mn) {
    TenmoEncodeTiledFn fn = reinterpret_cast<TenmoEncodeTiledFn>(ctx->encode_tiled);
    cuuint64_t dims[2] = {64, (cuuint64_t)o.blocks() * 512};
    cuuint64_t strides[1] = {128};
    cuuint32_t box[2] = {64, mn ? 64u : 128u};
    cuuint32_t step[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, o.img, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return tenmo_set_error(ctx, TENMO_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
    return TENMO_OK;
}

// Slices of the contraction: the number (at most 32, each at least 8 chunks) that finishes first by this count, in units of one 128-deep
// chunk of a 256 x 256 tile, 2.3 us at the measured rate: the rounds of tiles that the pairs need, and the partial results, which
// are written, read and folded at about 6 TB/s.  A shorter contraction can come out with more slices than a longer one (the rounds go by whole
// tiles), so scratch is asked for by every size that is used, and a count whose results do not fit `room` bytes is not taken.
size_t slice_bytes(int slices, int64_t M, int64_t N) { return (size_t)slices * (size_t)M * (size_t)((N + 3) / 4 * 4) * sizeof(float); }
int pick_slices(const tenmo_ctx* ctx, int64_t M, int64_t N, int64_t K, size_t room) {
    const int64_t tiles = ((M + 255) / 256) * ((N + 255) / 256), chunks = (K + 127) / 128;
    const int64_t pairs = (ctx->sm_count - ctx->reserve_sms) / 2 > 0 ? (ctx->sm_count - ctx->reserve_sms) / 2 : 1;
    const double traffic = 4.0 * M * N / 6e6 / 2.3;  // one pass over the result
    int best = 1;
    double best_cost = 1e300;
    for (int s = 1; s <= 32 && (s == 1 || (chunks >= 8 * s && slice_bytes(s, M, N) <= room)); ++s) {
        const int64_t rounds = (tiles * s + pairs - 1) / pairs;
        const double cost = (double)rounds * ((double)chunks / s + 1.0) + (s > 1 ? (2.0 * s + 1.0) * traffic + 2.0 : 0.0);
        if (cost < best_cost * 0.99) { best = s; best_cost = cost; }
    }
    return best;
}

}  // namespace

int tenmo_h3_make(tenmo_ctx* ctx, const float* src, int64_t rs, int64_t cs, const TenmoH3Operand& o, const void* labels, int is_i64, int64_t ignore) {
    if (o.blocks() > 0x7fffffffLL / 512) return tenmo_set_error(ctx, TENMO_ERR_UNSUPPORTED, "operand of %lld x %lld is too large", (long long)o.rows, (long long)o.cols);
    const int vec = cs == 1 && rs % 4 == 0 && ((uintptr_t)src & 15u) == 0;
    h3_make_kernel<<<(unsigned)o.blocks(), 512, 0, ctx->stream>>>(src, rs, cs, o.rows, o.cols, vec, labels, is_i64, ignore, o.img, o.inverse, (int)o.block_cols());
    TENMO_LAUNCH_CHECK(ctx, "h3_make_kernel");
    return TENMO_OK;
}

size_t tenmo_h3_partial_bytes(const tenmo_ctx* ctx, int64_t M, int64_t N, int64_t K) {
    const int s = pick_slices(ctx, M, N, K, SIZE_MAX);
    return s > 1 ? slice_bytes(s, M, N) : 0;
}

int tenmo_h3_gemm(tenmo_ctx* ctx, int64_t M, int64_t N, int64_t K, const TenmoH3Operand& A, bool a_rows_are_k, const TenmoH3Operand& B,
                  bool b_rows_are_k, const TenmoH3Epilogue& e, void* partial, size_t partial_bytes) {
    int st = tenmo_tma_init(ctx);
    if (st != TENMO_OK) return st;
    CUtensorMap ma, mb;
    if ((st = encode(ctx, &ma, A, a_rows_are_k)) != TENMO_OK || (st = encode(ctx, &mb, B, b_rows_are_k)) != TENMO_OK) return st;
    H3Params p = {};
    p.e = e;
    p.M = M; p.N = N;
    p.vec = e.ldc % 4 == 0 && ((uintptr_t)e.C & 15u) == 0;
    p.chunks = (int)((K + 127) / 128);
    p.tiles_m = (int)((M + 255) / 256); p.tiles_n = (int)((N + 255) / 256);
    const bool plain = !e.stats;
    if (plain && (e.bias || e.blocked || !e.C)) return tenmo_set_error(ctx, TENMO_ERR_UNSUPPORTED, "h3_gemm: a bias and blocks go with the statistics");
    if (!plain && (!e.at_label || !e.labels || (e.C && !e.blocked) || a_rows_are_k)) return tenmo_set_error(ctx, TENMO_ERR_UNSUPPORTED, "h3_gemm: this epilogue is not built");
    p.slices = plain && partial ? pick_slices(ctx, M, N, K, partial_bytes) : 1;
    p.partial = (float*)partial;
    p.ldp = (N + 3) / 4 * 4;
    p.a_inv = A.inverse; p.b_inv = B.inverse;
    p.a_cb = (int)A.block_cols(); p.b_cb = (int)B.block_cols();
    p.a_mb = (int)((M + 127) / 128); p.b_nb = (int)((N + 127) / 128);
    p.status = ctx->dev_status;
    const int64_t units = (int64_t)p.tiles_m * p.tiles_n * p.slices;
    int64_t pairs = (ctx->sm_count - ctx->reserve_sms) / 2;
    if (pairs > units) pairs = units;
    if (pairs < 1) pairs = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * pairs));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    auto go = [&](auto kernel) -> int {
        TENMO_CUDA_TRY(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        TENMO_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, kernel, ma, mb, p));
        TENMO_LAUNCH_CHECK(ctx, "h3_gemm_kernel");
        return TENMO_OK;
    };
    if (a_rows_are_k && !b_rows_are_k) return tenmo_set_error(ctx, TENMO_ERR_UNSUPPORTED, "h3_gemm: this pair of layouts is not built");
    if (plain) st = a_rows_are_k ? go(h3_gemm_kernel<true, true, false>) : b_rows_are_k ? go(h3_gemm_kernel<false, true, false>) : go(h3_gemm_kernel<false, false, false>);
    else st = b_rows_are_k ? go(h3_gemm_kernel<false, true, true>) : go(h3_gemm_kernel<false, false, true>);
    if (st != TENMO_OK) return st;
    if (p.slices > 1) {
        h3_fold_kernel<<<tenmo_stream_grid(ctx, M * (p.ldp / 4), 256 * 2, 8), 256, 0, ctx->stream>>>(p.partial, p.slices, M, N, p.ldp, e.C, e.ldc, e.add);
        TENMO_LAUNCH_CHECK(ctx, "h3_fold_kernel");
    }
    return TENMO_OK;
}
