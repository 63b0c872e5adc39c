// Tensor-core attention, forward: tile images and the fused kernel.
//
// Kernel.  A CTA owns 128 rows of one head.  Its q rows are split into fp16 pairs (scaled per row) and kept in tensor memory as
// the left operand; k and v come as 128-row tile images through a ring of three slots (k_0, v_0, k_1, ...).  Per tile j:
//   S_j = q k_j^T          left operand and accumulator in tensor memory
//   P_j = exp2(S_j c - m)  by warpgroups, a row per thread, written over S_j as fp16 pairs: the next left operand
//   O_j = P_j v_j          a fresh accumulator, added to the row's registers (and rescaled) with rounding
// The running reference m is kept a whole number (the ceiling of the maximum), which makes every rescaling an exact power of two.  What is
// kept is 15 - m, rounded downwards: scores beyond 2^24, where not every whole number exists, then still keep P below 2^15.
// What bounds the kernel is not a pipe but the instructions around the products and the chain S -> maximum -> exponentials -> P -> O
// of a tile, thousands of cycles of latencies.  So tiles are wide (128 keys: the waits, fences and exchanges of a tile are paid half as
// often as with 64), their columns are shared by two warpgroups (dim up to 64; 64 columns of S, 32 of O a thread) or four (up to
// 128), which exchange their maxima through shared memory, and up to dim 64, where everything fits twice into an SM (96 KB,
// 256 columns), two CTAs fill each other's gaps: one's products run while the other's exponentials are taken.  Up to dim 128 one
// CTA has the SM and a second S buffer lets S_{j+1} run while P_j is made.  One warp issues the MMAs and (or
// another warp, with one CTA on the SM) the copies.
// S and P are handed over in halves of 64 keys, so the maximum of the first half is taken while the second is computed and O_j
// starts while the second half's exponentials are taken; O_{j-1} is added while S_j is computed.
// Floor: tensor pipe, 3 * 4 * rows * keys * dim flop; the images cost one read and one write of k and v in front.
// Measured at 384 heads of 512 rows and keys, dim 64: 119 us behind 26 us of images (25.8 GF, 47 us of tensor time).  A tile of 128 x 128
// takes 3900 cycles with one CTA on the SM, 3350 with two, where the products and the exponentials (measured apart) need 1540 each and do
// not slow each other; a CTA costs 14,000 cycles besides (q's way into tensor memory, the first tile's way to the exponentials, the
// output).  Tensor pipe 32 % busy, exponential unit 24 %: the chain of a tile decides.  Two sides per CTA under one issuer were slower
// (202 us for 167 in all at the time); tiles of 64 keys with two S buffers took 131 us.
#include "attention_tc.cuh"

namespace {

constexpr int ROWS = 128;
constexpr int T = 128;     // keys of a tile
constexpr int SLOTS = 3;   // of the ring
constexpr int RT = ATTN_TILE;  // rows of a tile with row numbers

// ---------------------------------------------------------------------------------------------------------------------
// Tile images.  A block makes one tile: 8 columns (a 16-byte chunk of each plane) per thread and step.
// ---------------------------------------------------------------------------------------------------------------------
// delta_i = sum_d go o and the saved statistics of a tile's rows (x: this thread's columns of go)
template <int DP, int T>
__device__ __forceinline__ void attn_row_numbers(const TenmoTileJobs& jobs, const TenmoTileJob& j, int64_t t, int b, int h, int tile, int rows,
                                                 const float (&x)[T * (DP / 8) / 256][8]) {
    constexpr int CHUNKS = DP / 8, STEPS = T * CHUNKS / 256;
    __shared__ float delta[T], most[2][2];
    const float* src = j.o.ptr + b * j.o.sb + h * j.o.sh + (int64_t)tile * T * j.o.sr;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int q = threadIdx.x + s * 256, r = q / CHUNKS, d = (q % CHUNKS) * 8;
        const float* p = src + r * j.o.sr + d;
        float sum = 0.f;
        if (r < rows && j.o_vec && d + 8 <= jobs.D) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(p)), c = __ldg(reinterpret_cast<const float4*>(p) + 1);
            sum = (x[s][0] * a.x + x[s][1] * a.y) + (x[s][2] * a.z + x[s][3] * a.w) + (x[s][4] * c.x + x[s][5] * c.y) + (x[s][6] * c.z + x[s][7] * c.w);
        } else if (r < rows) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (d + e < jobs.D) sum = fmaf(x[s][e], __ldg(p + e), sum);
        }
#pragma unroll
        for (int w = CHUNKS / 2; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        if (q % CHUNKS == 0) delta[r] = sum;
    }
    __syncthreads();
    const int r = threadIdx.x;
    float m = INFINITY, il = 0.f, dl = 0.f;
    if (r < T) {
        if (r < rows) {
            const float* st = j.stats + (((int64_t)b * j.heads + h) * j.rows + (int64_t)tile * T + r) * 2;
            if (st[1] != 0.f) {
                m = st[0];
                il = 1.f / st[1];
                dl = delta[r];
            }
        }
        const float a = tenmo_warp_max(tc::finite_abs(il)), c = tenmo_warp_max(tc::finite_abs(dl));
        if ((r & 31) == 0) { most[0][r >> 5] = a; most[1][r >> 5] = c; }
    }
    __syncthreads();
    if (r < T) {
        const float il_max = fmaxf(most[0][0], most[0][1]);
        const float ps = il_max > 0.f ? 32768.f * tc::pow2_below_inverse(il_max) : 1.f;
        float* info = j.info + t * ATTN_INFO;
        info[4 * (r >> 1) + (r & 1)] = -m;
        info[4 * (r >> 1) + 2 + (r & 1)] = il * ps;
        info[2 * T + r] = dl;
        if (r == 0) { info[3 * T] = ps; info[3 * T + 1] = fmaxf(most[1][0], most[1][1]); info[3 * T + 2] = 1.f / ps; }
    }
    __syncthreads();
}

template <int DP, int T>
__global__ void __launch_bounds__(256) attn_tiles_kernel(const TenmoTileJobs jobs) {
    constexpr int CHUNKS = DP / 8, STEPS = T * CHUNKS / 256;
    __shared__ float largest[8];
    const TenmoTileJob& j = jobs.job[blockIdx.y];
    const int64_t t = blockIdx.x;
    if (t >= (int64_t)jobs.B * j.heads * j.tiles) return;
    const int tile = (int)(t % j.tiles);
    const int64_t bh = t / j.tiles;
    const int h = (int)(bh % j.heads), b = (int)(bh / j.heads);
    int rows = tenmo_attn_rows(j.lengths, b, j.rows);
    if (j.seen_by) rows = min(rows, max(0, tenmo_attn_rows(j.q_lengths, b, j.seen_by) + j.offset));
    rows -= tile * T;
    if (rows <= 0) return;  // no kernel reads a tile behind the length
    const float* src = j.src.ptr + b * j.src.sb + h * j.src.sh + (int64_t)tile * T * j.src.sr;
    const int skip = j.first - tile * T;
    float x[STEPS][8];
    float mx = 0.f;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int q = threadIdx.x + s * 256, r = q / CHUNKS, d = (q % CHUNKS) * 8;
        const float* p = src + r * j.src.sr + d;
        if (r < rows && r >= skip && j.vec && d + 8 <= jobs.D) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(p)), c = __ldg(reinterpret_cast<const float4*>(p) + 1);
            x[s][0] = a.x; x[s][1] = a.y; x[s][2] = a.z; x[s][3] = a.w;
            x[s][4] = c.x; x[s][5] = c.y; x[s][6] = c.z; x[s][7] = c.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[s][e] = r < rows && r >= skip && d + e < jobs.D ? __ldg(p + e) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[s][e]));  // a NaN does not count
    }
    if (!(mx <= 3.402823466e38f)) {  // an infinity does not either
        mx = 0.f;
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, tc::finite_abs(x[s][e]));
    }
    if constexpr (T == RT) {
        if (j.o.ptr) attn_row_numbers<DP, T>(jobs, j, t, b, h, tile, rows, x);
    }
    mx = tenmo_warp_max(mx);
    if ((threadIdx.x & 31) == 0) largest[threadIdx.x >> 5] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) mx = fmaxf(mx, largest[w]);
    float inverse;
    const float scale = tc::block_scale(mx, &inverse);
    if (threadIdx.x == 0) j.inverse[t] = inverse;
    uint8_t* img = j.img + t * (T * DP * 4);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int q = threadIdx.x + s * 256, r = q / CHUNKS, c = q % CHUNKS;
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) tc::split_rounded(x[s][2 * e] * scale, x[s][2 * e + 1] * scale, hi[e], lo[e]);
        const int at = (c >> 3) * (T * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
        *reinterpret_cast<uint4*>(img + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(img + T * DP * 2 + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------------------------------------------------
struct FwdParams {
    TenmoAttnParams a;
    const uint8_t* k_img; const uint8_t* v_img;
    const float* k_inv; const float* v_inv;
    int tiles;    // tiles of a head of k
    int q_tiles;  // 128-row tiles of a head of q
    TenmoAttnOrder order;
    int q_vec, o_vec;
    uint32_t* status;
};

template <int DP>
struct FwdCfg {
    static constexpr int WGS = DP / 32;             // warpgroups that share a tile
    static constexpr bool OWN_LOADER = DP != 64;    // up to dim 64 the issuing warp copies too (119 us for 122 below)
    static constexpr int ISSUER = 4 * WGS, LOADER = OWN_LOADER ? ISSUER + 1 : ISSUER;
    static constexpr int THREADS = 32 * (LOADER + 1);
    static constexpr int HC = T / 2 / WGS, W = DP / WGS;  // columns of a half of S and of O of a thread
    static constexpr int NB = DP == 64 ? 1 : 2;     // S / P buffers
    static constexpr int PLANE = T * DP * 2;        // bytes of one plane of a tile
    static constexpr int IMG = 2 * PLANE;           // a tile's hi and lo plane, a slot of the ring
    static constexpr int Q_COLS = DP;               // hi DP/2, lo DP/2
    static constexpr int S_COL = Q_COLS, O_COL = Q_COLS + NB * T;
    static constexpr int TMEM = DP == 64 ? 256 : 512;
    static constexpr int RING = SLOTS * IMG;
    static constexpr int SMEM = RING + 2 * WGS * 128 * 4 + 512;
    static_assert(O_COL + DP <= TMEM, "tensor memory");
};

template <int DP>
__global__ void __launch_bounds__(FwdCfg<DP>::THREADS, DP == 64 ? 2 : 1) attn_fwd_tc_kernel(const __grid_constant__ FwdParams p) {
    using C = FwdCfg<DP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    float* const shared_f = reinterpret_cast<float*>(smem + C::RING);  // [2][WGS][128] row maxima
    const uint32_t bars = smem_u32(smem + C::RING + 2 * C::WGS * 128 * 4);
    auto full = [&](int slot) { return bars + 8u * slot; };
    auto empty = [&](int slot) { return bars + 8u * (3 + slot); };
    auto s_full = [&](int j, int half) { return bars + 8u * (6 + 2 * (j & 1) + half); };
    auto p_full = [&](int j, int half) { return bars + 8u * (10 + 2 * (j & 1) + half); };
    auto o_full = [&](int j) { return bars + 8u * (14 + (j & 1)); };
    const uint32_t o_free = bars + 8u * 16, drain = bars + 8u * 17;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + C::RING + 2 * C::WGS * 128 * 4 + 256);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const TenmoAttnParams& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // the longest rows of a causal head first: the last tiles have the most keys
    int q_tile, bh;
    tenmo_attn_block(p.order, blockIdx.x, &q_tile, &bh);
    q_tile = p.q_tiles - 1 - q_tile;
    const int h = bh % a.H, b = bh / a.H, kvh = h / (a.H / a.Hkv);
    const int q_rows = tenmo_attn_rows(a.q_lengths, b, a.Sq), keys = tenmo_attn_rows(a.k_lengths, b, a.Sk);
    // keys that the last row of the tile that takes part sees
    const int last = min(q_rows, (q_tile + 1) * ROWS) - 1;
    int seen = last >= q_tile * ROWS ? keys : 0;
    if (a.causal) seen = min(seen, max(0, last + a.Sk - a.Sq + 1));
    const int n_tiles = (seen + T - 1) / T;
    const int64_t tile0 = ((int64_t)b * a.Hkv + kvh) * p.tiles;
    if (n_tiles == 0) {  // rows behind the length, or none with a visible key
        const int row0 = q_tile * ROWS;
        tenmo_attn_zero_rows<DP>(a.o.ptr + b * a.o.sb + h * a.o.sh, a.o.sr, row0, a.Sq, a.D, p.o_vec);
        if (a.stats && threadIdx.x < ROWS && row0 + (int)threadIdx.x < a.Sq) {
            float* st = a.stats + (((int64_t)b * a.H + h) * a.Sq + row0 + threadIdx.x) * 2;
            st[0] = -INFINITY;
            st[1] = 0.f;
        }
        return;
    }

    // The ring (one thread): tiles in the order in which the products use them, each as soon as its slot's last product is done.
    // One S buffer: k_0, v_0, k_1, v_1, ...; two: k_0, k_1, v_0, k_2, v_1, ..., v_{n-1}.
    int fetched = 0, fetch_slot = 0, fetch_round = 0;
    auto fetch = [&](int until) {
        for (; fetched < until; ++fetched) {
            if (fetch_round && !mbar_wait(empty(fetch_slot), (uint32_t)(fetch_round - 1) & 1u, abort_flag)) return;
            const uint32_t bar = full(fetch_slot);
            mbar_expect_tx(bar, C::IMG);
            const bool v = C::NB == 1 ? (fetched & 1) != 0 : (fetched & 1) ? fetched == 2 * n_tiles - 1 : fetched != 0;
            const int t = C::NB == 1 ? fetched >> 1 : v ? (fetched - 1) >> 1 : (fetched + 1) >> 1;
            tc::bulk_load(smem_u32(smem) + fetch_slot * C::IMG, (v ? p.v_img : p.k_img) + (tile0 + t) * C::IMG, C::IMG, bar);
            if (++fetch_slot == SLOTS) { fetch_slot = 0; ++fetch_round; }
        }
    };
    if (threadIdx.x == 32 * C::LOADER) {  // the thread that copies: the first tiles are on their way before the block meets
        for (int s = 0; s < SLOTS; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int w = 0; w < 2; ++w) {
            for (int half = 0; half < 2; ++half) { mbar_init(s_full(w, half), 1); mbar_init(p_full(w, half), 4 * C::WGS); }
            mbar_init(o_full(w), 1);
        }
        mbar_init(o_free, 4 * C::WGS);
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tc::fence_proxy_async();
        fetch(min(2 * n_tiles, SLOTS - 1));  // the last slot is scratch for now
    }

    float x[C::W];  // q
    if (warp < C::ISSUER)
        tenmo_attn_fetch<DP, C::WGS>(x, a.q.ptr + b * a.q.sb + h * a.q.sh + (int64_t)q_tile * ROWS * a.q.sr, a.q.sr, q_rows - q_tile * ROWS, p.q_vec, a.D,
                                     reinterpret_cast<float*>(smem + (SLOTS - 1) * C::IMG));

    if (warp == C::ISSUER) tc::alloc(tmem_slot, C::TMEM);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *tmem_slot;

    // ---- q into tensor memory ----
    const int wg = warp >> 2, row = threadIdx.x & 127;
    const int64_t i = (int64_t)q_tile * ROWS + row;
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    float q_inv = 1.f;
    if (warp < C::ISSUER)  // the sign of the scale goes with q: the factor of the scores is then never negative
        q_inv = tenmo_attn_stationary<DP, false, C::WGS>(x, a.scale < 0.f, lane_base, nullptr, shared_f);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();

    if (warp >= C::ISSUER) {
        // every copy has landed before shared memory is given back (bounded): by now they are the last ones
        auto landed = [&]() {
            int never = 0;
            for (int t = max(0, fetched - SLOTS); t < fetched; ++t) mbar_wait(full(t % SLOTS), (uint32_t)(t / SLOTS) & 1u, &never);
        };
        if (C::OWN_LOADER && warp == C::LOADER) {
            if (lane == 0) {
                fetch(2 * n_tiles);
                landed();
            }
        } else if (warp == C::ISSUER) {
            auto refill = [&](int until) {  // without a loader
                if (lane == 0) fetch(min(2 * n_tiles, until));
                __syncwarp();
            };
            if (!C::OWN_LOADER) refill(SLOTS);

            const uint32_t tm = tc::uniform(tmem), stages = tc::uniform(smem_u32(smem));
            const int n = tc::uniform(n_tiles);
            constexpr uint32_t ID_S = tc::idesc_f16(T / 2, false), ID_O = tc::idesc_f16(DP, true);
            auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0; };
            int slot = 0, phase = 0;
            auto next_slot = [&]() { if (++slot == SLOTS) { slot = 0; phase ^= 1; } };
            // S_j, each half (64 keys: an accumulator of its own) handed over as soon as it is there
            auto scores = [&](int j) {
                tc::fence_after();
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t hi = stages + slot * C::IMG + half * 8192, d = tm + C::S_COL + (uint32_t)(j % C::NB) * T + 64 * half;
#pragma unroll
                    for (int c = 0; c < DP / 64; ++c) tc::mma4_ts<8, tc::STEP_K>(d, tm + DP / 2 + 32 * c, tc::desc_k(hi + c * T * 128), ID_S, c == 0);
#pragma unroll
                    for (int c = 0; c < DP / 64; ++c) tc::mma4_ts<8, tc::STEP_K>(d, tm + 32 * c, tc::desc_k(hi + C::PLANE + c * T * 128), ID_S, false);
#pragma unroll
                    for (int c = 0; c < DP / 64; ++c) tc::mma4_ts<8, tc::STEP_K>(d, tm + 32 * c, tc::desc_k(hi + c * T * 128), ID_S, false);
                    tc::commit(s_full(j, half));
                }
                tc::commit(empty(slot));
                next_slot();
            };
            // In each place the wait that ends last comes last: one that is over costs its latency all the same.
            bool ok = n == 0 || wait(full(slot), phase);
            if (ok && n) scores(0);
            for (int j = 0; ok && j < n; ++j) {
                if (C::NB == 2 && j + 1 < n) {  // S_{j+1} replaces P_{j-1}, whose product must be done
                    ok = wait(full(slot), phase) && (j == 0 || wait(o_full(j - 1), (uint32_t)((j - 1) >> 1) & 1u));
                    if (!ok) break;
                    scores(j + 1);
                }
                ok = wait(full(slot), phase) && (j == 0 || wait(o_free, (uint32_t)(j - 1) & 1u));
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    ok = ok && wait(p_full(j, half), (uint32_t)(j >> 1) & 1u);
                    if (!ok) break;
                    tc::fence_after();
                    // keys 16 k ..: eight columns of hi pairs from 16 k on, then eight of lo pairs
                    const uint32_t hi = stages + slot * C::IMG + half * 8192;
                    const uint32_t pr = tm + C::S_COL + (uint32_t)(j % C::NB) * T + 64 * half, d = tm + C::O_COL;
                    tc::mma4_ts<16, tc::STEP_MN>(d, pr + 8, tc::desc_mn(hi, T), ID_O, half == 0);
                    tc::mma4_ts<16, tc::STEP_MN>(d, pr, tc::desc_mn(hi + C::PLANE, T), ID_O, false);
                    tc::mma4_ts<16, tc::STEP_MN>(d, pr, tc::desc_mn(hi, T), ID_O, false);
                }
                if (!ok) break;
                tc::commit(o_full(j));
                tc::commit(empty(slot));
                next_slot();
                if (C::NB == 1 && j + 1 < n) {  // S_{j+1} replaces P_j
                    ok = wait(full(slot), phase) && wait(o_full(j), (uint32_t)(j >> 1) & 1u);
                    if (ok) scores(j + 1);
                    if (ok && !C::OWN_LOADER) refill(2 * j + 2 + SLOTS);  // S_j and O_j are done: their two slots
                }
            }
            // Every MMA is done before tensor memory is given back: the readers of O have seen to it; after a wait that ran out, wait
            // again (bounded) here.
            if (!ok) {
                int never = 0;
                tc::commit(drain);
                mbar_wait(drain, 0, &never);
            }
            if (!C::OWN_LOADER) {
                if (lane == 0) landed();
                __syncwarp();
            }
        }
    } else {
        constexpr int HC = C::HC, W = C::W, GW = 16;
        float ref = INFINITY, l = 0.f, o[W];  // ref: 15 - m, infinite until a key was seen; l: of this thread's columns
#pragma unroll
        for (int d = 0; d < W; ++d) o[d] = 0.f;
        const float c_row = fabsf(a.scale_log2) * q_inv;
        int n_row = i < q_rows ? keys : 0;
        if (a.causal) n_row = min(n_row, (int)max((int64_t)0, i + a.Sk - a.Sq + 1));
        bool ok = true;
        auto await = [&](uint32_t bar, int phase) { ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, (uint32_t)phase & 1u, abort_flag)); };
        auto sync_rows = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(128 * C::WGS) : "memory"); };
        float shrink = 0.f, v_inv = 0.f;  // of the tile whose output is next
        auto add_output = [&](int j) {    // o = o * shrink + O_j
            await(o_full(j), j >> 1);
            if (!ok) return;
            tc::fence_after();
            float t[W];
            tc::ldn(lane_base + C::O_COL + wg * W, t);
            tc::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(o_free);
            const uint64_t sh2 = tc::pack2(shrink, shrink), vi2 = tc::pack2(v_inv, v_inv);
            if (__all_sync(0xffffffffu, shrink == 1.f)) {
#pragma unroll
                for (int e = 0; e < W; e += 2) tc::unpack2(tc::fma2(tc::pack2(t[e], t[e + 1]), vi2, tc::pack2(o[e], o[e + 1])), o[e], o[e + 1]);
            } else {
#pragma unroll
                for (int e = 0; e < W; e += 2) {
                    const uint64_t add = tc::mul2(tc::pack2(t[e], t[e + 1]), vi2);
                    tc::unpack2(tc::fma2(tc::pack2(o[e], o[e + 1]), sh2, add), o[e], o[e + 1]);
                }
            }
        };
        // the tiles' scales come from L2: loaded a tile ahead
        float k_ahead = n_tiles ? __ldg(p.k_inv + tile0) : 1.f, v_ahead = n_tiles ? __ldg(p.v_inv + tile0) : 1.f;
        for (int j = 0; j < n_tiles; ++j) {
            const float c = c_row * k_ahead, v_next = v_ahead;
            if (j + 1 < n_tiles) {
                k_ahead = __ldg(p.k_inv + tile0 + j + 1);
                v_ahead = __ldg(p.v_inv + tile0 + j + 1);
            }
            if (C::NB == 1 && j > 0) add_output(j - 1);  // its product is done before S_j begins: taken while S_j is computed
            const uint32_t s_addr = lane_base + C::S_COL + (uint32_t)(j % C::NB) * T + wg * HC;  // and 64 columns further for the second half
            const int lim = n_row - j * T - wg * HC;  // visible columns from there on
            const bool whole = __all_sync(0xffffffffu, lim >= 64 + HC);
            float mx = -INFINITY;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                await(s_full(j, half), j >> 1);
                tc::fence_after();
                float s[HC];
                tc::ldn(s_addr + 64 * half, s);
                if (whole) {
#pragma unroll
                    for (int e = 0; e < HC; e += 4) mx = fmaxf(mx, fmaxf(fmaxf(s[e], s[e + 1]), fmaxf(s[e + 2], s[e + 3])));
                } else {
#pragma unroll
                    for (int e = 0; e < HC; ++e) mx = fmaxf(mx, 64 * half + e < lim ? s[e] : -INFINITY);
                }
            }
            float* const row_max = shared_f + (j & 1) * (C::WGS * 128) + row;
            row_max[wg * 128] = mx;
            sync_rows();  // reached by all in every tile, also when a wait has run out
#pragma unroll
            for (int w = 0; w < C::WGS; ++w) mx = fmaxf(mx, row_max[w * 128]);
            if (!ok) continue;
            const float ref_new = mx == -INFINITY ? ref : fminf(ref, __fsub_rd(15.f, ceilf(mx * c)));
            const float shrink_next = ref == INFINITY ? 0.f : tc::ex2(ref_new - ref);
            ref = ref_new;
            // p = 2^15 exp2(s c - m): the factor 2^15 brings p into fp16's range and divides out with l
            const float base = ref == INFINITY ? 0.f : ref;
            const uint64_t c2 = tc::pack2(c, c), b2 = tc::pack2(base, base);
            // From 2^22 on the rounding of m, which an exact s c would leave in P, matters: there s c is rounded like m was.
            const bool plain = __all_sync(0xffffffffu, whole && fabsf(base) < 4194304.f);
            uint64_t sum2 = 0;
            auto hand_over = [&](int half) {
                tc::st_wait();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(j, half));
            };
            if (plain) {  // two loops: a choice inside would cost every element its instructions
#pragma unroll
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int g = 0; g < HC / GW; ++g) {
                        float s[GW];  // loaded again: with the sums of O the registers do not hold all columns
                        tc::ldn(s_addr + 64 * half + GW * g, s);
#pragma unroll
                        for (int e = 0; e < GW; e += 2) {
                            float x, y;
                            tc::unpack2(tc::fma2(tc::pack2(s[e], s[e + 1]), c2, b2), x, y);
                            s[e] = tc::ex2(x);
                            s[e + 1] = tc::ex2(y);
                            sum2 = tc::add2(sum2, tc::pack2(s[e], s[e + 1]));
                        }
                        tc::st_split(s_addr + 64 * half + GW * g, s);  // over the scores that they come from
                    }
                    hand_over(half);
                }
            } else {
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
#pragma unroll 1
                    for (int g = 0; g < HC / GW; ++g) {
                        const int col = 64 * half + GW * g;
                        float s[GW];
                        tc::ldn(s_addr + col, s);
#pragma unroll
                        for (int e = 0; e < GW; ++e) {
                            const float x = tc::ex2(__fadd_rn(__fmul_rn(s[e], c), base));
                            s[e] = col + e < lim ? x : 0.f;
                        }
#pragma unroll
                        for (int e = 0; e < GW; e += 2) sum2 = tc::add2(sum2, tc::pack2(s[e], s[e + 1]));
                        tc::st_split(s_addr + col, s);
                    }
                    hand_over(half);
                }
            }
            float x, y;
            tc::unpack2(sum2, x, y);
            l = fmaf(l, shrink_next, x + y);
            if (C::NB == 2 && j > 0) add_output(j - 1);  // the tile before: its product ran meanwhile
            shrink = shrink_next;
            v_inv = v_next;
        }
        if (ok && n_tiles > 0) add_output(n_tiles - 1);

        // ---- the sum over the warpgroups' columns, and the output through the stages: all products are done ----
        sync_rows();
        shared_f[wg * 128 + row] = l;
        sync_rows();
        l = 0.f;
#pragma unroll
        for (int w = 0; w < C::WGS; ++w) l += shared_f[w * 128 + row];
        // rows without keys: sum 0, output 0; a NaN in the sum reaches the output
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int d = 0; d < W; ++d) o[d] = l == 0.f ? 0.f : o[d] * inv;  // (0 times a NaN that other rows of the tile see)
        if (wg == 0 && a.stats && i < a.Sq) {
            float* st = a.stats + (((int64_t)b * a.H + h) * a.Sq + i) * 2;
            const float m = 15.f - ref;
            st[0] = m;
            st[1] = l == 0.f ? 0.f : l * exp2f(-(m + ref));  // 2^-15, but for the rounding of m
        }
        const int row0 = q_tile * ROWS + 32 * (warp & 3);
        tenmo_attn_write_rows<W>(o, a.o.ptr + b * a.o.sb + h * a.o.sh + (int64_t)row0 * a.o.sr + wg * W, a.o.sr, a.Sq - row0, a.D - wg * W, p.o_vec,
                                 false, reinterpret_cast<float*>(smem) + warp * (32 * W));
    }
    tc::fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag) atomicOr(p.status, TENMO_DEV_TIMEOUT);
    if (warp == C::ISSUER) {
        tc::fence_after();
        tc::dealloc(tmem, C::TMEM);
    }
}

size_t align_up(size_t n) { return (n + 1023) & ~(size_t)1023; }

}  // namespace

bool tenmo_attn_row_vec(const TenmoHeadsView& v, int D) {
    return D % 4 == 0 && v.sb % 4 == 0 && v.sh % 4 == 0 && v.sr % 4 == 0 && ((uintptr_t)v.ptr & 15u) == 0;
}

void tenmo_attn_causal_keys(const TenmoAttnParams& a, TenmoTileJob* j) {
    if (!a.causal) return;
    j->q_lengths = a.q_lengths;
    j->seen_by = a.Sq;
    j->offset = a.Sk - a.Sq;
}

int tenmo_attn_make_tiles(tenmo_ctx* ctx, const TenmoTileJobs& jobs, int count, int dp, int tile_rows) {
    int64_t most = 0;
    for (int c = 0; c < count; ++c) {
        const int64_t n = (int64_t)jobs.B * jobs.job[c].heads * jobs.job[c].tiles;
        if (n > most) most = n;
    }
    const dim3 grid((unsigned)most, (unsigned)count);
    if (dp == 64 && tile_rows == 64) attn_tiles_kernel<64, 64><<<grid, 256, 0, ctx->stream>>>(jobs);
    else if (dp == 64) attn_tiles_kernel<64, 128><<<grid, 256, 0, ctx->stream>>>(jobs);
    else if (tile_rows == 64) attn_tiles_kernel<128, 64><<<grid, 256, 0, ctx->stream>>>(jobs);
    else attn_tiles_kernel<128, 128><<<grid, 256, 0, ctx->stream>>>(jobs);
    TENMO_LAUNCH_CHECK(ctx, "attn_tiles_kernel");
    return TENMO_OK;
}

// Which kernels, from both sides measured over 4 .. 256 heads, dims 32 .. 128 and 16 .. 3000 rows and keys (one to three heads take the same rule
// without a measurement of their own; the tensor-core kernels never cut the keys, so few heads of few rows leave SMs idle).
// Forward: the few-row kernel takes about 10 us plus 3.7 ns for every row and 128 keys (dim 64), the tensor-core one 14 us plus the
// split of k and v, so it pays from some 2500 rows x 128 keys on (32 heads of 96x96: 15 us against 27; of 64x64: 15 against 13) -- but not for a
// few rows per head, which leave its 128-row tiles empty (256 heads of 4 rows and 3000 keys: 228 against 110).
// Backward: the row kernels take a warp through all keys (rows) of its row (key), the tensor-core ones 24 us at least: level at 64
// rows or keys with few heads (4 heads of 64x64: 24 us against 28) and at some 65,000 pairs with many (256 heads of 16x16: 40 against
// 32, of 32x32: 44 against 105).
bool tenmo_attn_tc_profitable(const TenmoAttnParams& p, bool backward) {
    const int64_t rows = (int64_t)p.B * p.H * p.Sq;
    if (rows == 0 || p.Sk == 0) return false;
    if (!backward) return p.Sq >= 16 && rows * ((p.Sk + 127) / 128) >= 2560;
    return p.Sq >= 64 || p.Sk >= 64 || rows * p.Sk > 65536;
}

int tenmo_attn_tc_fwd(tenmo_ctx* ctx, const TenmoAttnParams& a) {
    const int dp = tenmo_attn_padded(a.D);
    FwdParams p = {};
    p.a = a;
    p.tiles = (a.Sk + T - 1) / T;
    p.q_tiles = (a.Sq + ROWS - 1) / ROWS;
    p.q_vec = tenmo_attn_row_vec(a.q, a.D);
    p.o_vec = tenmo_attn_row_vec(a.o, a.D);
    p.status = ctx->dev_status;
    const int64_t n = (int64_t)a.B * a.Hkv * p.tiles;
    const size_t img = align_up((size_t)n * T * dp * 4), inv = align_up((size_t)n * sizeof(float));
    p.order = tenmo_attn_order(a, p.q_tiles, 2 * img);
    void* ws = nullptr;
    int st = tenmo_op_workspace(ctx, 2 * (img + inv), &ws);
    if (st != TENMO_OK) return st;
    uint8_t* w = (uint8_t*)ws;
    p.k_img = w;
    p.v_img = w + img;
    p.k_inv = (float*)(w + 2 * img);
    p.v_inv = (float*)(w + 2 * img + inv);
    TenmoTileJobs jobs = {};
    jobs.B = a.B;
    jobs.D = a.D;
    jobs.job[0] = TenmoTileJob{a.k, a.k_lengths, w, (float*)p.k_inv, a.Hkv, a.Sk, p.tiles, tenmo_attn_row_vec(a.k, a.D)};
    jobs.job[1] = TenmoTileJob{a.v, a.k_lengths, w + img, (float*)p.v_inv, a.Hkv, a.Sk, p.tiles, tenmo_attn_row_vec(a.v, a.D)};
    for (int e = 0; e < 2; ++e) tenmo_attn_causal_keys(a, &jobs.job[e]);
    if ((st = tenmo_attn_make_tiles(ctx, jobs, 2, dp, T)) != TENMO_OK) return st;
    const unsigned grid = (unsigned)((int64_t)a.B * a.H * p.q_tiles);
    if (dp == 64) {
        constexpr int THREADS = FwdCfg<64>::THREADS;
        TENMO_CUDA_TRY(ctx, cudaFuncSetAttribute(attn_fwd_tc_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, FwdCfg<64>::SMEM));
        attn_fwd_tc_kernel<64><<<grid, THREADS, FwdCfg<64>::SMEM, ctx->stream>>>(p);
    } else {
        constexpr int THREADS = FwdCfg<128>::THREADS;
        TENMO_CUDA_TRY(ctx, cudaFuncSetAttribute(attn_fwd_tc_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, FwdCfg<128>::SMEM));
        attn_fwd_tc_kernel<128><<<grid, THREADS, FwdCfg<128>::SMEM, ctx->stream>>>(p);
    }
    TENMO_LAUNCH_CHECK(ctx, "attn_fwd_tc_kernel");
    return TENMO_OK;
}
