// Tensor-core attention, backward: one kernel template for dq and for dk / dv.
//
// Two passes recompute the scores, one with the rows of q stationary and one with the keys: seven products instead of the five of
// a single pass, but no gradient is added by atomics (results repeat bit for bit) and no score tile crosses shared memory.
//   dq pass    X1 = q, X2 = go (128 rows, tensor memory), tiles of Y1 = k, Y2 = v:   S = X1 Y1^T, dP = X2 Y2^T,
//              dS = exp2(S c - m) (dP - delta),  dq += dS Y1
//   dkv pass   X1 = k, X2 = v (128 keys), tiles of Y1 = q, Y2 = go:  the same transposed, and  dv += P^T Y2,  dk += dS^T Y1
// P and dS are written as fp16 pairs over S and dP in tensor memory, where they are the next products' left operand; the tile
// images serve both as the right operand over the columns (S, dP) and over the rows (gradients).  The gradients of a tile are
// fresh accumulators that the warpgroups add to their registers with rounding.
// fp16 range of dS: |dP - delta| is bounded by the operands' scales (dim * 2^30 times the two inverse scales) and by the largest
// |delta|; a power of two from that bound brings dS to at most 2^15, exactly taken back when the tile is added.  The bound lies some 2^6 to
// 2^8 above the largest dS of normal data (dim times two maxima for a sum of random signs), so the pair's 22 bits end at 2^-11 of that dS
// and its error at 2^-31 of it; a bound from the rows' norms would be closer but would need them per row and key.
// One warp issues the MMAs, one the copies.  As in the forward pass the chain of a tile (S -> P -> dP -> dS -> sums) decides, so its
// columns are shared by four warpgroups (16 of the 64 columns of S a thread, a quarter of the gradient's; the dkv pass of dim 128, whose
// sums take 256 registers a row, has two).  Up to dim 64 S and dP have two buffers: the scores of tiles j + 1 and j + 2 are computed
// while tile j is worked on.  Up to dim 128 there is one of each and v of the dkv pass moves to shared memory; the products still
// follow each other without large gaps because each has one of another kind between itself and what it waits for.
// Shared key / value heads: the dkv pass works per query head into the workspace and a last kernel adds the heads of a group
// in order (per group it would leave most SMs idle behind the longest).
// Bound: tensor pipe, 3 * 14 * rows * keys * dim flop.
// Measured: 384 heads of 512x64, dq pass 193 us, dkv pass 245 us, pipe 31 to 33 % busy (a tile's chain and what a block costs besides); 16 heads of
// 4001x128 causal, 288 and 394 us, pipe 58 and 55 %.
#include "attention_tc.cuh"

namespace {

constexpr int ROWS = 128;
constexpr int T = ATTN_TILE;

struct BwdParams {
    TenmoAttnParams a;
    const uint8_t* y1_img; const uint8_t* y2_img;
    const float* y1_inv; const float* y2_inv;
    const float* info;   // row numbers per 64-row tile of q
    int tiles;           // tiles of a head of Y
    int q_info_tiles;    // 64-row tiles of a head of q
    int x_tiles;         // 128-row tiles of a head of X
    TenmoAttnOrder order;
    TenmoHeadsView x1, x2, out1, out2;  // out1: dq or dk, out2: dv
    int x1_vec, x2_vec, out1_vec, out2_vec;
    float beta;
    uint32_t* status;
};

template <int DP, bool DKV>
struct BwdCfg {
    static constexpr int WGS = DKV && DP == 128 ? 2 : 4;              // warpgroups that share a tile
    static constexpr int THREADS = WGS == 2 ? 384 : 128 * WGS + 64;  // two: the issuing warpgroup's registers go to them
    static constexpr int ISSUER = 4 * WGS, LOADER = ISSUER + 1;
    static constexpr int NC = T / WGS, W = DP / WGS;                 // columns of S and of the gradient of a thread
    static constexpr int NB = DP == 64 ? 2 : 1;                      // buffers of S and dP
    static constexpr bool X2S = DKV && DP == 128;  // X2 in shared memory
    static constexpr int STAGES = DP == 64 ? 5 : X2S ? 2 : 3;
    static constexpr int PLANE = T * DP * 2;
    static constexpr int STAGE = 4 * PLANE + (DKV ? 1024 : 0);  // Y1 hi, lo, Y2 hi, lo, row numbers
    static constexpr int X2_BYTES = X2S ? ROWS * DP * 4 : 0;
    static constexpr int X2_COL = DP;
    static constexpr int S_COL = X2S ? DP : 2 * DP, P_COL = S_COL + NB * T, A1_COL = P_COL + NB * T, A2_COL = A1_COL + DP;
    static constexpr int TMEM = 512;
    static_assert(A1_COL + (DKV ? 2 : 1) * DP <= TMEM, "tensor memory");
    static constexpr int TILES = STAGES * STAGE + X2_BYTES;
    static constexpr int SMEM = TILES + 2048 + 512;
    static_assert(STAGES * STAGE >= ROWS * DP * 4, "the output goes through the stages");
};

template <int DP, bool DKV>
__global__ void __launch_bounds__(BwdCfg<DP, DKV>::THREADS, 1) attn_bwd_tc_kernel(const __grid_constant__ BwdParams p) {
    using C = BwdCfg<DP, DKV>;
    constexpr int NB = C::NB, NC = C::NC, W = C::W;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* const x2_plane = smem + C::STAGES * C::STAGE;
    float* const exchange = reinterpret_cast<float*>(smem + C::TILES);
    const uint32_t bars = smem_u32(smem + C::TILES + 2048);
    auto full = [&](int slot) { return bars + 8u * (16 + slot); };
    auto empty = [&](int slot) { return bars + 8u * (24 + slot); };
    auto s_full = [&](int j) { return bars + 8u * (j & 1); };
    auto d_full = [&](int j) { return bars + 8u * (2 + (j & 1)); };
    // a warp may be a tile ahead of another one: what warps arrive on has a barrier for even and one for odd tiles
    auto p_full = [&](int j) { return bars + 8u * (7 + (j & 1)); };
    auto ds_full = [&](int j) { return bars + 8u * (9 + (j & 1)); };
    auto s_read = [&](int j) { return bars + 8u * (4 + (j & 1)); };
    auto acc_full = [&](int j) { return bars + 8u * (11 + (j & 1)); };
    auto acc_free = [&](int j) { return bars + 8u * (13 + (j & 1)); };
    const uint32_t pv_done = bars + 8u * 15, drain = bars + 8u * 6;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + C::TILES + 2048 + 256);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const TenmoAttnParams& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wg = warp >> 2, row = threadIdx.x & 127;
    // causal: the last rows of q see the most keys, the first keys are seen by the most rows; those blocks start first
    int x_tile, bh;
    tenmo_attn_block(p.order, blockIdx.x, &x_tile, &bh);
    if (!DKV) x_tile = p.x_tiles - 1 - x_tile;
    const int h = bh % a.H, b = bh / a.H, kvh = h / (a.H / a.Hkv);
    const int q_rows = tenmo_attn_rows(a.q_lengths, b, a.Sq), keys = tenmo_attn_rows(a.k_lengths, b, a.Sk);
    const int off = a.Sk - a.Sq;  // causal: key j is visible to row i when j <= i + off
    const int x_rows = DKV ? keys : q_rows;
    const int64_t i = (int64_t)x_tile * ROWS + row;  // this thread's row of X
    // tiles of Y that this block needs: [first, first + n)
    int first = 0, n = 0;
    const int top = min(x_rows, (x_tile + 1) * ROWS) - 1;  // last row of X that takes part
    if (top >= x_tile * ROWS) {
        if (DKV) {
            if (a.causal) first = max(0, x_tile * ROWS - off) / T;
            n = max(0, (q_rows + T - 1) / T - first);
        } else {
            int seen = keys;
            if (a.causal) seen = min(seen, max(0, top + off + 1));
            n = (seen + T - 1) / T;
        }
    }
    const int yh = DKV ? h : kvh, y_heads = DKV ? a.H : a.Hkv;
    const int64_t tile0 = ((int64_t)b * y_heads + yh) * p.tiles + first;
    if (n == 0) {  // nothing to add: rows (keys) behind the length, or none that sees (is seen by) another
        if (p.beta == 0.f) {
            tenmo_attn_zero_rows<DP>(p.out1.ptr + b * p.out1.sb + h * p.out1.sh, p.out1.sr, x_tile * ROWS, DKV ? a.Sk : a.Sq, a.D, p.out1_vec);
            if (DKV) tenmo_attn_zero_rows<DP>(p.out2.ptr + b * p.out2.sb + h * p.out2.sh, p.out2.sr, x_tile * ROWS, a.Sk, a.D, p.out2_vec);
        }
        return;
    }

    // the ring of tiles (one thread): a slot is refilled when all products of its tile are done
    int fetched = 0, fetch_slot = 0, fetch_round = 0;
    auto fetch = [&](int until) {
        for (; fetched < until; ++fetched) {
            if (fetch_round && !mbar_wait(empty(fetch_slot), (uint32_t)(fetch_round - 1) & 1u, abort_flag)) return;
            const uint32_t dst = smem_u32(smem) + fetch_slot * C::STAGE, bar = full(fetch_slot);
            mbar_expect_tx(bar, 4 * C::PLANE + (DKV ? 1024u : 0u));
            tc::bulk_load(dst, p.y1_img + (tile0 + fetched) * (2 * C::PLANE), 2 * C::PLANE, bar);
            tc::bulk_load(dst + 2 * C::PLANE, p.y2_img + (tile0 + fetched) * (2 * C::PLANE), 2 * C::PLANE, bar);
            if (DKV) tc::bulk_load(dst + 4 * C::PLANE, p.info + (tile0 + fetched) * ATTN_INFO, 1024, bar);
            if (++fetch_slot == C::STAGES) { fetch_slot = 0; ++fetch_round; }
        }
    };
    if (threadIdx.x == 32 * C::LOADER) {  // the thread that copies: the first tiles are on their way before the block meets
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int w = 0; w < 2; ++w) {
            mbar_init(s_full(w), 1);
            mbar_init(d_full(w), 1);
            mbar_init(acc_full(w), 1);
            mbar_init(s_read(w), 4 * C::WGS);
            mbar_init(p_full(w), 4 * C::WGS);
            mbar_init(ds_full(w), 4 * C::WGS);
            mbar_init(acc_free(w), 4 * C::WGS);
        }
        mbar_init(pv_done, 1);
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tc::fence_proxy_async();
        fetch(min(n, C::STAGES - 1));  // the last slot is scratch for now
    }

    auto fetch_x = [&](const TenmoHeadsView& v, bool vec, float (&x)[W]) {
        const int64_t x0 = (int64_t)x_tile * ROWS;
        tenmo_attn_fetch<DP, C::WGS>(x, v.ptr + b * v.sb + (DKV ? kvh : h) * v.sh + x0 * v.sr, v.sr, x_rows - x_tile * ROWS, vec, a.D,
                                     reinterpret_cast<float*>(smem + (C::STAGES - 1) * C::STAGE));
    };
    constexpr bool BOTH = W <= 32;  // as the registers allow
    float x1[W], x2[W];
    if (warp < C::ISSUER) {
        fetch_x(p.x1, p.x1_vec, x1);
        if (BOTH) fetch_x(p.x2, p.x2_vec, x2);
    }

    if (warp == C::ISSUER) tc::alloc(tmem_slot, C::TMEM);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);


    float x1_inv = 1.f, x2_inv = 1.f;
    if (warp < C::ISSUER) {
        x1_inv = tenmo_attn_stationary<DP, false, C::WGS>(x1, a.scale < 0.f, lane_base, nullptr, exchange);
        if (!BOTH) fetch_x(p.x2, p.x2_vec, x2);
        x2_inv = tenmo_attn_stationary<DP, C::X2S, C::WGS>(x2, false, lane_base + C::X2_COL, x2_plane, exchange);
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();

    if (warp >= C::ISSUER) {
        if (C::WGS == 2) tc::regs_down<88>();
        if (warp == C::LOADER) {
            if (lane == 0) {
                fetch(n);
                // every copy has landed before shared memory is given back (bounded)
                int never = 0;
                for (int t = max(0, fetched - C::STAGES); t < fetched; ++t) mbar_wait(full(t % C::STAGES), (uint32_t)(t / C::STAGES) & 1u, &never);
            }
        } else if (warp == C::ISSUER) {
            const uint32_t tm = tc::uniform(tmem), stages = tc::uniform(smem_u32(smem));
            const int tiles = tc::uniform(n);
            constexpr uint32_t ID_S = tc::idesc_f16(T, false), ID_G = tc::idesc_f16(DP, true);
            auto wait = [&](uint32_t bar, int phase) { return __all_sync(0xffffffffu, mbar_wait(bar, (uint32_t)phase & 1u, abort_flag)) != 0; };
            // S or dP: D = X Y^T over the columns; x: tensor memory (hi, then lo DP / 2 columns further)
            auto over_columns = [&](uint32_t d, uint32_t x, uint32_t hi) {
#pragma unroll
                for (int c = 0; c < DP / 64; ++c) tc::mma4_ts<8, tc::STEP_K>(d, x + DP / 2 + 32 * c, tc::desc_k(hi + c * T * 128), ID_S, c == 0);
#pragma unroll
                for (int c = 0; c < DP / 64; ++c) tc::mma4_ts<8, tc::STEP_K>(d, x + 32 * c, tc::desc_k(hi + C::PLANE + c * T * 128), ID_S, false);
#pragma unroll
                for (int c = 0; c < DP / 64; ++c) tc::mma4_ts<8, tc::STEP_K>(d, x + 32 * c, tc::desc_k(hi + c * T * 128), ID_S, false);
            };
            int s_slot = 0, s_phase = 0;  // of the next S
            auto arrived = [&]() { return wait(full(s_slot), s_phase); };  // asked before the wait that ends last: one that is over costs its latency too
            auto scores = [&](int j) {
                tc::fence_after();
                over_columns(tm + C::S_COL + (uint32_t)(j % NB) * T, tm, stages + s_slot * C::STAGE);
                tc::commit(s_full(j));
            };
            auto grads = [&](int j) {  // dP_j; its tile has arrived: S_j was issued before
                const uint32_t hi = stages + s_slot * C::STAGE + 2 * C::PLANE, d = tm + C::P_COL + (uint32_t)(j % NB) * T;
                if (C::X2S) {
                    const uint32_t xh = stages + C::STAGES * C::STAGE, xl = xh + ROWS * DP * 2;
#pragma unroll
                    for (int c = 0; c < DP / 64; ++c)
                        tc::mma4_ss<tc::STEP_K, tc::STEP_K>(d, tc::desc_k(xl + c * ROWS * 128), tc::desc_k(hi + c * T * 128), ID_S, c == 0);
#pragma unroll
                    for (int c = 0; c < DP / 64; ++c)
                        tc::mma4_ss<tc::STEP_K, tc::STEP_K>(d, tc::desc_k(xh + c * ROWS * 128), tc::desc_k(hi + C::PLANE + c * T * 128), ID_S, false);
#pragma unroll
                    for (int c = 0; c < DP / 64; ++c)
                        tc::mma4_ss<tc::STEP_K, tc::STEP_K>(d, tc::desc_k(xh + c * ROWS * 128), tc::desc_k(hi + c * T * 128), ID_S, false);
                } else {
                    over_columns(d, tm + C::X2_COL, hi);
                }
                tc::commit(d_full(j));
                if (++s_slot == C::STAGES) { s_slot = 0; s_phase ^= 1; }
            };
            // D = A Y over the rows of the tile; A: rows 16 k .. in eight columns of hi pairs from 16 k on, then eight of lo pairs
            auto over_rows = [&](uint32_t d, uint32_t x, uint32_t hi) {
                tc::mma4_ts<16, tc::STEP_MN>(d, x + 8, tc::desc_mn(hi, T), ID_G, true);
                tc::mma4_ts<16, tc::STEP_MN>(d, x, tc::desc_mn(hi + C::PLANE, T), ID_G, false);
                tc::mma4_ts<16, tc::STEP_MN>(d, x, tc::desc_mn(hi, T), ID_G, false);
            };
            // Order: the products of tile j that use P_j and dS_j, then S and dP of tile j + NB, which replace them.  Each waits for
            // something that is done while another product runs: S for P_j v (dkv) or for S_j's readers (dq), dP for the products of dS_j.
            bool ok = true;
            for (int j = 0; ok && j < min(tiles, NB); ++j) {
                ok = arrived();
                if (ok) { scores(j); grads(j); }
            }
            int slot = 0;  // of tile j
            for (int j = 0; ok && j < tiles; ++j) {
                const uint32_t s = tm + C::S_COL + (uint32_t)(j % NB) * T, ds = tm + C::P_COL + (uint32_t)(j % NB) * T, y1 = stages + slot * C::STAGE;
                const bool more = j + NB < tiles;
                auto sums_taken = [&]() { return j == 0 || wait(acc_free(j - 1), (j - 1) >> 1); };
                if (NB == 1 && !DKV && more) {  // one buffer: S_{j+1} runs while the warpgroups make dS_j
                    ok = arrived() && wait(s_read(j), j >> 1);
                    if (!ok) break;
                    scores(j + 1);
                }
                if (DKV) {
                    ok = wait(p_full(j), j >> 1) && sums_taken();
                    if (!ok) break;
                    tc::fence_after();
                    over_rows(tm + C::A2_COL, s, y1 + 2 * C::PLANE);
                    tc::commit(pv_done);
                }
                ok = wait(ds_full(j), j >> 1) && (DKV || sums_taken());
                if (!ok) break;
                tc::fence_after();
                over_rows(tm + C::A1_COL, ds, y1);
                tc::commit(acc_full(j));
                tc::commit(empty(slot));  // the tile is over
                if (++slot == C::STAGES) slot = 0;
                if (more) {
                    if (DKV || NB == 2) {  // P_j has been read (dkv), or S_j has, before dS_j was there
                        ok = arrived() && (!DKV || wait(pv_done, j));
                        if (!ok) break;
                        scores(j + NB);
                    }
                    ok = wait(acc_full(j), j >> 1);  // dS_j has been read
                    if (!ok) break;
                    tc::fence_after();
                    grads(j + NB);
                }
            }
            if (!ok) {  // a wait ran out: see the MMAs in flight to their end (bounded) before tensor memory is given back
                tc::commit(drain);
                int never = 0;
                mbar_wait(drain, 0, &never);
            }
        }
    } else {
        if (C::WGS == 2) tc::regs_up<208>();
        constexpr int W2 = DKV ? W : 2;   // the dq pass has no second gradient
        constexpr int LD = W < 32 ? W : 32;  // columns at a time
        float acc1[W], acc2[W2];
#pragma unroll
        for (int d = 0; d < W; ++d) acc1[d] = 0.f;
#pragma unroll
        for (int d = 0; d < W2; ++d) acc2[d] = 0.f;
        const float c_row = fabsf(a.scale_log2) * x1_inv;
        // dq pass: the row's numbers
        float negm_row = -INFINITY, il_row = 0.f, delta_row = 0.f;
        int n_row = 0;
        if (!DKV && i < q_rows) {
            const float* info = p.info + (((int64_t)b * a.H + h) * p.q_info_tiles + (i >> 6)) * ATTN_INFO;
            const int r = (int)(i & 63);
            negm_row = info[4 * (r >> 1) + (r & 1)];
            il_row = info[4 * (r >> 1) + 2 + (r & 1)] * info[3 * T + 2];
            delta_row = info[2 * T + r];
            n_row = keys;
            if (a.causal) n_row = min(n_row, (int)max((int64_t)0, i + off + 1));
        }
        bool ok = true;
        auto await = [&](uint32_t bar, int phase) { ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, (uint32_t)phase & 1u, abort_flag)); };
        // factors that the tile in flight in the accumulators is added with
        float f1 = 0.f, f2 = 0.f;
        auto add_tile = [&](int j) {  // registers += accumulators of tile j
            await(acc_full(j), j >> 1);
            if (!ok) return;
            tc::fence_after();
            const uint64_t g1 = tc::pack2(f1, f1), g2 = tc::pack2(f2, f2);
#pragma unroll
            for (int g = 0; g < W / LD; ++g) {
                float t[LD];
                tc::ldn(lane_base + C::A1_COL + wg * W + LD * g, t);
#pragma unroll
                for (int e = 0; e < LD; e += 2)
                    tc::unpack2(tc::fma2(tc::pack2(t[e], t[e + 1]), g1, tc::pack2(acc1[LD * g + e], acc1[LD * g + e + 1])), acc1[LD * g + e],
                                acc1[LD * g + e + 1]);
                if (DKV) {
                    tc::ldn(lane_base + C::A2_COL + wg * W + LD * g, t);
#pragma unroll
                    for (int e = 0; e < LD; e += 2)
                        tc::unpack2(tc::fma2(tc::pack2(t[e], t[e + 1]), g2, tc::pack2(acc2[(LD * g + e) % W2], acc2[(LD * g + e + 1) % W2])),
                                    acc2[(LD * g + e) % W2], acc2[(LD * g + e + 1) % W2]);
                }
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_free(j));
        };
        // What a tile's elements need besides S and dP: P = exp2(S c + (-m)) (il), dS = P (dP f G - delta G).  G, a power of two, brings dS
        // to at most 2^15; PS is the power of two in il (dkv pass).
        struct Tile {
            uint64_t c2, fg2, ng2;  // c, f * G, -G (dkv) or -delta * G (dq)
            float G, ps_inv;
            const float* info;
            int lim;                // first visible column (dkv) or their number (dq), of this thread's columns
            bool whole;             // no column is masked, and the scores' rounding cannot lift P far above 1
        };
        // |S| <= DP 2^30 and a recomputed S c differs from the forward pass's by 2^-19 of that times c at most: below 1?
        auto rounding = [](float c) { return c * (DP * 2048.f) < 1.f; };
        auto set_up = [&](int j, float y1_inv, float y2_inv) {
            Tile t;
            const float c = c_row * y1_inv, f = x2_inv * y2_inv;  // dP = f * accumulator
            const int col0 = NC * wg;
            t.c2 = tc::pack2(c, c);
            if (DKV) {
                t.info = reinterpret_cast<const float*>(smem + (j % C::STAGES) * C::STAGE + 4 * C::PLANE);
                t.ps_inv = t.info[3 * T + 2];  // read before dS is handed over: the stage may be refilled from then on
                t.G = tc::pow2_below_inverse(fmaf((float)DP * 1073741824.f, f, t.info[3 * T + 1]));
                t.ng2 = tc::pack2(-t.G, -t.G);
                t.lim = a.causal ? (int)max((int64_t)-1, min((int64_t)T, i - off - (int64_t)(first + j) * T)) - col0 : 0;
                t.whole = __all_sync(0xffffffffu, t.lim <= 0 && rounding(c));
            } else {
                t.info = nullptr;
                t.ps_inv = 1.f;
                t.G = 32768.f * tc::pow2_below_inverse(fmaf((float)DP * 1073741824.f, f, fabsf(delta_row)));
                t.ng2 = tc::pack2(-delta_row * t.G, -delta_row * t.G);
                t.lim = n_row - j * T - col0;
                t.whole = __all_sync(0xffffffffu, t.lim >= NC && rounding(c));
            }
            t.fg2 = tc::pack2(f * t.G, f * t.G);
            return t;
        };
        const uint64_t negm2 = tc::pack2(negm_row, negm_row);
        // columns u, u + 1 (of this thread's; info0: their rows' place in the tile): P, and its masking
        auto prob2 = [&](const Tile& t, float x, float y, int u, int info0, bool whole) {
            uint64_t v;
            if (DKV) {
                const float4 mi = *reinterpret_cast<const float4*>(t.info + 2 * info0);
                v = tc::fma2(tc::pack2(x, y), t.c2, tc::pack2(mi.x, mi.y));
                tc::unpack2(v, x, y);
                v = tc::mul2(tc::pack2(tc::ex2(x), tc::ex2(y)), tc::pack2(mi.z, mi.w));
            } else {
                v = tc::fma2(tc::pack2(x, y), t.c2, negm2);
                tc::unpack2(v, x, y);
                v = tc::pack2(tc::ex2(x), tc::ex2(y));
            }
            if (!whole) {
                tc::unpack2(v, x, y);
                const float most = DKV ? 32768.f : 1.f;  // (a NaN stays)
                x = (DKV ? u >= t.lim : u < t.lim) ? (x > most ? most : x) : 0.f;
                y = (DKV ? u + 1 >= t.lim : u + 1 < t.lim) ? (y > most ? most : y) : 0.f;
                v = tc::pack2(x, y);
            }
            return v;
        };
        auto dscore2 = [&](const Tile& t, uint64_t prob, float x, float y, int info0) {
            uint64_t shift = t.ng2;
            if (DKV) {
                const float2 d = *reinterpret_cast<const float2*>(t.info + 2 * T + info0);
                shift = tc::mul2(tc::pack2(d.x, d.y), t.ng2);
            }
            return tc::mul2(prob, tc::fma2(tc::pack2(x, y), t.fg2, shift));
        };
        auto factors = [&](const Tile& t, float y1_inv, float y2_inv) {
            f1 = a.scale * y1_inv * tc::pow2_inverse(t.G) * (DKV ? t.ps_inv : il_row);
            f2 = y2_inv * t.ps_inv;
        };
        // the tiles' scales come from L2: loaded a tile ahead
        float y1_next = n ? __ldg(p.y1_inv + tile0) : 1.f, y2_next = n ? __ldg(p.y2_inv + tile0) : 1.f;
        for (int j = 0; j < n; ++j) {
            const float y1_inv = y1_next, y2_inv = y2_next;
            if (j + 1 < n) {
                y1_next = __ldg(p.y1_inv + tile0 + j + 1);
                y2_next = __ldg(p.y2_inv + tile0 + j + 1);
            }
            const uint32_t s_addr = lane_base + C::S_COL + (uint32_t)(j % NB) * T + NC * wg, d_addr = s_addr + (C::P_COL - C::S_COL);
            // one buffer, dkv pass: the sums of tile j - 1 are taken first, while S_j is being computed
            if (NB == 1 && DKV && j >= 1) add_tile(j - 1);
            if (DKV) await(full(j % C::STAGES), j / C::STAGES);  // the row numbers that came with the tile
            await(s_full(j), j >> 1);
            if (!ok) break;
            tc::fence_after();
            const Tile t = set_up(j, y1_inv, y2_inv);
            float e[NC];
            tc::ldn(s_addr, e);
            if (!DKV) {  // nothing is written over S
                tc::fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_read(j));
            }
            if (t.whole) {  // two loops: a choice inside would cost every element its instructions
#pragma unroll
                for (int u = 0; u < NC; u += 2) tc::unpack2(prob2(t, e[u], e[u + 1], u, NC * wg + u, true), e[u], e[u + 1]);
            } else {
#pragma unroll
                for (int u = 0; u < NC; u += 2) tc::unpack2(prob2(t, e[u], e[u + 1], u, NC * wg + u, false), e[u], e[u + 1]);
            }
            if (DKV) {
                tc::st_split(s_addr, e);
                tc::st_wait();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(j));
            } else if (NB == 1 && j >= 1) {
                add_tile(j - 1);  // while dP_j is being computed
            }
            await(d_full(j), j >> 1);
            if (!ok) break;
            tc::fence_after();
            {
                float v[NC];
                tc::ldn(d_addr, v);
#pragma unroll
                for (int u = 0; u < NC; u += 2) tc::unpack2(dscore2(t, tc::pack2(e[u], e[u + 1]), v[u], v[u + 1], NC * wg + u), v[u], v[u + 1]);
                tc::st_split(d_addr, v);
            }
            tc::st_wait();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ds_full(j));
            if (NB == 2 && j >= 1) add_tile(j - 1);
            factors(t, y1_inv, y2_inv);
            if (!ok) break;
        }
        if (ok && n > 0) add_tile(n - 1);

        // ---- to memory, through the stages ----
        // rows that see no key, keys that no row sees: zeros, whatever their neighbours in the tile hold
        const bool valid = i < x_rows && (DKV ? !a.causal || i <= (int64_t)q_rows - 1 + off : n_row > 0);
        const int row0 = x_tile * ROWS + 32 * (warp & 3), here = (DKV ? a.Sk : a.Sq) - row0;
        auto out_row = [&](const TenmoHeadsView& out) { return out.ptr + b * out.sb + h * out.sh + (int64_t)row0 * out.sr; };
        float* const scratch = reinterpret_cast<float*>(smem) + warp * (32 * W);  // all products are done: the stages are free
#pragma unroll
        for (int d = 0; d < W; ++d) acc1[d] = valid ? acc1[d] : 0.f;
        tenmo_attn_write_rows<W>(acc1, out_row(p.out1) + wg * W, p.out1.sr, here, a.D - wg * W, p.out1_vec, p.beta != 0.f, scratch);
        if constexpr (DKV) {
#pragma unroll
            for (int d = 0; d < W; ++d) acc2[d] = valid ? acc2[d] : 0.f;
            tenmo_attn_write_rows<W>(acc2, out_row(p.out2) + wg * W, p.out2.sr, here, a.D - wg * W, p.out2_vec, p.beta != 0.f, scratch);
        }
    }
    tc::fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag) atomicOr(p.status, TENMO_DEV_TIMEOUT);
    if (warp == C::ISSUER) {
        tc::fence_after();
        tc::dealloc(tmem, C::TMEM);
    }
}

// dk, dv (+)= the sums of the partial gradients of a group's heads, in order.  A warp is a key; VEC: 16 bytes a lane.
// Bound: HBM.  16 heads on 4, 4001 keys, dim 128: 65 MB read.
template <bool VEC>
__global__ void __launch_bounds__(256) attn_fold_kernel(const float* dk_part, const float* dv_part, const TenmoAttnParams a) {
    const int group = a.H / a.Hkv, lane = threadIdx.x & 31;
    const int64_t per_head = (int64_t)a.Sk * a.D;
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= (int64_t)a.B * a.Hkv * a.Sk) return;
    const int64_t bh = row / a.Sk, j = row - bh * a.Sk;
    const int b = (int)(bh / a.Hkv), kvh = (int)(bh % a.Hkv);
    const float* src = (blockIdx.y ? dv_part : dk_part) + ((int64_t)b * a.H + (int64_t)kvh * group) * per_head + j * a.D;
    const TenmoHeadsView& out = blockIdx.y ? a.dv : a.dk;
    float* dst = out.ptr + b * out.sb + kvh * out.sh + j * out.sr;
    if (VEC) {
        const int d = 4 * lane;  // D <= 128: one step
        if (d >= a.D) return;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int g = 0; g < group; ++g) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(src + g * per_head + d));
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        if (a.beta != 0.f) {
            const float4 o = *reinterpret_cast<const float4*>(dst + d);
            s.x += o.x; s.y += o.y; s.z += o.z; s.w += o.w;
        }
        *reinterpret_cast<float4*>(dst + d) = s;
    } else {
        for (int d = lane; d < a.D; d += 32) {
            float s = 0.f;
#pragma unroll 4
            for (int g = 0; g < group; ++g) s += __ldg(src + g * per_head + d);
            dst[d] = a.beta != 0.f ? dst[d] + s : s;
        }
    }
}

size_t align_up(size_t n) { return (n + 1023) & ~(size_t)1023; }

template <int DP, bool DKV>
int launch(tenmo_ctx* ctx, const BwdParams& p) {
    const int smem = BwdCfg<DP, DKV>::SMEM;
    TENMO_CUDA_TRY(ctx, cudaFuncSetAttribute(attn_bwd_tc_kernel<DP, DKV>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    const unsigned grid = (unsigned)((int64_t)p.a.B * p.a.H * p.x_tiles);
    attn_bwd_tc_kernel<DP, DKV><<<grid, BwdCfg<DP, DKV>::THREADS, smem, ctx->stream>>>(p);
    TENMO_LAUNCH_CHECK(ctx, "attn_bwd_tc_kernel");
    return TENMO_OK;
}

}  // namespace

int tenmo_attn_tc_bwd(tenmo_ctx* ctx, const TenmoAttnParams& a) {
    const int dp = tenmo_attn_padded(a.D);
    const int k_tiles = (a.Sk + T - 1) / T, q_tiles = (a.Sq + T - 1) / T;
    const int64_t nk = (int64_t)a.B * a.Hkv * k_tiles, nq = (int64_t)a.B * a.H * q_tiles;
    const size_t k_img = align_up((size_t)nk * T * dp * 4), q_img = align_up((size_t)nq * T * dp * 4);
    const size_t k_inv = align_up((size_t)nk * sizeof(float)), q_inv = align_up((size_t)nq * sizeof(float));
    const size_t info = align_up((size_t)nq * ATTN_INFO * sizeof(float));
    const bool grouped = a.H != a.Hkv;
    const size_t part = grouped ? align_up((size_t)a.B * a.H * a.Sk * a.D * sizeof(float)) : 0;
    void* ws = nullptr;
    int st = tenmo_op_workspace(ctx, 2 * (k_img + q_img + k_inv + q_inv + part) + info, &ws);
    if (st != TENMO_OK) return st;
    uint8_t* w = (uint8_t*)ws;
    uint8_t *ik = w, *iv = ik + k_img, *iq = iv + k_img, *ig = iq + q_img;
    float* vk = (float*)(ig + q_img);
    float* vv = (float*)((uint8_t*)vk + k_inv);
    float* vq = (float*)((uint8_t*)vv + k_inv);
    float* vg = (float*)((uint8_t*)vq + q_inv);
    float* in = (float*)((uint8_t*)vg + q_inv);
    float* pk = (float*)((uint8_t*)in + info);
    float* pv = (float*)((uint8_t*)pk + part);
    TenmoTileJobs jobs = {};
    jobs.B = a.B;
    jobs.D = a.D;
    jobs.job[0] = TenmoTileJob{a.k, a.k_lengths, ik, vk, a.Hkv, a.Sk, k_tiles, tenmo_attn_row_vec(a.k, a.D)};
    jobs.job[1] = TenmoTileJob{a.v, a.k_lengths, iv, vv, a.Hkv, a.Sk, k_tiles, tenmo_attn_row_vec(a.v, a.D)};
    for (int e = 0; e < 2; ++e) tenmo_attn_causal_keys(a, &jobs.job[e]);
    const int first = a.causal && a.Sq > a.Sk ? a.Sq - a.Sk : 0;  // the first row that sees a key
    jobs.job[2] = TenmoTileJob{a.q, a.q_lengths, iq, vq, a.H, a.Sq, q_tiles, tenmo_attn_row_vec(a.q, a.D), first};
    jobs.job[3] = TenmoTileJob{a.go, a.q_lengths, ig, vg, a.H, a.Sq, q_tiles, tenmo_attn_row_vec(a.go, a.D), first};
    jobs.job[3].o = a.o;
    jobs.job[3].o_vec = tenmo_attn_row_vec(a.o, a.D);
    jobs.job[3].stats = a.stats;
    jobs.job[3].info = in;
    if ((st = tenmo_attn_make_tiles(ctx, jobs, 4, dp, T)) != TENMO_OK) return st;

    BwdParams p = {};
    p.a = a;
    p.info = in;
    p.q_info_tiles = q_tiles;
    p.status = ctx->dev_status;
    // dq
    p.y1_img = ik; p.y2_img = iv; p.y1_inv = vk; p.y2_inv = vv;
    p.tiles = k_tiles;
    p.x_tiles = (a.Sq + ROWS - 1) / ROWS;
    p.order = tenmo_attn_order(a, p.x_tiles, 2 * k_img);
    p.x1 = a.q; p.x2 = a.go; p.out1 = a.dq; p.out2 = a.dq;
    p.x1_vec = tenmo_attn_row_vec(a.q, a.D); p.x2_vec = tenmo_attn_row_vec(a.go, a.D);
    p.out1_vec = p.out2_vec = tenmo_attn_row_vec(a.dq, a.D);
    p.beta = a.beta;
    if ((st = dp == 64 ? launch<64, false>(ctx, p) : launch<128, false>(ctx, p)) != TENMO_OK) return st;
    // dk, dv
    p.y1_img = iq; p.y2_img = ig; p.y1_inv = vq; p.y2_inv = vg;
    p.tiles = q_tiles;
    p.x_tiles = (a.Sk + ROWS - 1) / ROWS;
    p.order = tenmo_attn_order(a, p.x_tiles, 2 * q_img);
    p.x1 = a.k; p.x2 = a.v;
    p.x1_vec = tenmo_attn_row_vec(a.k, a.D); p.x2_vec = tenmo_attn_row_vec(a.v, a.D);
    if (grouped) {
        const int64_t per = (int64_t)a.Sk * a.D;
        p.out1 = TenmoHeadsView{pk, per * a.H, per, a.D};
        p.out2 = TenmoHeadsView{pv, per * a.H, per, a.D};
        p.beta = 0.f;
    } else {
        p.out1 = a.dk;
        p.out2 = a.dv;
    }
    p.out1_vec = tenmo_attn_row_vec(p.out1, a.D);
    p.out2_vec = tenmo_attn_row_vec(p.out2, a.D);
    if ((st = dp == 64 ? launch<64, true>(ctx, p) : launch<128, true>(ctx, p)) != TENMO_OK) return st;
    if (grouped) {
        const dim3 grid((unsigned)(((int64_t)a.B * a.Hkv * a.Sk + 7) / 8), 2);
        if (tenmo_attn_row_vec(a.dk, a.D) && tenmo_attn_row_vec(a.dv, a.D)) attn_fold_kernel<true><<<grid, 256, 0, ctx->stream>>>(pk, pv, a);
        else attn_fold_kernel<false><<<grid, 256, 0, ctx->stream>>>(pk, pv, a);
        TENMO_LAUNCH_CHECK(ctx, "attn_fold_kernel");
    }
    return TENMO_OK;
}
