// Fifth-generation tensor core pieces shared by the fp16-pair kernels: fp32 products on fp16 tensor cores.
//
// Arithmetic.  A block of an fp32 operand is scaled by a power of two 2^e (its largest finite entry comes to lie in
// [2^14, 2^15)) and written as hi + lo, two fp16 numbers: hi = fp16(x 2^e), lo = fp16(x 2^e - hi).  That keeps 22 bits of an
// entry down to 2^-18 of the block's largest one and an absolute 2^-40 of it below.  A product of two such operands is
// lo.hi + hi.lo + hi.hi, three tcgen05.mma of kind::f16 into one fp32 accumulator; the dropped lo.lo is at most 2^-22 of the
// term, or 2^-21 where an operand made inside a loop is cut instead of rounded.  The powers of two come off in fp32, exactly.  fp16 runs at twice the rate of TF32 and its planes are half as
// large, which is why these kernels do not use the three TF32 products of the dense GEMM.
// The tensor core adds into its accumulator with truncation, so a chain is kept short (one tile) and tiles are added in
// registers with rounding; within a chain the two small products go first, while the accumulator is small.
//
// Tile image.  A tile of R rows x DP columns (DP a multiple of 64) is stored as the hi plane and then the lo plane, each as
// DP / 64 panels of R rows x 128 bytes, 16-byte chunk c of row r at chunk c ^ (r & 7): the 128-byte swizzle the tensor core
// reads.  The image is made once in global memory, so one plain bulk copy brings a tile in and no tensor map is needed.
// The same image serves a product over the columns (rows are M or N, "K-major") and one over the rows ("MN-major").
#pragma once
#include <cuda_fp16.h>

#include "op_util.cuh"
#include "tma_util.cuh"

namespace tc {

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// generic-proxy writes to shared memory become visible to the tensor core and the copy engine
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void alloc(uint32_t* slot, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void dealloc(uint32_t base, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}
// MMAs and commits are written for a whole converged warp, and one elected lane (always the same) executes them: what they are
// computed from then is uniform over the warp and the compiler keeps it in uniform registers, where the tensor core wants it.  Issued
// from a branch that a single thread takes, every MMA cost about 85 cycles of register moves, more than most take to run.
// arrives on `bar` when all MMAs issued so far are done
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
        : "memory");
}
// Four steps of a product (64 of the contraction): D[tmem] (+)= A . B, B in shared memory.  A tensor-memory operand (TS) holds row r
// in lane r, two fp16 per 32-bit column, and a step is AS columns further; of a shared-memory operand (SS), as of B, a step is
// AS / BS units of 16 bytes, an addition to the descriptor's low word (the address; a tile ends below 256 KB).  `first`: the first
// step overwrites D.  One election serves the four; the high words are constants.
struct Desc { uint32_t lo, hi; };
template <int AS, int BS>
__device__ __forceinline__ void mma4_ts(uint32_t d, uint32_t a, Desc b, uint32_t idesc, bool first) {
    asm volatile(
        "{\n\t.reg .pred e, p, q;\n\t.reg .b64 b0, b1, b2, b3;\n\t.reg .b32 l1, l2, l3, a1, a2, a3;\n\t"
        "add.u32 l1, %2, %6;\n\tadd.u32 l2, %2, %7;\n\tadd.u32 l3, %2, %8;\n\t"
        "add.u32 a1, %1, %9;\n\tadd.u32 a2, %1, %10;\n\tadd.u32 a3, %1, %11;\n\t"
        "mov.b64 b0, {%2, %3};\n\tmov.b64 b1, {l1, %3};\n\tmov.b64 b2, {l2, %3};\n\tmov.b64 b3, {l3, %3};\n\t"
        "setp.eq.b32 p, %5, 0;\n\tsetp.eq.b32 q, 0, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b0, %4, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %4, q;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %4, q;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %4, q;\n\t}"
        ::"r"(d), "r"(a), "r"(b.lo), "r"(b.hi), "r"(idesc), "r"((uint32_t)first), "n"(BS), "n"(2 * BS), "n"(3 * BS), "n"(AS), "n"(2 * AS), "n"(3 * AS)
        : "memory");
}
template <int AS, int BS>
__device__ __forceinline__ void mma4_ss(uint32_t d, Desc a, Desc b, uint32_t idesc, bool first) {
    asm volatile(
        "{\n\t.reg .pred e, p, q;\n\t.reg .b64 a0, a1, a2, a3, b0, b1, b2, b3;\n\t.reg .b32 l1, l2, l3, m1, m2, m3;\n\t"
        "add.u32 l1, %3, %7;\n\tadd.u32 l2, %3, %8;\n\tadd.u32 l3, %3, %9;\n\t"
        "add.u32 m1, %1, %10;\n\tadd.u32 m2, %1, %11;\n\tadd.u32 m3, %1, %12;\n\t"
        "mov.b64 b0, {%3, %4};\n\tmov.b64 b1, {l1, %4};\n\tmov.b64 b2, {l2, %4};\n\tmov.b64 b3, {l3, %4};\n\t"
        "mov.b64 a0, {%1, %2};\n\tmov.b64 a1, {m1, %2};\n\tmov.b64 a2, {m2, %2};\n\tmov.b64 a3, {m3, %2};\n\t"
        "setp.eq.b32 p, %6, 0;\n\tsetp.eq.b32 q, 0, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a0, b0, %5, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %5, q;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %5, q;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %5, q;\n\t}"
        ::"r"(d), "r"(a.lo), "r"(a.hi), "r"(b.lo), "r"(b.hi), "r"(idesc), "r"((uint32_t)first), "n"(BS), "n"(2 * BS), "n"(3 * BS), "n"(AS),
        "n"(2 * AS), "n"(3 * AS)
        : "memory");
}
// a value that is the same in all lanes, known as such to the compiler
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
// instruction descriptor: fp32 accumulator, fp16 operands, 128 rows
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool b_mn_major) {
    return (1u << 4) | (b_mn_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
// shared-memory operand: 128-byte swizzle, descriptor version 1; offsets in bytes
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)((lbo >> 4) & 0x3FFF) << 16) | ((uint64_t)((sbo >> 4) & 0x3FFF) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ Desc desc2(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return Desc{((addr >> 4) & 0x3FFF) | ((lbo >> 4) << 16), ((sbo >> 4) & 0x3FFF) | (1u << 14) | (2u << 29)};
}
// a panel (64 columns, rows 128 bytes apart) as an operand over its columns; a step of 16 columns is 2 units
constexpr int STEP_K = 2;
__device__ __forceinline__ Desc desc_k(uint32_t panel) { return desc2(panel, 16u, 1024u); }
// `rows`-row panels side by side as an operand over their rows, from a row on; a step of 16 rows is 128 units
constexpr int STEP_MN = 128;
__device__ __forceinline__ Desc desc_mn(uint32_t plane, int rows) { return desc2(plane, (uint32_t)(rows * 128), 1024u); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// packed pairs: two round-to-nearest operations per instruction
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// fp16 pairs (first value in the low half)
__device__ __forceinline__ uint32_t half_pair(float a, float b) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(a), "f"(b));
    return r;
}
// the same, what lies beyond fp16's range as its largest number (infinities too; a NaN stays one)
__device__ __forceinline__ uint32_t half_pair_finite(float a, float b) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(a), "f"(b));
    return r;
}
// hi / lo of two scaled entries of an operand: hi rounded to fp16, lo the difference, rounded.  |lo| <= 2^-11 |x|; together they miss
// x by at most 2^-23 of it, or 2^-25 where fp16 ends.
__device__ __forceinline__ void split_rounded(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = half_pair(a, b);
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    lo = half_pair(a - h.x, b - h.y);
}
// The same inside the loops (P, dS), where instructions count: hi is the value cut to 11 significant bits, a logical AND instead of a
// conversion back; fp16 holds it exactly down to 2^-14, and below that the pair is good to 2^-25 absolute, like lo.  |lo| < 2^-10 |x|, of whose at
// most 13 bits fp16 keeps 11: together they miss x by at most 2^-22 of it.
__device__ __forceinline__ void split_cut(float a, float b, uint32_t& hi, uint32_t& lo) {
    const float ah = __uint_as_float(__float_as_uint(a) & 0xFFFFE000u), bh = __uint_as_float(__float_as_uint(b) & 0xFFFFE000u);
    hi = half_pair_finite(ah, bh);
    float al, bl;
    unpack2(fma2(pack2(ah, bh), pack2(-1.f, -1.f), pack2(a, b)), al, bl);  // both differences, exact, in one instruction
    lo = half_pair(al, bl);
}

// 32 / 16 consecutive columns of this warp's 32 lanes; the wait is part of the instruction, so nothing reads too early
__device__ __forceinline__ void ld32(uint32_t addr, float (&f)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void ld16(uint32_t addr, float (&f)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void st8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
// N values as fp16 pairs over the N columns that they came from: of every 16 columns eight of hi pairs, then eight of lo pairs
template <int N>
__device__ __forceinline__ void st_split(uint32_t addr, const float (&x)[N]) {
#pragma unroll
    for (int g = 0; g < N / 16; ++g) {
        uint32_t r[16];
#pragma unroll
        for (int e = 0; e < 8; ++e) split_cut(x[16 * g + 2 * e], x[16 * g + 2 * e + 1], r[e], r[8 + e]);
        st16(addr + 16 * g, r);
    }
}
template <int N>
__device__ __forceinline__ void ldn(uint32_t addr, float (&f)[N]) {
    if constexpr (N == 16) ld16(addr, f);
    else ld32(addr, f);
}
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A warpgroup's share of the registers that the block was launched with.
template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// a contiguous copy from global memory that completes on an mbarrier (16-byte aligned, size a multiple of 16)
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
}

// 2^e that brings `largest` (finite, >= 0) into [2^14, 2^15), and its inverse.  0 and what is too small to be brought there
// without leaving fp32's range take the nearest factor that has an inverse.
__device__ __forceinline__ float block_scale(float largest, float* inverse) {
    const int ex = (int)((__float_as_uint(largest) >> 23) & 255u) - 127;
    const int e = largest > 0.f ? min(14 - ex, 120) : 0;
    *inverse = __uint_as_float((uint32_t)(127 - e) << 23);
    return __uint_as_float((uint32_t)(127 + e) << 23);
}
// the largest power of two (2^-121 .. 2^100) that is at most 1 / x, for x > 0
__device__ __forceinline__ float pow2_below_inverse(float x) {
    const int ex = (int)((__float_as_uint(x) >> 23) & 255u) - 127;
    const int e = max(-121, min(100, -(ex + 1)));
    return __uint_as_float((uint32_t)(127 + e) << 23);
}
// 1 / x of a power of two in 2^-126 .. 2^126
__device__ __forceinline__ float pow2_inverse(float x) { return __uint_as_float((254u << 23) - __float_as_uint(x)); }
// |x| for the search of the largest entry: infinities and NaN do not count
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.f;
}

}  // namespace tc
