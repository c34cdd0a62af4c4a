// tcgen05.cuh -- inline-PTX helpers of the 5th-generation tensor cores (tcgen05, TMEM) shared
// by the kernels that use them.
#pragma once

#include <cuda.h>

#include <cstdint>

namespace mlzc {
namespace tc05 {

// Orders this thread's generic-proxy shared-memory writes before later async-proxy reads.
__device__ __forceinline__ void fence_proxy_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tma_prefetch_desc(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// UMMA shared-memory descriptor of a K-major tile written by TMA with 128-byte swizzle:
// rows of 128 bytes, 8-row (1024-byte) swizzle atoms stacked along M/N.
__device__ __forceinline__ uint64_t umma_desc_sw128(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);   // start address        [0, 14)
    d |= (uint64_t)1 << 16;                     // leading byte offset  [16, 30) (unused: swizzled K-major)
    d |= (uint64_t)(1024 >> 4) << 32;           // stride byte offset   [32, 46): 8 rows x 128 B
    d |= (uint64_t)1 << 46;                     // descriptor version   [46, 48) = 1 on sm_100
    d |= (uint64_t)2 << 61;                     // layout: SWIZZLE_128B [61, 64)
    return d;
}

// Instruction descriptor, kind::f16: A = B = f16, D = f32, both K-major, M x N.
__host__ __device__ constexpr uint32_t umma_idesc_f16(int M, int N) {
    return (1u << 4)                             // D format f32        [4, 6)
           | (0u << 7) | (0u << 10)              // A, B format f16     [7, 10), [10, 13)
           | (0u << 15) | (0u << 16)             // A, B K-major        15, 16
           | ((uint32_t)(N >> 3) << 17)          // N / 8               [17, 23)
           | ((uint32_t)(M >> 4) << 24);         // M / 16              [24, 29)
}

__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        " .reg .pred p;\n"
        " setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}

__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Loads / stores 16 consecutive 32-bit columns of this thread's lane.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
        "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
                 : "memory");
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory descriptors in halves, for issue loops: K-major tiles as in umma_desc_sw128, and
// tiles whose M/N axis is contiguous (64-element rows of 128 bytes, one row a k value:
// `block_bytes` from one 64-element block of the M/N axis to the next, 1024 bytes from 8 k values
// to the next 8).  The upper words are alike (8 rows of 128
// bytes a swizzle atom, version, layout), and stepping through a tile is a 32-bit addition to
// the lower one (addresses count 16 bytes and stay below 2^14).
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr16, uint32_t block_bytes = 16) { return saddr16 | ((block_bytes >> 4) << 16); }
__device__ __forceinline__ void umma_f16_lo(uint32_t d_tmem, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n"
        " .reg .pred p;\n"
        " .reg .b64 x, y;\n"
        " mov.b64 x, {%1, %4};\n"
        " mov.b64 y, {%2, %4};\n"
        " setp.ne.b32 p, %5, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "r"(a), "r"(b), "r"(idesc), "r"(kDescHi), "r"((uint32_t)accumulate));
}
// A (f16, two k values per 32-bit column, one row a lane) in TMEM.
__device__ __forceinline__ void umma_f16_ta_lo(uint32_t d_tmem, uint32_t a_tmem, uint32_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n"
        " .reg .pred p;\n"
        " .reg .b64 y;\n"
        " mov.b64 y, {%2, %4};\n"
        " setp.ne.b32 p, %5, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b), "r"(idesc), "r"(kDescHi), "r"((uint32_t)accumulate));
}
constexpr uint32_t kIdescBMnMajor = 1u << 16;   // instruction descriptor: B with its N axis contiguous

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}

// One lane of a converged warp, in a form that the compiler knows to be a single lane.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n"
        " .reg .pred p;\n"
        " elect.sync _|p, 0xffffffff;\n"
        " selp.b32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(p));
    return p != 0;
}
// The value of lane 0, known to the compiler to be the same in all lanes: what instructions
// that take uniform registers (tcgen05.mma's descriptors) are computed from.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void tmem_alloc(uint32_t holder, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(holder), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t base, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}

// Pairs of f32 in one 64-bit register: two operations an instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
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
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 2^x of two values on the FMA pipe, for kernels bound by the exponential unit: x = n + f with
// |f| <= 1/2 (adding 1.5 * 2^23 rounds to an integer, left in the low bits), 2^f by its minimax
// polynomial of degree 5 with constant term 1 (relative error 1.6e-7 with f32 rounding; f = 0 is
// exact), n added to the exponent.  At and below -127 the result is exactly 0.
__device__ __forceinline__ void exp2_poly(uint64_t x, float& r0, float& r1) {
    float a, b, t0, t1;
    unpair(x, a, b);
    x = pair(fmaxf(a, -127.0f), fmaxf(b, -127.0f));
    const float kRound = 12582912.0f;
    const uint64_t t = add2(x, pair(kRound, kRound));
    const uint64_t n = add2(t, pair(-kRound, -kRound));
    const uint64_t f = fma2(n, pair(-1.0f, -1.0f), x);
    uint64_t p = pair(0.0013274633092805743f, 0.0013274633092805743f);
    p = fma2(p, f, pair(0.009671961888670921f, 0.009671961888670921f));
    p = fma2(p, f, pair(0.055506784468889236f, 0.055506784468889236f));
    p = fma2(p, f, pair(0.24022234976291656f, 0.24022234976291656f));
    p = fma2(p, f, pair(0.6931470632553101f, 0.6931470632553101f));
    p = fma2(p, f, pair(1.0f, 1.0f));
    unpair(t, t0, t1);
    unpair(p, a, b);
    r0 = __uint_as_float(__float_as_uint(a) + (__float_as_uint(t0) << 23));
    r1 = __uint_as_float(__float_as_uint(b) + (__float_as_uint(t1) << 23));
}

// cap * tanh(t) for |t| <= 1: the odd minimax polynomial of tanh there (degree 13, Remez; 1.7e-7
// relative with f32 rounding).
__device__ __forceinline__ float cap_near(float t, float cap) {
    const float q = t * t;
    float p = fmaf(0.0010582648683339357f, q, -0.006259339861571789f);
    p = fmaf(p, q, 0.020359760150313377f);
    p = fmaf(p, q, -0.053498707711696625f);
    p = fmaf(p, q, 0.13326409459114075f);
    p = fmaf(p, q, -0.33332985639572144f);
    p = fmaf(p, q, 1.0f);
    return t * cap * p;
}
// cap * tanh(t) for |t| > 1: cap (1 - e) / (1 + e), e = exp(-2 |t|) < 0.14, so that 1 - e loses nothing.
__device__ __forceinline__ float cap_far(float t, float cap) {
    const float e = ex2(fabsf(t) * (-2.0f * 1.4426950408889634f));
    return copysignf(__fdividef(1.0f - e, 1.0f + e) * cap, t);
}

// N scores to cap * tanh(s * in), in = scale / cap, each by the form for its own size: a score's
// bits depend on nothing beside it.  The far form's two more uses of the exponential unit a score
// would be the bound, so a warp passes it over where none of its lanes has a score for it (lanes
// and columns that do not count may decide that: it changes the time alone).
template <int N>
__device__ __forceinline__ void cap_scores(float (&x)[N], float in, float cap) {
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] *= in;
#pragma unroll
    for (int j = 0; j < N; j += 2) top = max3(top, fabsf(x[j]), fabsf(x[j + 1]));
    if (__all_sync(~0u, top <= 1.0f)) {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = cap_near(x[j], cap);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = fabsf(x[j]) <= 1.0f ? cap_near(x[j], cap) : cap_far(x[j], cap);
    }
}

}  // namespace tc05
}  // namespace mlzc
