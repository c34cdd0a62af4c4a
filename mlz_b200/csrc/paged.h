// paged.h -- the paged KV cache as its kernels see it (paged_*.cu): device view, length rules
// and the host-side argument checks.
#pragma once

#include "internal.h"
#ifdef __CUDACC__
#include "ptx.cuh"
#endif

namespace mlzc {
namespace paged {

// Division of 0 <= n < 2^31 by a divisor known at the call: q = n * mul / 2^shift (mul the
// reciprocal rounded up, exact for all such n), instead of a division's 20 instructions.
struct Div {
    uint32_t d, mul, shift;
    void set(uint32_t x) {
        d = x;
        shift = 0;
        while ((1ull << shift) < x) ++shift;
        mul = x == 1 ? 0 : (uint32_t)(((1ull << 32) * ((1ull << shift) - x)) / x + 1);
    }
#ifdef __CUDACC__
    __device__ __forceinline__ int quot(int n) const {
        const uint32_t hi = __umulhi((uint32_t)n, mul);
        return (int)((hi + (uint32_t)n) >> shift);
    }
    __device__ __forceinline__ int rem(int n) const { return n - quot(n) * (int)d; }
#endif
};

// Pools, block table and lengths of one call.  Strides in bytes.
struct View {
    char* k;
    char* v;
    size_t k_row, k_head, k_page, v_row, v_head, v_page;
    const int* table;
    size_t table_nb;
    const int* kv_len;
    const int* q_start;
    int page, max_pages, n_pages, n_head_kv, batch, n_tokens, cap;   // cap = max_pages * page
    Div by_page;
    unsigned int* err;
};

// A sequence's share of the call: `rows` new tokens from packed row `row0`, `kv` slots.  New
// token i has slot kv - rows + i (negative: none).
struct Seq {
    int row0, rows, kv;
};

#ifdef __CUDACC__
__device__ __forceinline__ int ld_int(const int* p) {
    int v;
    asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}

// Reads a sequence's lengths and cuts them to the tensors (see mlzc_paged_cache).
__device__ __forceinline__ Seq load_seq(const View& c, int b, bool with_rows = true) {
    Seq s;
    const int kv = ld_int(c.kv_len + b);
    s.kv = min(max(kv, 0), c.cap);
    bool bad = s.kv != kv;
    s.row0 = s.rows = 0;
    if (with_rows) {
        const int q0 = ld_int(c.q_start + b), q1 = ld_int(c.q_start + b + 1);
        s.row0 = min(max(q0, 0), c.n_tokens);
        const int end = min(max(q1, s.row0), c.n_tokens);
        s.rows = end - s.row0;
        bad |= s.row0 != q0 || end != q1;
    }
    if (bad) atomicOr(c.err, MLZC_DEVERR_BAD_INDEX);
    return s;
}

// Page of index `i` of sequence b, or -1 (and the error bit) where it is outside the pools.
__device__ __forceinline__ int load_page(const View& c, int b, int i) {
    const int p = ld_int(reinterpret_cast<const int*>(reinterpret_cast<const char*>(c.table) + (size_t)b * c.table_nb) + i);
    if ((unsigned)p < (unsigned)c.n_pages) return p;
    atomicOr(c.err, MLZC_DEVERR_BAD_INDEX);
    return -1;
}
// Bounded wait as ptx::mbar_wait, all inline: kernels that move registers between warpgroups
// cannot call functions.  The timer, slow to read, is looked at after some polls only.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort, unsigned int* err) {
    uint64_t t0 = 0;
    for (uint32_t i = 1;; ++i) {
        if (ptx::mbar_try_wait(bar, parity)) return true;
        if ((i & 31) == 0) {
            if (*abort) return false;
            const uint64_t t = ptx::global_ns();
            if (!t0) t0 = t;
            if (t - t0 > ptx::kWaitNs) {
                atomicOr(err, MLZC_DEVERR_WAIT_TIMEOUT);
                *abort = 1;
                return false;
            }
        }
    }
}
#endif

// Fills `out` from `cache` after checking it; `rows`: the call reads q_start and n_tokens.
int make_view(const mlzc_paged_cache* cache, bool rows, const DeviceCtx* c, View* out);
int check_cache(const mlzc_paged_cache* cache, bool rows);
// q / dst / lse of the attention and weights calls.
int check_attn(const mlzc_paged_cache* cache, const mlzc_paged_attn_desc* d, bool weights);
// Tensor map of a pool (K or V): dims head_dim, row, head, page; boxes of 64 values x box_rows
// rows in the 128-byte swizzle.
int encode_pool(CUtensorMap* map, const mlzc_paged_cache* cache, bool v, int box_rows);
// Tensor map of packed f16 rows [token][head][D]: dims D, head, token; boxes of 64 values x
// `heads` heads x `tokens` tokens in the 128-byte swizzle.
int encode_rows(CUtensorMap* map, const void* p, int64_t D, int64_t n_heads, int64_t n_tokens, size_t head_nb,
                size_t token_nb, int heads, int tokens);
// A packed [token][head][head_dim] tensor on 16-byte boundaries.
int check_rows(const char* what, const void* p, const size_t* nb, int64_t heads, int64_t tokens, size_t row_bytes,
               size_t elem);

}  // namespace paged
}  // namespace mlzc
