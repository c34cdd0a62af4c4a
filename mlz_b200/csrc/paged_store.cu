// paged_store.cu -- new tokens into the paged KV cache: rotary positions with one to four axes
// on q and k, k and v rounded to f16 into their pages (mlzc_paged_store_dev).
//
// Rotation of pair j by angle a = pos * freq_scale * base^(-2j / n_rot):
//   (x, y) -> (x cos a - y sin a, x sin a + y cos a).
// The angle is carried as a fraction of a turn in 64-bit fixed point.  With
// F_j = freq_j / 2 pi * 2^64 (computed once on the host in extended precision and passed as a
// kernel argument), pos * F_j modulo 2^64 IS the fraction: the integer product drops whole
// turns exactly, so a position of two million is nearly as exact as position two (f32 angles of far
// positions lose all their bits).  What lies beyond the nearest quarter turn goes to sincospi: within
// an eighth of a turn f32 holds it to 2^-28 of one (2^-26 over the whole turn).
//
// Bound by HBM (each row read once, written once; in f32 6 bytes a k or v value, 8 a q value)
// and, for a decode step, by launch latency.  One block handles one token and a range of its
// heads: the token's n_rot / 2 sines are computed once into shared memory and serve every head of
// the range.  8000 tokens of 32 + 2 x 8 heads of 128 dims, three axes: 52 us, 6.1 TB/s; 16 tokens: 3.7 us.
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "paged.h"
#include "ptx.cuh"

namespace mlzc {
namespace {

using paged::Seq;
using paged::View;

constexpr int kThreads = 256;

struct StoreArgs {
    View c;
    const char *q, *k, *v;
    char* q_dst;
    size_t q_head, q_tok, k_head, k_tok, v_head, v_tok, d_head, d_tok;
    const int* pos;
    size_t pos_nb;
    int n_head_q, D, half, axes, heads_per_block;
    uint8_t axis[128];      // position axis of pair j
    uint64_t turn[128];     // F_j
};

// Four consecutive values of a row.
template <typename T>
__device__ __forceinline__ float4 load4(const char* p) {
    if constexpr (sizeof(T) == 4) {
        return ptx::ld_act(reinterpret_cast<const float4*>(p));
    } else {
        const uint2 u = ptx::ld_act(reinterpret_cast<const uint2*>(p));
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
}
template <typename T>
__device__ __forceinline__ void store4(char* p, float4 x) {
    if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4*>(p) = x;
    else
        *reinterpret_cast<uint2*>(p) = make_uint2(ptx::pack_h2(x.x, x.y), ptx::pack_h2(x.z, x.w));
}

// The sequence that owns packed row t, or -1: q_start is ascending, so every thread of the
// block halves the range (the loads are the same for all and hit L1 after the first).
__device__ __forceinline__ int owner(const View& c, int t) {
    int lo = 0, hi = c.batch;   // the first b with q_start[b + 1] > t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (paged::ld_int(c.q_start + mid + 1) > t) hi = mid;
        else lo = mid + 1;
    }
    return lo < c.batch && paged::ld_int(c.q_start + lo) <= t ? lo : -1;
}

template <typename T, bool HALVES>
__global__ void __launch_bounds__(kThreads) store_kernel(const __grid_constant__ StoreArgs a) {
    __shared__ float2 cs[128];
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    const View& c = a.c;
    const int t = blockIdx.x;
    const int b = owner(c, t);
    if (b < 0) return;
    const Seq s = paged::load_seq(c, b);
    // an out-of-range kv_len still names the slots; only those inside the table are written
    const int64_t slot = (int64_t)paged::ld_int(c.kv_len + b) - s.rows + (t - s.row0);
    int page = -1;
    if (slot >= 0 && slot < c.cap) page = paged::load_page(c, b, (int)(slot / c.page));
    for (int j = threadIdx.x; j < a.half; j += kThreads) {
        const int64_t pos = paged::ld_int(reinterpret_cast<const int*>(reinterpret_cast<const char*>(a.pos) + a.axis[j] * a.pos_nb) + t);
        const uint64_t turns = (uint64_t)pos * a.turn[j];
        const uint32_t quarter = (uint32_t)((turns + (1ull << 61)) >> 62);
        float sn, cn;
        sincospif((float)(int64_t)(turns - ((uint64_t)quarter << 62)) * 0x1p-63f, &sn, &cn);
        const float2 at = quarter & 1 ? make_float2(-sn, cn) : make_float2(cn, sn);
        cs[j] = quarter & 2 ? make_float2(-at.x, -at.y) : at;
    }
    __syncthreads();
    const int heads = a.n_head_q + 2 * c.n_head_kv;
    const int h0 = blockIdx.y * a.heads_per_block, h1 = min(h0 + a.heads_per_block, heads);
    // a work item: 8 values of a head -- with HALVES the pairs' first and second dims lie half
    // a rotation apart, 4 + 4; otherwise (and past n_rot) 8 in a row
    const int per_head = a.D / 8, rot_items = a.half / 4;
    const int row = page < 0 ? 0 : (int)(slot % c.page);
    for (int i = threadIdx.x; i < (h1 - h0) * per_head; i += kThreads) {
        const int h = h0 + i / per_head, e = i % per_head;
        const bool is_q = h < a.n_head_q, is_v = h >= a.n_head_q + c.n_head_kv;
        const int hk = h - a.n_head_q - (is_v ? c.n_head_kv : 0);
        if (!is_q && page < 0) continue;
        const char* src = is_q ? a.q + (size_t)t * a.q_tok + (size_t)h * a.q_head
                               : (is_v ? a.v + (size_t)t * a.v_tok + (size_t)hk * a.v_head
                                       : a.k + (size_t)t * a.k_tok + (size_t)hk * a.k_head);
        const bool turned = !is_v && e < rot_items;
        const int d0 = HALVES && turned ? 4 * e : 8 * e;
        const int d1 = HALVES && turned ? d0 + a.half : d0 + 4;
        float4 x = load4<T>(src + (size_t)d0 * sizeof(T)), y = load4<T>(src + (size_t)d1 * sizeof(T));
        if (turned) {
            const float2* w = cs + 4 * e;
            if (HALVES) {
                const float4 p = x, r = y;
                x = make_float4(p.x * w[0].x - r.x * w[0].y, p.y * w[1].x - r.y * w[1].y, p.z * w[2].x - r.z * w[2].y,
                                p.w * w[3].x - r.w * w[3].y);
                y = make_float4(p.x * w[0].y + r.x * w[0].x, p.y * w[1].y + r.y * w[1].x, p.z * w[2].y + r.z * w[2].x,
                                p.w * w[3].y + r.w * w[3].x);
            } else {
                x = make_float4(x.x * w[0].x - x.y * w[0].y, x.x * w[0].y + x.y * w[0].x, x.z * w[1].x - x.w * w[1].y,
                                x.z * w[1].y + x.w * w[1].x);
                y = make_float4(y.x * w[2].x - y.y * w[2].y, y.x * w[2].y + y.y * w[2].x, y.z * w[3].x - y.w * w[3].y,
                                y.z * w[3].y + y.w * w[3].x);
            }
        }
        if (is_q) {
            char* dst = a.q_dst + (size_t)t * a.d_tok + (size_t)h * a.d_head;
            store4<T>(dst + (size_t)d0 * sizeof(T), x);
            store4<T>(dst + (size_t)d1 * sizeof(T), y);
        } else {
            char* dst = is_v ? c.v + (size_t)page * c.v_page + (size_t)hk * c.v_head + (size_t)row * c.v_row
                             : c.k + (size_t)page * c.k_page + (size_t)hk * c.k_head + (size_t)row * c.k_row;
            store4<__half>(dst + (size_t)d0 * 2, x);
            store4<__half>(dst + (size_t)d1 * 2, y);
        }
    }
}

}  // namespace
}  // namespace mlzc

using namespace mlzc;

extern "C" int mlzc_paged_store_dev(const mlzc_paged_cache* cache, const mlzc_paged_store_desc* d, void* stream) {
    int st = paged::check_cache(cache, true);
    if (st != MLZC_OK) return st;
    if (!d) return fail(MLZC_ERR_INVALID, "paged store: null descriptor");
    if (d->type != MLZC_TYPE_F32 && d->type != MLZC_TYPE_F16)
        return fail(MLZC_ERR_UNSUPPORTED, "paged store: type %d (F32 = 0, F16 = 1)", d->type);
    if (d->n_head_q < 0 || d->n_head_q > 65535) return fail(MLZC_ERR_INVALID, "paged store: n_head_q %lld", (long long)d->n_head_q);
    if (d->n_rot < 0 || d->n_rot % 8 || d->n_rot > cache->head_dim)
        return fail(MLZC_ERR_INVALID, "paged store: n_rot %d (a multiple of 8 up to head_dim)", d->n_rot);
    if (d->pairs != MLZC_ROPE_ADJACENT && d->pairs != MLZC_ROPE_HALVES)
        return fail(MLZC_ERR_INVALID, "paged store: pairs %d", d->pairs);
    StoreArgs a{};
    const int64_t T = cache->n_tokens;
    if (d->n_rot) {
        if (d->n_axes < 1 || d->n_axes > 4) return fail(MLZC_ERR_INVALID, "paged store: n_axes %d (1 to 4)", d->n_axes);
        if (!(d->freq_base > 0.0f) || !std::isfinite(d->freq_base) || !std::isfinite(d->freq_scale))
            return fail(MLZC_ERR_INVALID, "paged store: freq_base must be positive, freq_scale finite");
        int64_t sum = 0;
        for (int i = 0; i < d->n_axes; ++i) {
            if (d->sections[i] < 0) return fail(MLZC_ERR_INVALID, "paged store: negative section");
            sum += d->sections[i];
        }
        if (sum != d->n_rot / 2)
            return fail(MLZC_ERR_INVALID, "paged store: sections add up to %lld, n_rot / 2 is %d", (long long)sum, d->n_rot / 2);
        if (T > 0 && (!d->positions || (uintptr_t)d->positions % 4 || d->positions_nb % 4 ||
                      (d->n_axes > 1 && d->positions_nb < (size_t)T * 4)))
            return fail(MLZC_ERR_INVALID, "paged store: positions null, misaligned or overlapping");
        const long double two_pi = 6.283185307179586476925286766559005768L;
        // powers of the step between pairs from two short tables (a dozen roundings of 2^-64)
        const long double step = powl((long double)d->freq_base, -2.0L / d->n_rot);
        long double fine[8] = {1.0L}, coarse = (long double)d->freq_scale / two_pi;
        for (int i = 1; i < 8; ++i) fine[i] = fine[i - 1] * step;
        int j = 0;
        for (int ax = 0; ax < d->n_axes; ++ax)
            for (int i = 0; i < d->sections[ax]; ++i, ++j) {
                if (j > 0 && j % 8 == 0) coarse *= fine[7] * step;
                a.axis[j] = (uint8_t)ax;
                const long double turns = coarse * fine[j % 8];
                a.turn[j] = (uint64_t)ldexpl(turns - floorl(turns), 64);   // whole turns a position step drop out
            }
    }
    if (T == 0) return MLZC_OK;
    const size_t elem = d->type == MLZC_TYPE_F32 ? 4 : 2, rb = (size_t)cache->head_dim * elem;
    st = paged::check_rows("paged store: k", d->k, d->k_nb, cache->n_head_kv, T, rb, elem);
    if (st == MLZC_OK) st = paged::check_rows("paged store: v", d->v, d->v_nb, cache->n_head_kv, T, rb, elem);
    if (st == MLZC_OK && d->n_head_q) st = paged::check_rows("paged store: q", d->q, d->q_nb, d->n_head_q, T, rb, elem);
    if (st == MLZC_OK && d->n_head_q) st = paged::check_rows("paged store: q_dst", d->q_dst, d->q_dst_nb, d->n_head_q, T, rb, elem);
    if (st != MLZC_OK) return st;
    if (d->n_head_q && d->q == d->q_dst && ((d->n_head_q > 1 && d->q_nb[1] != d->q_dst_nb[1]) || (T > 1 && d->q_nb[2] != d->q_dst_nb[2])))
        return fail(MLZC_ERR_INVALID, "paged store: q_dst in place with other strides");
    DeviceCtx* c = current_ctx();
    if (!c) return MLZC_ERR_CUDA;
    st = paged::make_view(cache, true, c, &a.c);
    if (st != MLZC_OK) return st;
    a.q = static_cast<const char*>(d->q);
    a.k = static_cast<const char*>(d->k);
    a.v = static_cast<const char*>(d->v);
    a.q_dst = static_cast<char*>(d->q_dst);
    a.q_head = d->q_nb[1]; a.q_tok = d->q_nb[2];
    a.k_head = d->k_nb[1]; a.k_tok = d->k_nb[2];
    a.v_head = d->v_nb[1]; a.v_tok = d->v_nb[2];
    a.d_head = d->q_dst_nb[1]; a.d_tok = d->q_dst_nb[2];
    a.pos = d->positions;
    a.pos_nb = d->positions_nb;
    a.n_head_q = (int)d->n_head_q;
    a.D = (int)cache->head_dim;
    a.half = d->n_rot / 2;
    a.axes = d->n_axes;
    const int heads = a.n_head_q + 2 * a.c.n_head_kv;
    // few tokens: a token's heads are spread over several blocks, about two blocks an SM
    const int most = (heads * (a.D / 8) + kThreads - 1) / kThreads;
    const int split = (int)std::max<int64_t>(1, std::min<int64_t>(most, 2 * c->sm_count / std::max<int64_t>(T, 1)));
    a.heads_per_block = (heads + split - 1) / split;
    const dim3 grid((unsigned)T, (unsigned)((heads + a.heads_per_block - 1) / a.heads_per_block));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool halves = d->pairs == MLZC_ROPE_HALVES;
    if (elem == 4)
        MLZC_CUDA_TRY(launch_pdl(halves ? store_kernel<float, true> : store_kernel<float, false>, grid, dim3(kThreads), 0, s, a));
    else
        MLZC_CUDA_TRY(launch_pdl(halves ? store_kernel<__half, true> : store_kernel<__half, false>, grid, dim3(kThreads), 0, s, a));
    MLZC_CUDA_TRY(cudaGetLastError());
    count_launch();
    return MLZC_OK;
}
