// paged_attn.cu -- attention of new tokens over a paged KV cache (mlzc_paged_attn_dev).
//
// One warp a query row: online softmax over the slots the row sees, the head's dims spread over
// the lanes.
#include <cuda_fp16.h>

#include <cmath>

#include "paged.h"
#include "ptx.cuh"

namespace mlzc {
namespace {

using paged::Seq;
using paged::View;

struct AttnArgs {
    View c;
    const char* q;
    char* dst;
    size_t q_head, q_tok, d_head, d_tok, lse_head, lse_tok;
    char* lse;
    int n_head_q, f32;
    float scale, softcap;
};

constexpr int kWarps = 8;

template <int D>
__global__ void __launch_bounds__(kWarps * 32) attn_kernel(const __grid_constant__ AttnArgs a) {
    constexpr int E = D / 32;
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    const View& c = a.c;
    const int lane = threadIdx.x & 31;
    const int64_t r = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int t = (int)(r / a.n_head_q), h = (int)(r % a.n_head_q);
    if (t >= c.n_tokens) return;
    int lo = 0, hi = c.batch;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (paged::ld_int(c.q_start + mid + 1) > t) hi = mid;
        else lo = mid + 1;
    }
    if (lo >= c.batch || paged::ld_int(c.q_start + lo) > t) return;
    const Seq s = paged::load_seq(c, lo);
    const int hk = h / (a.n_head_q / c.n_head_kv);
    float q[E], o[E];
    const char* qr = a.q + (size_t)t * a.q_tok + (size_t)h * a.q_head;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int d = lane * E + e;
        q[e] = a.f32 ? reinterpret_cast<const float*>(qr)[d] : __half2float(reinterpret_cast<const __half*>(qr)[d]);
        o[e] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    const int seen = s.kv - s.rows + (t - s.row0) + 1;
    for (int j = 0; j < seen; ++j) {
        const int page = paged::load_page(c, lo, j / c.page);
        const __half* kr = reinterpret_cast<const __half*>(c.k + (size_t)page * c.k_page + (size_t)hk * c.k_head + (size_t)(j % c.page) * c.k_row);
        const __half* vr = reinterpret_cast<const __half*>(c.v + (size_t)page * c.v_page + (size_t)hk * c.v_head + (size_t)(j % c.page) * c.v_row);
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) x += page < 0 ? 0.0f : q[e] * __half2float(kr[lane * E + e]);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(~0u, x, d);
        x *= a.scale;
        if (a.softcap > 0.0f) x = a.softcap * tanhf(x / a.softcap);
        const float mn = fmaxf(m, x), al = expf(m - mn), p = expf(x - mn);
        l = l * al + p;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * al + (page < 0 ? 0.0f : p * __half2float(vr[lane * E + e]));
        m = mn;
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    char* dr = a.dst + (size_t)t * a.d_tok + (size_t)h * a.d_head;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int d = lane * E + e;
        if (a.f32) reinterpret_cast<float*>(dr)[d] = o[e] * inv;
        else reinterpret_cast<__half*>(dr)[d] = __float2half_rn(o[e] * inv);
    }
    if (a.lse && lane == 0)
        *reinterpret_cast<float*>(a.lse + (size_t)t * a.lse_tok + (size_t)h * a.lse_head) = l > 0.0f ? m + logf(l) : -INFINITY;
}

}  // namespace
}  // namespace mlzc

using namespace mlzc;

extern "C" int mlzc_paged_attn_workspace_bytes(const mlzc_paged_cache* cache, const mlzc_paged_attn_desc* d,
                                               size_t* out_bytes) {
    if (!out_bytes) return fail(MLZC_ERR_INVALID, "paged attention: null out_bytes");
    *out_bytes = 0;
    return paged::check_attn(cache, d, false);
}

extern "C" int mlzc_paged_attn_dev(const mlzc_paged_cache* cache, const mlzc_paged_attn_desc* d, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    int st = paged::check_attn(cache, d, false);
    if (st != MLZC_OK || cache->n_tokens == 0) return st;
    DeviceCtx* c = current_ctx();
    if (!c) return MLZC_ERR_CUDA;
    AttnArgs a{};
    st = paged::make_view(cache, true, c, &a.c);
    if (st != MLZC_OK) return st;
    a.q = static_cast<const char*>(d->q);
    a.dst = static_cast<char*>(d->dst);
    a.q_head = d->q_nb[1]; a.q_tok = d->q_nb[2];
    a.d_head = d->dst_nb[1]; a.d_tok = d->dst_nb[2];
    a.lse = reinterpret_cast<char*>(d->lse);
    a.lse_head = d->lse_nb[0]; a.lse_tok = d->lse_nb[1];
    a.n_head_q = (int)d->n_head_q;
    a.f32 = d->type == MLZC_TYPE_F32;
    a.scale = d->scale;
    a.softcap = (d->mode & MLZC_FA_MODE_SOFTCAP) ? d->logit_softcap : 0.0f;
    const int64_t rows = cache->n_tokens * d->n_head_q;
    const int D = (int)cache->head_dim;
    MLZC_CUDA_TRY(launch_pdl(D == 64 ? attn_kernel<64> : (D == 128 ? attn_kernel<128> : attn_kernel<256>),
                             dim3((unsigned)((rows + kWarps - 1) / kWarps)), dim3(kWarps * 32), 0,
                             static_cast<cudaStream_t>(stream), a));
    MLZC_CUDA_TRY(cudaGetLastError());
    count_launch();
    return MLZC_OK;
}
