// paged_weights.cu -- the attention weight that each slot of a paged KV cache received from the
// new tokens (mlzc_paged_weights_dev).
//
// One warp a slot: the sum of exp(score - lse) over the query rows that see it.
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "paged.h"
#include "ptx.cuh"

namespace mlzc {
namespace {

using paged::Seq;
using paged::View;

struct WeightArgs {
    View c;
    const char* q;
    size_t q_head, q_tok, lse_head, lse_tok;
    const char* lse;
    const char* acc;
    char* out;
    size_t a_head, a_seq, o_head, o_seq;
    int n_head_q, f32;
    float scale, softcap;
};

constexpr int kWarps = 8;

template <int D>
__global__ void __launch_bounds__(kWarps * 32) weights_kernel(const __grid_constant__ WeightArgs a) {
    constexpr int E = D / 32;
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    const View& c = a.c;
    const int lane = threadIdx.x & 31, hk = blockIdx.y, b = blockIdx.z;
    const Seq s = paged::load_seq(c, b);
    const int G = a.n_head_q / c.n_head_kv;
    for (int j = blockIdx.x * kWarps + (threadIdx.x >> 5); j < s.kv; j += gridDim.x * kWarps) {
        const int page = paged::load_page(c, b, j / c.page);
        float k[E];
        const __half* kr = reinterpret_cast<const __half*>(c.k + (size_t)page * c.k_page + (size_t)hk * c.k_head + (size_t)(j % c.page) * c.k_row);
#pragma unroll
        for (int e = 0; e < E; ++e) k[e] = page < 0 ? 0.0f : __half2float(kr[lane * E + e]);
        float sum = 0.0f;
        for (int i = std::max(0, j - (s.kv - s.rows)); i < s.rows; ++i)
            for (int g = 0; g < G; ++g) {
                const int t = s.row0 + i, h = hk * G + g;
                const char* qr = a.q + (size_t)t * a.q_tok + (size_t)h * a.q_head;
                float x = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int d = lane * E + e;
                    x += k[e] * (a.f32 ? reinterpret_cast<const float*>(qr)[d] : __half2float(reinterpret_cast<const __half*>(qr)[d]));
                }
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(~0u, x, d);
                x *= a.scale;
                if (a.softcap > 0.0f) x = a.softcap * tanhf(x / a.softcap);
                const float lse = *reinterpret_cast<const float*>(a.lse + (size_t)t * a.lse_tok + (size_t)h * a.lse_head);
                if (lse != -INFINITY) sum += expf(x - lse);
            }
        if (lane == 0) {
            const float* in = reinterpret_cast<const float*>(a.acc + (size_t)b * a.a_seq + (size_t)hk * a.a_head);
            float* out = reinterpret_cast<float*>(a.out + (size_t)b * a.o_seq + (size_t)hk * a.o_head);
            out[j] = (a.acc ? in[j] : 0.0f) + sum;
        }
    }
}

int check_table(const char* what, const void* p, const size_t* nb, int64_t heads, int64_t batch, size_t row) {
    if (!p || !nb || (uintptr_t)p % 4) return fail(MLZC_ERR_INVALID, "paged weights: %s null or misaligned", what);
    if (nb[0] != 4 || nb[1] % 4 || nb[2] % 4 || (heads > 1 && nb[1] < row) || (batch > 1 && nb[2] < row))
        return fail(MLZC_ERR_INVALID, "paged weights: %s strides (rows of floats that do not overlap)", what);
    return MLZC_OK;
}

}  // namespace
}  // namespace mlzc

using namespace mlzc;

extern "C" int mlzc_paged_weights_workspace_bytes(const mlzc_paged_cache* cache, const mlzc_paged_attn_desc* d,
                                                  size_t* out_bytes) {
    if (!out_bytes) return fail(MLZC_ERR_INVALID, "paged weights: null out_bytes");
    *out_bytes = 0;
    return paged::check_attn(cache, d, true);
}

extern "C" int mlzc_paged_weights_dev(const mlzc_paged_cache* cache, const mlzc_paged_attn_desc* d, const float* acc,
                                      const size_t acc_nb[3], float* out, const size_t out_nb[3], void* workspace,
                                      size_t workspace_bytes, void* stream) {
    int st = paged::check_attn(cache, d, true);
    if (st != MLZC_OK) return st;
    const size_t row = (size_t)cache->max_pages * cache->page_size * 4;
    if (acc) st = check_table("acc", acc, acc_nb, cache->n_head_kv, cache->batch_size, row);
    if (st == MLZC_OK) st = check_table("out", out, out_nb, cache->n_head_kv, cache->batch_size, row);
    if (st != MLZC_OK) return st;
    if (acc == out && (acc_nb[1] != out_nb[1] || acc_nb[2] != out_nb[2]))
        return fail(MLZC_ERR_INVALID, "paged weights: acc and out in place with other strides");
    if (cache->batch_size > 65535) return fail(MLZC_ERR_UNSUPPORTED, "paged weights: batch_size above 65535");
    DeviceCtx* c = current_ctx();
    if (!c) return MLZC_ERR_CUDA;
    WeightArgs a{};
    st = paged::make_view(cache, true, c, &a.c);
    if (st != MLZC_OK) return st;
    a.q = static_cast<const char*>(d->q);
    a.q_head = d->q_nb[1]; a.q_tok = d->q_nb[2];
    a.lse = reinterpret_cast<const char*>(d->lse);
    a.lse_head = d->lse_nb[0]; a.lse_tok = d->lse_nb[1];
    a.acc = reinterpret_cast<const char*>(acc);
    a.out = reinterpret_cast<char*>(out);
    if (acc) { a.a_head = acc_nb[1]; a.a_seq = acc_nb[2]; }
    a.o_head = out_nb[1]; a.o_seq = out_nb[2];
    a.n_head_q = (int)d->n_head_q;
    a.f32 = d->type == MLZC_TYPE_F32;
    a.scale = d->scale;
    a.softcap = (d->mode & MLZC_FA_MODE_SOFTCAP) ? d->logit_softcap : 0.0f;
    const int D = (int)cache->head_dim;
    const unsigned gx = (unsigned)std::min(1024, (a.c.cap + kWarps - 1) / kWarps);
    MLZC_CUDA_TRY(launch_pdl(D == 64 ? weights_kernel<64> : (D == 128 ? weights_kernel<128> : weights_kernel<256>),
                             dim3(gx, a.c.n_head_kv, a.c.batch), dim3(kWarps * 32), 0, static_cast<cudaStream_t>(stream), a));
    MLZC_CUDA_TRY(cudaGetLastError());
    count_launch();
    return MLZC_OK;
}
