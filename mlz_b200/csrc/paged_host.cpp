// paged_host.cpp -- argument checks of the paged-cache entry points (mlzc_paged_*).
#include <cmath>

#include "paged.h"

namespace mlzc {
namespace paged {

namespace {
constexpr int64_t kMaxInt = (1ll << 31) - 1;
constexpr size_t kMaxStride = (size_t)1 << 40;   // tensor-map limit
}  // namespace

int check_rows(const char* what, const void* p, const size_t* nb, int64_t heads, int64_t tokens, size_t row_bytes,
               size_t elem) {
    if (!p) return fail(MLZC_ERR_INVALID, "%s: null pointer", what);
    if ((uintptr_t)p % 16) return fail(MLZC_ERR_INVALID, "%s: rows must start on 16-byte boundaries", what);
    if (nb[0] != elem) return fail(MLZC_ERR_INVALID, "%s: rows must be contiguous (element stride %zu)", what, nb[0]);
    if (heads > 1 && (nb[1] % 16 || nb[1] < row_bytes || nb[1] >= kMaxStride))
        return fail(MLZC_ERR_INVALID, "%s: head stride %zu", what, nb[1]);
    if (tokens > 1 && (nb[2] % 16 || nb[2] < row_bytes || nb[2] >= kMaxStride))
        return fail(MLZC_ERR_INVALID, "%s: token stride %zu", what, nb[2]);
    return MLZC_OK;
}

int check_cache(const mlzc_paged_cache* c, bool rows) {
    if (!c) return fail(MLZC_ERR_INVALID, "paged cache: null descriptor");
    if (c->kv_type != MLZC_TYPE_F16) return fail(MLZC_ERR_UNSUPPORTED, "paged cache: type %d (F16 = 1 supported)", c->kv_type);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(MLZC_ERR_UNSUPPORTED, "paged cache: head_dim %lld (64, 128, 256 supported)", (long long)c->head_dim);
    if (c->page_size < 8 || c->page_size % 8)
        return fail(MLZC_ERR_UNSUPPORTED, "paged cache: page_size %d (multiples of 8 supported)", c->page_size);
    if (c->n_pages < 1 || c->n_head_kv < 1 || c->batch_size < 1 || c->max_pages < 1)
        return fail(MLZC_ERR_INVALID, "paged cache: empty or negative dimension");
    if (c->n_pages > kMaxInt || c->n_head_kv > 65535 || c->batch_size > (1 << 24) || c->max_pages > kMaxInt ||
        c->max_pages * c->page_size > kMaxInt - 4096)
        return fail(MLZC_ERR_INVALID, "paged cache: dimension too large");
    if (!c->k || !c->v || !c->block_table || !c->kv_len) return fail(MLZC_ERR_INVALID, "paged cache: null pointer");
    const size_t row = (size_t)c->head_dim * 2;
    for (int i = 0; i < 2; ++i) {
        const size_t* nb = i ? c->v_nb : c->k_nb;
        const char* what = i ? "v" : "k";
        if ((uintptr_t)(i ? c->v : c->k) % 16) return fail(MLZC_ERR_INVALID, "paged cache: %s not 16-byte aligned", what);
        if (nb[0] != 2) return fail(MLZC_ERR_INVALID, "paged cache: %s rows must be contiguous f16", what);
        for (int d = 1; d < 4; ++d) {
            const bool stepped = d == 1 || (d == 2 ? c->n_head_kv : c->n_pages) > 1;
            if (stepped && (nb[d] % 16 || nb[d] < row || nb[d] >= kMaxStride))
                return fail(MLZC_ERR_INVALID, "paged cache: %s stride %d is %zu bytes", what, d, nb[d]);
        }
    }
    if ((uintptr_t)c->block_table % 4 || (uintptr_t)c->kv_len % 4 || c->block_table_nb % 4 ||
        (c->batch_size > 1 && c->block_table_nb < (size_t)c->max_pages * 4))
        return fail(MLZC_ERR_INVALID, "paged cache: block table or lengths misaligned, or table rows overlap");
    if (rows) {
        if (!c->q_start || (uintptr_t)c->q_start % 4) return fail(MLZC_ERR_INVALID, "paged cache: q_start null or misaligned");
        if (c->n_tokens < 0 || c->n_tokens > kMaxInt) return fail(MLZC_ERR_INVALID, "paged cache: n_tokens %lld", (long long)c->n_tokens);
    }
    return MLZC_OK;
}

int make_view(const mlzc_paged_cache* cache, bool rows, const DeviceCtx* ctx, View* out) {
    const int st = check_cache(cache, rows);
    if (st != MLZC_OK) return st;
    View& v = *out;
    v.k = static_cast<char*>(cache->k);
    v.v = static_cast<char*>(cache->v);
    v.k_row = cache->k_nb[1]; v.k_head = cache->k_nb[2]; v.k_page = cache->k_nb[3];
    v.v_row = cache->v_nb[1]; v.v_head = cache->v_nb[2]; v.v_page = cache->v_nb[3];
    v.table = cache->block_table;
    v.table_nb = cache->block_table_nb;
    v.kv_len = cache->kv_len;
    v.q_start = rows ? cache->q_start : nullptr;
    v.page = cache->page_size;
    v.max_pages = (int)cache->max_pages;
    v.n_pages = (int)cache->n_pages;
    v.n_head_kv = (int)cache->n_head_kv;
    v.batch = (int)cache->batch_size;
    v.n_tokens = rows ? (int)cache->n_tokens : 0;
    v.cap = (int)(cache->max_pages * cache->page_size);
    v.by_page.set((uint32_t)v.page);
    v.err = ctx ? ctx->err : nullptr;
    return MLZC_OK;
}

namespace {
int encode(CUtensorMap* map, const void* p, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    auto enc = tensor_map_encoder();
    if (!enc) return fail(MLZC_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(p), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(MLZC_ERR_UNSUPPORTED, "paged cache: strides not expressible as a tensor map (%d)", (int)r);
    return MLZC_OK;
}
}  // namespace

int encode_pool(CUtensorMap* map, const mlzc_paged_cache* c, bool v, int box_rows) {
    const size_t* nb = v ? c->v_nb : c->k_nb;
    const cuuint64_t dims[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->page_size, (cuuint64_t)c->n_head_kv, (cuuint64_t)c->n_pages};
    // the stride of a dimension of extent 1 is never stepped: any legal one
    const cuuint64_t strides[3] = {nb[1], c->n_head_kv > 1 ? nb[2] : nb[1], c->n_pages > 1 ? nb[3] : nb[1]};
    const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1};
    return encode(map, v ? c->v : c->k, 4, dims, strides, box);
}

int encode_rows(CUtensorMap* map, const void* p, int64_t D, int64_t n_heads, int64_t n_tokens, size_t head_nb,
                size_t token_nb, int heads, int tokens) {
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)n_heads, (cuuint64_t)n_tokens};
    const cuuint64_t row = (cuuint64_t)D * 2;
    const cuuint64_t strides[2] = {n_heads > 1 ? (cuuint64_t)head_nb : row, n_tokens > 1 ? (cuuint64_t)token_nb : row};
    const cuuint32_t box[3] = {64, (cuuint32_t)heads, (cuuint32_t)tokens};
    return encode(map, p, 3, dims, strides, box);
}

int check_attn(const mlzc_paged_cache* cache, const mlzc_paged_attn_desc* d, bool weights) {
    const int st = check_cache(cache, true);
    if (st != MLZC_OK) return st;
    if (!d) return fail(MLZC_ERR_INVALID, "paged attention: null descriptor");
    if (d->type != MLZC_TYPE_F32 && d->type != MLZC_TYPE_F16)
        return fail(MLZC_ERR_UNSUPPORTED, "paged attention: q type %d (F32 = 0, F16 = 1)", d->type);
    if (d->mode & ~(uint32_t)MLZC_FA_MODE_SOFTCAP)
        return fail(MLZC_ERR_UNSUPPORTED, "paged attention: mode 0x%x (SOFTCAP only)", d->mode);
    if (d->n_head_q < 1 || d->n_head_q % cache->n_head_kv || d->n_head_q / cache->n_head_kv > 128)
        return fail(MLZC_ERR_UNSUPPORTED, "paged attention: %lld query heads on %lld kv heads (a multiple, at most 128 times)",
                    (long long)d->n_head_q, (long long)cache->n_head_kv);
    // their products and quotients with one another and with scores stay inside f32
    auto usable = [](float x) { return x >= 0x1p-40f && x <= 0x1p40f; };
    if (!usable(d->scale)) return fail(MLZC_ERR_INVALID, "paged attention: scale %g (2^-40 to 2^40)", (double)d->scale);
    if ((d->mode & MLZC_FA_MODE_SOFTCAP) && !usable(d->logit_softcap))
        return fail(MLZC_ERR_INVALID, "paged attention: SOFTCAP mode with softcap %g (2^-40 to 2^40)", (double)d->logit_softcap);
    if (cache->n_tokens == 0) return MLZC_OK;
    if (cache->n_tokens * d->n_head_q > kMaxInt) return fail(MLZC_ERR_INVALID, "paged attention: too many query rows");
    const size_t elem = d->type == MLZC_TYPE_F32 ? 4 : 2, row = (size_t)cache->head_dim * elem;
    int e = check_rows("paged attention: q", d->q, d->q_nb, d->n_head_q, cache->n_tokens, row, elem);
    if (e == MLZC_OK && !weights) e = check_rows("paged attention: dst", d->dst, d->dst_nb, d->n_head_q, cache->n_tokens, row, elem);
    if (e != MLZC_OK) return e;
    if (weights && !d->lse) return fail(MLZC_ERR_INVALID, "paged weights: null lse");
    if (d->lse && ((uintptr_t)d->lse % 4 || d->lse_nb[0] % 4 || d->lse_nb[1] % 4 || (d->n_head_q > 1 && !d->lse_nb[0]) ||
                   (cache->n_tokens > 1 && !d->lse_nb[1])))
        return fail(MLZC_ERR_INVALID, "paged attention: lse strides must be multiples of 4 bytes");
    return MLZC_OK;
}

}  // namespace paged
}  // namespace mlzc
