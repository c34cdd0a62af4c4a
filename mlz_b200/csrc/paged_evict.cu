// paged_evict.cu -- the paged KV cache cut down to a budget of slots a head, by accumulated
// attention weight (mlzc_paged_evict_dev).
//
// Per (sequence, kv head) with n > budget slots: the first n_sink and the last n_recent stay,
// and of the candidates between them the m = budget - n_sink - n_recent of the largest weight,
// ties to the lowest slot.  Two launches:
//   select: the m-th largest key by a radix select (weights mapped to integers of the same
//           order), then one pass in slot order that numbers the freed slots below the budget
//           (holes) and the kept ones behind it (movers).  There are as many of the one as of
//           the other, so mover r goes to hole r.
//   move:   rows of K and V from movers to holes.  Every source lies at or behind the budget
//           and every target before it, so rows move in place, in any order, and only those
//           that have to (order-keeping compaction would move nearly all of them).
#include <algorithm>

#include "paged.h"
#include "ptx.cuh"

namespace mlzc {
namespace {

using paged::View;

constexpr int kSelThreads = 1024;
constexpr int kItems = 4;                     // slots a thread takes per ordered step
constexpr int kBins = 2048;                   // 11 bits a radix pass: 11 + 11 + 10

struct EvictArgs {
    View c;
    int budget, sink, recent, D;
    const char* w;
    char* w_out;
    char* kept;
    int* kv_len_out;
    int* holes;                               // workspace: [batch][head][budget]
    size_t w_head, w_seq, o_head, o_seq, kept_head, kept_seq;
};

// Integer of the same order as the float: -0 equals 0, NaN below everything.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Inclusive sums of (a, b) over the block's threads in order; totals in *ta, *tb.  sh: 64 ints.
__device__ __forceinline__ void block_scan2(int& a, int& b, int* ta, int* tb, int* sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(~0u, a, o), y = __shfl_up_sync(~0u, b, o);
        if (lane >= o) { a += x; b += y; }
    }
    if (lane == 31) { sh[warp] = a; sh[32 + warp] = b; }
    __syncthreads();
    if (warp == 0) {
        int x = sh[lane], y = sh[32 + lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int p = __shfl_up_sync(~0u, x, o), q = __shfl_up_sync(~0u, y, o);
            if (lane >= o) { x += p; y += q; }
        }
        sh[lane] = x;
        sh[32 + lane] = y;
    }
    __syncthreads();
    if (warp > 0) { a += sh[warp - 1]; b += sh[32 + warp - 1]; }
    *ta = sh[31];
    *tb = sh[63];
    __syncthreads();
}

__global__ void __launch_bounds__(kSelThreads) select_kernel(const __grid_constant__ EvictArgs a) {
    __shared__ int hist[kBins];
    __shared__ int sh[64];
    __shared__ int found[2];                  // the digit, and how many keys lie above it
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int n = paged::load_seq(a.c, b, false).kv;
    const int size = min(n, a.budget);
    const float* w = reinterpret_cast<const float*>(a.w + (size_t)b * a.w_seq + (size_t)h * a.w_head);
    float* wo = reinterpret_cast<float*>(a.w_out + (size_t)b * a.o_seq + (size_t)h * a.o_head);
    int* kept = reinterpret_cast<int*>(a.kept + (size_t)b * a.kept_seq + (size_t)h * a.kept_head);
    int* holes = a.holes + ((size_t)b * a.c.n_head_kv + h) * a.budget;
    for (int i = size + tid; i < a.budget; i += kSelThreads) kept[i] = -1;
    if (n <= a.budget) {
        for (int i = tid; i < n; i += kSelThreads) {
            kept[i] = i;
            if (wo != w) wo[i] = ptx::ld_act(w + i);
        }
        return;
    }
    const int lo = a.sink, hi = n - a.recent;          // candidates
    int need = a.budget - a.sink - a.recent;           // of which so many stay (fewer than hi - lo)
    uint32_t prefix = 0, mask = 0;
    if (need > 0) {
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11, bins = 1 << bits;
            for (int i = tid; i < bins; i += kSelThreads) hist[i] = 0;
            __syncthreads();
            for (int i = lo + tid; i < hi; i += kSelThreads) {
                const uint32_t k = order_key(ptx::ld_act(w + i));
                if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1);
            }
            __syncthreads();
            // from the top: the digit whose keys hold the need-th largest; each thread owns two
            const int d0 = bins - 1 - 2 * tid;
            const int c0 = 2 * tid < bins ? hist[d0] : 0, c1 = 2 * tid < bins ? hist[d0 - 1] : 0;
            int upto = c0 + c1, unused = 0, t0, t1;
            block_scan2(upto, unused, &t0, &t1, sh);
            const int before = upto - c0 - c1;
            if (before < need && need <= upto) {
                const bool second = need > before + c0;
                found[0] = second ? d0 - 1 : d0;
                found[1] = second ? before + c0 : before;
            }
            __syncthreads();
            prefix |= (uint32_t)found[0] << shift;
            mask |= (uint32_t)(bins - 1) << shift;
            need -= found[1];
            __syncthreads();
        }
    }
    // keys above `prefix` stay, and the first `need` equal to it
    int equal_seen = 0, hole_seen = 0, mover_seen = 0;
    for (int base = 0; base < n; base += kSelThreads * kItems) {
        const int i0 = base + tid * kItems;
        float x[kItems];
        bool eq[kItems], stay[kItems];
        int ne = 0;
#pragma unroll
        for (int j = 0; j < kItems; ++j) {
            const int i = i0 + j;
            x[j] = i < n ? ptx::ld_act(w + i) : 0.0f;
            const uint32_t k = order_key(x[j]);
            const bool cand = i >= lo && i < hi;
            eq[j] = cand && a.budget > a.sink + a.recent && k == prefix;
            stay[j] = i < n && (!cand || (a.budget > a.sink + a.recent && k > prefix));
            ne += eq[j];
        }
        int ie = ne, unused = 0, te, t1;
        block_scan2(ie, unused, &te, &t1, sh);
        int r = equal_seen + ie - ne;
        int nh = 0, nm = 0;
#pragma unroll
        for (int j = 0; j < kItems; ++j) {
            if (eq[j] && r++ < need) stay[j] = true;
            nh += i0 + j < size && !stay[j];
            nm += i0 + j >= size && stay[j];
        }
        equal_seen += te;
        int ih = nh, im = nm, th, tm;
        block_scan2(ih, im, &th, &tm, sh);
        int rh = hole_seen + ih - nh, rm = mover_seen + im - nm;
#pragma unroll
        for (int j = 0; j < kItems; ++j) {
            const int i = i0 + j;
            if (i < size) {
                if (stay[j]) {
                    kept[i] = i;
                    if (wo != w) wo[i] = x[j];
                } else {
                    holes[rh++] = i;
                }
            }
        }
        __syncthreads();                      // holes of this step before its movers
#pragma unroll
        for (int j = 0; j < kItems; ++j) {
            const int i = i0 + j;
            if (i >= size && stay[j]) {
                const int to = holes[rm++];
                kept[to] = i;
                wo[to] = x[j];
            }
        }
        hole_seen += th;
        mover_seen += tm;
    }
    __syncthreads();                          // in place: every weight has been read
    for (int i = size + tid; i < n; i += kSelThreads) wo[i] = 0.0f;
}

constexpr int kMoveWarps = 8;
constexpr int kMoveSlots = kMoveWarps * 32;

template <int D>
__global__ void __launch_bounds__(kMoveWarps * 32) move_kernel(const __grid_constant__ EvictArgs a) {
    constexpr int kChunks = D * 2 / 16;       // 16-byte pieces of a row: a warp copies 32 / kChunks rows at a time
    constexpr int kRows = 32 / kChunks;
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    const View& c = a.c;
    const int h = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) {
        const int kv = paged::ld_int(c.kv_len + b);
        a.kv_len_out[b] = min(min(max(kv, 0), c.cap), a.budget);
    }
    const int slot = blockIdx.x * kMoveSlots + warp * 32 + lane;
    const int* kept = reinterpret_cast<const int*>(a.kept + (size_t)b * a.kept_seq + (size_t)h * a.kept_head);
    const int from = slot < a.budget ? paged::ld_int(kept + slot) : -1;
    const bool moves = from >= 0 && from != slot;
    int pf = -1, pt = -1;
    if (moves) {
        pf = paged::load_page(c, b, from / c.page);
        pt = paged::load_page(c, b, slot / c.page);
    }
    const bool go = pf >= 0 && pt >= 0;
    // byte offsets of this lane's row, source and target
    size_t sk = 0, sv = 0, tk = 0, tv = 0;
    if (go) {
        const int rf = from % c.page, rt = slot % c.page;
        sk = (size_t)pf * c.k_page + (size_t)h * c.k_head + (size_t)rf * c.k_row;
        sv = (size_t)pf * c.v_page + (size_t)h * c.v_head + (size_t)rf * c.v_row;
        tk = (size_t)pt * c.k_page + (size_t)h * c.k_head + (size_t)rt * c.k_row;
        tv = (size_t)pt * c.v_page + (size_t)h * c.v_head + (size_t)rt * c.v_row;
    }
    uint32_t todo = __ballot_sync(~0u, go);
    const int sub = lane / kChunks, piece = (lane % kChunks) * 16;
    while (todo) {
        constexpr int U = 4;                  // row groups in flight
        uint4 xk[U], xv[U];
        size_t ok[U], ov[U];
        bool on[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            int mine = -1;
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const int l = __ffs(todo) - 1;
                if (todo) todo &= todo - 1;
                if (r == sub) mine = l;
            }
            on[u] = mine >= 0;
            const int src = on[u] ? mine : 0;
            const size_t fk = __shfl_sync(~0u, sk, src), fv = __shfl_sync(~0u, sv, src);
            ok[u] = __shfl_sync(~0u, tk, src);
            ov[u] = __shfl_sync(~0u, tv, src);
            if (on[u]) {
                xk[u] = ptx::ld_act(reinterpret_cast<const uint4*>(c.k + fk + piece));
                xv[u] = ptx::ld_act(reinterpret_cast<const uint4*>(c.v + fv + piece));
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (on[u]) {
                *reinterpret_cast<uint4*>(c.k + ok[u] + piece) = xk[u];
                *reinterpret_cast<uint4*>(c.v + ov[u] + piece) = xv[u];
            }
    }
}

size_t evict_workspace(const mlzc_paged_cache* cache, const mlzc_paged_evict_desc* d) {
    return ((size_t)cache->batch_size * cache->n_head_kv * d->budget * 4 + 15) / 16 * 16;
}

int check_table(const char* what, const void* p, const size_t* nb, int64_t heads, int64_t batch, size_t row) {
    if (!p || (uintptr_t)p % 4) return fail(MLZC_ERR_INVALID, "paged evict: %s null or misaligned", what);
    if (nb[0] != 4 || nb[1] % 4 || nb[2] % 4 || (heads > 1 && nb[1] < row) || (batch > 1 && nb[2] < row))
        return fail(MLZC_ERR_INVALID, "paged evict: %s strides (rows of 4-byte entries that do not overlap)", what);
    return MLZC_OK;
}

int check_evict(const mlzc_paged_cache* cache, const mlzc_paged_evict_desc* d) {
    int st = paged::check_cache(cache, false);
    if (st != MLZC_OK) return st;
    if (!d) return fail(MLZC_ERR_INVALID, "paged evict: null descriptor");
    if (d->budget < 1 || d->budget > (1ll << 30)) return fail(MLZC_ERR_INVALID, "paged evict: budget %lld", (long long)d->budget);
    if (d->n_sink < 0 || d->n_recent < 0 || d->n_sink > d->budget || d->n_recent > d->budget - d->n_sink)
        return fail(MLZC_ERR_INVALID, "paged evict: n_sink %lld + n_recent %lld over budget %lld", (long long)d->n_sink,
                    (long long)d->n_recent, (long long)d->budget);
    if (cache->batch_size > 65535) return fail(MLZC_ERR_UNSUPPORTED, "paged evict: batch_size above 65535");
    return MLZC_OK;
}

}  // namespace
}  // namespace mlzc

using namespace mlzc;

extern "C" int mlzc_paged_evict_workspace_bytes(const mlzc_paged_cache* cache, const mlzc_paged_evict_desc* d,
                                                size_t* out_bytes) {
    if (!out_bytes) return fail(MLZC_ERR_INVALID, "paged evict: null out_bytes");
    *out_bytes = 0;
    const int st = check_evict(cache, d);
    if (st == MLZC_OK) *out_bytes = evict_workspace(cache, d);
    return st;
}

extern "C" int mlzc_paged_evict_dev(const mlzc_paged_cache* cache, const mlzc_paged_evict_desc* d, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    int st = check_evict(cache, d);
    if (st != MLZC_OK) return st;
    const size_t row = (size_t)cache->max_pages * cache->page_size * 4;
    st = check_table("weights", d->weights, d->weights_nb, cache->n_head_kv, cache->batch_size, row);
    if (st == MLZC_OK) st = check_table("weights_out", d->weights_out, d->weights_out_nb, cache->n_head_kv, cache->batch_size, row);
    if (st == MLZC_OK) st = check_table("kept", d->kept, d->kept_nb, cache->n_head_kv, cache->batch_size, (size_t)d->budget * 4);
    if (st != MLZC_OK) return st;
    if (d->weights == d->weights_out &&
        (d->weights_nb[1] != d->weights_out_nb[1] || d->weights_nb[2] != d->weights_out_nb[2]))
        return fail(MLZC_ERR_INVALID, "paged evict: weights_out in place with other strides");
    if (!d->kv_len_out || (uintptr_t)d->kv_len_out % 4) return fail(MLZC_ERR_INVALID, "paged evict: kv_len_out null or misaligned");
    const size_t need = evict_workspace(cache, d);
    if (!workspace || workspace_bytes < need)
        return fail(MLZC_ERR_NOMEM, "paged evict: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    if ((uintptr_t)workspace % 16) return fail(MLZC_ERR_INVALID, "paged evict: workspace not 16-byte aligned");
    DeviceCtx* c = current_ctx();
    if (!c) return MLZC_ERR_CUDA;
    EvictArgs a{};
    st = paged::make_view(cache, false, c, &a.c);
    if (st != MLZC_OK) return st;
    a.budget = (int)d->budget;
    a.sink = (int)d->n_sink;
    a.recent = (int)d->n_recent;
    a.D = (int)cache->head_dim;
    a.w = reinterpret_cast<const char*>(d->weights);
    a.w_out = reinterpret_cast<char*>(d->weights_out);
    a.kept = reinterpret_cast<char*>(d->kept);
    a.kv_len_out = d->kv_len_out;
    a.holes = static_cast<int*>(workspace);
    a.w_head = d->weights_nb[1]; a.w_seq = d->weights_nb[2];
    a.o_head = d->weights_out_nb[1]; a.o_seq = d->weights_out_nb[2];
    a.kept_head = d->kept_nb[1]; a.kept_seq = d->kept_nb[2];
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    MLZC_CUDA_TRY(launch_pdl(select_kernel, dim3(a.c.n_head_kv, a.c.batch), dim3(kSelThreads), 0, s, a));
    MLZC_CUDA_TRY(cudaGetLastError());
    // slots past the table's capacity cannot be kept
    const int slots = std::min(a.budget, a.c.cap);
    const dim3 g((unsigned)((slots + kMoveSlots - 1) / kMoveSlots), (unsigned)a.c.n_head_kv, (unsigned)a.c.batch);
    MLZC_CUDA_TRY(launch_pdl(a.D == 64 ? move_kernel<64> : (a.D == 128 ? move_kernel<128> : move_kernel<256>), g,
                             dim3(kMoveWarps * 32), 0, s, a));
    MLZC_CUDA_TRY(cudaGetLastError());
    count_launch(2);
    return MLZC_OK;
}
