// paged_evict.cu -- the paged KV cache cut down to a budget of slots a head, by accumulated
// attention weight (mlzc_paged_evict_dev).
//
// Per (sequence, kv head) with n > budget slots: the first n_sink and the last n_recent stay,
// and of the candidates between them the m = budget - n_sink - n_recent of the largest weight,
// ties to the lowest slot.  Two launches:
//   select: the m-th largest key by a radix select (weights mapped to integers of the same
//           order, three passes of 11, 11 and 10 bits), then the freed slots below the budget
//           (holes) and the kept ones behind it (movers) numbered in slot order.  There are as
//           many of the one as of the other, so mover r goes to hole r.
//   move:   rows of K and V from movers to holes.  Every source lies at or behind the budget
//           and every target before it, so rows move in place, in any order, and only those
//           that have to (order-keeping compaction would move nearly all of them).
// Measured: 16 sequences of 512 to 8192 slots x 8 heads x 128 dims cut to 1000 take 29.6 us, half of it
// the move of 43 MB (and as much back, most of it to L2), bound by HBM and its own three dependent
// loads.  The selection is bound by latency, by passes that depend on one another and
// cost some twenty instructions a slot and pass on the one SM that has the head: 15 us for 8192
// slots (20 before its keys, bits and holes lay in shared memory).  Where heads are few, a cluster
// of up to 8 CTAs shares one, its counts read over distributed shared memory: 18 us for 32768
// slots (41 with one CTA).
#include <cooperative_groups.h>

#include <algorithm>

#include "paged.h"
#include "ptx.cuh"

namespace mlzc {
namespace {

using paged::View;

constexpr int kSelThreads = 1024, kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048;                   // 11 bits a radix pass
constexpr int kHeldSlots = 32768;             // keys of so many slots fit in a CTA's shared memory,
constexpr int kHeldHoles = 8192;              // and the holes of such a budget beside them

struct EvictArgs {
    View c;
    int budget, sink, recent, D;
    const char* w;
    char* w_out;
    char* kept;
    int* kv_len_out;
    int* holes;                               // workspace: [batch][head][budget], for heads of several CTAs
    uint32_t* words;                          // workspace: [batch][head][n_words], a bit a slot that stays, for long heads
    int n_words;
    int held, held_holes;                     // slots and holes that shared memory has room for
    size_t w_head, w_seq, o_head, o_seq, kept_head, kept_seq;
};

// Integer of the same order as the float: -0 equals 0, NaN below everything.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

namespace cg = cooperative_groups;

constexpr int kRanks = 8;                     // CTAs of a cluster at most (the portable size)
constexpr int kShare = 4096;                  // slots worth a CTA of a cluster (its barriers cost 1 us each)

// Shared memory of a selecting CTA.
struct Sel {
    int4 hist[3][kBins / 4];                  // of each pass
    int coarse[3][kSelWarps];                 // the same in blocks of 64 digits
    int sums[3][kSelWarps];                   // warps' sums, a row a scan
    int found[3][3];                          // the digit, how many keys lie above it, how many have it
    int count[3];                             // this CTA's equals, holes, movers
    int listed;
    uint32_t list[2048];                      // keys with the first digit found, where they are few
};
constexpr int kList = 2048;
constexpr uint32_t kForced = 0xFFFFFFFFu;     // key of a slot that stays anyway: above every weight's

__device__ __forceinline__ int warp_sum(int x) { return __reduce_add_sync(~0u, x); }

// Sum of a warp-wide value over the warps before this one, and over all: sh is a row of sums.
__device__ __forceinline__ int warps_before(int mine, int* total, int* sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) sh[warp] = mine;
    __syncthreads();
    const int x = sh[lane];
    *total = warp_sum(x);
    return warp_sum(lane < warp ? x : 0);
}

// Of 32 x K counts, K a lane in ascending order, the place of the need-th from the top: its index
// (warp-wide), the counts above it, its own.
template <int K>
__device__ __forceinline__ int3 find_from_top(const int (&c)[K], int need) {
    const int lane = threadIdx.x & 31;
    int mine = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) mine += c[i];
    int upto = mine;                          // of this lane and those above
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_down_sync(~0u, upto, o);
        if (lane + o < 32) upto += y;
    }
    const int at = 31 - __clz(__ballot_sync(~0u, upto >= need));
    int above = upto - mine, k = K - 1, have = c[K - 1];
#pragma unroll
    for (int i = K - 2; i >= 0; --i)
        if (above + have < need) { above += have; have = c[i]; k = i; }
    return make_int3(__shfl_sync(~0u, lane * K + k, at), __shfl_sync(~0u, above, at), __shfl_sync(~0u, have, at));
}

__global__ void __launch_bounds__(kSelThreads) select_kernel(const __grid_constant__ EvictArgs a) {
    __shared__ Sel sel;
    extern __shared__ uint32_t held[];        // keys, bits of the slots that stay, holes
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const int n = paged::load_seq(a.c, b, false).kv;
    for (int i = tid; i < 3 * kBins / 4; i += kSelThreads) sel.hist[0][i] = make_int4(0, 0, 0, 0);
    if (tid == 0) sel.listed = 0;
    const int size = min(n, a.budget);
    const float* w = reinterpret_cast<const float*>(a.w + (size_t)b * a.w_seq + (size_t)h * a.w_head);
    float* wo = reinterpret_cast<float*>(a.w_out + (size_t)b * a.o_seq + (size_t)h * a.o_head);
    int* kept = reinterpret_cast<int*>(a.kept + (size_t)b * a.kept_seq + (size_t)h * a.kept_head);
    auto sync = [&]() {
        if (ranks == 1) __syncthreads();
        else cluster.sync();
    };
    const int all = kSelThreads * ranks, me = rank * kSelThreads + tid;
    for (int i = size + me; i < a.budget; i += all) kept[i] = -1;
    if (n <= a.budget) {                      // alike for the whole cluster
        for (int i = me; i < n; i += all) {
            kept[i] = i;
            if (wo != w) wo[i] = ptx::ld_act(w + i);
        }
        return;
    }
    // This CTA's run of slots (whole words of 32), and each warp's within it: lane l of a warp has
    // every 32nd slot, so that loads and stores are whole lines and a slot's rank is a count of
    // ballot bits.  Short loops on purpose: each phase runs once a launch, and with 16 slots a
    // lane unrolled the selection of 8 heads of 32768 slots took 35 us.
    const int lane = tid & 31, warp = __shfl_sync(~0u, tid >> 5, 0), log_ranks = 31 - __clz(ranks);
    const int share = (((n + ranks - 1) >> log_ranks) + 31) & ~31, s0 = min(n, rank * share), s1 = min(n, s0 + share);
    const int run = (share / kSelWarps + 31) & ~31, w0 = min(s1, s0 + warp * run), w1 = min(s1, w0 + run);
    const bool hold = share <= a.held;
    const uint32_t below = (1u << lane) - 1;
    const int lo = a.sink, hi = n - a.recent;          // candidates
    int need = a.budget;                               // with the forced ones; fewer than n
    const size_t head = (size_t)b * a.c.n_head_kv + h;
    uint32_t* words = hold ? held + a.held : a.words + head * a.n_words + (s0 >> 5);
    int* holes = ranks == 1 && a.budget <= a.held_holes ? reinterpret_cast<int*>(held + a.held + a.held / 32) : a.holes + head * a.budget;
    auto key_of = [&](int i) {
        const uint32_t k = order_key(ptx::ld_act(w + i));
        return i < lo || i >= hi ? kForced : k;
    };
    if (hold) {
        for (int i = w0 + lane; i < w1; i += 128) {    // read by the same lane alone
            uint32_t k[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) k[u] = key_of(min(i + 32 * u, w1 - 1));
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + 32 * u < w1) held[i + 32 * u - s0] = k[u];
        }
    }
    // f(slot, key) for this lane's slots; every lane of the warp comes along (slots at or past w1
    // are none of its)
    auto each = [&](auto f) {
#pragma unroll 2
        for (int i = w0 + lane; i - lane < w1; i += 32) f(i, i < w1 ? (hold ? held[i - s0] : key_of(i)) : 0u);
    };
    __syncthreads();
    uint32_t prefix = 0, mask = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), digits = pass == 2 ? 1023 : 2047;
        int* hist = reinterpret_cast<int*>(sel.hist[pass]);
        const bool few = pass > 0 && sel.found[0][2] <= kList;
        if (few && pass == 2) {
            for (int i = tid; i < sel.listed; i += kSelThreads)
                if ((sel.list[i] & mask) == prefix) atomicAdd(&hist[sel.list[i] & digits], 1);
        } else {
            each([&](int i, uint32_t k) {
                const bool in = i < w1 && (k & mask) == prefix;
                if (in) atomicAdd(&hist[(k >> shift) & digits], 1);
                if (few && in) sel.list[atomicAdd(&sel.listed, 1)] = k;
            });
        }
        // the digit whose keys hold the need-th largest: its block of 64 first, then the digit, so
        // that a cluster's CTAs read little of one another's
        __syncthreads();
        const int2 mine = reinterpret_cast<const int2*>(hist)[tid];
        const int sum = warp_sum(mine.x + mine.y);
        if (lane == 0) sel.coarse[pass][warp] = sum;
        sync();
        if (warp == 0) {
            int c[1] = {0}, d[2] = {0, 0};
            if (ranks == 1) {
                c[0] = sel.coarse[pass][lane];
            } else {
#pragma unroll
                for (int r = 0; r < kRanks; ++r) c[0] += r < ranks ? *cluster.map_shared_rank(&sel.coarse[pass][lane], r) : 0;
            }
            const int3 block = find_from_top(c, need);
            const int2* fine = reinterpret_cast<const int2*>(hist) + block.x * 32 + lane;
            if (ranks == 1) {
                d[0] = fine->x;
                d[1] = fine->y;
            } else {
                int2 v[kRanks];
#pragma unroll
                for (int r = 0; r < kRanks; ++r) v[r] = r < ranks ? *cluster.map_shared_rank(fine, r) : make_int2(0, 0);
#pragma unroll
                for (int r = 0; r < kRanks; ++r) { d[0] += v[r].x; d[1] += v[r].y; }
            }
            const int3 digit = find_from_top(d, need - block.y);
            if (lane == 0) {
                sel.found[pass][0] = block.x * 64 + digit.x;
                sel.found[pass][1] = block.y + digit.y;
                sel.found[pass][2] = digit.z;
            }
        }
        __syncthreads();
        prefix |= (uint32_t)sel.found[pass][0] << shift;
        mask |= (uint32_t)digits << shift;
        need -= sel.found[pass][1];
    }
    // Keys above `prefix` stay, and the first `need` equal to it.  Counts of the CTAs before this
    // one come from their shared memory.
    auto from_others = [&](int which) {
        int sum = 0;
        if (ranks > 1) {
#pragma unroll
            for (int r = 0; r < kRanks; ++r) sum += r < rank ? *cluster.map_shared_rank(&sel.count[which], r) : 0;
        }
        return sum;
    };
    // equal keys need counting in order only where not all of them stay
    const bool ties = sel.found[2][2] > need;
    int equals = 0, total;
    if (ties) {
        int mine = 0;
        each([&](int i, uint32_t k) { mine += i < w1 && k == prefix; });
        equals = warps_before(warp_sum(mine), &total, sel.sums[0]);
        if (tid == 0) sel.count[0] = total;
        sync();
        equals += from_others(0);
    }
    // which slots stay, and how many are holes and movers
    int nh = 0, nm = 0;
    each([&](int i, uint32_t k) {
        bool s = i < w1 && k >= prefix;
        if (ties) {
            const bool eq = i < w1 && k == prefix;
            const uint32_t bits = __ballot_sync(~0u, eq);
            if (eq) s = equals + __popc(bits & below) < need;
            equals += __popc(bits);
        }
        const uint32_t stay = __ballot_sync(~0u, s);
        if (lane == 0) words[(i - s0) >> 5] = stay;
        nh += i < min(w1, size) && !s;
        nm += i >= size && s;
    });
    __syncwarp();
    int th, tm;
    int rh = warps_before(warp_sum(nh), &th, sel.sums[1]), rm = warps_before(warp_sum(nm), &tm, sel.sums[2]);
    if (tid == 0) {
        sel.count[1] = th;
        sel.count[2] = tm;
    }
    sync();
    rh += from_others(1);
    rm += from_others(2);
#pragma unroll 1
    for (int i = w0 + lane; i - lane < min(w1, size); i += 32) {
        const bool mine = i < min(w1, size), s = words[(i - s0) >> 5] >> lane & 1;
        const uint32_t bits = __ballot_sync(~0u, mine && !s);
        if (mine && !s) holes[rh + __popc(bits & below)] = i;
        rh += __popc(bits);
        if (mine && s) {
            kept[i] = i;
            if (wo != w) wo[i] = ptx::ld_act(w + i);
        }
    }
    sync();                                   // every hole is listed, every count read
    // four words at a time, their holes and weights on the way together
    constexpr int U = 4;
    const int from = max(w0, size & ~31);
#pragma unroll 1
    for (int i0 = from + lane; i0 - lane < w1; i0 += 32 * U) {
        int to[U];
        float x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + 32 * u;
            const uint32_t stay = i - lane < w1 ? words[(i - s0) >> 5] : 0;
            const bool mover = i >= size && (stay >> lane & 1);
            const uint32_t bits = __ballot_sync(~0u, mover);
            to[u] = mover ? holes[rm + __popc(bits & below)] : -1;
            x[u] = mover ? ptx::ld_act(w + i) : 0.0f;
            rm += __popc(bits);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + 32 * u;
            if (to[u] >= 0) {
                kept[to[u]] = i;
                wo[to[u]] = x[u];
            }
            if (i >= size && i < w1) wo[i] = 0.0f;
        }
    }
}

constexpr int kMoveWarps = 8;
// Slots a warp looks after: with 32 a warp's rows come in four dependent steps (16 sequences to 1000
// 30.5 us for 29.6, 32768 slots 24.0 for 22.6), with 8 large batches pay for the blocks' starts (64
// sequences of 2000 to 4000 to 1500: 104 us for 92).
constexpr int kWarpSlots = 16;
constexpr int kMoveSlots = kMoveWarps * kWarpSlots;

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
    const int slot = blockIdx.x * kMoveSlots + warp * kWarpSlots + lane;
    const int* kept = reinterpret_cast<const int*>(a.kept + (size_t)b * a.kept_seq + (size_t)h * a.kept_head);
    const int from = lane < kWarpSlots && slot < a.budget ? paged::ld_int(kept + slot) : -1;
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

int launch_select(EvictArgs& a, const DeviceCtx* c, cudaStream_t s) {
    // CTAs of kShare slots, as long as every head's are on the GPU together
    int ranks = 1;
    while (ranks < kRanks && (int64_t)a.c.n_head_kv * a.c.batch * 2 * ranks <= c->sm_count && a.c.cap > ranks * kShare) ranks *= 2;
    a.held = std::min(kHeldSlots, ((a.c.cap + ranks - 1) / ranks + 31) / 32 * 32);
    a.held_holes = ranks == 1 ? std::min(kHeldHoles, a.budget) : 0;
    const size_t smem = (size_t)a.held * 4 + a.held / 8 + (size_t)a.held_holes * 4;
    static bool set[64] = {};
    const int dev = c->device < 64 ? c->device : 63;
    if (!set[dev] || c->device >= 64) {
        MLZC_CUDA_TRY(cudaFuncSetAttribute(select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           kHeldSlots * 4 + kHeldSlots / 8 + kHeldHoles * 4));
        set[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ranks, a.c.n_head_kv, a.c.batch);
    cfg.blockDim = dim3(kSelThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_mode() == MLZC_OVERLAP_OFF ? 1 : 2;
    MLZC_CUDA_TRY(cudaLaunchKernelEx(&cfg, select_kernel, a));
    MLZC_CUDA_TRY(cudaGetLastError());
    return MLZC_OK;
}

size_t evict_words(const mlzc_paged_cache* cache) { return ((size_t)cache->max_pages * cache->page_size + 31) / 32; }
size_t evict_workspace(const mlzc_paged_cache* cache, const mlzc_paged_evict_desc* d) {
    return ((size_t)cache->batch_size * cache->n_head_kv * (d->budget + evict_words(cache)) * 4 + 15) / 16 * 16;
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
    a.n_words = (int)evict_words(cache);
    a.words = reinterpret_cast<uint32_t*>(a.holes + (size_t)a.c.batch * a.c.n_head_kv * a.budget);
    a.w_head = d->weights_nb[1]; a.w_seq = d->weights_nb[2];
    a.o_head = d->weights_out_nb[1]; a.o_seq = d->weights_out_nb[2];
    a.kept_head = d->kept_nb[1]; a.kept_seq = d->kept_nb[2];
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    st = launch_select(a, c, s);
    if (st != MLZC_OK) return st;
    // slots past the table's capacity cannot be kept
    const int slots = std::min(a.budget, a.c.cap);
    const dim3 g((unsigned)((slots + kMoveSlots - 1) / kMoveSlots), (unsigned)a.c.n_head_kv, (unsigned)a.c.batch);
    MLZC_CUDA_TRY(launch_pdl(a.D == 64 ? move_kernel<64> : (a.D == 128 ? move_kernel<128> : move_kernel<256>), g,
                             dim3(kMoveWarps * 32), 0, s, a));
    MLZC_CUDA_TRY(cudaGetLastError());
    count_launch(2);
    return MLZC_OK;
}
