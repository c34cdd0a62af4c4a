// paged_weights.cu -- the attention weight that each slot of a paged KV cache received from the
// new tokens (mlzc_paged_weights_dev), on the 5th-generation tensor cores.
//
//   out[j] = acc[j] + sum over the rows r that see slot j of 2^(c s_jr - lse2_r),
//   s_jr = <k_j, q_r>,  c = scale * log2 e,  lse2 = lse * log2 e,
// for every (sequence, KV head); the rows are its new tokens x the query heads of the head.
//
// The scores are recomputed (storing them would cost 4 bytes a score) as S^T = K Q^T: slots on
// the lanes, rows on the columns.  A slot's sum then stays in one thread, so nothing is added
// across threads and nothing atomically, and the softmax's statistics, known from the
// attention, enter as one constant a column: one FMA, one exponential and one add a score.  Of a
// long chunk's time the exponential unit (1024 clocks a 128 x 128 tile; the products take 512) is
// busy 72 %, the tensor cores 36 % (counters, 2048 tokens of 8192, 8 heads of 4).  The unit is the
// nearest bound, but not alone what takes the time: moving one exponential in four to the FMA pipe
// gained nothing (175 us either way); each step waits for its 32 columns before it computes.  Decode
// reads K at 4 TB/s with no unit busy (HBM 46 %, tensor cores 7 %, exponentials 15 %).
//
// A piece of work is what one operand is held for: a slot tile (K) and its query tiles, or,
// where a sequence's rows fill one query tile at most (decode), that tile (Q) and a run of slot
// tiles.  The held operand and the passing one share a ring of shared-memory units: loader warp
// (K by one TMA box a page piece, Q by one box a 64-dim block), MMA warp (scores into four TMEM
// buffers, as many columns as there are rows), two lse warps (a tile's lse2 into shared memory),
// four warpgroups that take turns at the tiles (with two
// the exponential unit idled half of the time: 205 us for 2048 tokens of 8192).  f32 queries come
// as f16 hi + lo from a small preparing launch, low products summed first.
//
// Measured (device times): 2048 tokens of 8192 slots, 8 heads of 4, 128 dims: f16 172 us, f32 231 (twice
// the products); masked columns become -inf before the common code (selected after the exponentials
// instead: 175 and 235); decode of 16 sequences of 512 to 8192: 38 us (152 MB), of one of 32768: 18 us.
//
// lse2 is rounded to f32 once a row (4e-7 of a weight at lse 10).  Carrying what that drops as a
// factor a column made no weight better (the products' own sums are as far off) and cost 12 %.
//
// Slot tiles x query tiles of a call form one list cut into equal shares, as in paged_attn.cu;
// a cut slot tile's 128 partial sums are merged in order by a last launch.
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstring>
#include <numeric>

#include "paged.h"
#include "ptx.cuh"
#include "tcgen05.cuh"

namespace mlzc {
namespace {

using paged::mbar_wait;
using paged::Seq;
using paged::View;
using ptx::mbar_arrive;
using ptx::mbar_expect_tx;
using ptx::mbar_init;
using ptx::smem_u32;
using namespace tc05;

constexpr int kSmemMax = 232448;
constexpr int kBN = 128;               // slots a tile
constexpr int kBufs = 4;               // score buffers in TMEM (128 columns each) and lse tiles
constexpr int kBarBytes = 640;
constexpr int kTurns = 4;              // warpgroups that take turns at the tiles
constexpr int kFixed = kBarBytes + kBufs * 128 * 4 + 2 * (kTurns - 1) * 128 * 4;   // barriers, lse tiles, sums handed over
constexpr int kEpiWarps = 4 * kTurns;
constexpr int kThreads = (kEpiWarps + 4) * 32;
constexpr float kLog2e = 1.4426950408889634f;

struct WeightArgs {
    View c;
    CUtensorMap mk, mkp, mq, mql;      // K pool in boxes of `box` rows, of a page (where `whole`); q rows (hi), lo
    const char* lse;
    const char* acc;
    char* out;
    size_t lse_head, lse_tok, a_head, a_seq, o_head, o_seq;
    int G, tq, box, whole, n_ctas;
    paged::Div by_tq, by_g;
    float scale, softcap;
    float* rec;                        // [cta][2][128]: 0 continues a cut slot tile, 1 begins one
    int4* head;                        // [cta]: sequence (-1: none), kv head, slot tile, last CTA of the tile begun
};

template <int D_, bool HL_, bool CAP_>
struct Cfg {
    static constexpr int D = D_;
    static constexpr bool HL = HL_;                   // f32 queries: hi + lo
    static constexpr bool CAP = CAP_;                 // scores are capped
    static constexpr int DU = D < 128 ? D : 128;      // dims of a ring unit (128 rows)
    static constexpr int UN = D / DU;
    static constexpr int SUBS = DU / 64;
    static constexpr uint32_t kSub = 128 * 128;
    static constexpr uint32_t kUnit = kSub * SUBS;
    static constexpr int kFit = (kSmemMax - 1024 - kFixed) / (int)kUnit;
    static constexpr int ST = kFit > 12 ? 12 : kFit;
    static constexpr size_t kSmem = 1024 + kFixed + (size_t)ST * kUnit;
    static constexpr int QU = UN * (HL ? 2 : 1);      // units of a Q tile
    static_assert(ST >= QU + 2 && ST >= UN + 2, "ring");
};

// Address of element i of a barrier array, from the base address `bars` at hand.
#define MLZC_BAR(member, i) (bars + (uint32_t)offsetof(Bars, member) + 8u * (uint32_t)(i))

struct Bars {
    uint64_t full[12], empty[12], s_full[kBufs], s_empty[kBufs], lse_full[kBufs], hand_full[2], hand_empty[2];
    uint32_t tmem;
    int abort;
    long long first, count, total;
    int b, h, t, tile;
    long long scan[kThreads / 32];
};
static_assert(sizeof(Bars) <= kBarBytes, "barriers");

// Query tiles of slot tile t: from the first one with a row that sees slot 128 t on; one at
// least, so that every slot below kv_len is written.
__device__ __forceinline__ int first_tile(const WeightArgs& a, const Seq& s, int t) {
    return a.by_tq.quot(max(0, t * kBN - (s.kv - s.rows)));
}
__device__ __forceinline__ int tiles_of(const WeightArgs& a, const Seq& s, int t) {
    return max(1, a.by_tq.quot(s.rows + a.tq - 1) - first_tile(a, s, t));
}
// The sum of tiles_of over a sequence's slot tiles: all alike up to the chunk's own slots.
struct Tiles {
    int alike, all;            // slot tiles [0, alike) have `each` query tiles
    int each;
    long long sum;
    __device__ Tiles(const WeightArgs& a, const Seq& s) {
        all = (s.kv + kBN - 1) / kBN;
        each = tiles_of(a, s, 0);
        const int off = max(0, s.kv - s.rows);
        alike = min(all, off / kBN + 1);
        sum = (long long)alike * each;
        for (int t = alike; t < all; ++t) sum += tiles_of(a, s, t);
    }
};

struct Walk {
    int b, h, t, tile, n;      // sequence, kv head, slot tile, query tile (after first_tile), tiles
    bool wide;                 // tiles of one query tile: slot tiles t .. t + n - 1
    int lead, tiles, all;      // first_tile and tiles_of of slot tile t; slot tiles of the head
    long long left;
    Seq s;
    bool first;
    __device__ Walk(const Bars* B) : b(B->b), h(B->h), t(B->t), tile(B->tile), n(0), wide(false), left(B->count), first(true) {}
    __device__ bool next(const WeightArgs& a) {
        if (left <= 0) return false;
        if (first) {
            s = paged::load_seq(a.c, b);
            first = false;
        } else {
            tile = 0;
            t += wide ? n : 1;
            if (t >= all) {
                t = 0;
                if (++h == a.c.n_head_kv) {
                    h = 0;
                    do {
                        s = paged::load_seq(a.c, ++b);
                    } while (s.kv == 0);
                }
            }
        }
        all = (s.kv + kBN - 1) / kBN;
        wide = s.rows <= a.tq;
        lead = wide ? 0 : first_tile(a, s, t);
        tiles = wide ? 1 : tiles_of(a, s, t);
        n = (int)min((long long)(wide ? all - t : tiles - tile), left);
        left -= n;
        return true;
    }
    __device__ bool whole() const { return wide || (tile == 0 && n == tiles); }
    // of the piece's tile i: slot tile, first token, columns, slots
    __device__ int slot_tile(int i) const { return wide ? t + i : t; }
    __device__ int tok0(const WeightArgs& a, int i) const { return wide ? 0 : (lead + tile + i) * a.tq; }
    __device__ int cols(const WeightArgs& a, int i) const { return max(0, min(a.tq, s.rows - tok0(a, i))) * a.G; }
    __device__ int slots(int i) const { return min(kBN, s.kv - slot_tile(i) * kBN); }
};

__device__ void plan(const WeightArgs& a, Bars* B) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (a.c.batch + kThreads - 1) / kThreads;
    const int b0 = tid * per, b1 = min(b0 + per, a.c.batch);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) mine += Tiles(a, paged::load_seq(a.c, b)).sum * a.c.n_head_kv;
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) B->scan[warp] = upto;
    __syncthreads();
    long long total = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) upto += B->scan[w];
        total += B->scan[w];
    }
    const long long n = min((long long)a.n_ctas, total), c = blockIdx.x;
    const long long lo = c < n ? total * c / n : 0, hi = c < n ? total * (c + 1) / n : 0;
    if (tid == 0) { B->first = lo; B->count = hi - lo; B->total = total; }
    if (hi > lo && lo >= upto - mine && lo < upto) {
        long long r = lo - (upto - mine);
        for (int b = b0; b < b1; ++b) {
            const Seq s = paged::load_seq(a.c, b);
            const Tiles k(a, s);
            if (r >= k.sum * a.c.n_head_kv) { r -= k.sum * a.c.n_head_kv; continue; }
            B->b = b;
            B->h = (int)(r / k.sum);
            r %= k.sum;
            int t = (int)min((long long)k.alike, r / k.each);
            r -= (long long)t * k.each;
            while (r >= tiles_of(a, s, t)) r -= tiles_of(a, s, t++);
            B->t = t;
            B->tile = (int)r;
            break;
        }
    }
    __syncthreads();
}

// Sums the weights of tile after tile; thread = slot.
template <class C>
__device__ __forceinline__ void sum_role(const WeightArgs& a, Bars* B, const float* lse2, float* handed, uint32_t tmem, int warp, int lane) {
    const int turn = warp >> 2;
    const int slot = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const float c2 = C::CAP ? kLog2e : a.scale * kLog2e;
    const float cap_in = C::CAP ? a.scale / a.softcap : 0.0f;
    const uint32_t bars = smem_u32(B);
    volatile int* abort = &B->abort;
    uint32_t g = 0, item = 0;
    Walk w(B);
    while (w.next(a)) {
        const bool whole = w.whole();
        // a slot tile with several query tiles: the warpgroups hand their sums to the first
        const bool shared = !w.wide && w.n > 1;
        const char* acc = a.acc ? a.acc + (size_t)w.b * a.a_seq + (size_t)w.h * a.a_head : nullptr;
        float* out = reinterpret_cast<float*>(a.out + (size_t)w.b * a.o_seq + (size_t)w.h * a.o_head);
        const int past = w.s.kv - w.s.rows;
        float total = 0.0f, before = 0.0f;
        bool mine = false;                    // this warpgroup had a tile of the piece
        if (!w.wide && whole && acc && slot < w.slots(0) && (!shared || turn == 0))
            before = ptx::ld_act(reinterpret_cast<const float*>(acc) + w.t * kBN + slot);
        for (int it = 0; it < w.n; ++it, ++g) {
            if ((int)(g % kTurns) != turn) continue;
            const int buf = g % kBufs, slots = w.slots(it), j = w.slot_tile(it) * kBN + slot;
            const uint32_t par = (g / kBufs) & 1;
            if (w.wide && acc && slot < slots) before = ptx::ld_act(reinterpret_cast<const float*>(acc) + j);
            mine = true;
            if (!mbar_wait(MLZC_BAR(s_full, buf), par, abort, a.c.err)) return;
            if (!mbar_wait(MLZC_BAR(lse_full, buf), par, abort, a.c.err)) return;
            tc_fence_after();
            const int cols = w.cols(a, it);
            if ((warp & 3) * 32 < slots && cols > 0) {
                // columns [from, cols) see this thread's slot; outside them a score may hold anything
                const int gap = j - past - w.tok0(a, it);
                const int from = gap > 0 ? min(gap, a.tq) * a.G : 0;
                auto counts = [&](int i) { return (uint32_t)(i - from) < (uint32_t)max(0, cols - from); };
                const float* lt = lse2 + buf * 128;
                const uint32_t s_col = lanes + buf * 128;
                uint64_t sum[2] = {0, 0};
                const bool some_cols = __any_sync(~0u, from > 0);
                const uint64_t c22 = pair(c2, c2);
#pragma unroll 1
                for (int i = 0; i < cols; i += 32) {
                    float x[32];
                    tmem_ld32(s_col + i, *reinterpret_cast<uint32_t(*)[32]>(x));
                    tmem_ld_wait();
                    if (C::CAP) cap_scores(x, cap_in, a.softcap);
                    if (some_cols || i + 32 > cols) {
#pragma unroll
                        for (int k = 0; k < 32; ++k) x[k] = counts(i + k) ? x[k] : -INFINITY;
                    }
#pragma unroll
                    for (int k = 0; k < 32; k += 4) {
                        const float4 L = *reinterpret_cast<const float4*>(lt + i + k);
                        float y0, y1, y2, y3;
                        unpair(fma2(pair(x[k], x[k + 1]), c22, pair(L.x, L.y)), y0, y1);
                        unpair(fma2(pair(x[k + 2], x[k + 3]), c22, pair(L.z, L.w)), y2, y3);
                        sum[0] = add2(sum[0], pair(ex2(y0), ex2(y1)));
                        sum[1] = add2(sum[1], pair(ex2(y2), ex2(y3)));
                    }
                }
                float s0, s1;
                unpair(add2(sum[0], sum[1]), s0, s1);
                float s = s0 + s1;
                // A sum that is not a number is taken again, in the same order, from the rows that add
                // something alone: one with lse = -inf (lt = -inf) does not, whatever its q, nor one that does
                // not see the slot, whatever its lse.
                if (__any_sync(~0u, s != s && slot < slots)) {
                    sum[0] = sum[1] = 0;
#pragma unroll 1
                    for (int i = 0; i < cols; i += 32) {
                        float x[32];
                        tmem_ld32(s_col + i, *reinterpret_cast<uint32_t(*)[32]>(x));
                        tmem_ld_wait();
                        if (C::CAP) cap_scores(x, cap_in, a.softcap);
#pragma unroll
                        for (int k = 0; k < 32; ++k) x[k] = counts(i + k) && lt[i + k] != -INFINITY ? ex2(fmaf(x[k], c2, lt[i + k])) : 0.0f;
#pragma unroll
                        for (int k = 0; k < 32; k += 2) sum[k >> 1 & 1] = add2(sum[k >> 1 & 1], pair(x[k], x[k + 1]));
                    }
                    unpair(add2(sum[0], sum[1]), s0, s1);
                    s = s0 + s1;
                }
                total += s;
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(MLZC_BAR(s_empty, buf));
            if (w.wide) {
                if (slot < slots) out[j] = before + total;
                total = 0.0f;
                before = 0.0f;
            }
        }
        if (w.wide) continue;
        if (shared) {
            float* there = handed + (item & 1) * (kTurns - 1) * 128 + slot;
            const uint32_t full = MLZC_BAR(hand_full, item & 1), empty = MLZC_BAR(hand_empty, item & 1), par = (item >> 1) & 1;
            ++item;
            if (turn > 0) {
                if (!mbar_wait(empty, par ^ 1, abort, a.c.err)) return;
                there[(turn - 1) * 128] = total;
                __syncwarp();
                if (lane == 0) mbar_arrive(full);
                continue;
            }
            if (!mbar_wait(full, par, abort, a.c.err)) return;
#pragma unroll
            for (int i = 0; i < kTurns - 1; ++i) total += there[i * 128];
            __syncwarp();
            if (lane == 0) mbar_arrive(empty);
        } else if (!mine) {
            continue;
        }
        if (!whole) a.rec[((size_t)blockIdx.x * 2 + (w.tile == 0 ? 1 : 0)) * 128 + slot] = total;
        else if (slot < w.slots(0)) out[w.t * kBN + slot] = before + total;
    }
}

// The order in which loader and MMA warp go round the ring: slots that hold the operand at hand
// are passed over.  A slot's phase is the parity of its uses.
template <int ST>
struct Ring {
    uint32_t next = 0, uses = 0, held = 0;
    // the next slot and the parity of its use
    __device__ __forceinline__ void step(uint32_t& st, uint32_t& par) {
        while ((held >> next) & 1) next = next + 1 == ST ? 0 : next + 1;
        st = next;
        par = (uses >> st) & 1;
        uses ^= 1u << st;
        next = st + 1 == ST ? 0 : st + 1;
    }
};

template <class C>
__device__ __forceinline__ void load_role(const WeightArgs& a, Bars* B, uint32_t ring, int lane) {
    const uint32_t bars = smem_u32(B);
    volatile int* abort = &B->abort;
    Ring<C::ST> r;
    uint32_t begun = 0;                                 // slots with a copy issued
    bool ok = true;
    auto slot = [&](uint32_t& st) {
        uint32_t par;
        r.step(st, par);
        if (!mbar_wait(MLZC_BAR(empty, st), par ^ 1, abort, a.c.err)) {
            r.uses ^= 1u << st;
            return false;
        }
        begun |= 1u << st;
        return true;
    };
    // the page of this lane's box of slot tile t
    auto page_of = [&](const Walk& w, int t) {
        const int j = t * kBN + lane * a.box;
        return lane * a.box < kBN && j < w.s.kv ? paged::load_page(a.c, w.b, a.c.by_page.quot(j)) : -1;
    };
    auto load_k = [&](const Walk& w, int t, int page, uint32_t& taken) {
        const int n = (min(kBN, w.s.kv - t * kBN) + a.box - 1) / a.box;
        const int row = a.c.by_page.rem(t * kBN + lane * a.box);
        // a page whose rows all lie in the tile: its first box's lane fetches them
        const int start = lane * a.box - row;
        const bool inside = a.whole && start >= 0 && start + a.c.page <= kBN, first = inside && row == 0;
        const bool copies = lane < n && (first || !inside);
        const int rows = __popc(__ballot_sync(~0u, copies && first)) * a.c.page + __popc(__ballot_sync(~0u, copies && !first)) * a.box;
        const CUtensorMap* map = first ? &a.mkp : &a.mk;
        const int pg = page < 0 ? a.c.n_pages : page;   // outside the map: zeros
#pragma unroll
        for (int unit = 0; unit < C::UN; ++unit) {
            uint32_t st;
            if (!slot(st)) return false;
            const uint32_t bar = MLZC_BAR(full, st);
            if (lane == 0) mbar_expect_tx(bar, (uint32_t)rows * 128 * C::SUBS);
            __syncwarp();
            if (copies) {
#pragma unroll
                for (int u = 0; u < C::SUBS; ++u)
                    tma_load_4d(ring + st * C::kUnit + u * C::kSub + lane * a.box * 128, map, bar, (unit * C::SUBS + u) * 64, row, w.h, pg);
            }
            taken |= 1u << st;
        }
        return true;
    };
    auto load_q = [&](const Walk& w, int i, uint32_t& taken) {
        const int row = w.s.row0 + w.tok0(a, i);
#pragma unroll
        for (int unit = 0; unit < C::QU; ++unit) {
            uint32_t st;
            if (!slot(st)) return false;
            if (lane == 0) {
                const uint32_t bar = MLZC_BAR(full, st);
                mbar_expect_tx(bar, (uint32_t)a.tq * a.G * 128 * C::SUBS);
                // lo first (see the MMA warp)
                const CUtensorMap* map = C::HL && unit < C::UN ? &a.mql : &a.mq;
#pragma unroll
                for (int u = 0; u < C::SUBS; ++u)
                    tma_load_3d(ring + st * C::kUnit + u * C::kSub, map, bar, ((unit % C::UN) * C::SUBS + u) * 64, w.h * a.G, row);
            }
            taken |= 1u << st;
        }
        return true;
    };
    Walk w(B);
    while (ok && w.next(a)) {
        uint32_t held = 0, passing = 0;
        r.held = 0;
        int page = page_of(w, w.t);
        if (w.wide) {
            if (w.s.rows > 0) ok = load_q(w, 0, held);
            r.held = held;
            for (int it = 0; ok && it < w.n; ++it) {
                const int next = it + 1 < w.n ? page_of(w, w.t + it + 1) : -1;
                ok = load_k(w, w.t + it, page, passing);
                page = next;
            }
        } else {
            ok = load_k(w, w.t, page, held);
            r.held = held;
            for (int it = 0; ok && it < w.n; ++it)
                if (w.cols(a, it) > 0) ok = load_q(w, it, passing);
        }
    }
    if (!ok) {
        // the copies already issued land before this CTA's shared memory goes away
        for (int i = 0; i < C::ST; ++i) {
            const uint64_t t0 = ptx::global_ns();
            while ((begun >> i & 1) && !ptx::mbar_try_wait(MLZC_BAR(full, i), (r.uses >> i & 1) ^ 1) && ptx::global_ns() - t0 < ptx::kWaitNs) {
            }
        }
    }
}

// Minus the lse2 of each query tile's rows; two warps take turns, so that one's loads are under
// way while the other waits.  Of a wide piece the rows are the same for every tile.
__device__ __forceinline__ void lse_role(const WeightArgs& a, Bars* B, float* lse2, int turn, int lane) {
    const uint32_t bars = smem_u32(B);
    volatile int* abort = &B->abort;
    uint32_t g = 0;
    Walk w(B);
    while (w.next(a)) {
        float v[4];
        bool have = false;
        for (int it = 0; it < w.n; ++it, ++g) {
            if ((int)(g & 1) != turn) continue;
            const int buf = g % kBufs;
            if (!w.wide || !have) {
                const int cols = w.cols(a, it), t0 = w.s.row0 + w.tok0(a, it);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = lane + 32 * i;
                    v[i] = c < cols ? ptx::ld_act(reinterpret_cast<const float*>(a.lse + (size_t)(t0 + a.by_g.quot(c)) * a.lse_tok +
                                                                                 (size_t)(w.h * a.G + a.by_g.rem(c)) * a.lse_head))
                                    : -INFINITY;
                    // a row that saw nothing adds nothing
                    v[i] = v[i] == -INFINITY ? -INFINITY : v[i] * -kLog2e;
                }
                have = true;
            }
            if (!mbar_wait(MLZC_BAR(s_empty, buf), ((g / kBufs) & 1) ^ 1, abort, a.c.err)) return;
#pragma unroll
            for (int i = 0; i < 4; ++i) lse2[buf * 128 + lane + 32 * i] = v[i];
            __syncwarp();
            if (lane == 0) mbar_arrive(MLZC_BAR(lse_full, buf));
        }
    }
}

template <class C>
__device__ __forceinline__ void mma_role(const WeightArgs& a, Bars* B, uint32_t ring, uint32_t tmem_base) {
    const uint32_t bars = uniform(smem_u32(B)), ring16 = uniform(ring >> 4), tmem = uniform(tmem_base);
    volatile int* abort = &B->abort;
    Ring<C::ST> r;
    uint32_t g = 0, last_bar = 0, last_par = 0;
    bool ok = true;
    auto take = [&](uint32_t& st) {
        uint32_t par;
        r.step(st, par);
        st = uniform(st);
        if (!mbar_wait(MLZC_BAR(full, st), par, abort, a.c.err)) return false;
        tc_fence_after();
        return true;
    };
    auto commit = [&](uint32_t bar) {
        if (elect_one()) umma_commit(bar);
    };
    auto release = [&](uint32_t st) {
        last_bar = MLZC_BAR(empty, st);
        last_par = (r.uses >> st & 1) ^ 1;
        commit(last_bar);
    };
    // the products of K unit ks and Q unit qs into buffer buf; `add` to what it holds
    auto products = [&](int buf, uint32_t idesc, uint32_t ks, uint32_t qs, bool add) {
        const uint32_t k = desc_lo(ring16 + ks * (C::kUnit >> 4)), q = desc_lo(ring16 + qs * (C::kUnit >> 4)), d = tmem + buf * 128;
        if (elect_one()) {
#pragma unroll
            for (int i = 0; i < C::DU / 16; ++i) {
                const uint32_t o = ((i >> 2) * C::kSub + (i & 3) * 32) >> 4;
                umma_f16_lo(d, k + o, q + o, idesc, add || i > 0);
            }
        }
    };
    // as many columns as there are rows (multiples of 16)
    auto idesc_of = [&](int cols) { return uniform(umma_idesc_f16(128, 0) | ((uint32_t)((cols + 15) / 16 * 16 >> 3) << 17)); };
    Walk w(B);
    while (ok && w.next(a)) {
        uint32_t held = 0;
        r.held = 0;
        if (w.wide) {
            const int cols = w.cols(a, 0);
            const uint32_t idesc = idesc_of(cols);
            uint32_t qs[C::QU];
#pragma unroll
            for (int unit = 0; unit < C::QU; ++unit)
                if (ok && cols > 0) {
                    ok = take(qs[unit]);
                    held |= 1u << qs[unit];
                }
            r.held = held;
            for (int it = 0; ok && it < w.n; ++it, ++g) {
                const int buf = (int)uniform(g % kBufs);
                if (!(ok = mbar_wait(MLZC_BAR(s_empty, buf), ((g / kBufs) & 1) ^ 1, abort, a.c.err))) break;
                tc_fence_after();
#pragma unroll
                for (int unit = 0; unit < C::UN; ++unit) {
                    uint32_t ks;
                    if (ok) ok = take(ks);
                    if (!ok) break;
                    if (cols > 0) {
                        // low products first: the tensor cores' sums are cut, not rounded, at the
                        // sum's own size
#pragma unroll
                        for (int part = 0; part < C::QU / C::UN; ++part) products(buf, idesc, ks, qs[part * C::UN + unit], unit > 0 || part > 0);
                    }
                    release(ks);
                }
                if (!ok) break;
                commit(MLZC_BAR(s_full, buf));
            }
            if (!ok) break;
#pragma unroll
            for (int unit = 0; unit < C::QU; ++unit)
                if (cols > 0) release(qs[unit]);
        } else {
            uint32_t ks[C::UN];
#pragma unroll
            for (int unit = 0; unit < C::UN; ++unit)
                if (ok) {
                    ok = take(ks[unit]);
                    held |= 1u << ks[unit];
                }
            r.held = held;
            for (int it = 0; ok && it < w.n; ++it, ++g) {
                const int buf = (int)uniform(g % kBufs);
                if (!(ok = mbar_wait(MLZC_BAR(s_empty, buf), ((g / kBufs) & 1) ^ 1, abort, a.c.err))) break;
                tc_fence_after();
                const int cols = w.cols(a, it);
                if (cols > 0) {
                    const uint32_t idesc = idesc_of(cols);
#pragma unroll
                    for (int unit = 0; unit < C::QU; ++unit) {
                        uint32_t qs;
                        if (ok) ok = take(qs);
                        if (!ok) break;
                        products(buf, idesc, ks[unit % C::UN], qs, unit > 0);
                        release(qs);
                    }
                    if (!ok) break;
                }
                commit(MLZC_BAR(s_full, buf));
            }
            if (!ok) break;
#pragma unroll
            for (int unit = 0; unit < C::UN; ++unit) release(ks[unit]);
        }
    }
    if (!ok && last_bar && elect_one()) {
        umma_commit(last_bar);
        const uint64_t t0 = ptx::global_ns();
        while (!ptx::mbar_try_wait(last_bar, last_par) && ptx::global_ns() - t0 < ptx::kWaitNs) {
        }
    }
}

// Notes the slot tile that begins in this CTA's share and ends in a later one.
__device__ __forceinline__ void head_role(const WeightArgs& a, Bars* B) {
    int4 hd = make_int4(-1, 0, 0, 0);
    long long at = B->first;
    Walk w(B);
    while (w.next(a)) {
        if (!w.wide && w.tile == 0 && w.n < w.tiles) {
            const long long n = min((long long)a.n_ctas, B->total), end = at + w.tiles;
            hd = make_int4(w.b, w.h, w.t, (int)((end * n - 1) / B->total));
        }
        at += w.n;
    }
    a.head[blockIdx.x] = hd;
}

template <class C>
__global__ void __launch_bounds__(kThreads, 1) weights_kernel(const __grid_constant__ WeightArgs a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t ring = smem_u32(smem);
    uint8_t* fixed = smem + (size_t)C::ST * C::kUnit;
    Bars* B = reinterpret_cast<Bars*>(fixed);
    float* lse2 = reinterpret_cast<float*>(fixed + kBarBytes);
    float* handed = lse2 + kBufs * 128;
    // the loading and issuing warps come first (a scheduler prefers its lower warps)
    const int warp = (int)uniform(threadIdx.x >> 5) - 4, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::ST; ++i) {
            mbar_init(smem_u32(&B->full[i]), 1);
            mbar_init(smem_u32(&B->empty[i]), 1);
        }
        for (int i = 0; i < kBufs; ++i) {
            mbar_init(smem_u32(&B->s_full[i]), 1);
            mbar_init(smem_u32(&B->s_empty[i]), 4);
            mbar_init(smem_u32(&B->lse_full[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&B->hand_full[i]), kEpiWarps - 4);
            mbar_init(smem_u32(&B->hand_empty[i]), 4);
        }
        B->abort = 0;
        ptx::mbar_init_fence();
        tma_prefetch_desc(&a.mk);
        tma_prefetch_desc(&a.mq);
    }
    if (warp == -3) tmem_alloc(smem_u32(&B->tmem), 512);
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    plan(a, B);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = B->tmem;
    if (warp >= 0) {
        sum_role<C>(a, B, lse2, handed, tmem, warp, lane);
    } else if (warp == -4) {
        load_role<C>(a, B, ring, lane);
    } else if (warp == -3) {
        mma_role<C>(a, B, ring, tmem);
    } else {
        lse_role(a, B, lse2, warp + 2, lane);
        if (warp == -1 && lane == 0) head_role(a, B);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == -3) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Block c: the slot tile begun by CTA c and cut, its records added in order.
__global__ void __launch_bounds__(128) merge_kernel(const __grid_constant__ WeightArgs a) {
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    const int c = blockIdx.x, slot = threadIdx.x;
    const int b = paged::ld_int(&a.head[c].x);
    if (b < 0) return;
    const int h = paged::ld_int(&a.head[c].y), t = paged::ld_int(&a.head[c].z), last = paged::ld_int(&a.head[c].w);
    const Seq s = paged::load_seq(a.c, b);
    const int j = t * kBN + slot;
    if (j >= s.kv) return;
    float total = 0.0f;
    for (int i = c; i <= last; ++i) total += ptx::ld_act(&a.rec[((size_t)i * 2 + (i == c ? 1 : 0)) * 128 + slot]);
    const float before = a.acc ? ptx::ld_act(reinterpret_cast<const float*>(a.acc + (size_t)b * a.a_seq + (size_t)h * a.a_head) + j) : 0.0f;
    reinterpret_cast<float*>(a.out + (size_t)b * a.o_seq + (size_t)h * a.o_head)[j] = before + total;
}

// f32 q rows -> f16 hi + lo, dense [token][head][D].  8 values a thread.
__global__ void __launch_bounds__(256) split_kernel(const char* q, size_t q_head, size_t q_tok, int n_head, int per_row, int64_t items,
                                                    uint4* hi, uint4* lo) {
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < items; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / per_row;
        const char* p = q + (size_t)(r / n_head) * q_tok + (size_t)(r % n_head) * q_head + (size_t)(i % per_row) * 32;
        const float4 v0 = ptx::ld_act(reinterpret_cast<const float4*>(p)), v1 = ptx::ld_act(reinterpret_cast<const float4*>(p + 16));
        uint4 x, y;
        ptx::split_h2(v0.x, v0.y, x.x, y.x);
        ptx::split_h2(v0.z, v0.w, x.y, y.y);
        ptx::split_h2(v1.x, v1.y, x.z, y.z);
        ptx::split_h2(v1.z, v1.w, x.w, y.w);
        hi[i] = x;
        lo[i] = y;
    }
}

struct Plan {
    size_t q, rec, total;
};
Plan make_plan(const mlzc_paged_cache* cache, const mlzc_paged_attn_desc* d, int ctas) {
    Plan p{};
    p.q = d->type == MLZC_TYPE_F32 ? (size_t)cache->n_tokens * d->n_head_q * cache->head_dim * 2 : 0;
    p.rec = (size_t)ctas * 2 * 128 * 4;
    p.total = 2 * p.q + p.rec + (size_t)ctas * 16;
    return p;
}

template <class C>
int launch(const WeightArgs& a, const DeviceCtx* c, cudaStream_t s) {
    static bool set[64] = {};
    const int dev = c->device < 64 ? c->device : 63;
    if (!set[dev] || c->device >= 64) {
        MLZC_CUDA_TRY(cudaFuncSetAttribute(weights_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem));
        set[dev] = true;
    }
    MLZC_CUDA_TRY(launch_pdl(weights_kernel<C>, dim3(a.n_ctas), dim3(kThreads), C::kSmem, s, a));
    MLZC_CUDA_TRY(cudaGetLastError());
    count_launch();
    // no sequence can have a second query tile: no slot tile is cut
    if (a.c.n_tokens <= a.tq) return MLZC_OK;
    MLZC_CUDA_TRY(launch_pdl(merge_kernel, dim3(a.n_ctas), dim3(128), 0, s, a));
    MLZC_CUDA_TRY(cudaGetLastError());
    count_launch();
    return MLZC_OK;
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
    const int st = paged::check_attn(cache, d, true);
    if (st != MLZC_OK) return st;
    DeviceCtx* c = current_ctx();
    if (!c) return MLZC_ERR_CUDA;
    *out_bytes = make_plan(cache, d, c->sm_count).total;
    return MLZC_OK;
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
    DeviceCtx* c = current_ctx();
    if (!c) return MLZC_ERR_CUDA;
    const Plan p = make_plan(cache, d, c->sm_count);
    if (!workspace || workspace_bytes < p.total)
        return fail(MLZC_ERR_NOMEM, "paged weights: workspace of %zu bytes needed, %zu given", p.total, workspace_bytes);
    if ((uintptr_t)workspace % 16) return fail(MLZC_ERR_INVALID, "paged weights: workspace not 16-byte aligned");
    WeightArgs a{};
    st = paged::make_view(cache, true, c, &a.c);
    if (st != MLZC_OK) return st;
    char* ws = static_cast<char*>(workspace);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int64_t T = cache->n_tokens, H = d->n_head_q, D = cache->head_dim;
    const bool f32 = d->type == MLZC_TYPE_F32;
    a.G = (int)(H / cache->n_head_kv);
    a.tq = 128 / a.G;
    a.by_tq.set((uint32_t)a.tq);
    a.by_g.set((uint32_t)a.G);
    a.box = std::gcd(cache->page_size, kBN);
    if ((st = paged::encode_pool(&a.mk, cache, false, a.box)) != MLZC_OK) return st;
    a.whole = cache->page_size < kBN && a.box < cache->page_size;
    if (a.whole && (st = paged::encode_pool(&a.mkp, cache, false, cache->page_size)) != MLZC_OK) return st;
    if (T > 0) {
        // checked after every argument: from here on work is issued
        if (f32) {
            if ((st = paged::encode_rows(&a.mq, ws, D, H, T, D * 2, H * D * 2, a.G, a.tq)) != MLZC_OK) return st;
            if ((st = paged::encode_rows(&a.mql, ws + p.q, D, H, T, D * 2, H * D * 2, a.G, a.tq)) != MLZC_OK) return st;
            const int64_t items = T * H * (D / 8);
            const unsigned grid = (unsigned)std::min<int64_t>((items + 255) / 256, (int64_t)c->sm_count * 8);
            MLZC_CUDA_TRY(launch_pdl(split_kernel, dim3(grid), dim3(256), 0, s, static_cast<const char*>(d->q), d->q_nb[1], d->q_nb[2],
                                     (int)H, (int)(D / 8), items, reinterpret_cast<uint4*>(ws), reinterpret_cast<uint4*>(ws + p.q)));
            MLZC_CUDA_TRY(cudaGetLastError());
            count_launch();
        } else if ((st = paged::encode_rows(&a.mq, d->q, D, H, T, d->q_nb[1], d->q_nb[2], a.G, a.tq)) != MLZC_OK) {
            return st;
        }
    } else {
        a.mq = a.mk;   // not read
    }
    a.lse = reinterpret_cast<const char*>(d->lse);
    a.lse_head = d->lse_nb[0]; a.lse_tok = d->lse_nb[1];
    a.acc = reinterpret_cast<const char*>(acc);
    a.out = reinterpret_cast<char*>(out);
    if (acc) { a.a_head = acc_nb[1]; a.a_seq = acc_nb[2]; }
    a.o_head = out_nb[1]; a.o_seq = out_nb[2];
    a.scale = d->scale;
    a.softcap = (d->mode & MLZC_FA_MODE_SOFTCAP) ? d->logit_softcap : 0.0f;
    a.n_ctas = c->sm_count;
    a.rec = reinterpret_cast<float*>(ws + 2 * p.q);
    a.head = reinterpret_cast<int4*>(ws + 2 * p.q + p.rec);
    const bool cap = a.softcap > 0.0f;
#define MLZC_LAUNCH(DIM)                                                                                                \
    return f32 ? (cap ? launch<Cfg<DIM, true, true>>(a, c, s) : launch<Cfg<DIM, true, false>>(a, c, s))                 \
               : (cap ? launch<Cfg<DIM, false, true>>(a, c, s) : launch<Cfg<DIM, false, false>>(a, c, s))
    if (D == 64) MLZC_LAUNCH(64);
    if (D == 128) MLZC_LAUNCH(128);
    MLZC_LAUNCH(256);
#undef MLZC_LAUNCH
}
