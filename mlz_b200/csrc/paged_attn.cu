// paged_attn.cu -- attention of new tokens over a paged KV cache (mlzc_paged_attn_dev) on the
// 5th-generation tensor cores.
//
// One pass over a sequence's slots with the softmax's running maximum and sum:
//   S = Q K^T,  m' = max(m, row max S),  P = 2^(c (S - m')),  l' = a l + row sum P,
//   O' = a O + P V,  a = 2^(c (m - m')),  c = scale * log2 e;  out = O / l, lse = m scale + ln l.
// The query rows of a sequence that share a KV head (its new tokens x the head's G query heads)
// are packed into tiles of up to 128 rows, so K and V are read once for G heads: rows of a
// tile are (token, head in group), tokens outermost.
//
// A CTA walks BN-slot tiles of K and V:
//   loader warp    K and V tiles by TMA into a ring, one box per page piece (box height
//                  gcd(page, BN), so a box never crosses a page, or the page where it lies whole in
//                  the tile: 24 mixed sequences with pages of 24 rows 75 us, 88 without); each lane
//                  looks up its own box's page in the block table and issues its own copies;
//   Q warp         the next piece's Q tile (f16: TMA; f32: split into f16 hi + lo);
//   MMA warp       S = Q K^T (operands in shared memory) and O += P V (P in TMEM, V as an
//                  N-contiguous B operand) with tcgen05.mma, accumulators in TMEM;
//   softmax warps  one thread a row: S from TMEM, P back over it.
// f16 calls (P rounded to f16 once: P V then carries the rounding that the output's type has
// anyway) keep O in TMEM; a softmax thread rescales it only when its row's maximum has risen by
// more than 8 in the exponent (P then stays below 2^8 times its offset), so in the steady state
// no thread touches O.  NS = 2: two query tiles with a softmax warpgroup each share every K and
// V tile, and the tensor cores work on one while the other is in the softmax; for calls with
// more than 128 query rows a sequence.  NS = 1: one tile and two S buffers; for decode (the time
// is that of reading K and V) and for head_dim 256 (whose O takes half of TMEM).
// f32 calls keep f32 precision: Q = Qhi + Qlo and P = Phi + Plo (f16 each, 22 bits), twice the
// products.  The tensor cores' f32 sums drop what lies below an addend's last place, always
// towards zero (measured: 1.4e-8 of the sum a step), so a long sum in TMEM drifts: over 2500
// steps it is off by 4e-5.  Here O therefore sums one slot tile in TMEM, low products first, and
// correction warps add the tiles up in registers, rounding to nearest.  Tiles are independent
// of one another (each has its own maximum and sum), so the softmax keeps no state.
// SPREAD (f32 decode): query tiles of up to 8 rows would leave most of the 128 rows of the products
// idle.  They lie there eight times instead: hi and lo as rows of their own, so that one pass
// gives both parts' scores and both parts' P V, and that four times, each softmax warp taking a
// quarter of the slots (P is 0 in the others); the correction warps add the copies up at the end
// of a piece.
//
// Measured (device times): 4096 new of 16384 slots, 8 KV heads of 4, 128 dims: f16 840-980 us (980-1140
// TFLOP/s, by the clock), f32 1510-1780 (540-640, each product twice); 4096 of 8192, 4 KV heads of 4, 256
// dims: f16 353 us, f32 775-850.  Decode of 64 sequences of 4096 slots: 173 us, 6.2 TB/s, f16 and f32 alike; of 16
// of 512 to 8192: 55 and 57 us (5.3 TB/s); of one: 10 us of latency.
//
// All (sequence, KV head, query tile, slot tile) of a call form one list, of which every CTA
// takes an equal contiguous share (few rows over a long cache and many rows over a short one
// balance alike).  A query tile that a share boundary cuts leaves partial (O, m, l) records in
// the workspace, merged in slot order by the combine launch: results repeat bit for bit.
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstring>
#include <numeric>
#include <type_traits>

#include "paged.h"
#include "paged_records.h"
#include "ptx.cuh"
#include "tcgen05.cuh"

namespace mlzc {
namespace {

using paged::Seq;
using paged::View;
using ptx::mbar_arrive;
using ptx::mbar_expect_tx;
using ptx::mbar_init;
using ptx::smem_u32;
using paged::mbar_wait;
using namespace tc05;

constexpr int kSmemMax = 232448;
constexpr int kBarBytes = 512;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// P carries a factor 2^6: f16 then holds weights down to 2^-20 of the largest at full
// precision, and with the rescaling threshold 2^8 the largest P is 2^14 (f16 ends at 2^16).
constexpr float kPOffset = 6.0f;
constexpr float kRescale = 8.0f;

struct AttnArgs {
    View c;
    CUtensorMap mk, mv, mq, mkp, mvp;   // pools in boxes of `box` rows, of a page (where `whole`)
    const char* q;
    char* dst;
    char* lse;
    size_t q_head, q_tok, d_head, d_tok, lse_head, lse_tok;
    int G, tq;                 // query heads a KV head; tokens a tile (tq * G <= 128)
    paged::Div by_g;
    int box;                   // rows of a K / V box
    int whole;                 // pages that lie whole in a tile come as one box
    float scale, softcap;      // softcap 0: none
    int n_ctas, rec_rows;
    float* rec;                // [cta][2][rec_rows][D]: 0 continues a cut tile, 1 begins one (paged_records.h)
    float2* ml;                // [cta][2][rec_rows]: exponent of the record's scale, sum
    int4* head;                // [cta]: of the query tile begun in record 1, packed row, tokens, kv head, last CTA (-1: none)
};

constexpr int BN = 128;        // slots a tile

template <int D_, int NS_, bool HL_, bool CAP_, bool SPREAD_ = false>
struct Cfg {
    static constexpr int D = D_, NS = NS_;
    static constexpr bool HL = HL_, CAP = CAP_;           // f32 queries (hi + lo); scores are capped
    // dims of a ring unit (a K or V tile is UN units); beside f32 queries of 256 dims (128 KB)
    // half units leave a ring of five
    static constexpr int DU = D == 64 || (HL && D == 256) ? 64 : 128;
    static constexpr int UN = D / DU;
    static constexpr int SUBS = DU / 64;
    static constexpr uint32_t kQSub = 128 * 128;          // bytes of a 64-value block of a Q tile
    static constexpr uint32_t kQTile = kQSub * (D / 64);
    static constexpr uint32_t kQBytes = kQTile * NS * (HL ? 2 : 1);   // [tile][hi, lo]
    static constexpr uint32_t kSub = BN * 128;            // bytes of a 64-value block of a unit
    static constexpr uint32_t kUnit = kSub * SUBS;
    static constexpr bool kSpread = SPREAD_;              // up to 8 rows lie eight times
    static constexpr int kPitch = D + 4;                  // floats of a staged row of O
    static constexpr uint32_t kStage = 4 * 8 * (kPitch + 2) * 4;
    static constexpr uint32_t kStats = HL ? 4 * 128 * 8 + (kSpread ? kStage : 0) : 0;
    static constexpr int kFit = (kSmemMax - 1024 - kBarBytes - (int)kStats - (int)kQBytes) / (int)kUnit;
    static constexpr int ST = kFit > 8 ? 8 : kFit;
    static constexpr size_t kSmem = 1024 + kBarBytes + kStats + kQBytes + (size_t)ST * kUnit;
    // warps: four that load and issue, softmax (f32 calls of 64 dims are bound by it: two
    // warpgroups take turns at the tiles), correction (f32; 128 dims a thread at most)
    static constexpr int kSoftWarps = 4 * (HL ? (D == 64 ? 2 : 1) : NS);
    static constexpr int CD = D < 128 ? D : 128;          // dims of a correction thread
    static constexpr int kCorrWarps = HL ? 4 * (D / CD) : 0;
    static constexpr int kThreads = (4 + kSoftWarps + kCorrWarps) * 32;
    // Measured on 4096 tokens of 16384 slots (8 KV heads of 4, f16):
    // steps of S a tile with two query tiles: 64 dims 673 us with two, 728 with one (a step's
    // products run beside the other's softmax); 128 dims 1027 with two (products of 64 columns
    // read Q twice as often), 855 with one
    static constexpr int H = NS == 2 && D == 64 ? 2 : 1;
    // one in so many pairs of exponentials on the FMA pipe (0: none): 128 dims 855 us with 4, 947
    // with none; 64 dims 712 and 673; 256 dims, where the products are the bound, 370 and 353
    static constexpr int kPoly = NS == 2 && D == 128 ? 4 : 0;
    static constexpr uint32_t kSCol = 0;                  // S of tile / buffer i at i * BN
    static constexpr uint32_t kOCol = 2 * BN;             // O of tile i at + i * D
    static_assert(2 * BN + NS * D <= 512, "TMEM");
    static_assert(ST >= 3, "ring");
    static_assert(!HL || NS == 1, "f32 calls take one query tile");
    static_assert(!kSpread || (HL && D <= 128), "one correction warpgroup");
};

// Barriers in shared memory.
struct Bars {
    uint64_t full[8], empty[8], q_full, q_empty, s_full[4], p_full[4], o_step[2], o_done[2], o_empty[2], stat_full[4], copies;
    uint32_t tmem;
    int abort;
    long long first, count, total;   // this CTA's share of the list; its start's place
    int b, h, t, at;
    long long scan[16];
};
static_assert(sizeof(Bars) <= kBarBytes, "barriers");

// Slots that query tile t of a sequence sees, and its slot tiles (one at least, so that rows
// which see nothing are written too).
__device__ __forceinline__ int visible(const Seq& s, int t, int tokens) {
    const int64_t e = (int64_t)(t + 1) * tokens;
    return max(0, s.kv - s.rows + (int)(e < s.rows ? e : s.rows));
}
__device__ __forceinline__ int tiles_of(const Seq& s, int t, int tokens) {
    return max(1, (visible(s, t, tokens) + BN - 1) / BN);
}

// What a query tile costs beside its slot tiles (its Q, filling and draining the pipeline), in slot
// tiles.  The list counts it in front of the tiles, so that CTAs with many short query tiles get
// fewer slot tiles (24 mixed sequences, 64 dims f32, before later steps: 127 us with 0, 90 with 2 to
// 4, 101 with 8).
constexpr int kStart = 3;

// A walk over this CTA's share: piece after piece (the tiles of one query tile).
template <class C>
struct Walk {
    int b, h, t, tile, n;      // the piece: slot tiles [tile, tile + n)
    int all;                   // of so many
    int at;                    // place in the query tile's part of the list
    long long left;
    Seq s;
    bool first;
    __device__ Walk(const Bars* B) : b(B->b), h(B->h), t(B->t), tile(0), n(0), all(0), at(B->at), left(B->count), first(true) {}
    // Moves to the next piece; false at the end.
    __device__ bool next(const AttnArgs& a) {
        const int tokens = a.tq * C::NS;
        do {
            if (left <= 0) return false;
            if (first) {
                s = paged::load_seq(a.c, b);
                first = false;
            } else {
                at = 0;
                if ((int64_t)(++t) * tokens >= s.rows) {
                    t = 0;
                    if (++h == a.c.n_head_kv) {
                        h = 0;
                        do {
                            s = paged::load_seq(a.c, ++b);
                        } while (s.rows == 0);   // the list ends at a sequence with rows
                    }
                }
            }
            all = tiles_of(s, t, tokens);
            const int to = (int)min((long long)(all + kStart), at + left);
            left -= to - at;
            tile = max(0, at - kStart);
            n = max(0, to - kStart) - tile;
        } while (n == 0);                        // no more than its start
        return true;
    }
    __device__ int tok0(const AttnArgs& a) const { return t * a.tq * C::NS; }
    __device__ int tiles(const AttnArgs& a) const { return C::NS == 2 && tok0(a) + a.tq < s.rows ? 2 : 1; }
    // Rows of the piece's (first) query tile, and whether they lie eight times in it: row r of
    // copy c at 32 c + r (hi) and 32 c + 16 + r (lo).
    __device__ int rows(const AttnArgs& a) const { return min(a.tq, s.rows - tok0(a)) * a.G; }
    __device__ bool spread(const AttnArgs& a) const { return C::kSpread && rows(a) <= 8; }
    __device__ bool ends() const { return tile + n == all; }
};

// Finds this CTA's share.  Threads own runs of sequences: their tile counts are summed over the
// block, then the owner of the share's first tile walks to it.
template <class C>
__device__ void plan(const AttnArgs& a, Bars* B) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (a.c.batch + C::kThreads - 1) / C::kThreads;
    const int b0 = tid * per, b1 = min(b0 + per, a.c.batch);
    const int tokens = a.tq * C::NS;
    long long mine = 0;
    for (int b = b0; b < b1; ++b) {
        const Seq s = paged::load_seq(a.c, b);
        long long one = 0;
        for (int t = 0; (int64_t)t * tokens < s.rows; ++t) one += tiles_of(s, t, tokens) + kStart;
        mine += one * a.c.n_head_kv;
    }
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) B->scan[warp] = upto;
    __syncthreads();
    long long total = 0;
    for (int w = 0; w < C::kThreads / 32; ++w) {
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
            long long one = 0;
            for (int t = 0; (int64_t)t * tokens < s.rows; ++t) one += tiles_of(s, t, tokens) + kStart;
            if (r >= one * a.c.n_head_kv) { r -= one * a.c.n_head_kv; continue; }
            B->b = b;
            B->h = (int)(r / one);
            r %= one;
            int t = 0;
            while (r >= tiles_of(s, t, tokens) + kStart) r -= tiles_of(s, t++, tokens) + kStart;
            B->t = t;
            B->at = (int)r;
            break;
        }
    }
    __syncthreads();
}

// 32 accumulator columns to a dst row (f16 or f32) or a record row.
__device__ __forceinline__ void put32(float* p, const float (&x)[32]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<float4*>(p)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
}
__device__ __forceinline__ void put32(__half* p, const float (&x)[32]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        reinterpret_cast<uint4*>(p)[i] = make_uint4(ptx::pack_h2(x[8 * i], x[8 * i + 1]), ptx::pack_h2(x[8 * i + 2], x[8 * i + 3]),
                                                    ptx::pack_h2(x[8 * i + 4], x[8 * i + 5]), ptx::pack_h2(x[8 * i + 6], x[8 * i + 7]));
}

// A query row's place: thread `row` of a query tile.
struct Row {
    int row, tok_of, head_of;            // token and head in the tile
    __device__ Row(const AttnArgs& a, int r) : row(r), tok_of(a.by_g.quot(r)), head_of(a.by_g.rem(r)) {}
    template <class C>
    __device__ int tok(const AttnArgs& a, const Walk<C>& w, int slot) const { return w.tok0(a) + slot * a.tq + tok_of; }
    template <class C>
    __device__ bool real(const AttnArgs& a, const Walk<C>& w, int slot) const {
        return row < a.tq * a.G && tok(a, w, slot) < w.s.rows;
    }
};

template <int N>
__device__ __forceinline__ float row_max(const float (&x)[N]) {
    float m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = max3(x[3 * i], x[3 * i + 1], x[3 * i + 2]);
#pragma unroll
    for (int i = 12; i + 1 < N; i += 2) m[(i >> 1) & 3] = max3(m[(i >> 1) & 3], x[i], x[i + 1]);
    return fmaxf(max3(m[0], m[1], m[2]), m[3]);
}

// Where a piece's rows go: dst and lse when it is the whole query tile, else a record.
template <class C>
struct Sink {
    bool whole;
    int t, h;
    size_t r;
    __device__ Sink(const AttnArgs& a, const Walk<C>& w, const Row& q, int slot) {
        whole = w.tile == 0 && w.ends();
        t = w.s.row0 + q.tok(a, w, slot);
        h = w.h * a.G + q.head_of;
        r = ((size_t)blockIdx.x * 2 + (w.tile == 0 ? 1 : 0)) * a.rec_rows + paged::record_row(slot, q.row, a.tq, a.G);
    }
    // the row's sum: of 2^(...) = 2^e2 * l
    __device__ void sums(const AttnArgs& a, float e2, float l) const {
        if (!whole)
            a.ml[r] = make_float2(e2, l);
        else if (a.lse)
            *reinterpret_cast<float*>(a.lse + (size_t)t * a.lse_tok + (size_t)h * a.lse_head) = l > 0.0f ? (e2 + log2f(l)) * kLn2 : -INFINITY;
    }
    // dims i .. i + 31 of O
    __device__ void put(const AttnArgs& a, int i, float (&o)[32], float inv) const {
        using Out = typename std::conditional<C::HL, float, __half>::type;
        if (whole) {
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] *= inv;
            put32(reinterpret_cast<Out*>(a.dst + (size_t)t * a.d_tok + (size_t)h * a.d_head) + i, o);
        } else {
            put32(a.rec + r * C::D + i, o);
        }
    }
};

// P = 2^(c2 x + off) of N scores, rounded to f16, back over them (32 scores a column pair block:
// their first 16 columns); returns the sum.
template <int POLY, int N>
__device__ __forceinline__ float weigh(const float (&x)[N], float c2, float off, uint32_t s_col) {
    const uint64_t c22 = pair(c2, c2), off2 = pair(off, off);
    uint64_t sum[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < N / 32; ++i) {
        uint32_t p[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const uint64_t y = fma2(pair(x[i * 32 + 2 * j], x[i * 32 + 2 * j + 1]), c22, off2);
            float p0, p1;
            if (POLY && j % (POLY ? POLY : 1) == POLY - 1) {
                exp2_poly(y, p0, p1);
            } else {
                unpair(y, p0, p1);
                p0 = ex2(p0);
                p1 = ex2(p1);
            }
            sum[j & 1] = add2(sum[j & 1], pair(p0, p1));
            p[j] = ptx::pack_h2(p0, p1);
        }
        tmem_st16(s_col + i * 32, p);
    }
    float s0, s1;
    unpair(add2(sum[0], sum[1]), s0, s1);
    return s0 + s1;
}

// f(i, 32 scores from column i on) for N scores at s_col, the next ones under way: a short loop,
// because code unrolled over a row outgrows the instruction cache (4096 of 16384, 128 dims f32:
// 1781 us for 1649; 1024 of 2048 capped, 256 dims: 233 for 113), with one copy of its body
// (two, to save the moves: 122).
template <int N, typename F>
__device__ __forceinline__ void each32(uint32_t s_col, F f) {
    float x[32], v[32];
    tmem_ld32(s_col, *reinterpret_cast<uint32_t(*)[32]>(x));
#pragma unroll 1
    for (int i = 0; i < N; i += 32) {
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = x[j];
        if (i + 32 < N) tmem_ld32(s_col + i + 32, *reinterpret_cast<uint32_t(*)[32]>(x));
        f(i, v);
    }
}

// A row's scores s go into P = 2^(c2 s + off), off = kPOffset - c2 m with their maximum m: one rounding
// a row and one a score.  The first is half a last place of c2 m: far from 0 it would move P by more
// than a few powers of two, until P and its sum leave their types.  There m is taken from the scores first.
constexpr float kFar = 0x1p22f;
__device__ __forceinline__ float offset(float m, float c2) { return m == -INFINITY ? 0.0f : kPOffset - m * c2; }
__device__ __forceinline__ bool is_far(float off) { return fabsf(off) > kFar; }

// N scores at s_col less the maximum m of a far row, back in place; the row's offset then.
template <int N>
__device__ __forceinline__ float shift_row(uint32_t s_col, float m, float off) {
    const float shift = is_far(off) ? m : 0.0f;
#pragma unroll 1
    for (int i = 0; i < N; i += 16) {
        float v[16];
        tmem_ld16(s_col + i, *reinterpret_cast<uint32_t(*)[16]>(v));
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] -= shift;
        tmem_st16(s_col + i, *reinterpret_cast<uint32_t(*)[16]>(v));
    }
    tmem_st_wait();
    return is_far(off) ? kPOffset : off;
}

// N scores at s_col capped, those past `limit` masked where `cut`, back in place; the largest.
template <int N>
__device__ __forceinline__ float cap_row(uint32_t s_col, float cap_in, float cap, bool cut, int limit) {
    float top = -INFINITY;
    each32<N>(s_col, [&](int i, float (&v)[32]) {
        cap_scores(v, cap_in, cap);
        if (cut) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = i + j > limit ? -INFINITY : v[j];
        }
        tmem_st16(s_col + i, *reinterpret_cast<uint32_t(*)[16]>(v));
        tmem_st16(s_col + i + 16, *reinterpret_cast<uint32_t(*)[16]>(v + 16));
        top = fmaxf(top, row_max(v));
    });
    tmem_st_wait();
    return top;
}

// Softmax of an f16 call, step by step (a tile, or half of one: Cfg::H).
template <class C>
__device__ __forceinline__ void softmax_role(const AttnArgs& a, Bars* B, uint32_t tmem, int warp, int lane) {
    constexpr int D = C::D, H = C::H, N = BN / H;        // steps a tile, scores a step
    const int slot = C::NS == 2 ? warp >> 2 : 0;         // query tile of this warpgroup
    const Row q(a, (warp & 3) * 32 + lane);
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t o_col = lanes + C::kOCol + slot * D;
    const float c2 = C::CAP ? kLog2e : a.scale * kLog2e;
    const float cap_in = C::CAP ? a.scale / a.softcap : 0.0f;
    const float rise = kRescale / c2;
    volatile int* abort = &B->abort;
    uint32_t g = 0, piece = 0;                           // steps, pieces
    Walk<C> w(B);
    while (w.next(a)) {
        if (slot >= w.tiles(a)) continue;
        const bool real = q.real(a, w, slot), busy = __any_sync(~0u, real);
        const int own = w.s.kv - w.s.rows + q.tok(a, w, slot);   // last slot this row sees
        float m = -INFINITY, l = 0.0f;
        float off = 0.0f;                                // of m
        for (int it = 0; it < w.n * H; ++it, ++g) {
            // barriers 2 * query tile + half, or the buffer; either way one phase in two steps
            const int buf = C::NS == 1 ? (int)(g & 1) : (H == 2 ? 2 * slot + (int)(g & 1) : slot);
            if (!mbar_wait(smem_u32(&B->s_full[buf]), (C::NS == 1 || H == 2 ? g >> 1 : g) & 1, abort, a.c.err)) return;
            tc_fence_after();
            if (busy) {
                const uint32_t s_col = lanes + C::kSCol + buf * N;
                const int limit = own - w.tile * BN - it * N;
                const bool cut = __any_sync(~0u, limit < N - 1);
                bool far = false;                        // some row of the warp is
                // the running maximum with a step's; O follows where it rises far (far rows come
                // by every time: a vote of their own cost 64 dims 3 %)
                auto raise = [&](float top) {
                    if (it == 0) {
                        m = top;
                        off = offset(m, c2);
                        far = __any_sync(~0u, is_far(off));
                    } else if (__any_sync(~0u, top - m > rise || is_far(off))) {
                        const float to = top - m > rise ? top : m;
                        const float al = m == -INFINITY ? 0.0f : ex2((m - to) * c2);
                        m = to;
                        l *= al;
                        off = offset(m, c2);
                        far = __any_sync(~0u, is_far(off));
                        // O has the products of the steps before the last (this S came after
                        // them); wait for the last's
                        if (!mbar_wait(smem_u32(&B->o_step[slot]), (g - 1) & 1, abort, a.c.err)) return false;
                        tc_fence_after();
#pragma unroll 1
                        for (int i = 0; i < D; i += 16) {
                            uint32_t o[16];
                            tmem_ld16(o_col + i, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * al);
                            tmem_st16(o_col + i, o);
                        }
                    }
                    return true;
                };
                if constexpr (C::CAP) {
                    const float top = cap_row<N>(s_col, cap_in, a.softcap, cut, limit);
                    if (!raise(top)) return;
                    const float add = far ? shift_row<N>(s_col, m, off) : off;
                    each32<N>(s_col, [&](int i, float (&v)[32]) { l += weigh<C::kPoly>(v, c2, add, s_col + i); });
                } else {
                    float x[N];
#pragma unroll
                    for (int i = 0; i < N / 32; ++i)
                        tmem_ld32(s_col + i * 32, *reinterpret_cast<uint32_t(*)[32]>(reinterpret_cast<uint32_t*>(x) + i * 32));
                    tmem_ld_wait();
                    if (cut) {
#pragma unroll
                        for (int i = 0; i < N; ++i) x[i] = i > limit ? -INFINITY : x[i];
                    }
                    if (!raise(row_max(x))) return;
                    float add = off;
                    if (far) {
                        const float shift = is_far(off) ? m : 0.0f;
                        const uint64_t sh = pair(-shift, -shift);
#pragma unroll
                        for (int i = 0; i < N; i += 2) unpair(add2(pair(x[i], x[i + 1]), sh), x[i], x[i + 1]);
                        add = is_far(off) ? kPOffset : off;
                    }
                    l += weigh<C::kPoly>(x, c2, add, s_col);
                }
                tmem_st_wait();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&B->p_full[buf]));
        }
        // the piece's O
        if (!mbar_wait(smem_u32(&B->o_done[slot]), piece & 1, abort, a.c.err)) return;
        tc_fence_after();
        if (busy) {
            const Sink<C> sink(a, w, q, slot);
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            if (real) sink.sums(a, m == -INFINITY ? -INFINITY : m * c2 - kPOffset, l);
#pragma unroll 1
            for (int i = 0; i < D; i += 32) {
                float o[32];
                tmem_ld32(o_col + i, *reinterpret_cast<uint32_t(*)[32]>(o));
                tmem_ld_wait();
                if (real) sink.put(a, i, o, inv);
            }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&B->o_empty[slot]));
        ++piece;
    }
}

// Softmax of an f32 call: a tile's rows by themselves.  Phi of 32 slots goes to the first 16
// columns of their scores, Plo to the other 16; (exponent of the row's scale, sum) to stats.
template <class C>
__device__ __forceinline__ void softmax_tile_role(const AttnArgs& a, Bars* B, float2* stats, uint32_t tmem, int warp, int lane) {
    constexpr int kTurns = C::kSoftWarps / 4;
    const int turn = warp >> 2;
    const int row = (warp & 3) * 32 + lane;              // of the products
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const float c2 = C::CAP ? kLog2e : a.scale * kLog2e;
    const float cap_in = C::CAP ? a.scale / a.softcap : 0.0f;
    volatile int* abort = &B->abort;
    uint32_t g = 0;
    Walk<C> w(B);
    while (w.next(a)) {
        const bool spread = w.spread(a);
        const Row q(a, spread ? lane & 15 : row);
        const bool busy = __any_sync(~0u, q.real(a, w, 0));
        const int own = w.s.kv - w.s.rows + q.tok(a, w, 0);
        for (int it = 0; it < w.n; ++it, ++g) {
            if (kTurns == 2 && (int)(g & 1) != turn) continue;
            const int buf = g & 1;
            if (!mbar_wait(smem_u32(&B->s_full[buf]), (g >> 1) & 1, abort, a.c.err)) return;
            tc_fence_after();
            if (busy) {
                const uint32_t s_col = lanes + C::kSCol + buf * BN;
                const int limit = own - (w.tile + it) * BN;
                const bool cut = __any_sync(~0u, limit < BN - 1);
                const uint64_t c22 = pair(c2, c2);
                uint64_t sum[2] = {0, 0};
                float m;
                auto clip = [&](float x, int i) { return i > limit ? -INFINITY : x; };
                if (C::kSpread && spread) {
                    // this warp's quarter of the slots; lane and lane ^ 16 have the parts of a score
                    const int c0 = (warp & 3) * 32;
                    float x[32];
                    tmem_ld32(s_col + c0, *reinterpret_cast<uint32_t(*)[32]>(x));
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) x[i] += __shfl_xor_sync(~0u, x[i], 16);
                    if (C::CAP) cap_scores(x, cap_in, a.softcap);
                    if (cut) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] = clip(x[i], c0 + i);
                    }
                    m = row_max(x);
                    float off = offset(m, c2);
                    if (__any_sync(~0u, is_far(off))) {
                        const float shift = is_far(off) ? m : 0.0f;
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] -= shift;
                        off = is_far(off) ? kPOffset : off;
                    }
                    uint32_t p[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        float p0, p1;
                        unpair(fma2(pair(x[2 * j], x[2 * j + 1]), c22, pair(off, off)), p0, p1);
                        p0 = ex2(p0);
                        p1 = ex2(p1);
                        sum[j & 1] = add2(sum[j & 1], pair(p0, p1));
                        const float h0 = __uint_as_float(__float_as_uint(p0) & 0xFFFFE000u), h1 = __uint_as_float(__float_as_uint(p1) & 0xFFFFE000u);
                        p[j] = lane < 16 ? ptx::pack_h2(h0, h1) : ptx::pack_h2(p0 - h0, p1 - h1);
                    }
                    tmem_st16(s_col + c0, p);
                    const uint32_t zero[16] = {};
#pragma unroll
                    for (int i = 0; i < BN; i += 32)
                        if (i != c0) tmem_st16(s_col + i, zero);
                } else {
                    // short loops, the scores read twice from TMEM (see each32)
                    m = -INFINITY;
                    if constexpr (C::CAP) {
                        m = cap_row<BN>(s_col, cap_in, a.softcap, cut, limit);
                    } else {
#pragma unroll 1
                        for (int i = 0; i < BN; i += 32) {
                            float v[32];
                            tmem_ld32(s_col + i, *reinterpret_cast<uint32_t(*)[32]>(v));
                            tmem_ld_wait();
                            if (cut) {
#pragma unroll
                                for (int j = 0; j < 32; ++j) v[j] = clip(v[j], i + j);
                                tmem_st16(s_col + i, *reinterpret_cast<uint32_t(*)[16]>(v));
                                tmem_st16(s_col + i + 16, *reinterpret_cast<uint32_t(*)[16]>(v + 16));
                            }
                            m = fmaxf(m, row_max(v));
                        }
                        if (cut) tmem_st_wait();
                    }
                    float x[16];                         // (under way during the vote: 256 dims 775 us for 800)
                    tmem_ld16(s_col, *reinterpret_cast<uint32_t(*)[16]>(x));
                    float off = offset(m, c2);
                    if (__any_sync(~0u, is_far(off))) {
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 16; ++j) asm volatile("" ::"f"(x[j]));   // until here the load's
                        off = shift_row<BN>(s_col, m, off);
                        tmem_ld16(s_col, *reinterpret_cast<uint32_t(*)[16]>(x));
                    }
                    tmem_ld_wait();
#pragma unroll 1
                    for (int i = 0; i < BN; i += 16) {
                        uint64_t y[8];
                        uint32_t hi[8], lo[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) y[j] = fma2(pair(x[2 * j], x[2 * j + 1]), c22, pair(off, off));
                        if (i + 16 < BN) tmem_ld16(s_col + i + 16, *reinterpret_cast<uint32_t(*)[16]>(x));
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            float p0, p1;
                            unpair(y[j], p0, p1);
                            p0 = ex2(p0);
                            p1 = ex2(p1);
                            const uint64_t p = pair(p0, p1);
                            sum[j & 1] = add2(sum[j & 1], p);
                            // hi: the first 11 bits (f16 holds them), lo: the rest, within 2^-22
                            const float h0 = __uint_as_float(__float_as_uint(p0) & 0xFFFFE000u);
                            const float h1 = __uint_as_float(__float_as_uint(p1) & 0xFFFFE000u);
                            hi[j] = ptx::pack_h2(h0, h1);
                            unpair(fma2(pair(h0, h1), pair(-1.0f, -1.0f), p), p0, p1);
                            lo[j] = ptx::pack_h2(p0, p1);
                        }
                        tmem_ld_wait();                  // lo lies over the scores just fetched
                        const uint32_t to = s_col + (i & ~31) + (i >> 1 & 15);
                        tmem_st8(to, hi);
                        tmem_st8(to + 16, lo);
                    }
                }
                float s0, s1;
                unpair(add2(sum[0], sum[1]), s0, s1);
                // (of a row that lies as hi and lo the hi lane has the sum)
                stats[(g & 3) * 128 + row] = make_float2(m == -INFINITY ? -INFINITY : m * c2 - kPOffset, spread && lane >= 16 ? 0.0f : s0 + s1);
                tmem_st_wait();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(smem_u32(&B->p_full[buf]));
                mbar_arrive(smem_u32(&B->stat_full[g & 3]));
            }
        }
    }
}

// Adds up the tiles of an f32 call: O += 2^(e - E) O_tile, rounded to nearest, with E the
// largest exponent so far (raised, and O rescaled, when a tile's lies more than 8 above it).
// stats has four places: the softmax fills that of tile g + 4 only after tile g + 1 was read.
template <class C>
__device__ __forceinline__ void correct_role(const AttnArgs& a, Bars* B, float2* stats, uint32_t tmem, int warp, int lane) {
    constexpr int CD = C::CD;
    const int part = (warp - C::kSoftWarps) >> 2;        // dims [part * CD, + CD)
    const int row = (warp & 3) * 32 + lane;              // of the products
    float* stage = reinterpret_cast<float*>(stats + 4 * 128);
    const uint32_t o_col = tmem + ((uint32_t)((warp & 3) * 32) << 16) + C::kOCol + part * CD;
    volatile int* abort = &B->abort;
    uint32_t g = 0, merges = 0;
    Walk<C> w(B);
    while (w.next(a)) {
        const bool spread = w.spread(a);
        const Row q(a, spread ? lane & 15 : row);
        const bool real = q.real(a, w, 0), busy = __any_sync(~0u, real);
        float o[CD], e = -INFINITY, l = 0.0f;
#pragma unroll
        for (int i = 0; i < CD; ++i) o[i] = 0.0f;
        for (int it = 0; it < w.n; ++it, ++g) {
            if (!mbar_wait(smem_u32(&B->stat_full[g & 3]), (g >> 2) & 1, abort, a.c.err)) return;
            float2 st = make_float2(-INFINITY, 0.0f);
            if (busy) st = stats[(g & 3) * 128 + row];
            if (!mbar_wait(smem_u32(&B->o_done[0]), g & 1, abort, a.c.err)) return;
            tc_fence_after();
            if (busy) {
                if (__any_sync(~0u, st.x > e + kRescale)) {
                    const float to = st.x > e + kRescale ? st.x : e;
                    const float f = e == -INFINITY ? 0.0f : ex2(e - to);
                    e = to;
                    l *= f;
#pragma unroll
                    for (int i = 0; i < CD; ++i) o[i] *= f;
                }
                const float f = st.x == -INFINITY ? 0.0f : ex2(st.x - e);
                l = fmaf(st.y, f, l);
#pragma unroll
                for (int i = 0; i < CD; i += 32) {
                    uint32_t r[32];
                    tmem_ld32(o_col + i, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[i + j] = fmaf(__uint_as_float(r[j]), f, o[i + j]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&B->o_empty[0]));
        }
        if (C::kSpread && spread) {
            // hi and lo, then the four copies through shared memory, a thread a few dims of a row
            auto meet = [&]() {
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&B->copies));
                return mbar_wait(smem_u32(&B->copies), merges++ & 1, abort, a.c.err);
            };
            float2* scale = reinterpret_cast<float2*>(stage + 32 * C::kPitch);
#pragma unroll
            for (int i = 0; i < CD; ++i) o[i] += __shfl_xor_sync(~0u, o[i], 16);
            if (lane < 8) {
                const int at = (warp & 3) * 8 + lane;
                scale[at] = make_float2(e, l);
#pragma unroll
                for (int i = 0; i < CD; i += 4)
                    *reinterpret_cast<float4*>(stage + at * C::kPitch + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            }
            if (!meet()) return;
            constexpr int N = CD / 16;
            const Row r(a, row >> 4);
            if (r.real(a, w, 0)) {
                float2 c[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) c[i] = scale[i * 8 + r.row];
                const float top = fmaxf(fmaxf(c[0].x, c[1].x), fmaxf(c[2].x, c[3].x));
                float x[N] = {}, sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float f = c[i].x == -INFINITY ? 0.0f : ex2(c[i].x - top);
                    sum = fmaf(f, c[i].y, sum);
                    const float* p = stage + (i * 8 + r.row) * C::kPitch + (row & 15) * N;
#pragma unroll
                    for (int j = 0; j < N; ++j) x[j] = fmaf(f, p[j], x[j]);
                }
                const Sink<C> sink(a, w, r, 0);
                if ((row & 15) == 0) sink.sums(a, top, sum);
                const float inv = sink.whole ? (sum > 0.0f ? 1.0f / sum : 0.0f) : 1.0f;
                float* to = (sink.whole ? reinterpret_cast<float*>(a.dst + (size_t)sink.t * a.d_tok + (size_t)sink.h * a.d_head)
                                        : a.rec + sink.r * C::D) + (row & 15) * N;
#pragma unroll
                for (int j = 0; j < N; j += 4)
                    *reinterpret_cast<float4*>(to + j) = make_float4(x[j] * inv, x[j + 1] * inv, x[j + 2] * inv, x[j + 3] * inv);
            }
            if (!meet()) return;                         // the staging place is free again
            continue;
        }
        if (real) {
            const Sink<C> sink(a, w, q, 0);
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            if (part == 0) sink.sums(a, e, l);
#pragma unroll
            for (int i = 0; i < CD; i += 32) sink.put(a, part * CD + i, *reinterpret_cast<float(*)[32]>(o + i), inv);
        }
    }
}

// Slots of tile `i` that some row of the piece sees.
template <class C>
__device__ __forceinline__ int tile_rows(const AttnArgs& a, const Walk<C>& w, int i) {
    return min(BN, max(0, visible(w.s, w.t, a.tq * C::NS) - i * BN));
}

template <class C>
__device__ __forceinline__ void load_role(const AttnArgs& a, Bars* B, uint32_t ring, int lane) {
    volatile int* abort = &B->abort;
    const int boxes = BN / a.box;             // <= 16
    uint32_t at = 0;
    bool ok = true;
    // the page of box `lane` of slot tile i
    auto page_of = [&](const Walk<C>& w, int i) {
        const int j = i * BN + lane * a.box;
        return lane < boxes && lane * a.box < tile_rows(a, w, i) ? paged::load_page(a.c, w.b, a.c.by_page.quot(j)) : -1;
    };
    auto load = [&](const Walk<C>& w, int i, int page, const CUtensorMap* map, const CUtensorMap* map_whole) {
        const int n = (tile_rows(a, w, i) + a.box - 1) / a.box;
        const int row = a.c.by_page.rem(i * BN + lane * a.box);
        // a page whose rows all lie in the tile: its first box's lane fetches them
        const int start = lane * a.box - row;
        const bool inside = a.whole && start >= 0 && start + a.c.page <= BN, first = inside && row == 0;
        const bool copies = lane < n && (first || !inside);
        const int rows = __popc(__ballot_sync(~0u, copies && first)) * a.c.page + __popc(__ballot_sync(~0u, copies && !first)) * a.box;
        if (first) map = map_whole;
        // a page outside the pools is a coordinate outside the map, which reads as zeros
        const int pg = page < 0 ? a.c.n_pages : page;
#pragma unroll
        for (int unit = 0; unit < C::UN; ++unit, ++at) {
            const uint32_t st = at % C::ST;
            if (!mbar_wait(smem_u32(&B->empty[st]), ((at / C::ST) & 1) ^ 1, abort, a.c.err)) return false;
            const uint32_t bar = smem_u32(&B->full[st]);
            if (lane == 0) {
                if (n) mbar_expect_tx(bar, (uint32_t)rows * 128 * C::SUBS);
                else mbar_arrive(bar);
            }
            __syncwarp();
            if (copies) {
#pragma unroll
                for (int u = 0; u < C::SUBS; ++u)
                    tma_load_4d(ring + st * C::kUnit + u * C::kSub + lane * a.box * 128, map, bar, (unit * C::SUBS + u) * 64, row, w.h, pg);
            }
        }
        return true;
    };
    Walk<C> w(B);
    while (ok && w.next(a)) {
        int cur = page_of(w, w.tile), nxt = -1;
        ok = load(w, w.tile, cur, &a.mk, &a.mkp);
        for (int it = 0; ok && it < w.n; ++it) {
            const int i = w.tile + it;
            const bool more = it + 1 < w.n;
            if (more) nxt = page_of(w, i + 1);
            // the order in which the MMA warp takes them
            if (C::NS == 1 && more) ok = load(w, i + 1, nxt, &a.mk, &a.mkp);
            if (ok) ok = load(w, i, cur, &a.mv, &a.mvp);
            if (C::NS == 2 && more && ok) ok = load(w, i + 1, nxt, &a.mk, &a.mkp);
            cur = nxt;
        }
    }
    if (!ok) {
        // the copies already issued land before this CTA's shared memory goes away
        for (uint32_t j = at > (uint32_t)C::ST ? at - C::ST : 0; j < at; ++j) {
            const uint64_t t0 = ptx::global_ns();
            while (!ptx::mbar_try_wait(smem_u32(&B->full[j % C::ST]), (j / C::ST) & 1) && ptx::global_ns() - t0 < ptx::kWaitNs) {
            }
        }
    }
}

// f16: one warp, by TMA.  f32: two warps split the rows into f16 hi + lo; a lane keeps its place
// in a row (8 values) and steps through rows, with kDeep rows' loads under way (one warp with a
// division a row took 31 000 clocks a tile of 128 x 128).
template <class C>
__device__ __forceinline__ void q_role(const AttnArgs& a, Bars* B, uint32_t qs, int part, int lane) {
    volatile int* abort = &B->abort;
    const uint32_t bar = smem_u32(&B->q_full);
    uint32_t piece = 0;
    bool ok = true;
    Walk<C> w(B);
    while (w.next(a)) {
        if (!(ok = mbar_wait(smem_u32(&B->q_empty), (piece & 1) ^ 1, abort, a.c.err))) break;
        const int nt = w.tiles(a);
        if constexpr (!C::HL) {
            if (lane == 0) {
                mbar_expect_tx(bar, (uint32_t)nt * a.tq * a.G * 128 * (C::D / 64));
                for (int i = 0; i < nt; ++i)
#pragma unroll
                    for (int u = 0; u < (C::D / 64); ++u)
                        tma_load_3d(qs + i * C::kQTile + u * C::kQSub, &a.mq, bar, u * 64, w.h * a.G, w.s.row0 + w.tok0(a) + i * a.tq);
            }
        } else {
            constexpr int kCh = C::D / 8, kStep = 64 / kCh, kDeep = 4;   // places a row; rows a step of both warps
            const int ch = lane % kCh, t0 = w.tok0(a);
            const int rows = w.rows(a);
            const bool spread = w.spread(a);
            const char* q0 = a.q + (size_t)(w.s.row0 + t0) * a.q_tok + (size_t)w.h * a.G * a.q_head + ch * 32;
            const uint32_t to0 = qs + (ch >> 3) * C::kQSub;
            for (int r0 = (lane + 32 * part) / kCh; r0 < rows; r0 += kStep * kDeep) {
                float4 v[kDeep][2];
#pragma unroll
                for (int k = 0; k < kDeep; ++k) {
                    const int r = r0 + k * kStep;
                    if (r < rows) {
                        const char* p = q0 + (size_t)a.by_g.quot(r) * a.q_tok + (size_t)a.by_g.rem(r) * a.q_head;
                        v[k][0] = ptx::ld_act(reinterpret_cast<const float4*>(p));
                        v[k][1] = ptx::ld_act(reinterpret_cast<const float4*>(p + 16));
                    }
                }
#pragma unroll
                for (int k = 0; k < kDeep; ++k) {
                    const int r = r0 + k * kStep;
                    if (r < rows) {
                        uint4 hi, lo;
                        ptx::split_h2(v[k][0].x, v[k][0].y, hi.x, lo.x);
                        ptx::split_h2(v[k][0].z, v[k][0].w, hi.y, lo.y);
                        ptx::split_h2(v[k][1].x, v[k][1].y, hi.z, lo.z);
                        ptx::split_h2(v[k][1].z, v[k][1].w, hi.w, lo.w);
                        const uint32_t to = to0 + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
                        auto put = [&](uint32_t at, const uint4& v) {
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
                        };
                        if (spread) {
                            for (int copy = 0; copy < 4; ++copy) {
                                put(to + copy * 32 * 128, hi);
                                put(to + copy * 32 * 128 + 16 * 128, lo);
                            }
                        } else {
                            put(to, hi);
                            put(to + C::kQTile, lo);
                        }
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        }
        __syncwarp();
        ++piece;
    }
    if (!C::HL && !ok && piece > 0 && lane == 0) {
        const uint64_t t0 = ptx::global_ns();
        while (!ptx::mbar_try_wait(bar, (piece - 1) & 1) && ptx::global_ns() - t0 < ptx::kWaitNs) {
        }
    }
}

// Everything that the issued instructions take is computed from values that the compiler knows
// to be uniform (one shuffle a ring unit), with 32-bit descriptor steps: the tensor cores hold
// only about four products in their queue, so what this warp does between two of them has to
// take less than four products' time.
template <class C>
__device__ __forceinline__ void mma_role(const AttnArgs& a, Bars* B, uint32_t qs, uint32_t ring, uint32_t tmem_base, int lane) {
    constexpr int NS = C::NS, DU = C::DU, PARTS = C::HL ? 2 : 1;
    constexpr int kCols = BN / C::H;                      // slots a step of S
    constexpr uint32_t idesc_s = umma_idesc_f16(128, kCols);
    constexpr uint32_t idesc_o = umma_idesc_f16(128, DU) | kIdescBMnMajor;
    const uint32_t bars = uniform(smem_u32(B)), q16 = uniform(qs >> 4), ring16 = uniform(ring >> 4), tmem = uniform(tmem_base);
#define MLZC_BAR(member, i) (bars + (uint32_t)offsetof(Bars, member) + 8u * (uint32_t)(i))
    volatile int* abort = &B->abort;
    uint32_t slot = 0, phase = 0, seg = 0, g[2] = {0, 0}, piece[2] = {0, 0};
    uint32_t last_bar = 0, last_par = 0;     // of the latest commit to a ring barrier
    auto wait = [&](uint32_t bar, uint32_t par) { return mbar_wait(bar, par, abort, a.c.err); };
    auto commit = [&](uint32_t bar) {
        if (elect_one()) umma_commit(bar);
    };
    // waits for the ring's next unit and takes it: its number (uniform) and phase
    struct Unit {
        uint32_t st, phase;
    };
    auto take = [&](Unit& u) {
        u.st = uniform(slot);
        u.phase = phase;
        if (!wait(MLZC_BAR(full, u.st), phase)) return false;
        tc_fence_after();
        if (++slot == C::ST) {
            slot = 0;
            phase ^= 1;
        }
        return true;
    };
    // frees a unit when the products issued so far are done
    auto release = [&](const Unit& u) {
        commit(MLZC_BAR(empty, u.st));
        last_bar = MLZC_BAR(empty, u.st);
        last_par = u.phase;
    };
    // S of query tile `tile` and the slots from `row` of the tile on, into buffer `buf`
    bool spread = false;                     // hi and lo are rows of one Q tile
    auto scores = [&](int tile, int buf, int unit, const Unit& u, int row) {
        const uint32_t k = desc_lo(ring16 + u.st * (C::kUnit >> 4) + row * 8);
        const uint32_t q = desc_lo(q16 + ((tile * PARTS * C::kQTile + unit * C::SUBS * C::kQSub) >> 4));
        const uint32_t d = tmem + C::kSCol + buf * kCols;
        if (elect_one()) {
#pragma unroll
            for (int part = PARTS - 1; part >= 0; --part) {    // lo, then hi
                if (C::kSpread && part > 0 && spread) continue;
#pragma unroll
                for (int i = 0; i < DU / 16; ++i)
                    umma_f16_lo(d, q + ((part * C::kQTile + (i >> 2) * C::kQSub + (i & 3) * 32) >> 4),
                                k + (((i >> 2) * C::kSub + (i & 3) * 32) >> 4), idesc_s,
                                unit > 0 || i > 0 || (part != PARTS - 1 && !spread));
            }
        }
    };
    // `steps` key steps of P V, from step i0 (even) on
    auto values = [&](int tile, int buf, int unit, const Unit& u, bool add, int i0, auto steps) {
        const uint32_t v = desc_lo(ring16 + u.st * (C::kUnit >> 4) + i0 * 128, C::kSub);
        const uint32_t d = tmem + C::kOCol + tile * C::D + unit * DU, p = tmem + C::kSCol + buf * BN + i0 * 16;
        if (elect_one()) {
#pragma unroll
            for (int part = PARTS - 1; part >= 0; --part) {
                if (C::kSpread && part > 0 && spread) continue;
#pragma unroll
                for (int i = 0; i < decltype(steps)::value; ++i)
                    umma_f16_ta_lo(d, p + (i >> 1) * 32 + (i & 1) * 8 + part * 16, v + i * 128, idesc_o,
                                   add || i > 0 || (part != PARTS - 1 && !spread));
            }
        }
    };
    constexpr std::integral_constant<int, BN / 16> all{};
    constexpr std::integral_constant<int, BN / 16 / C::H> step{};
    // V rows that no row of the piece sees may hold anything (a page's unused rows) or have not
    // been copied: P is 0 there, and 0 * NaN would be NaN
    auto blank = [&](const Walk<C>& w, int i, const Unit& u) {
        const int n = tile_rows(a, w, i);
        if (n == BN) return;
        for (int x = n * 8 + lane; x < BN * 8; x += 32)
#pragma unroll
            for (int k = 0; k < C::SUBS; ++k)
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(ring + u.st * C::kUnit + k * C::kSub + x * 16), "r"(0) : "memory");
        fence_proxy_async_smem();
        __syncwarp();
    };
    // S of one query tile (NS = 1): all units of K
    auto scores_all = [&](int buf) {
#pragma unroll
        for (int unit = 0; unit < C::UN; ++unit) {
            Unit u;
            if (!take(u)) return false;
            scores(0, buf, unit, u, 0);
            release(u);
        }
        commit(MLZC_BAR(s_full, buf));
        return true;
    };
    bool ok = true;
    Walk<C> w(B);
    while (ok && w.next(a)) {
        const int nt = w.tiles(a);
        spread = uniform(w.spread(a)) != 0;
        ok = wait(MLZC_BAR(q_full, 0), seg & 1);
        if (!ok) break;
        ++seg;
        tc_fence_after();
        if constexpr (NS == 1) {
            const int first = (int)uniform(g[0] & 1);
            if (!(ok = scores_all(first))) break;
            if (w.n == 1) commit(MLZC_BAR(q_empty, 0));
            for (int it = 0; it < w.n; ++it, ++g[0]) {
                const int buf = (int)uniform(g[0] & 1);
                if (it + 1 < w.n) {
                    if (!(ok = scores_all(buf ^ 1))) break;
                    if (it + 2 == w.n) commit(MLZC_BAR(q_empty, 0));
                }
                ok = wait(MLZC_BAR(p_full, buf), (g[0] >> 1) & 1);
                // O free: f32 calls empty it tile by tile, the others piece by piece
                const uint32_t turn = C::HL ? g[0] : piece[0];
                if (ok && (C::HL || it == 0)) ok = wait(MLZC_BAR(o_empty, 0), (turn & 1) ^ 1);
                if (!ok) break;
                const bool add = !C::HL && uniform(it) > 0;
#pragma unroll
                for (int unit = 0; unit < C::UN; ++unit) {
                    Unit u;
                    if (!(ok = take(u))) break;
                    blank(w, w.tile + it, u);
                    tc_fence_after();
                    values(0, buf, unit, u, add, 0, all);
                    release(u);
                }
                if (!ok) break;
                if (C::HL || it + 1 == w.n) commit(MLZC_BAR(o_done, 0));
                if (!C::HL) commit(MLZC_BAR(o_step, 0));
            }
        } else {
            Unit k, v;
            if (!(ok = take(k))) break;
#pragma unroll
            for (int h = 0; h < C::H; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (i < nt) {
                        scores(i, C::H * i + h, 0, k, h * kCols);
                        commit(MLZC_BAR(s_full, C::H * i + h));
                    }
            release(k);
            if (w.n == 1) commit(MLZC_BAR(q_empty, 0));
            for (int it = 0; ok && it < w.n; ++it) {
                const bool more = it + 1 < w.n, begun = uniform(it) > 0;
                if (!(ok = take(v))) break;
                blank(w, w.tile + it, v);
#pragma unroll
                for (int h = 0; h < C::H; ++h)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (!ok || i >= nt) continue;
                        const int buf = C::H * i + h;
                        ok = wait(MLZC_BAR(p_full, buf), (C::H == 2 ? g[i] >> 1 : g[i]) & 1);
                        if (ok && it == 0 && h == 0) ok = wait(MLZC_BAR(o_empty, i), (piece[i] & 1) ^ 1);
                        if (!ok) continue;
                        tc_fence_after();
                        values(i, i, 0, v, begun || h > 0, h * (BN / 16 / C::H), step);
                        commit(MLZC_BAR(o_step, i));
                        if (!more && h == C::H - 1) commit(MLZC_BAR(o_done, i));
                        if (more) {
                            if (h == 0 && i == 0 && !(ok = take(k))) continue;
                            scores(i, buf, 0, k, h * kCols);
                            commit(MLZC_BAR(s_full, buf));
                        }
                        ++g[i];
                    }
                if (!ok) break;
                release(v);
                if (more) {
                    release(k);
                    if (it + 2 == w.n) commit(MLZC_BAR(q_empty, 0));
                }
            }
        }
        for (int i = 0; i < nt; ++i) ++piece[i];
    }
#undef MLZC_BAR
    if (!ok && last_bar && elect_one()) {
        // the products already issued end before TMEM is released
        umma_commit(last_bar);
        const uint64_t t0 = ptx::global_ns();
        while (!ptx::mbar_try_wait(last_bar, last_par) && ptx::global_ns() - t0 < ptx::kWaitNs) {
        }
    }
}

// Notes for the merge launch the query tile that begins in this CTA's share and ends in a later one.
template <class C>
__device__ __forceinline__ void head_role(const AttnArgs& a, Bars* B) {
    int4 hd = make_int4(0, 0, 0, -1);
    Walk<C> w(B);
    while (w.next(a)) {
        if (w.tile == 0 && !w.ends()) {
            // the share's last piece: what is left of its query tile ends so many places on
            const long long n = min((long long)a.n_ctas, B->total), end = B->first + B->count + w.all - w.n;
            hd = make_int4(w.s.row0 + w.tok0(a), min(a.tq * C::NS, w.s.rows - w.tok0(a)), w.h, (int)((end * n - 1) / B->total));
        }
    }
    a.head[blockIdx.x] = hd;
}

template <int FROM, int TO>
__device__ __forceinline__ void set_registers() {
    if constexpr (TO > FROM) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TO));
    if constexpr (TO < FROM) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TO));
}

template <class C>
__global__ void __launch_bounds__(C::kThreads, 1) attn_kernel(const __grid_constant__ AttnArgs a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t qs = smem_u32(smem), ring = qs + C::kQBytes;
    uint8_t* fixed = smem + C::kQBytes + (size_t)C::ST * C::kUnit;
    Bars* B = reinterpret_cast<Bars*>(fixed);
    float2* stats = reinterpret_cast<float2*>(fixed + kBarBytes);
    // the loading and issuing warps come first (a scheduler prefers its lower warps), then the
    // softmax and correction warpgroups, numbered from 0 in their roles
    const int warp = (int)uniform(threadIdx.x >> 5) - 4, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::ST; ++i) {
            mbar_init(smem_u32(&B->full[i]), 1);
            mbar_init(smem_u32(&B->empty[i]), 1);
        }
        mbar_init(smem_u32(&B->q_full), C::HL ? 2 : 1);
        mbar_init(smem_u32(&B->q_empty), 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&B->o_step[i]), 1);
            mbar_init(smem_u32(&B->o_done[i]), 1);
            mbar_init(smem_u32(&B->o_empty[i]), C::HL ? C::kCorrWarps : 4);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(smem_u32(&B->s_full[i]), 1);
            mbar_init(smem_u32(&B->p_full[i]), 4);
        }
        for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&B->stat_full[i]), 4);
        mbar_init(smem_u32(&B->copies), 4);
        B->abort = 0;
        ptx::mbar_init_fence();
        tma_prefetch_desc(&a.mk);
        tma_prefetch_desc(&a.mv);
        if (!C::HL) tma_prefetch_desc(&a.mq);
    }
    if (warp == -3) tmem_alloc(smem_u32(&B->tmem), 512);
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    plan<C>(a, B);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = B->tmem;
    // Registers: the launch's share is 168 a thread with 384 threads and 128 with 512; a wait
    // for more than the launch's sum would not end.
    constexpr int kShare = C::kThreads == 512 ? 128 : (C::kThreads == 384 ? 168 : 255);
    constexpr int kSoft = C::HL ? (C::D == 64 ? 136 : (C::D == 128 ? 176 : 120)) : (C::NS == 2 ? 208 : 255);
    constexpr int kCorr = C::HL ? (C::D == 64 ? 136 : (C::D == 128 ? 216 : 160)) : 0;
    constexpr int kRest = C::HL ? (C::D == 256 ? 72 : (C::D == 128 ? 112 : 104)) : (C::NS == 2 ? 88 : 255);
    static_assert(kSoft * C::kSoftWarps + kCorr * C::kCorrWarps + kRest * 4 <= kShare * (C::kThreads / 32), "registers");
    if (warp >= 0 && warp < C::kSoftWarps) {
        set_registers<kShare, kSoft>();
        if constexpr (C::HL) softmax_tile_role<C>(a, B, stats, tmem, warp, lane);
        else softmax_role<C>(a, B, tmem, warp, lane);
    } else if (C::HL && warp >= 0) {
        if constexpr (C::HL) {
            set_registers<kShare, kCorr>();
            correct_role<C>(a, B, stats, tmem, warp, lane);
        }
    } else {
        set_registers<kShare, kRest>();
        if (warp == -4) load_role<C>(a, B, ring, lane);
        else if (warp == -3) mma_role<C>(a, B, qs, ring, tmem, lane);
        else if (C::HL || warp == -2) q_role<C>(a, B, qs, warp + 2, lane);
        if (warp == -1 && lane == 0) head_role<C>(a, B);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == -3) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Merges the records of each cut query tile: block (c, y) the tile begun by CTA c, 8 rows.
constexpr int kMergeRows = 8;
template <int D, typename Out>
__global__ void __launch_bounds__(kMergeRows * 32) merge_kernel(const __grid_constant__ AttnArgs a) {
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    const int c = blockIdx.x, lane = threadIdx.x & 31;
    const uint4 hd = ptx::ld_act(reinterpret_cast<const uint4*>(&a.head[c]));
    const int row0 = (int)hd.x, tokens = (int)hd.y, h = (int)hd.z, last = (int)hd.w;
    if (last < 0) return;
    const int row = blockIdx.y * kMergeRows + (threadIdx.x >> 5);
    const int tok = a.by_g.quot(row);
    if (row >= a.rec_rows || tok >= tokens) return;
    auto rec = [&](int i) { return ((size_t)i * 2 + (i == c ? 1 : 0)) * a.rec_rows + row; };
    // four records at a time, their loads under way together
    float top = -INFINITY, l = 0.0f, acc[D / 32] = {};
    for (int i0 = c; i0 <= last; i0 += 4) {
        uint2 m[4], v[4][D / 64];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i0 + k <= last) {
                const size_t r = rec(i0 + k);
                m[k] = ptx::ld_act(reinterpret_cast<const uint2*>(&a.ml[r]));
#pragma unroll
                for (int e = 0; e < D / 64; ++e) v[k][e] = ptx::ld_act(reinterpret_cast<const uint2*>(a.rec + r * D + e * 64 + lane * 2));
            }
        float to = top;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i0 + k <= last) to = fmaxf(to, __uint_as_float(m[k].x));
        if (to == -INFINITY) continue;
        const float f0 = ex2(top - to);
        top = to;
        l *= f0;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) acc[e] *= f0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i0 + k <= last) {
                const float f = ex2(__uint_as_float(m[k].x) - to);
                l = fmaf(f, __uint_as_float(m[k].y), l);
#pragma unroll
                for (int e = 0; e < D / 64; ++e) {
                    acc[2 * e] = fmaf(f, __uint_as_float(v[k][e].x), acc[2 * e]);
                    acc[2 * e + 1] = fmaf(f, __uint_as_float(v[k][e].y), acc[2 * e + 1]);
                }
            }
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const int q = row0 + tok, head = h * a.G + a.by_g.rem(row);
    char* dst = a.dst + (size_t)q * a.d_tok + (size_t)head * a.d_head;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) {
        if constexpr (sizeof(Out) == 4)
            reinterpret_cast<float2*>(dst)[e * 32 + lane] = make_float2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
        else
            reinterpret_cast<uint32_t*>(dst)[e * 32 + lane] = ptx::pack_h2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
    }
    if (a.lse && lane == 0)
        *reinterpret_cast<float*>(a.lse + (size_t)q * a.lse_tok + (size_t)head * a.lse_head) =
            l > 0.0f ? (top + log2f(l)) * kLn2 : -INFINITY;
}

struct Plan {
    int ns, rec_rows;
    size_t rec, ml, total;
};

Plan make_plan(const mlzc_paged_cache* cache, const mlzc_paged_attn_desc* d, int ctas) {
    Plan p{};
    const int64_t G = d->n_head_q / cache->n_head_kv, rows = cache->n_tokens * G;
    // two query tiles a CTA when the sequences fill more than one on average
    p.ns = d->type == MLZC_TYPE_F16 && cache->head_dim < 256 && rows > 128 * cache->batch_size ? 2 : 1;
    p.rec_rows = paged::record_rows(cache->n_tokens, (int)G, 128 / (int)G, p.ns);
    p.rec = (size_t)ctas * 2 * p.rec_rows * cache->head_dim * 4;
    p.ml = (size_t)ctas * 2 * p.rec_rows * 8;
    p.total = p.rec + p.ml + (size_t)ctas * 16;
    return p;
}

template <class C>
int launch(const AttnArgs& a, const DeviceCtx* c, cudaStream_t s) {
    static bool set[64] = {};
    const int dev = c->device < 64 ? c->device : 63;
    if (!set[dev] || c->device >= 64) {
        MLZC_CUDA_TRY(cudaFuncSetAttribute(attn_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem));
        set[dev] = true;
    }
    MLZC_CUDA_TRY(launch_pdl(attn_kernel<C>, dim3(a.n_ctas), dim3(C::kThreads), C::kSmem, s, a));
    MLZC_CUDA_TRY(cudaGetLastError());
    using Out = typename std::conditional<C::HL, float, __half>::type;
    const dim3 g(a.n_ctas, (a.rec_rows + kMergeRows - 1) / kMergeRows);
    MLZC_CUDA_TRY(launch_pdl(merge_kernel<C::D, Out>, g, dim3(kMergeRows * 32), 0, s, a));
    MLZC_CUDA_TRY(cudaGetLastError());
    count_launch(2);
    return MLZC_OK;
}

}  // namespace
}  // namespace mlzc

using namespace mlzc;

extern "C" int mlzc_paged_attn_workspace_bytes(const mlzc_paged_cache* cache, const mlzc_paged_attn_desc* d,
                                               size_t* out_bytes) {
    if (!out_bytes) return fail(MLZC_ERR_INVALID, "paged attention: null out_bytes");
    *out_bytes = 0;
    const int st = paged::check_attn(cache, d, false);
    if (st != MLZC_OK || cache->n_tokens == 0) return st;
    DeviceCtx* c = current_ctx();
    if (!c) return MLZC_ERR_CUDA;
    *out_bytes = make_plan(cache, d, c->sm_count).total;
    return MLZC_OK;
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
    const Plan p = make_plan(cache, d, c->sm_count);
    if (!workspace || workspace_bytes < p.total)
        return fail(MLZC_ERR_NOMEM, "paged attention: workspace of %zu bytes needed, %zu given", p.total, workspace_bytes);
    if ((uintptr_t)workspace % 16) return fail(MLZC_ERR_INVALID, "paged attention: workspace not 16-byte aligned");
    const bool f32 = d->type == MLZC_TYPE_F32;
    a.G = (int)(d->n_head_q / cache->n_head_kv);
    a.tq = 128 / a.G;
    a.by_g.set((uint32_t)a.G);
    a.box = std::gcd(cache->page_size, BN);
    if ((st = paged::encode_pool(&a.mk, cache, false, a.box)) != MLZC_OK) return st;
    if ((st = paged::encode_pool(&a.mv, cache, true, a.box)) != MLZC_OK) return st;
    // a page of 24 rows is three boxes of 8 where a tile cuts it, one of 24 elsewhere
    a.whole = cache->page_size < BN && a.box < cache->page_size;
    if (a.whole && (st = paged::encode_pool(&a.mkp, cache, false, cache->page_size)) != MLZC_OK) return st;
    if (a.whole && (st = paged::encode_pool(&a.mvp, cache, true, cache->page_size)) != MLZC_OK) return st;
    if (!f32 && (st = paged::encode_rows(&a.mq, d->q, cache->head_dim, d->n_head_q, cache->n_tokens, d->q_nb[1], d->q_nb[2],
                                         a.G, a.tq)) != MLZC_OK)
        return st;
    a.q = static_cast<const char*>(d->q);
    a.dst = static_cast<char*>(d->dst);
    a.q_head = d->q_nb[1]; a.q_tok = d->q_nb[2];
    a.d_head = d->dst_nb[1]; a.d_tok = d->dst_nb[2];
    a.lse = reinterpret_cast<char*>(d->lse);
    a.lse_head = d->lse_nb[0]; a.lse_tok = d->lse_nb[1];
    a.scale = d->scale;
    a.softcap = (d->mode & MLZC_FA_MODE_SOFTCAP) ? d->logit_softcap : 0.0f;
    a.n_ctas = c->sm_count;
    a.rec_rows = p.rec_rows;
    a.rec = static_cast<float*>(workspace);
    a.ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + p.rec);
    a.head = reinterpret_cast<int4*>(static_cast<char*>(workspace) + p.rec + p.ml);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool cap = a.softcap > 0.0f;
    // f32 decode: a token a sequence, at most 8 query rows a KV head
    const bool spread = f32 && cache->n_tokens <= cache->batch_size && a.G <= 8;
    if (spread && cache->head_dim == 128) return cap ? launch<Cfg<128, 1, true, true, true>>(a, c, s) : launch<Cfg<128, 1, true, false, true>>(a, c, s);
    if (spread && cache->head_dim == 64) return cap ? launch<Cfg<64, 1, true, true, true>>(a, c, s) : launch<Cfg<64, 1, true, false, true>>(a, c, s);
#define MLZC_LAUNCH(DIM, NS)                                                                                            \
    return f32 ? (cap ? launch<Cfg<DIM, 1, true, true>>(a, c, s) : launch<Cfg<DIM, 1, true, false>>(a, c, s))           \
               : (cap ? launch<Cfg<DIM, NS, false, true>>(a, c, s) : launch<Cfg<DIM, NS, false, false>>(a, c, s))
    if (cache->head_dim == 256) MLZC_LAUNCH(256, 1);
    if (p.ns == 2 && cache->head_dim == 128) MLZC_LAUNCH(128, 2);
    if (p.ns == 2) MLZC_LAUNCH(64, 2);
    if (cache->head_dim == 128) MLZC_LAUNCH(128, 1);
    MLZC_LAUNCH(64, 1);
#undef MLZC_LAUNCH
}
