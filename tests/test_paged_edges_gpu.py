"""GPU: calls of the paged KV cache at the edges of what its contract allows, against the plain
64-bit forms."""
import math

import pytest
import torch

import mlz_b200
from tests import paged_ref as ref
from tests.test_paged_gpu import _check_attn

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


# ------------------------------------------------------------------ records of two query tiles

@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("behind", [300, 5000])
@pytest.mark.parametrize("group,tokens", [(3, (43, 44, 48, 51, 84, 85)), (5, (26, 27, 28, 50, 51)), (6, (22, 23, 42)),
                                          (7, (19, 20, 21, 36)), (12, (11, 12, 20)), (33, (4, 5, 6)), (100, (2, 3))])
def test_attn_one_sequence_with_groups_that_do_not_divide_a_tile(dev, group, tokens, behind, D):
    """A chunk of one sequence that fills one query tile and part of a second one, its slots shared
    out to many CTAs: every row of both tiles comes back from the records."""
    for T in tokens:
        _check_attn(ref.make(dev, [T], [T + behind], hkv=2, group=group, D=D, page=64, dtype=F16, seed=T))


# ------------------------------------------------------------------ capped scores

def _unused_rows(c):
    """Rows of the pools that lie past every sequence's length."""
    u = torch.ones((c.k.shape[0], c.page), dtype=torch.bool)
    table = c.table.cpu()
    for b, n in enumerate(c.kv_len):
        for j in range(n):
            u[table[b, j // c.page], j % c.page] = False
    return u[:, None, :, None].expand_as(c.k).to(c.k.device)


@pytest.mark.parametrize("softcap", [0.0, 9.0])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q_len,kv_len", [([5, 1], [100, 333]), ([1, 1, 1], [40, 200, 1001]), ([200], [500])])
def test_what_does_not_count_changes_no_bit(dev, q_len, kv_len, D, dtype, softcap):
    """Attention and weights with other contents of the pages' unused rows, of the rows behind the
    last sequence and, left by other calls, of shared and tensor memory."""
    c = ref.make(dev, q_len, kv_len, D=D, dtype=dtype, seed=7, tail=5, junk=False)
    unused, cache, first = _unused_rows(c), ref.handle(c), None
    for junk in (0.0, 3.0e4, -7.0, math.nan):
        c.k[unused] = c.v[unused] = junk
        c.q[c.T:] = junk
        o = ref.make(dev, [130, 64], [700, 400], D=D, dtype=dtype, seed=3, q_scale=0.1 if junk == 0 else 300.0)
        other = ref.handle(o)
        _, lse = mlz_b200.paged_attn(other, o.q, o.scale, return_lse=True)
        mlz_b200.paged_weights(other, o.q, lse, o.scale)
        out, lse = mlz_b200.paged_attn(cache, c.q, c.scale, softcap=softcap, return_lse=True)
        w = mlz_b200.paged_weights(cache, c.q, lse, c.scale, softcap=softcap)
        got = out[:c.T].clone(), lse[:c.T].clone(), w
        first = first or got
        for a, b, what in zip(first, got, ("out", "lse", "weights")):
            assert torch.equal(a, b), f"{what} with {junk} in what does not count"


@pytest.mark.parametrize("cap", [50.0, 1000.0, 2.0 ** 14])
@pytest.mark.parametrize("q_len,kv_len", [([4], [40]), ([1, 1], [300, 77]), ([150], [150])])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_small_capped_scores_beside_large_ones(dev, D, q_len, kv_len, cap):
    """f32: one head's scores reach past the cap, the others' stay below 1.  q and k have one dim,
    so the products are exact and the bound is that of the capping alone."""
    c = ref.make(dev, q_len, kv_len, hkv=1, group=4, D=D, seed=1, junk=False)
    g = torch.Generator(device=dev).manual_seed(5)
    c.q.zero_()
    c.k.zero_()
    c.q[:, :, 3] = torch.rand(c.q.shape[:2], generator=g, device=dev) - 0.5
    c.q[::2, 1, 3] = 3 * cap
    c.k[..., 3] = (torch.rand(c.k.shape[:3], generator=g, device=dev) * 2 - 1).half()
    c.scale = 1.1
    cache = ref.handle(c)
    _, lse = mlz_b200.paged_attn(cache, c.q, c.scale, softcap=cap, return_lse=True)
    _, want, _, _ = ref.attn(c, cap)
    # q as hi + lo (2^-22), scale / cap and its product with the score (2^-24 each), tanh (1.7e-7),
    # two products with the cap's (2^-24 each): below 2^-20 of a score, which is below 1 in heads 0, 2 and 3
    # and below cap in head 1; then the exponentials (2^-22) and their sum, in f32, and the lse from the
    # maximum less an offset of 6 and the logarithm of a sum below 2^20, each rounded twice
    n = max(kv_len)
    for h in range(4):
        most = cap if h == 1 else 1.0
        bound = 2.0 ** -20 * most + (8 + n ** 0.5) * 2.0 ** -24 + 4 * 2.0 ** -24 * (most + 6 + 20)
        worst = float((lse[:, h].double() - want[:, h]).abs().max())
        assert worst <= bound, f"head {h}: lse off by {worst:.2e}, bound {bound:.2e}"
    # weights of the small heads with lse = 0: exp(score), its relative error that of the score, of the
    # exponential and of the sums of T x 4 terms
    zero = torch.zeros_like(lse)
    zero[:, 1] = -math.inf
    got = mlz_b200.paged_weights(cache, c.q, zero, c.scale, softcap=cap)
    want, _ = ref.weights(c, zero, cap)
    real = ~torch.isnan(want)
    bound = 2.0 ** -20 + 2.0 ** -22 + (8 + (4 * c.T) ** 0.5) * 2.0 ** -24
    assert float(((got.double() - want) / want)[real].abs().max()) <= bound


# ------------------------------------------------------------------ workspaces

@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("q_len", [[1, 1], [150, 1], [0, 0]])
def test_workspaces_of_the_stated_sizes(dev, q_len, dtype):
    """The stated sizes are enough and needed, asked for before the first call or after it."""
    for before in (True, False):
        c = ref.make(dev, q_len, [400, 90], hkv=3, dtype=dtype, seed=61)
        cache, q = ref.handle(c), c.q[:c.T]
        if not before:
            _, lse = mlz_b200.paged_attn(cache, q, c.scale, return_lse=True)
            w = mlz_b200.paged_weights(cache, q, lse, c.scale)
            mlz_b200.paged_evict(cache, w, 100, kv_len_out=c.lens.clone())
        sizes = (mlz_b200.paged_attn_workspace_bytes(cache, q), mlz_b200.paged_weights_workspace_bytes(cache, q),
                 mlz_b200.paged_evict_workspace_bytes(cache, 100))
        assert (sizes[0] > 0) == (c.T > 0) and sizes[1] > 0 and sizes[2] > 0
        room = [torch.empty(max(16, n), dtype=torch.uint8, device=dev) for n in sizes]
        attn = lambda ws: mlz_b200.paged_attn(cache, q, c.scale, return_lse=True, workspace=ws)  # noqa: E731
        _, lse = attn(room[0])
        weigh = lambda ws: mlz_b200.paged_weights(cache, q, lse, c.scale, workspace=ws)  # noqa: E731
        w = weigh(room[1])
        evict = lambda ws: mlz_b200.paged_evict(cache, w.clone(), 100, kv_len_out=c.lens.clone(), workspace=ws)  # noqa: E731
        evict(room[2])
        torch.cuda.synchronize()
        for call, ws, n in zip((attn, weigh, evict), room, sizes):
            if n:
                with pytest.raises(mlz_b200.MlzcError, match="workspace"):
                    call(ws[:n - 1])


# ------------------------------------------------------------------ tokens that are to add nothing

@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("softcap", [0.0, 8.0])
def test_weights_of_tokens_without_lse_add_nothing_whatever_their_q(dev, dtype, softcap):
    c = ref.make(dev, [3, 150, 1, 1], [20, 400, 30, 300], dtype=dtype, seed=9)
    _, lse, _, _ = ref.attn(c, softcap)
    lse = lse.float().contiguous()
    dead = torch.zeros(c.T, dtype=torch.bool, device=dev)
    dead[[1, 77, 130, 153]] = True
    lse[dead] = -math.inf
    c.q[dead] = 0.0
    want, bound = ref.weights(c, lse, softcap)
    real = ~torch.isnan(want)
    for x in (0.0, math.nan, math.inf, -math.inf):
        c.q[dead] = x
        got = mlz_b200.paged_weights(ref.handle(c), c.q, lse, c.scale, softcap=softcap)
        assert ((got.double() - want).abs() <= bound)[real].all(), f"q = {x}"
        first = got if x == 0.0 else first
        assert torch.equal(got, first), f"q = {x}"
        assert (got[2, :, :30] == 0).all()   # a sequence whose only token adds nothing


# ------------------------------------------------------------------ scores of any size

def _check_far_scores(c, softcap, scales):
    """q and k of c have one dim of a few bits, so products and differences of scores are exact; no
    two different scores are within 2^-11 of one another."""
    vmax = float(c.v.abs().max())
    for e in scales:
        c.scale = 1.37 * 2.0 ** e
        # (softmax by differences of scores: at 2^44 the lse's own 64-bit rounding is 2^-10)
        want, want_lse = torch.zeros(c.q.shape, dtype=torch.float64, device=c.q.device), torch.zeros(c.q.shape[:2], dtype=torch.float64, device=c.q.device)
        for r in range(c.group):
            x, _ = ref.score_rows(c, 0, 0, r, softcap)
            want[:, r], want_lse[:, r] = torch.softmax(x, dim=-1) @ ref.rows(c, c.v, 0, 0), torch.logsumexp(x, dim=-1)
        top = float(want_lse.abs().max())
        if softcap and top > 2.0 ** 36:   # of cap 2^40: nearer to it, f32 does not hold the scores apart
            continue
        out, lse = mlz_b200.paged_attn(ref.handle(c), c.q, c.scale, softcap=softcap, return_lse=True)
        # a weight is off by its score's rounded difference from the largest, d: 2^-24 of the scale, its
        # product with log2 e and the difference's, below 2^-20 of d, and d exp(-d) < 0.37; then as in every
        # call.  With a cap also by each score's own 2^-20, which past 2^15 moves no weight off 0 or 1
        own = 2.0 ** -20 * top if softcap and top < 2.0 ** 15 else 0.0
        worst = float((out.double() - want).abs().nan_to_num(math.inf).max())
        bound = vmax * (2.0 ** -18 + 4 * own + (0.0 if c.q.dtype == F32 else 2.0 ** -10))
        assert worst <= bound, f"scale 2^{e}: out off by {worst:.2e}, bound {bound:.2e}"
        worst = float(((lse.double() - want_lse) / want_lse.abs().clamp(min=8)).abs().nan_to_num(math.inf).max())
        assert worst <= 2.0 ** -19, f"scale 2^{e}: lse off by {worst:.2e}"


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("softcap", [0.0, 2.0 ** 40])
@pytest.mark.parametrize("q", [1.3125, -1.3125, 20000.0])
@pytest.mark.parametrize("T", [1, 140])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attn_of_scores_past_f32s_fractions(dev, D, T, q, softcap, dtype):
    """Scores of 2^26 to 2^56 are weights of 1 for the largest and 0 for the others."""
    c = ref.make(dev, [T], [300], hkv=1, group=2, D=D, seed=1, junk=False, dtype=dtype)
    rank = torch.randperm(300, generator=torch.Generator().manual_seed(2)).to(dev)
    slot = torch.arange(300, device=dev)
    c.q.zero_()
    c.k.zero_()
    c.q[:, :, 3] = q
    c.k[c.table[0].long()[slot // c.page], 0, slot % c.page, 3] = ((rank + 100) / 32).half()
    _check_far_scores(c, softcap, (0, 9, 16, 19, 20, 21, 22, 24, 26, 28, 32, 38))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("softcap", [0.0, 2.0 ** 40])
@pytest.mark.parametrize("T", [1, 150])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attn_of_far_scores_that_rise_from_tile_to_tile(dev, D, T, softcap, dtype):
    """Several slot tiles a CTA, each with larger scores than the one before."""
    n = 60000
    c = ref.make(dev, [T], [n], hkv=1, group=2, D=D, page=128, seed=1, junk=False, dtype=dtype)
    slot = torch.arange(n, device=dev)
    c.q.zero_()
    c.k.zero_()
    c.q[:, :, 3] = 1.3125
    c.k[c.table[0].long()[slot // c.page], 0, slot % c.page, 3] = ((slot // 64 + 100) / 32).half()
    _check_far_scores(c, softcap, (9, 18, 20, 22, 24, 28, 31, 38))


# ------------------------------------------------------------------ the exponentials

@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_lse_has_the_precision_of_f32_exponentials(dev, D, dtype):
    """Row r: one slot with score 0 and eight, in places where any form of the exponential may be
    used, with score -q_r; everything else counts for nothing.  q and k have one dim of few bits."""
    T = 150
    c = ref.make(dev, [T], [300], hkv=1, group=1, D=D, page=64, seed=1, junk=False, dtype=dtype)
    q = (1.0 + torch.arange(T, device=dev) / 512).to(dtype)
    k = torch.full((300,), -60000.0, device=dev)
    k[0], k[[6, 7, 14, 15, 22, 23, 30, 31]] = 0.0, -1.0
    slot = torch.arange(300, device=dev)
    c.q.zero_()
    c.k.zero_()
    c.q[:, 0, 3] = q
    c.k[c.table[0].long()[slot // c.page], 0, slot % c.page, 3] = k.half()
    _, lse = mlz_b200.paged_attn(ref.handle(c), c.q, 1.0, return_lse=True)
    want = torch.log1p(8 * torch.exp(-q.double()))
    # an exponent below 8 rounded (2^-22 ln 2) with log2 e's own rounding (2^-24 of 1.3), the
    # exponential (2^-22), nine additions (2^-24 each), log2 of a sum below 2^8 to one last place
    # (2^-21 ln 2), its sum with the offset and the product with ln 2 (values below 2: 2^-23 in all)
    ln2 = math.log(2.0)
    bound = 2.0 ** -22 * ln2 + 1.3 * 2.0 ** -24 + 2.0 ** -22 + 9 * 2.0 ** -24 + 2.0 ** -21 * ln2 + 2.0 ** -23
    worst = float((lse[:, 0].double() - want).abs().max())
    assert worst <= bound, f"lse off by {worst:.2e}, bound {bound:.2e}"


# ------------------------------------------------------------------ angles

@pytest.mark.parametrize("pairs", ["halves", "adjacent"])
@pytest.mark.parametrize("first,base", [(0, 10000.0), (10 ** 6, 500000.0), (2 ** 31 - 5000, 10000.0), (-2 ** 31, 500000.0)])
def test_store_angles(dev, first, base, pairs):
    """Pairs (1, 0) become (cos, sin) themselves."""
    from fractions import Fraction
    T, D, half = 600, 128, 64
    c = ref.make(dev, [T], [T], hkv=1, group=1, D=D, page=64, seed=71, junk=False)
    g = torch.Generator().manual_seed(3)
    pos = (first + torch.randint(0, 4000, (T,), generator=g)).to(torch.int32)
    one = torch.zeros((T, 1, D), device=dev)
    one[..., slice(0, half) if pairs == "halves" else slice(0, D, 2)] = 1.0
    got = mlz_b200.paged_store(ref.handle(c), one, one, q=one, positions=pos.to(dev), n_rot=D, pairs=pairs, freq_base=base)
    got = got[:, 0].double().cpu()
    co, si = (got[:, :half], got[:, half:]) if pairs == "halves" else (got[:, ::2], got[:, 1::2])
    # turns of a position, rounded to 2^-100 (the powers of base by square roots of rationals)
    one100 = 1 << 100
    two_pi = Fraction(6283185307179586476925286766559005768394, 10 ** 39)
    step, x = Fraction(int(base)), []
    for _ in range(6):   # base ^ (1 / 64)
        step = Fraction(math.isqrt(int(step * one100 * one100)), one100)
    freq = Fraction(1)
    for _ in range(half):
        x.append(round(freq / two_pi * one100))
        freq = Fraction(int(freq / step * one100), one100)
    # 2^-27 of a turn; the functions to one last place of values below 1
    bound = 2 * math.pi * 2.0 ** -27 + 2.0 ** -24
    for j in range(half):
        turn = torch.tensor([((int(p) * x[j]) % one100) / one100 for p in pos], dtype=torch.float64) * (2 * math.pi)
        worst = max(float((co[:, j] - torch.cos(turn)).abs().max()), float((si[:, j] - torch.sin(turn)).abs().max()))
        assert worst <= bound, f"pair {j}: off by {worst:.2e}, bound {bound:.2e}"
