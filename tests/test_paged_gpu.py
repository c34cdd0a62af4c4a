"""GPU parity of the paged KV cache (store, attention, weights, eviction) with plain 64-bit
forms, at the sizes, masks and layouts where each can go wrong."""
import math

import pytest
import torch

import mlz_b200
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def _within(got, want, bound, what):
    got = got.double()
    real = ~torch.isnan(want)
    assert torch.equal(torch.isinf(got[real]), torch.isinf(want[real])), what
    fin = real & ~torch.isinf(want)
    assert torch.isfinite(got[fin]).all(), f"{what}: not finite"
    over = (got[fin] - want[fin]).abs() / bound[fin].clamp(min=1e-30)
    assert over.numel() == 0 or float(over.max()) <= 1.0, f"{what}: {float(over.max()):.2f} of the bound"


def _attn(c, softcap=0.0, **kw):
    sent = 7.0   # rows of no sequence keep it
    out, lse = torch.full_like(c.q, sent), torch.full(c.q.shape[:2], sent, device=c.q.device)
    mlz_b200.paged_attn(ref.handle(c), c.q, c.scale, softcap=softcap, out=out, lse=lse, **kw)
    torch.cuda.synchronize()
    assert (out[c.T:] == sent).all() and (lse[c.T:] == sent).all()
    return out, lse


def _check_attn(c, softcap=0.0, **kw):
    out, lse = _attn(c, softcap, **kw)
    w_out, w_lse, e_out, e_lse = ref.attn(c, softcap)
    _within(out, w_out, e_out, "out")
    _within(lse, w_lse, e_lse, "lse")
    return out, lse


# ------------------------------------------------------------------ attention

@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129, 255, 257, 1000])
def test_attn_single_token_lengths(dev, n, D, dtype):
    _check_attn(ref.make(dev, [1, 1], [n, 2 * n + 1], D=D, dtype=dtype, seed=n))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q_len,kv_len", [
    ([5], [5]), ([33], [33]), ([128], [128]), ([129], [300]), ([257], [700]), ([64], [1000]),
    ([1, 40, 0, 7], [900, 40, 17, 130]), ([300, 1, 1, 65], [512, 511, 1, 66])])
def test_attn_chunks(dev, q_len, kv_len, D, dtype):
    _check_attn(ref.make(dev, q_len, kv_len, D=D, dtype=dtype, seed=sum(kv_len), tail=3))


@pytest.mark.parametrize("hkv,group", [(1, 1), (3, 1), (2, 3), (1, 5), (2, 7), (1, 16), (2, 33), (1, 100), (1, 128)])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_attn_head_groups(dev, hkv, group, dtype):
    _check_attn(ref.make(dev, [3, 1, 17], [200, 65, 17], hkv=hkv, group=group, D=64, dtype=dtype, seed=group))


@pytest.mark.parametrize("group", [1, 3, 8, 9])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("softcap", [0.0, 6.0])
@pytest.mark.parametrize("q_len,kv_len", [([1] * 7, [1, 40, 128, 129, 1000, 3000, 5]), ([3, 0, 1, 0, 0, 2], [700, 9, 333, 0, 50, 64]),
                                          ([20] + [0] * 19, [900] + [3] * 19)])
def test_attn_f32_decode_batches(dev, q_len, kv_len, softcap, D, group):
    """As many tokens as sequences, or fewer: few query rows a head (which f32 calls lay out
    apart), and sequences with more among them."""
    _check_attn(ref.make(dev, q_len, kv_len, hkv=2, group=group, D=D, dtype=F32, seed=group + D), softcap=softcap)


@pytest.mark.parametrize("page", [8, 16, 24, 40, 64, 72, 128, 136, 256, 512])
@pytest.mark.parametrize("layout", ["hpd", "phd"])
def test_attn_pages(dev, page, layout):
    _check_attn(ref.make(dev, [70, 1, 9], [333, 257, 9], page=page, layout=layout, dtype=F32, seed=page))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attn_softcap(dev, D, dtype):
    _check_attn(ref.make(dev, [150, 1], [400, 300], D=D, dtype=dtype, seed=3, q_scale=6.0), softcap=5.0)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_attn_scores_of_wide_range(dev, dtype):
    """Scores over hundreds: one key carries a row, and the running maximum moves by more than
    the range that an unscaled sum bears."""
    _check_attn(ref.make(dev, [200, 1], [900, 700], dtype=dtype, seed=4, q_scale=60.0))


@pytest.mark.parametrize("dtype", [F32, F16])
def test_attn_rising_scores(dev, dtype):
    """Keys sorted so that every tile raises the maximum."""
    c = ref.make(dev, [130], [1100], hkv=1, group=1, page=64, dtype=dtype, seed=5, junk=False)
    c.q[:] = c.q[:1] * 4
    flat = c.k[c.table[0, :18].long(), 0].reshape(-1, c.D)
    order = (flat[:1100].double() @ c.q[0, 0].double()).argsort()
    flat[:1100] = flat[:1100][order]
    c.k[c.table[0, :18].long(), 0] = flat.reshape(18, 64, c.D)
    _check_attn(c)


def test_attn_rows_without_a_slot(dev):
    """More new tokens than slots: the first ones have none; and sequences of length 0."""
    c = ref.make(dev, [6, 2, 3], [4, 0, 3], seed=6)
    out, lse = _attn(c)
    w_out, w_lse, e_out, e_lse = ref.attn(c)
    assert (out[:2] == 0).all() and torch.isinf(lse[:2]).all()
    assert (out[6:8] == 0).all() and (lse[6:8] == -math.inf).all()
    keep = torch.isfinite(w_lse)
    _within(lse[keep], w_lse[keep], e_lse[keep], "lse")
    _within(out[keep], w_out[keep], e_out[keep], "out")


def test_attn_strided_q_out_lse(dev):
    c = ref.make(dev, [40, 1], [90, 300], D=64, seed=7)
    T, H, D = c.q.shape
    wide = torch.zeros((T, H + 2, 2 * D), device=dev)
    wide[:, 1:H + 1, :D] = c.q
    o = torch.full((H, T, D + 4), 9.0, device=dev)
    l = torch.full((H, T), 9.0, device=dev)
    qs = wide[:, 1:H + 1, :D]
    mlz_b200.paged_attn(ref.handle(c), qs, c.scale, out=o.transpose(0, 1)[..., :D], lse=l.T)
    w_out, w_lse, e_out, e_lse = ref.attn(c)
    _within(o.transpose(0, 1)[..., :D], w_out, e_out, "out")
    _within(l.T, w_lse, e_lse, "lse")
    assert (o[..., D:] == 9.0).all()


def test_attn_many_sequences(dev):
    g = torch.Generator().manual_seed(8)
    kv = torch.randint(1, 90, (700,), generator=g).tolist()
    q = [min(n, int(x)) for n, x in zip(kv, torch.randint(0, 4, (700,), generator=g))]
    _check_attn(ref.make(dev, q, kv, hkv=1, group=2, D=64, page=8, dtype=F16, seed=8))


def test_attn_repeats_bit_for_bit(dev):
    c = ref.make(dev, [1] * 5 + [300], [2000, 1999, 50, 700, 4000, 3000], dtype=F32, seed=9)
    a, b = _attn(c), _attn(c)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_attn_long_cache_past_32_bit_offsets(dev):
    """Pools of 2.4 GB each: byte offsets of the last pages pass 2^31 (and 2^32 across both)."""
    n_pages, page, D = 18500, 512, 128
    pool = torch.zeros((n_pages, 1, page, D), dtype=F16, device=dev)
    pool2 = torch.zeros_like(pool)
    c = ref.make(dev, [1, 9], [700, 1030], hkv=1, group=8, page=page, seed=10, junk=False)
    far = torch.arange(n_pages - c.k.shape[0], n_pages, device=dev)
    pool[far], pool2[far] = c.k, c.v
    c.table = torch.where(c.table < c.k.shape[0], c.table + (n_pages - c.k.shape[0]), 0).int()
    c.k, c.v = pool, pool2
    _check_attn(c)


def test_attn_bad_pages_and_lengths_are_not_followed(dev):
    c = ref.make(dev, [1, 1, 1], [40, 40, 40], page=16, seed=11, junk=False)
    c.table[1, 1] = -5
    c.table[2, 0] = c.k.shape[0]
    out, _ = _attn(c)
    assert mlz_b200.device_errors(0) == mlz_b200.DEVERR_BAD_INDEX
    assert torch.isfinite(out).all()
    w_out, _, e_out, _ = ref.attn(_first(c))
    _within(out[:1], w_out, e_out, "untouched sequence")
    c.lens[0] = 1 << 30
    c.q_start[3] = 100
    c.table[:] = 0
    out, _ = _attn(c)
    assert mlz_b200.device_errors(0) == mlz_b200.DEVERR_BAD_INDEX


def _first(c):
    from types import SimpleNamespace
    d = SimpleNamespace(**vars(c))
    d.q_len, d.kv_len, d.q = c.q_len[:1], c.kv_len[:1], c.q[:c.starts[1]]
    return d


# ------------------------------------------------------------------ weights

def _check_weights(c, softcap=0.0, with_acc=True, in_place=False):
    _, lse, _, _ = ref.attn(c, softcap)
    lse = lse.nan_to_num(nan=-math.inf, neginf=-math.inf).float()
    g = torch.Generator(device=c.q.device).manual_seed(1)
    acc = torch.rand((len(c.kv_len), c.hkv, c.cap), generator=g, device=c.q.device) if with_acc else None
    want, bound = ref.weights(c, lse, softcap, acc)
    out = acc if in_place else torch.full((len(c.kv_len), c.hkv, c.cap), 5.0, device=c.q.device)
    before = out.clone()
    mlz_b200.paged_weights(ref.handle(c), c.q, lse, c.scale, softcap=softcap, acc=acc, out=out)
    torch.cuda.synchronize()
    past = torch.isnan(want)
    assert torch.equal(out[past], before[past])
    _within(out, want, bound, "weights")
    return out


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q_len,kv_len", [
    ([1], [1]), ([1, 1], [127, 129]), ([1, 1, 1], [1000, 64, 65]), ([33], [33]), ([129], [300]), ([257], [700]),
    ([1, 40, 0, 7], [900, 40, 17, 130]), ([4], [3])])
def test_weights(dev, q_len, kv_len, D, dtype):
    _check_weights(ref.make(dev, q_len, kv_len, D=D, dtype=dtype, seed=sum(kv_len), tail=2))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_weights_many_query_tiles(dev, D, dtype):
    """Slot tiles with far more query tiles than a CTA holds at a time, and cut between CTAs."""
    _check_weights(ref.make(dev, [1900, 900], [2100, 900], hkv=2, group=8, D=D, dtype=dtype, seed=33))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attn_many_tiles(dev, D, dtype):
    """Query tiles over far more slot tiles than the ring holds, several to a CTA, some cut."""
    _check_attn(ref.make(dev, [1700, 1300], [9000, 1300], hkv=2, group=4, D=D, dtype=dtype, seed=34))


@pytest.mark.parametrize("hkv,group", [(1, 1), (2, 3), (1, 7), (2, 33), (1, 100), (1, 128)])
def test_weights_head_groups(dev, hkv, group):
    _check_weights(ref.make(dev, [3, 1, 17], [200, 65, 17], hkv=hkv, group=group, D=64, seed=group))


@pytest.mark.parametrize("page", [8, 24, 64, 136, 256])
@pytest.mark.parametrize("layout", ["hpd", "phd"])
def test_weights_pages(dev, page, layout):
    _check_weights(ref.make(dev, [70, 1, 9], [333, 257, 9], page=page, layout=layout, dtype=F16, seed=page))


@pytest.mark.parametrize("with_acc,in_place", [(False, False), (True, True)])
def test_weights_start_and_in_place(dev, with_acc, in_place):
    _check_weights(ref.make(dev, [20, 1], [200, 90], seed=12), softcap=8.0, with_acc=with_acc, in_place=in_place)


def test_weights_without_new_tokens_copies(dev):
    c = ref.make(dev, [0, 0], [20, 0], seed=13)
    _check_weights(c)


def test_weights_sum_is_the_number_of_rows(dev):
    """Each row spreads a weight of 1: a head's slots sum to rows x group."""
    c = ref.make(dev, [50, 1], [400, 200], dtype=F16, seed=14)
    _, lse = _attn(c)
    out = mlz_b200.paged_weights(ref.handle(c), c.q, lse, c.scale)
    total = out.double().sum(dim=-1)
    for b, n in enumerate(c.q_len):
        # every weight within 2^-14 of itself at these scores (see score_error), so is their sum
        assert (total[b] / (n * c.group) - 1).abs().max() < 2.0 ** -14


# ------------------------------------------------------------------ eviction

def _check_evict(c, w, budget, sink, recent, **kw):
    kept, wout = ref.evict(c, w, budget, sink, recent)
    k0, v0 = c.k.clone(), c.v.clone()
    own = kw.get("weights_out", w)
    before = own.clone()
    lens = c.lens.clone()
    got, gw, gl = mlz_b200.paged_evict(ref.handle(c), w, budget, n_sink=sink, n_recent=recent, kv_len_out=lens, **kw)
    torch.cuda.synchronize()
    assert gl.tolist() == [min(n, budget) for n in c.kv_len]
    assert got.reshape(-1, budget).tolist() == kept
    ek, ev = k0.clone(), v0.clone()
    for b, n in enumerate(c.kv_len):
        for h in range(c.hkv):
            kp = kept[b * c.hkv + h]
            for to, fr in enumerate(kp):
                if fr >= 0 and fr != to:
                    p0, p1 = int(c.table[b, fr // c.page]), int(c.table[b, to // c.page])
                    ek[p1, h, to % c.page], ev[p1, h, to % c.page] = k0[p0, h, fr % c.page], v0[p0, h, fr % c.page]
            want = torch.tensor(wout[b * c.hkv + h], device=w.device)
            assert torch.equal(gw[b, h, :n].nan_to_num(-9.0), want.nan_to_num(-9.0).float())
            assert torch.equal(gw[b, h, n:].nan_to_num(-9.0), before[b, h, n:].nan_to_num(-9.0))
    assert torch.equal(c.k.view(torch.int16), ek.view(torch.int16))
    assert torch.equal(c.v.view(torch.int16), ev.view(torch.int16))


def _weights_of(c, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    shape = (len(c.kv_len), c.hkv, c.cap)
    if kind == "spread":
        w = torch.randn(shape, generator=g).mul(3).exp()
    elif kind == "ties":
        w = torch.randint(0, 4, shape, generator=g).float()
    elif kind == "equal":
        w = torch.full(shape, 0.25)
    elif kind == "close":      # keys that differ in the last bits alone
        w = 1.0 + torch.randint(0, 50, shape, generator=g) * 2.0 ** -23
    else:                      # signs, zeros of both signs, infinities, NaN, subnormals
        w = torch.randn(shape, generator=g)
        pick = torch.randint(0, 9, shape, generator=g)
        for i, x in enumerate((0.0, -0.0, math.inf, -math.inf, math.nan, 1e-42, -1e-42)):
            w[pick == i] = x
    return w.to(c.k.device)


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "close", "odd"])
@pytest.mark.parametrize("D,page", [(64, 8), (128, 24), (256, 64)])
def test_evict(dev, D, page, kind):
    c = ref.make(dev, [0] * 5, [300, 1, 77, 0, 150], hkv=3, D=D, page=page, seed=page)
    _check_evict(c, _weights_of(c, kind), 77, 3, 10)


@pytest.mark.parametrize("n,budget,sink,recent", [
    (5000, 1000, 4, 64), (9000, 8999, 0, 0), (9000, 1, 0, 0), (9000, 1, 1, 0), (9000, 1, 0, 1), (700, 300, 300, 0),
    (700, 300, 0, 300), (700, 300, 100, 200), (4097, 4096, 1, 1), (10, 4000, 4, 4), (33000, 12000, 16, 1000)])
def test_evict_sizes(dev, n, budget, sink, recent):
    c = ref.make(dev, [0], [n], hkv=2, D=64, page=64, seed=n)
    _check_evict(c, _weights_of(c, "spread", n), budget, sink, recent)


@pytest.mark.parametrize("hkv,n,budget", [
    (75, 33000, 500),      # a CTA a head, keys past its shared memory
    (75, 9500, 9000),      # a CTA a head, holes past its shared memory
    (2, 300000, 3000)])    # a cluster a head, keys past its CTAs' shared memory
def test_evict_long_heads(dev, hkv, n, budget):
    c = ref.make(dev, [0], [n], hkv=hkv, D=64, page=128, seed=n)
    w = _weights_of(c, "spread", n)
    k0 = c.k.clone()
    kept, wout = ref.evict(c, w, budget, 4, 64)
    got, gw, gl = mlz_b200.paged_evict(ref.handle(c), w, budget, n_sink=4, n_recent=64, kv_len_out=c.lens.clone())
    assert gl.tolist() == [budget]
    assert torch.equal(got.cpu(), torch.tensor(kept, dtype=torch.int32).view(1, hkv, budget))
    assert torch.equal(gw[0, :, :n].cpu(), torch.tensor(wout).view(hkv, n))
    fr, to = got[0].long(), torch.arange(budget, device=dev)
    page = lambda x: c.table[0].long()[x // c.page]  # noqa: E731
    h = torch.arange(hkv, device=dev)[:, None]
    assert torch.equal(c.k[page(to), h, to % c.page], k0[page(fr), h, fr % c.page])


def test_evict_into_other_weights_and_layout(dev):
    c = ref.make(dev, [0, 0], [500, 900], hkv=2, page=16, layout="phd", seed=15)
    w = _weights_of(c, "ties")
    _check_evict(c, w, 200, 2, 20, weights_out=torch.full_like(w, 3.0))


# ------------------------------------------------------------------ store

def _check_store(dev, q_len, kv_len, *, D=128, hkv=2, group=3, page=16, dtype=F32, n_rot=None, sections=None, pairs="halves",
                 base=10000.0, scale=1.0, first=0, layout="hpd", in_place=False, q=True, seed=0):
    c = ref.make(dev, q_len, kv_len, D=D, hkv=hkv, group=group, page=page, dtype=dtype, seed=seed, layout=layout, tail=2)
    n_rot = D if n_rot is None else n_rot
    sections = [n_rot // 2] if sections is None else sections
    g = torch.Generator(device=dev).manual_seed(seed)
    T = c.q.shape[0]
    kn, vn = (torch.randn((T, hkv, D), generator=g, device=dev).to(dtype) for _ in range(2))
    pos = torch.stack([first + torch.randint(0, 3000, (T,), generator=g, device=dev) * (a + 1) for a in range(len(sections))]).int()
    k0, v0, q0 = c.k.clone(), c.v.clone(), c.q.clone()
    qo = c.q if in_place else torch.full_like(c.q, 7.0)
    rest = qo[c.T:].clone()
    kw = dict(q=c.q, q_out=qo) if q else {}
    mlz_b200.paged_store(ref.handle(c), kn, vn, positions=pos, sections=sections, n_rot=n_rot, pairs=pairs, freq_base=base,
                         freq_scale=scale, **kw)
    torch.cuda.synchronize()
    rk, rq = ref.rope(kn, pos, sections, n_rot, pairs, base, scale), ref.rope(q0, pos, sections, n_rot, pairs, base, scale)
    # a sine or cosine within 2^-22 (angle to 2^-25 of a half turn, the function 2 steps),
    # two products and a sum in f32, then one rounding to the output's type
    ew = lambda x, half: 2.0 ** -20 * x.double().abs().amax(dim=-1, keepdim=True) + half  # noqa: E731
    if q:
        _within(qo[:c.T], rq[:c.T], ew(q0, 0)[:c.T] + (2.0 ** -24 if dtype == F32 else 2.0 ** -11) * rq[:c.T].abs() + 2.0 ** -25, "q")
        assert torch.equal(qo[c.T:], rest)
    touched = torch.zeros(c.k.shape[:1] + c.k.shape[2:3], dtype=torch.bool, device=dev)
    for b, (a, n) in enumerate(zip(q_len, kv_len)):
        for i in range(a):
            slot, t = n - a + i, c.starts[b] + i
            if slot < 0:
                continue
            p, r = int(c.table[b, slot // page]), slot % page
            touched[p, r] = True
            _within(c.k[p, :, r], rk[t], (ew(kn, 0)[t] + 2.0 ** -11 * rk[t].abs() + 2.0 ** -25), "k")
            assert torch.equal(c.v[p, :, r], vn[t].half())
    same = ~touched[:, None, :, None].expand_as(c.k)
    assert torch.equal(c.k.view(torch.int16)[same], k0.view(torch.int16)[same])
    assert torch.equal(c.v.view(torch.int16)[same], v0.view(torch.int16)[same])


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("pairs", ["halves", "adjacent"])
@pytest.mark.parametrize("D,n_rot,sections", [(128, 128, [64]), (128, 128, [16, 24, 24]), (64, 64, [20, 12]), (256, 64, [8, 8, 8, 8]),
                                              (128, 40, [20]), (64, 8, [0, 4]), (128, 0, [0])])
def test_store(dev, D, n_rot, sections, pairs, dtype):
    _check_store(dev, [1, 7, 0, 30], [33, 7, 5, 70], D=D, n_rot=n_rot, sections=sections, pairs=pairs, dtype=dtype, seed=D + n_rot)


@pytest.mark.parametrize("first", [-5000, 10 ** 6, 2 ** 30])
def test_store_far_positions(dev, first):
    _check_store(dev, [20], [20], first=first, base=500000.0, seed=21)


def test_store_scaled_frequencies(dev):
    _check_store(dev, [20], [50], scale=0.25, base=1e6, seed=22)
    _check_store(dev, [20], [50], scale=-9.5, first=12345, seed=23)


def test_store_layouts_in_place_and_without_q(dev):
    _check_store(dev, [9, 1], [9, 80], layout="phd", in_place=True, seed=24)
    _check_store(dev, [9, 1], [9, 80], page=24, q=False, seed=25)
    _check_store(dev, [500], [700], hkv=5, group=1, page=64, seed=26)


def test_store_tokens_without_a_slot(dev):
    _check_store(dev, [6, 1], [4, 3], seed=27)


def test_store_bad_pages_are_not_written(dev):
    c = ref.make(dev, [2, 2], [20, 20], seed=28)
    k0 = c.k.clone()
    c.table[0, 1] = c.k.shape[0] + 3
    kn = torch.ones((4, c.hkv, c.D), device=dev)
    mlz_b200.paged_store(ref.handle(c), kn, kn)
    assert mlz_b200.device_errors(0) == mlz_b200.DEVERR_BAD_INDEX
    p = int(c.table[1, 1])
    changed = (c.k != k0) & ~(torch.isnan(c.k) & torch.isnan(k0))
    assert changed.any() and not changed[torch.arange(len(k0), device=dev) != p].any()


# ------------------------------------------------------------------ together

def _loop(dev, stream=None, graph=False):
    """A prompt in two chunks, an eviction, then decode steps: store, attend, accumulate."""
    D, hkv, group, page, budget = 64, 2, 2, 16, 40
    g = torch.Generator(device=dev).manual_seed(31)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    pools = [torch.zeros((20, hkv, page, D), dtype=F16, device=dev) for _ in range(2)]
    table = torch.arange(20, dtype=torch.int32, device=dev).reshape(2, 10)[:, torch.randperm(10)].contiguous()
    lens = torch.zeros(2, dtype=torch.int32, device=dev)
    start = torch.zeros(3, dtype=torch.int32, device=dev)
    acc = torch.zeros((2, hkv, 160), device=dev)
    cache = mlz_b200.PagedCache(*pools, table, lens, start)
    # the same cache as plain lists of rows
    K, V, W = ([[[] for _ in range(hkv)] for _ in range(2)] for _ in range(3))
    pos_of, worst = [0, 0], 0.0
    for step, q_len in enumerate([(50, 33), (20, 41), None, (1, 1), (1, 1), (3, 0), None, (1, 1)]):
        if q_len is None:
            mlz_b200.paged_evict(cache, acc, budget, n_sink=2, n_recent=8)
            for b in range(2):
                for h in range(hkv):
                    n = len(W[b][h])
                    row = acc_now[b, h, :n].tolist()
                    size = min(n, budget)
                    rank = sorted(range(n), key=lambda i: (not (i < 2 or i >= n - 8), -row[i], i))
                    stay = set(rank[:size])
                    mv = iter(sorted(i for i in stay if i >= size))
                    src = [i if i in stay else next(mv) for i in range(size)]
                    for L in (K, V, W):
                        L[b][h] = [L[b][h][i] for i in src]
            acc_now = acc.clone()
            continue
        T = sum(q_len)
        q, k, v = rnd(T, hkv * group, D), rnd(T, hkv, D), rnd(T, hkv, D)
        lens += torch.tensor(q_len, dtype=torch.int32, device=dev)
        start.copy_(torch.tensor([0, q_len[0], T], dtype=torch.int32))
        pos = torch.cat([torch.arange(pos_of[b], pos_of[b] + q_len[b]) for b in range(2)]).int().to(dev)
        qr = mlz_b200.paged_store(cache, k, v, q=q, positions=pos, n_rot=D)
        out, lse = mlz_b200.paged_attn(cache, qr, 0.2, return_lse=True)
        mlz_b200.paged_weights(cache, qr, lse, 0.2, acc=acc, out=acc)
        acc_now = acc.clone()
        rq, rk = ref.rope(q, pos[None], [D // 2], D, "halves", 1e4), ref.rope(k, pos[None], [D // 2], D, "halves", 1e4)
        t0 = 0
        for b in range(2):
            for i in range(q_len[b]):
                for h in range(hkv):
                    K[b][h].append(rk[t0 + i, h].half().double())
                    V[b][h].append(v[t0 + i, h].half().double())
                    W[b][h].append(0.0)
                    kk, vv = torch.stack(K[b][h]), torch.stack(V[b][h])
                    for r in range(group):
                        p = torch.softmax(kk @ rq[t0 + i, h * group + r] * 0.2, 0)
                        worst = max(worst, float((out[t0 + i, h * group + r].double() - p @ vv).abs().max()))
                        for j, x in enumerate(p.tolist()):
                            W[b][h][j] += x
            t0 += q_len[b]
            pos_of[b] += q_len[b]
        for b in range(2):
            for h in range(hkv):
                want = torch.tensor(W[b][h], device=dev, dtype=torch.float64)
                worst = max(worst, float((acc[b, h, :len(want)].double() - want).abs().max()))
                assert (acc[b, h, len(want):] == 0).all()
    return worst


def test_serving_loop(dev):
    # the rotated k's f32 value may fall to the other side of an f16 rounding than the 64-bit
    # one: a score moves by up to one step of one k component, 2^-10 * 4 * 4 * 0.2, a weight or
    # an output (|v| < 5) by the same share
    assert _loop(dev) < 5 * 2.0 ** -10 * 16 * 0.2


def test_calls_on_a_side_stream_and_captured(dev):
    """The three calls of a decode step on another stream, then captured in two graphs that
    share a workspace and replay with lengths that changed since."""
    c = ref.make(dev, [1, 1], [100, 60], seed=41)
    cache = ref.handle(c)
    want, lse0 = _attn(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out, lse = mlz_b200.paged_attn(cache, c.q, c.scale, return_lse=True, stream=side)
    w = mlz_b200.paged_weights(cache, c.q, lse, c.scale, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, lse0)
    ws = torch.empty(max(1, mlz_b200.paged_attn_workspace_bytes(cache, c.q)), dtype=torch.uint8, device=dev)
    outs = [torch.zeros_like(c.q) for _ in range(2)]
    accs = [torch.zeros_like(w) for _ in range(2)]
    graphs = []
    for o, a in zip(outs, accs):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            mlz_b200.paged_attn(cache, c.q, c.scale, out=o, lse=lse, workspace=ws)
            mlz_b200.paged_weights(cache, c.q, lse, c.scale, acc=a, out=a)
        graphs.append(gr)
    for gr in graphs + graphs:
        gr.replay()
    torch.cuda.synchronize()
    for o, a in zip(outs, accs):
        assert torch.equal(o, want)
        assert torch.allclose(a, 2 * w, rtol=2.0 ** -22, atol=0)
    c.lens.sub_(13)
    c.kv_len = [n - 13 for n in c.kv_len]
    graphs[1].replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    w_out, _, e_out, _ = ref.attn(c)
    for o in outs:
        _within(o, w_out, e_out, "replayed")


def test_attn_without_tokens(dev):
    c = ref.make(dev, [0, 0], [40, 9], seed=43)
    out, lse = mlz_b200.paged_attn(ref.handle(c), c.q[:0], c.scale, return_lse=True)
    assert out.shape == (0,) + c.q.shape[1:] and lse.shape[0] == 0


def test_two_streams_at_once(dev):
    """Attention, weights and eviction of two caches on two streams, again and again with nothing
    between them: the same bits as one after the other."""
    cs = [ref.make(dev, [1, 90, 3], [900, 300, 2000], hkv=2, page=16, dtype=t, seed=51 + i) for i, t in enumerate((F32, F16))]
    streams = [torch.cuda.Stream() for _ in cs]

    def step(c, stream):
        h = ref.handle(c)
        out, lse = mlz_b200.paged_attn(h, c.q, c.scale, return_lse=True, stream=stream)
        w = mlz_b200.paged_weights(h, c.q, lse, c.scale, stream=stream)
        kept, wo, _ = mlz_b200.paged_evict(h, w, 500, n_sink=2, n_recent=9, weights_out=acc[id(c)], kv_len_out=spare[id(c)], stream=stream)
        return out[:c.T], lse[:c.T], w, kept

    acc = {id(c): torch.zeros((3, 2, c.cap), device=dev) for c in cs}
    spare = {id(c): c.lens.clone() for c in cs}
    pools = [(c.k.clone(), c.v.clone()) for c in cs]

    def restore(c, p):
        c.k.copy_(p[0])
        c.v.copy_(p[1])

    want = []
    for c, p in zip(cs, pools):
        want.append(step(c, None))
        torch.cuda.synchronize()
        restore(c, p)
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for c, p, st in zip(cs, pools, streams):
            got.append(step(c, st))
            with torch.cuda.stream(st):
                restore(c, p)
        for st in streams:
            st.synchronize()
        for g, x in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, x))
