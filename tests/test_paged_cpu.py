"""CPU: the paged-cache entry points refuse what they do not take, with a status and a message
that names it, before they touch a device."""
import ctypes as C

import pytest
import torch

import mlz_b200
from mlz_b200 import _lib

INVALID, UNSUPPORTED, NOMEM = -1, -2, -4
P = 1 << 20   # an aligned address that nothing reads


def cache(**kw):
    d = _lib.PagedCacheDesc()
    d.kv_type, d.page_size, d.n_pages, d.head_dim = 1, 16, 10, 128
    d.n_head_kv, d.batch_size, d.max_pages, d.n_tokens = 2, 3, 4, 5
    d.k = d.v = d.block_table = d.kv_len = d.q_start = P
    for nb in (d.k_nb, d.v_nb):
        nb[:] = (2, 256, 16 * 256, 2 * 16 * 256)
    d.block_table_nb = 16
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(d, k)[:] = v
        else:
            setattr(d, k, v)
    return d


def attn(**kw):
    d = _lib.PagedAttnDesc()
    d.type, d.n_head_q, d.scale = 0, 8, 0.1
    d.q = d.dst = d.lse = P
    d.q_nb[:] = d.dst_nb[:] = (4, 512, 8 * 512)
    d.lse_nb[:] = (4, 32)
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(d, k)[:] = v
        else:
            setattr(d, k, v)
    return d


def store(**kw):
    d = _lib.PagedStoreDesc()
    d.type, d.pairs, d.n_rot, d.n_axes, d.freq_base, d.freq_scale = 0, 1, 128, 2, 10000.0, 1.0
    d.sections[:2] = (40, 24)
    d.positions, d.positions_nb, d.n_head_q = P, 20, 8
    d.q = d.k = d.v = d.q_dst = P
    d.q_nb[:] = d.q_dst_nb[:] = (4, 512, 8 * 512)
    d.k_nb[:] = d.v_nb[:] = (4, 512, 2 * 512)
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(d, k)[:len(v)] = v
        else:
            setattr(d, k, v)
    return d


def evict(**kw):
    d = _lib.PagedEvictDesc()
    d.budget, d.n_sink, d.n_recent = 32, 2, 8
    d.weights, d.weights_out, d.kept, d.kv_len_out = P, 2 * P, P, P
    d.weights_nb[:] = d.weights_out_nb[:] = (4, 256, 512)
    d.kept_nb[:] = (4, 128, 256)
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(d, k)[:] = v
        else:
            setattr(d, k, v)
    return d


def calls(c):
    """Every entry point on one cache descriptor."""
    L = mlz_b200.lib()
    n = C.c_size_t(0)
    nb = (C.c_size_t * 3)(4, 256, 512)
    yield L.mlzc_paged_store_dev(C.byref(c), C.byref(store()), None)
    yield L.mlzc_paged_attn_workspace_bytes(C.byref(c), C.byref(attn()), C.byref(n))
    yield L.mlzc_paged_attn_dev(C.byref(c), C.byref(attn()), None, 0, None)
    yield L.mlzc_paged_weights_workspace_bytes(C.byref(c), C.byref(attn()), C.byref(n))
    yield L.mlzc_paged_weights_dev(C.byref(c), C.byref(attn()), None, nb, P, nb, None, 0, None)
    yield L.mlzc_paged_evict_workspace_bytes(C.byref(c), C.byref(evict()), C.byref(n))
    yield L.mlzc_paged_evict_dev(C.byref(c), C.byref(evict()), None, 0, None)


@pytest.mark.parametrize("kw,status,says", [
    (dict(kv_type=8), UNSUPPORTED, "type 8"), (dict(head_dim=96), UNSUPPORTED, "head_dim 96"),
    (dict(page_size=12), UNSUPPORTED, "page_size 12"), (dict(page_size=0), UNSUPPORTED, "page_size 0"),
    (dict(page_size=-8), UNSUPPORTED, "page_size -8"),
    (dict(n_pages=0), INVALID, "dimension"), (dict(batch_size=0), INVALID, "dimension"), (dict(max_pages=0), INVALID, "dimension"),
    (dict(n_head_kv=-1), INVALID, "dimension"), (dict(max_pages=1 << 28), INVALID, "too large"),
    (dict(k=None), INVALID, "null"), (dict(kv_len=None), INVALID, "null"), (dict(k=P + 8), INVALID, "16-byte"),
    (dict(k_nb=(4, 256, 4096, 8192)), INVALID, "contiguous"), (dict(v_nb=(2, 264, 4096, 8192)), INVALID, "stride 1"),
    (dict(v_nb=(2, 256, 0, 8192)), INVALID, "stride 2"), (dict(k_nb=(2, 128, 4096, 8192)), INVALID, "stride 1"),
    (dict(k_nb=(2, 256, 4096, 1 << 41)), INVALID, "stride 3"), (dict(block_table_nb=12), INVALID, "table"),
    (dict(block_table=P + 2), INVALID, "misaligned")])
def test_cache_refusals(kw, status, says):
    for st in calls(cache(**kw)):
        assert st == status and says in mlz_b200.last_error(), mlz_b200.last_error()


@pytest.mark.parametrize("kw,status,says", [
    (dict(type=12), UNSUPPORTED, "type 12"), (dict(mode=8), UNSUPPORTED, "mode 0x8"), (dict(n_head_q=7), UNSUPPORTED, "7 query"),
    (dict(n_head_q=0), UNSUPPORTED, "0 query"), (dict(n_head_q=2 * 129), UNSUPPORTED, "258 query"), (dict(scale=0.0), INVALID, "scale"),
    (dict(scale=float("nan")), INVALID, "scale"), (dict(scale=float("inf")), INVALID, "scale"), (dict(mode=16), INVALID, "softcap"),
    (dict(q=None), INVALID, "null"), (dict(q=P + 4), INVALID, "16-byte"), (dict(q_nb=(2, 512, 4096)), INVALID, "contiguous"),
    (dict(q_nb=(4, 256, 4096)), INVALID, "head stride"), (dict(q_nb=(4, 512, 4100)), INVALID, "token stride"),
    (dict(lse=P + 2), INVALID, "lse"), (dict(lse_nb=(6, 32)), INVALID, "lse"), (dict(lse_nb=(4, 0)), INVALID, "lse")])
def test_attn_refusals(kw, status, says):
    L, n, nb = mlz_b200.lib(), C.c_size_t(0), (C.c_size_t * 3)(4, 256, 512)
    c, d = cache(), attn(**kw)
    for st in (L.mlzc_paged_attn_workspace_bytes(C.byref(c), C.byref(d), C.byref(n)),
               L.mlzc_paged_attn_dev(C.byref(c), C.byref(d), None, 0, None),
               L.mlzc_paged_weights_workspace_bytes(C.byref(c), C.byref(d), C.byref(n)),
               L.mlzc_paged_weights_dev(C.byref(c), C.byref(d), None, nb, P, nb, None, 0, None)):
        assert st == status and says in mlz_b200.last_error(), mlz_b200.last_error()


@pytest.mark.parametrize("kw,says", [(dict(scale=2.0 ** -41), "scale"), (dict(scale=2.0 ** 41), "scale"),
                                     (dict(mode=16, logit_softcap=2.0 ** -41), "softcap"), (dict(mode=16, logit_softcap=2.0 ** 41), "softcap")])
def test_scales_outside_f32s_room_are_refused(kw, says):
    """Products of such a scale with scores, or its inverse, would leave f32."""
    L = mlz_b200.lib()
    assert L.mlzc_paged_attn_dev(C.byref(cache()), C.byref(attn(**kw)), None, 0, None) == INVALID and says in mlz_b200.last_error()


def test_rotation_in_place_with_other_strides_is_refused():
    L = mlz_b200.lib()
    for nb in ((4, 1024, 8 * 1024), (4, 512, 16 * 512)):
        assert L.mlzc_paged_store_dev(C.byref(cache()), C.byref(store(q_dst_nb=nb)), None) == INVALID
        assert "in place" in mlz_b200.last_error()


def test_attn_and_weights_own_refusals():
    L, nb = mlz_b200.lib(), (C.c_size_t * 3)(4, 256, 512)
    c = cache()
    assert L.mlzc_paged_attn_dev(C.byref(c), C.byref(attn(dst=None)), None, 0, None) == INVALID
    assert L.mlzc_paged_attn_dev(C.byref(c), None, None, 0, None) == INVALID
    assert L.mlzc_paged_attn_dev(None, C.byref(attn()), None, 0, None) == INVALID
    assert L.mlzc_paged_attn_workspace_bytes(C.byref(c), C.byref(attn()), None) == INVALID
    w = lambda d, acc, anb, out, onb: L.mlzc_paged_weights_dev(C.byref(c), C.byref(d), acc, anb, out, onb, None, 0, None)  # noqa: E731
    assert w(attn(lse=None), None, None, P, nb) == INVALID
    assert w(attn(), None, None, None, nb) == INVALID
    assert w(attn(), None, None, P, (C.c_size_t * 3)(8, 256, 512)) == INVALID
    assert w(attn(), None, None, P, (C.c_size_t * 3)(4, 252, 512)) == INVALID
    assert w(attn(), P, (C.c_size_t * 3)(4, 256, 1024), P, nb) == INVALID and "in place" in mlz_b200.last_error()
    for kw in (dict(n_tokens=-1), dict(q_start=None), dict(n_tokens=1 << 31)):
        assert L.mlzc_paged_attn_dev(C.byref(cache(**kw)), C.byref(attn()), None, 0, None) == INVALID
        assert L.mlzc_paged_store_dev(C.byref(cache(**kw)), C.byref(store()), None) == INVALID


@pytest.mark.parametrize("kw,says", [
    (dict(type=7), "type 7"), (dict(pairs=2), "pairs"), (dict(n_rot=12), "n_rot"), (dict(n_rot=136), "n_rot"), (dict(n_rot=-8), "n_rot"),
    (dict(n_axes=0), "n_axes"), (dict(n_axes=5), "n_axes"), (dict(sections=(40, 20)), "sections"), (dict(sections=(70, -6)), "negative"),
    (dict(freq_base=0.0), "freq_base"), (dict(freq_scale=float("nan")), "freq_scale"), (dict(positions=None), "positions"),
    (dict(positions_nb=16), "positions"), (dict(k=None), "k: null"), (dict(v=P + 4), "v: rows"), (dict(q_dst=None), "q_dst"),
    (dict(q_nb=(4, 512, 2048 + 8)), "q: token"), (dict(n_head_q=-1), "n_head_q")])
def test_store_refusals(kw, says):
    st = mlz_b200.lib().mlzc_paged_store_dev(C.byref(cache()), C.byref(store(**kw)), None)
    assert st in (INVALID, UNSUPPORTED) and says in mlz_b200.last_error(), mlz_b200.last_error()


@pytest.mark.parametrize("kw,says", [
    (dict(budget=0), "budget"), (dict(n_sink=-1), "n_sink"), (dict(n_sink=30), "n_sink"), (dict(n_recent=1 << 62, n_sink=1 << 62), "n_sink"),
    (dict(weights=None), "weights"), (dict(weights_out_nb=(4, 252, 512)), "weights_out"), (dict(kept=P + 1), "kept"),
    (dict(kept_nb=(4, 100, 256)), "kept"), (dict(kv_len_out=None), "kv_len_out"), (dict(weights_out=P, weights_out_nb=(4, 256, 1024)), "in place")])
def test_evict_refusals(kw, says):
    st = mlz_b200.lib().mlzc_paged_evict_dev(C.byref(cache()), C.byref(evict(**kw)), P, 1 << 20, None)
    assert st == INVALID and says in mlz_b200.last_error(), mlz_b200.last_error()


def test_evict_workspace():
    L, n, c, d = mlz_b200.lib(), C.c_size_t(0), cache(q_start=None), evict()
    assert L.mlzc_paged_evict_workspace_bytes(C.byref(c), C.byref(d), C.byref(n)) == 0
    assert n.value >= 3 * 2 * 32 * 4
    assert L.mlzc_paged_evict_dev(C.byref(c), C.byref(d), None, 0, None) == NOMEM
    assert L.mlzc_paged_evict_dev(C.byref(c), C.byref(d), P, n.value - 1, None) == NOMEM
    assert L.mlzc_paged_evict_dev(C.byref(c), C.byref(d), P + 4, n.value, None) == INVALID


def test_no_tokens_needs_no_device():
    L, c = mlz_b200.lib(), cache(n_tokens=0)
    assert L.mlzc_paged_attn_dev(C.byref(c), C.byref(attn(q=None, dst=None)), None, 0, None) == 0
    assert L.mlzc_paged_store_dev(C.byref(c), C.byref(store(q=None, k=None, v=None, positions=None)), None) == 0


def test_handle_refusals():
    k = torch.zeros((4, 2, 16, 64), dtype=torch.float16)
    t, n, s = torch.zeros((1, 3), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for args, e in (((k, k[:3], t, n, s), ValueError), ((k.float(), k.float(), t, n, s), TypeError), ((k, k, t.long(), n, s), TypeError),
                    ((k, k, t, torch.zeros(2, dtype=torch.int32), s), ValueError), ((k, k, t, n, n), ValueError),
                    ((k, k, t[0], n, s), ValueError), ((k, k, t, n, s), ValueError)):   # the last: not on a CUDA device
        with pytest.raises(e):
            mlz_b200.PagedCache(*args)
