"""The paged KV cache: the mlzc_paged_* entry points over torch device tensors.

A :class:`PagedCache` names the pools, the block table and the lengths of a batch; the calls
work on it in a serving loop's order: :func:`paged_store` (rotary positions, new K and V into
the pages), :func:`paged_attn` (attention of the new tokens over their sequences' slots),
:func:`paged_weights` (attention weight received by each slot) and :func:`paged_evict` (the
cache cut down to its heaviest slots).  include/mlzc.h states each operation.

Every call runs on the cache's device; ``stream`` is a torch stream or a raw handle, by
default that device's current stream.  No counterpart in the reference, whose attention reads
one contiguous cache (src/simd/flash_attention.h:65-114).
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from ._lib import (FA_MODE_SOFTCAP, ROPE_ADJACENT, ROPE_HALVES, TYPE_F16, TYPE_F32, PagedAttnDesc, PagedCacheDesc,
                   PagedEvictDesc, PagedStoreDesc, check, lib)

_F32, _F16, _I32, _U8 = torch.float32, torch.float16, torch.int32, torch.uint8
# the descriptors, packed in one go (a field by field fill costs more than a small kernel runs)
_ATTN = struct.Struct("iIqff2Q3Q3QQ2Q")
_STORE = struct.Struct("8i2fQQq4Q12Q")
_EVICT = struct.Struct("3q2Q6QQ3QQ")
assert [x.size for x in (_ATTN, _STORE, _EVICT)] == [C.sizeof(x) for x in (PagedAttnDesc, PagedStoreDesc, PagedEvictDesc)]


# the current stream's handle by device index (current_stream builds a Stream object around it)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


class _Launch:
    """The device and stream of one call, and where its outputs and workspaces come from: torch
    hands their memory to nobody else until the call's stream is past it."""

    __slots__ = ("device", "other", "given", "handle")

    def __init__(self, device, stream):
        self.device = device
        self.other = torch.cuda.current_device() != device.index
        self.given = None
        if stream is None:
            self.handle = _raw_stream(device.index)
        elif hasattr(stream, "cuda_stream"):
            self.given, self.handle = stream, stream.cuda_stream
        else:
            self.handle = int(stream)
            self.given = torch.cuda.ExternalStream(self.handle, device=device) if self.handle else torch.cuda.default_stream(device)

    def empty(self, shape, dtype, like):
        """An uninitialised tensor beside `like` (new_empty costs half of torch.empty here)."""
        if self.given is None:
            return like.new_empty(shape, dtype=dtype)
        with torch.cuda.stream(self.given):
            return torch.empty(shape, dtype=dtype, device=self.device)

    def run(self, f, *args):
        if self.other:
            with torch.cuda.device(self.device):
                return check(f(*args))
        return check(f(*args))


def _rows(what, t, cache, heads, dtype=None):
    """Checks a packed (tokens, heads, head_dim) tensor; its byte strides element, head, token."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != cache.head_dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{what}: shape {tuple(shape)}, expected (tokens, {heads or 'heads'}, {cache.head_dim})")
    if t.device != cache.device:
        raise ValueError(f"{what} is on {t.device}, the cache on {cache.device}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{what}: {t.dtype}, expected {dtype}")
    e = t.element_size()
    st = t.stride()
    return st[2] * e, st[1] * e, st[0] * e


def _type_of(what, t):
    if t.dtype == _F32:
        return TYPE_F32
    if t.dtype == _F16:
        return TYPE_F16
    raise TypeError(f"{what}: {t.dtype}, expected float32 or float16")


def _table(what, t, cache, last, dtype):
    """Checks a (batch, n_head_kv, >= last) table; its byte strides entry, head, sequence."""
    shape = t.shape
    if len(shape) != 3 or shape[0] != cache.batch or shape[1] != cache.n_head_kv or shape[2] < last:
        raise ValueError(f"{what}: shape {tuple(shape)}, expected ({cache.batch}, {cache.n_head_kv}, {last})")
    if t.dtype != dtype or t.device != cache.device:
        raise TypeError(f"{what}: {t.dtype} on {t.device}, expected {dtype} on {cache.device}")
    st = t.stride()
    return st[2] * 4, st[1] * 4, st[0] * 4


class PagedCache:
    """Handle of a paged KV cache.

    k, v: pools (n_pages, n_head_kv, page_size, head_dim) float16 (any strides with contiguous
    rows; a pool laid out (n_pages, page_size, n_head_kv, head_dim) is passed transposed).
    block_table: (batch, max_pages) int32; kv_len: (batch,) int32, slots of each sequence with
    its new tokens; q_start: (batch + 1,) int32, first packed row of each sequence's new tokens.
    The handle keeps references; the kernels read block_table, kv_len and q_start at each call,
    so their contents may change between calls.
    """

    def __init__(self, k, v, block_table, kv_len, q_start=None):
        if k.dim() != 4 or v.shape != k.shape:
            raise ValueError(f"pools {tuple(k.shape)} and {tuple(v.shape)}: expected two (pages, heads, rows, head_dim)")
        if k.dtype != _F16 or v.dtype != _F16:
            raise TypeError(f"pools: {k.dtype}, {v.dtype}, expected float16")
        if block_table.dim() != 2 or block_table.stride(1) != 1:
            raise ValueError("block_table: expected (batch, max_pages) with contiguous rows")
        B = block_table.shape[0]
        for what, t, n in (("kv_len", kv_len, B), ("q_start", q_start, B + 1)):
            if t is not None and (tuple(t.shape) != (n,) or not t.is_contiguous()):
                raise ValueError(f"{what}: expected a contiguous ({n},) tensor, got {tuple(t.shape)}")
        for what, t in (("block_table", block_table), ("kv_len", kv_len), ("q_start", q_start)):
            if t is not None and t.dtype != torch.int32:
                raise TypeError(f"{what}: {t.dtype}, expected int32")
        for t in (v, block_table, kv_len, q_start):
            if t is not None and t.device != k.device:
                raise ValueError(f"cache tensors on {k.device} and {t.device}")
        if k.device.type != "cuda":
            raise ValueError(f"cache on {k.device}: expected a CUDA device")
        self.k, self.v, self.block_table, self.kv_len, self.q_start = k, v, block_table, kv_len, q_start
        self.device, self.batch, self.max_pages = k.device, B, block_table.shape[1]
        self.n_pages, self.n_head_kv, self.page_size, self.head_dim = k.shape
        self.capacity = self.max_pages * self.page_size
        d = self._desc = PagedCacheDesc()
        d.kv_type, d.page_size, d.n_pages, d.head_dim = TYPE_F16, self.page_size, self.n_pages, self.head_dim
        d.n_head_kv, d.batch_size, d.max_pages = self.n_head_kv, B, self.max_pages
        d.k, d.v = k.data_ptr(), v.data_ptr()
        for nb, t in ((d.k_nb, k), (d.v_nb, v)):
            nb[:] = [t.stride(i) * 2 for i in (3, 2, 1, 0)]
        d.block_table, d.block_table_nb = block_table.data_ptr(), block_table.stride(0) * 4
        d.kv_len = kv_len.data_ptr()
        d.q_start = q_start.data_ptr() if q_start is not None else None

        self._last = (-1, None)
        self._sizes = {}

    def _with(self, n_tokens):
        """The descriptor of a call with so many packed rows."""
        n, d = self._last
        if n != n_tokens:
            d = PagedCacheDesc.from_buffer_copy(self._desc)
            d.n_tokens = n_tokens
            self._last = (n_tokens, d)
        return d

    def _workspace(self, L, query, key, *args):
        """Bytes of workspace by the sizes that decide them (the library's answer, asked once)."""
        n = self._sizes.get(key)
        if n is None:
            out = C.c_size_t(0)
            L.run(query, *args, C.byref(out))
            if len(self._sizes) >= 64:
                self._sizes.clear()
            n = self._sizes[key] = out.value
        return n


def paged_store(cache, k, v, *, q=None, q_out=None, positions=None, sections=None, n_rot=0, pairs="halves",
                freq_base=10000.0, freq_scale=1.0, stream=None):
    """Writes new tokens' k and v (tokens, n_head_kv, head_dim) float32 / float16 into the cache,
    k rotated; q (tokens, n_head_q, head_dim) is rotated into q_out (made if None; may be q)
    and returned.  positions: (axes, tokens) or (tokens,) int32; sections: pairs of each axis,
    n_rot / 2 in all (one axis: may be None); pairs: "halves" (j, j + n_rot / 2) or "adjacent"
    (2j, 2j + 1)."""
    T = k.shape[0]
    kind = _type_of("k", k)
    if pairs not in ("halves", "adjacent"):
        raise ValueError(f"pairs {pairs!r}: expected 'halves' or 'adjacent'")
    knb = _rows("k", k, cache, cache.n_head_kv)
    vnb = _rows("v", v, cache, cache.n_head_kv, k.dtype)
    if v.shape[0] != T or (q is not None and q.shape[0] != T):
        raise ValueError("k, v and q differ in their tokens")
    n_axes, sec, pos, pos_nb = 0, (0, 0, 0, 0), 0, 0
    if n_rot:
        if positions is None:
            raise ValueError("n_rot without positions")
        if positions.dim() == 1:
            positions = positions[None]
        if positions.dtype != _I32 or positions.device != cache.device:
            raise TypeError(f"positions: {positions.dtype} on {positions.device}, expected int32 on {cache.device}")
        sec = (n_rot // 2,) if sections is None else tuple(sections)
        n_axes = len(sec)
        if positions.dim() != 2 or positions.shape[1] != T or positions.shape[0] != n_axes:
            raise ValueError(f"positions {tuple(positions.shape)}: expected ({n_axes}, {T})")
        if T > 1 and positions.stride(1) != 1:
            raise ValueError("positions of an axis must be contiguous")
        if n_axes > 4:
            raise ValueError("at most 4 position axes")
        sec += (0,) * (4 - n_axes)
        pos, pos_nb = positions.data_ptr(), positions.stride(0) * 4
    L = _Launch(cache.device, stream)
    hq, qp, qo, qnb, onb = 0, 0, 0, (0, 0, 0), (0, 0, 0)
    if q is not None:
        hq, qnb = q.shape[1], _rows("q", q, cache, None, k.dtype)
        if q_out is None:
            q_out = L.empty(q.shape, q.dtype, q)
        if q_out.shape != q.shape:
            raise ValueError(f"q_out {tuple(q_out.shape)}, q {tuple(q.shape)}")
        onb = _rows("q_out", q_out, cache, None, k.dtype)
        qp, qo = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q")
    d = PagedStoreDesc.from_buffer_copy(_STORE.pack(
        kind, ROPE_HALVES if pairs == "halves" else ROPE_ADJACENT, n_rot, n_axes, *sec, freq_base, freq_scale, pos, pos_nb, hq,
        qp, k.data_ptr(), v.data_ptr(), qo, *qnb, *knb, *vnb, *onb))
    L.run(lib().mlzc_paged_store_dev, C.byref(cache._with(T)), C.byref(d), L.handle)
    return q_out


def _attn_desc(cache, q, scale, softcap, out=None, lse=None):
    """Descriptor of the attention and weights calls, its tensors checked."""
    kind = _type_of("q", q)
    qnb = _rows("q", q, cache, None)
    dst, dnb, lp, lnb = 0, (0, 0, 0), 0, (0, 0)
    if out is not None:
        if out.shape != q.shape:
            raise ValueError(f"out {tuple(out.shape)}, q {tuple(q.shape)}")
        dst, dnb = out.data_ptr(), _rows("out", out, cache, None, q.dtype)
    if lse is not None:
        if lse.shape != q.shape[:2] or lse.dtype != _F32 or lse.device != cache.device:
            raise ValueError(f"lse: {lse.dtype} {tuple(lse.shape)} on {lse.device}, expected float32 {tuple(q.shape[:2])} on {cache.device}")
        st = lse.stride()
        lp, lnb = lse.data_ptr(), (st[1] * 4, st[0] * 4)
    return PagedAttnDesc.from_buffer_copy(_ATTN.pack(kind, FA_MODE_SOFTCAP if softcap else 0, q.shape[1], scale, softcap,
                                                     q.data_ptr(), dst, *qnb, *dnb, lp, *lnb))


def _given(workspace, need, L, like):
    """(pointer, bytes, owner) of the caller's workspace, or of one made here."""
    if workspace is None:
        if not need:
            return None, 0, None
        workspace = L.empty(need, _U8, like)
    elif workspace.device != L.device or not workspace.is_contiguous():
        raise ValueError(f"workspace: a contiguous tensor on {L.device} is expected")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size(), workspace


def paged_attn_workspace_bytes(cache, q, scale=1.0, *, softcap=0.0):
    """Bytes of workspace that :func:`paged_attn` needs for these tensors."""
    L = _Launch(cache.device, None)
    d = _attn_desc(cache, q, scale, softcap, q)
    return cache._workspace(L, lib().mlzc_paged_attn_workspace_bytes, ("attn", q.shape[0], q.shape[1], q.dtype),
                            C.byref(cache._with(q.shape[0])), C.byref(d))


def paged_attn(cache, q, scale, *, softcap=0.0, out=None, lse=None, return_lse=False, workspace=None, stream=None):
    """Attention of the new tokens q (tokens, n_head_q, head_dim), float32 or float16, over
    their sequences' slots: out of q's shape and type; with lse given (tokens, n_head_q)
    float32 or return_lse, (out, lse).  Rows that belong to no sequence are left as they were."""
    L = _Launch(cache.device, stream)
    if out is None:
        out = L.empty(q.shape, q.dtype, q)
    if lse is None and return_lse:
        lse = L.empty(q.shape[:2], _F32, q)
    d = C.byref(_attn_desc(cache, q, scale, softcap, out, lse))
    T = q.shape[0]
    cd = C.byref(cache._with(T))
    need = cache._workspace(L, lib().mlzc_paged_attn_workspace_bytes, ("attn", T, q.shape[1], q.dtype), cd, d)
    ws, n, owner = _given(workspace, need, L, q)
    L.run(lib().mlzc_paged_attn_dev, cd, d, ws, n, L.handle)
    return (out, lse) if lse is not None else out


def paged_weights_workspace_bytes(cache, q, scale=1.0, *, softcap=0.0):
    """Bytes of workspace that :func:`paged_weights` needs for these tensors."""
    L = _Launch(cache.device, None)
    d = _attn_desc(cache, q, scale, softcap)
    d.lse, d.lse_nb[:] = q.data_ptr(), (4, 4 * q.shape[1])   # any lse: its place does not change the size
    return cache._workspace(L, lib().mlzc_paged_weights_workspace_bytes, ("weights", q.shape[0], q.shape[1], q.dtype),
                            C.byref(cache._with(q.shape[0])), C.byref(d))


def paged_weights(cache, q, lse, scale, *, softcap=0.0, acc=None, out=None, workspace=None, stream=None):
    """Attention weight that each slot received from the new tokens, summed over them and the
    query heads of each kv head, added to acc (batch, n_head_kv, capacity) float32 (None: from
    0): out (acc itself to accumulate in place; made, with zeros past kv_len, if None).  q,
    scale, softcap and lse as given to and returned by :func:`paged_attn`."""
    L = _Launch(cache.device, stream)
    d = C.byref(_attn_desc(cache, q, scale, softcap, None, lse))
    if out is None:
        out = L.empty((cache.batch, cache.n_head_kv, cache.capacity), _F32, q)
        if L.given is None:
            out.zero_()
        else:
            with torch.cuda.stream(L.given):
                out.zero_()
    nb = C.c_size_t * 3
    onb = nb(*_table("out", out, cache, cache.capacity, _F32))
    anb = nb(*_table("acc", acc, cache, cache.capacity, _F32)) if acc is not None else None
    T = q.shape[0]
    cd = C.byref(cache._with(T))
    need = cache._workspace(L, lib().mlzc_paged_weights_workspace_bytes, ("weights", T, q.shape[1], q.dtype), cd, d)
    ws, n, owner = _given(workspace, need, L, q)
    L.run(lib().mlzc_paged_weights_dev, cd, d, acc.data_ptr() if acc is not None else None, anb, out.data_ptr(), onb, ws, n, L.handle)
    return out


def paged_evict_workspace_bytes(cache, budget):
    """Bytes of workspace that :func:`paged_evict` needs for this cache and budget."""
    d = PagedEvictDesc()
    d.budget = budget
    return cache._workspace(_Launch(cache.device, None), lib().mlzc_paged_evict_workspace_bytes, ("evict", budget),
                            C.byref(cache._desc), C.byref(d))


def paged_evict(cache, weights, budget, *, n_sink=0, n_recent=0, weights_out=None, kept=None, kv_len_out=None,
                workspace=None, stream=None):
    """Cuts each sequence down to `budget` slots a head by weights (batch, n_head_kv, capacity)
    float32, keeping the first n_sink and the last n_recent.  Returns (kept, weights_out,
    kv_len): kept (batch, n_head_kv, budget) int32 the former slot of each slot (-1 past the
    new length), weights_out the kept slots' weights (weights itself unless given), kv_len the
    new lengths (cache.kv_len itself is updated unless kv_len_out is given)."""
    L = _Launch(cache.device, stream)
    if weights_out is None:
        weights_out = weights
    if kept is None:
        kept = L.empty((cache.batch, cache.n_head_kv, budget), _I32, weights)
    if kv_len_out is None:
        kv_len_out = cache.kv_len
    if tuple(kv_len_out.shape) != (cache.batch,) or kv_len_out.dtype != _I32 or not kv_len_out.is_contiguous() or \
            kv_len_out.device != cache.device:
        raise ValueError("kv_len_out: expected a contiguous (batch,) int32 tensor beside the cache")
    d = C.byref(PagedEvictDesc.from_buffer_copy(_EVICT.pack(
        budget, n_sink, n_recent, weights.data_ptr(), weights_out.data_ptr(), *_table("weights", weights, cache, cache.capacity, _F32),
        *_table("weights_out", weights_out, cache, cache.capacity, _F32), kept.data_ptr(), *_table("kept", kept, cache, budget, _I32),
        kv_len_out.data_ptr())))
    cd = C.byref(cache._desc)
    ws, n, owner = _given(workspace, cache._workspace(L, lib().mlzc_paged_evict_workspace_bytes, ("evict", budget), cd, d), L, weights)
    L.run(lib().mlzc_paged_evict_dev, cd, d, ws, n, L.handle)
    return kept, weights_out, kv_len_out


__all__ = ["PagedCache", "paged_store", "paged_attn", "paged_attn_workspace_bytes", "paged_weights",
           "paged_weights_workspace_bytes", "paged_evict", "paged_evict_workspace_bytes"]
