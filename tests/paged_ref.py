"""Plain 64-bit forms of the paged-cache operators, and the cases' tensors, for the tests.

Everything is a loop over sequences and heads in float64 (torch, on the inputs' device); the
bounds on a kernel's error follow from its number formats (see ``attn_bounds``).
"""
import math
from types import SimpleNamespace

import torch

HALF16 = 2.0 ** -11      # half a step of f16, relative
HALF32 = 2.0 ** -24      # half a step of f32


def make(dev, q_len, kv_len, *, hkv=2, group=4, D=128, page=16, dtype=torch.float32, seed=0, layout="hpd", spare=2,
         junk=True, tail=0, q_scale=1.5):
    """A cache with shuffled pages and the packed q of a ragged batch.  junk: rows past each
    sequence's length, and pages of nobody, hold NaN; table entries past the needed pages are
    far out of range.  tail: packed rows that belong to no sequence."""
    g = torch.Generator().manual_seed(1000 + seed)
    B = len(kv_len)
    need = [-(-n // page) for n in kv_len]
    n_pages, max_pages = sum(need) + spare, max(1, max(need)) + 1
    order = torch.randperm(n_pages, generator=g)
    table = torch.full((B, max_pages), 1 << 30, dtype=torch.int32)
    shape = (n_pages, hkv, page, D)
    k, v = (torch.randn(shape, generator=g) for _ in range(2))
    k, v = k.half(), v.half()
    used = torch.zeros((n_pages, page), dtype=torch.bool)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].int()
        at += n
        for j in range(kv_len[b]):
            used[table[b, j // page], j % page] = True
    if junk:
        for pool in (k, v):
            pool.masked_fill_(~used[:, None, :, None], float("nan"))
    T = sum(q_len)
    q = (torch.randn((T + tail, hkv * group, D), generator=g) * q_scale).to(dtype)
    starts = [0]
    for n in q_len:
        starts.append(starts[-1] + n)
    put = lambda t: t.to(dev)  # noqa: E731
    if layout == "phd":   # rows of all heads of a token together
        k, v = (put(t.transpose(1, 2).contiguous()).transpose(1, 2) for t in (k, v))
    else:
        k, v = put(k), put(v)
    c = SimpleNamespace(q_len=list(q_len), kv_len=list(kv_len), hkv=hkv, group=group, D=D, page=page, starts=starts, T=T,
                        k=k, v=v, q=put(q), table=put(table), lens=put(torch.tensor(kv_len, dtype=torch.int32)),
                        q_start=put(torch.tensor(starts, dtype=torch.int32)), scale=1.0 / math.sqrt(D), cap=max_pages * page)
    return c


def handle(c):
    import mlz_b200
    return mlz_b200.PagedCache(c.k, c.v, c.table, c.lens, c.q_start)


def rows(c, pool, b, h):
    """The slots of (sequence, head) in float64."""
    n = c.kv_len[b]
    if n == 0:
        return torch.zeros((0, c.D), dtype=torch.float64, device=pool.device)
    ids = c.table[b, :-(-n // c.page)].long()
    return pool[ids, h].reshape(-1, c.D)[:n].double()


def score_rows(c, b, h, r, softcap):
    """(new tokens, slots) scores of query head r, -inf where not seen; also sum |q k| * scale."""
    a, n = c.q_len[b], c.kv_len[b]
    q = c.q[c.starts[b]:c.starts[b + 1], r].double()
    k = rows(c, c.k, b, h)
    x = (q @ k.T) * c.scale
    mass = (q.abs() @ k.abs().T) * c.scale
    if softcap:
        x = softcap * torch.tanh(x / softcap)
    slot = torch.arange(n, device=x.device)[None]
    own = n - a + torch.arange(a, device=x.device)[:, None]
    return x.masked_fill(slot > own, -math.inf), mass


def attn(c, softcap=0.0):
    """(out, lse, bounds on |out error| and |lse error| per element), rows of no sequence NaN."""
    dev, f32 = c.q.device, c.q.dtype == torch.float32
    full = lambda *s: torch.full(s, math.nan, dtype=torch.float64, device=dev)  # noqa: E731
    hq = c.hkv * c.group
    out, lse, eo, el = full(*c.q.shape), full(c.q.shape[0], hq), full(*c.q.shape), full(c.q.shape[0], hq)
    for b in range(len(c.kv_len)):
        t = slice(c.starts[b], c.starts[b + 1])
        for h in range(c.hkv):
            v = rows(c, c.v, b, h)
            for r in range(h * c.group, (h + 1) * c.group):
                x, mass = score_rows(c, b, h, r, softcap)
                L = torch.logsumexp(x, dim=-1) if x.shape[1] else torch.full((x.shape[0],), -math.inf, dtype=torch.float64, device=dev)
                p = torch.exp(x - L[:, None]).nan_to_num(0.0)
                out[t, r], lse[t, r] = p @ v, L
                es, vmax = score_error(c, x, mass, f32), float(v.abs().max()) if v.numel() else 0.0
                # weights: exp of a score es off, the exponential itself (2 steps of f32), the sum;
                # f32 weights go on as hi + lo (2^-22), f16 ones are rounded once
                ep = 2 * es + (8 + math.sqrt(max(1, x.shape[1]))) * HALF32 + (2.0 ** -21 if f32 else HALF16)
                eo[t, r] = ep[:, None] * (p @ v.abs() + 2.0 ** -16 * vmax) + (HALF32 if f32 else HALF16) * out[t, r].abs() + (
                    0.0 if f32 else 2.0 ** -25)
                el[t, r] = es + (8 + math.sqrt(max(1, x.shape[1]))) * HALF32 + 2 * HALF32 * L.abs().nan_to_num(0, 0, 0)
    return out, lse, eo, el


def score_error(c, x, mass, f32):
    """Bound on a score's absolute error by query row: f32 sums of D exact products (q as hi +
    lo within 2^-22), each partial sum within the row's sum of |q k|; the scaled score and its
    difference from the maximum rounded in f32."""
    if mass.shape[1] == 0:
        return torch.zeros(mass.shape[0], dtype=torch.float64, device=mass.device)
    m = mass.amax(dim=1)
    return m * ((c.D + 4) * HALF32 + (2.0 ** -22 if f32 else 0.0)) + 2.0 ** -22


def weights(c, lse, softcap=0.0, acc=None):
    """(weights, error bound): NaN past each sequence's length."""
    dev, f32 = c.q.device, c.q.dtype == torch.float32
    out = torch.full((len(c.kv_len), c.hkv, c.cap), math.nan, dtype=torch.float64, device=dev)
    err = out.clone()
    for b, n in enumerate(c.kv_len):
        t = slice(c.starts[b], c.starts[b + 1])
        for h in range(c.hkv):
            w = acc[b, h, :n].double().clone() if acc is not None else torch.zeros(n, dtype=torch.float64, device=dev)
            e = HALF32 * w.abs()
            for r in range(h * c.group, (h + 1) * c.group):
                x, mass = score_rows(c, b, h, r, softcap)
                L = lse[t, r].double()[:, None]
                p = torch.where(torch.isinf(L), torch.zeros_like(x), torch.exp(x - L))
                es = score_error(c, x, mass, f32)[:, None] + 2 * HALF32 * L.abs().nan_to_num(0, 0, 0)
                w = w + p.sum(dim=0)
                e = e + (p * (2 * es + 8 * HALF32)).sum(dim=0)
            out[b, h, :n], err[b, h, :n] = w, e + w.abs() * HALF32 * (8 + math.sqrt(max(1, c.T * c.group)))
    return out, err


def rope(x, positions, sections, n_rot, pairs, base, scale=1.0):
    """x (tokens, heads, D) rotated, float64."""
    half = n_rot // 2
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    y = x.double().clone()
    if not half:
        return y
    freq = torch.tensor([scale * base ** (-2.0 * j / n_rot) for j in range(half)], dtype=torch.float64, device=x.device)
    ang = positions.double()[axis].T * freq[None]
    co, si = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    i0, i1 = (slice(0, half), slice(half, n_rot)) if pairs == "halves" else (slice(0, n_rot, 2), slice(1, n_rot, 2))
    a, b = y[..., i0].clone(), y[..., i1].clone()
    y[..., i0], y[..., i1] = a * co - b * si, a * si + b * co
    return y


def evict(c, w, budget, sink, recent):
    """(kept lists, weights): plain Python per (sequence, head)."""
    kept, wout = [], []
    for b, n in enumerate(c.kv_len):
        for h in range(c.hkv):
            row = w[b, h, :n].tolist()
            size = min(n, budget)
            rank = lambda i: (0,) if i < sink or i >= n - recent else (1, row[i] != row[i], -row[i] if row[i] == row[i] else 0.0, i)  # noqa: E731
            stay = set(sorted(range(n), key=rank)[:size])
            movers = iter(sorted(i for i in stay if i >= size))
            kp = [i if i in stay else next(movers) for i in range(size)]
            kept.append(kp + [-1] * (budget - size))
            wout.append([row[i] for i in kp] + [0.0] * (n - size))
    return kept, wout
