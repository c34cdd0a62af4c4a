"""The operators of the paged KV cache, as they are measured: each in a plain form of
elementary torch operations, and through the calls of this package (where ``own`` is set).

* ``store``   -- the new tokens' rotary positions (one to four axes), K and V written to their
                 pages, Q rotated beside them;
* ``attn``    -- attention of the new tokens of a ragged batch over their cached pages;
* ``weights`` -- the attention weight that each cached token received, accumulated;
* ``evict``   -- the cache cut down to a budget of tokens a head, by that weight.

A cache: pools k, v (n_pages, n_head_kv, page, head_dim) f16, a block table (batch, max_pages),
kv_len (batch) cached tokens with the new ones, q_start (batch + 1) first rows of the new tokens.
New token i of sequence b has slot kv_len[b] - (q_start[b + 1] - q_start[b]) + i and sees the
slots up to its own.
"""
import math
import random

import torch

own = False

F16 = torch.float16
TYPES = {"f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one user's decode step: nothing but latency
        dict(name="attn decode 1 seq", op="attn", batch=1, q_lo=1, q_hi=1, kv_lo=777, kv_hi=777, hkv=8, group=4, dim=128,
             page=16, type="f16", softcap=0.0, lens=1),
        # the framework's batched decode (16 sequences of 512 to 8192 tokens), at its f32 contract
        dict(name="attn decode 16 seqs f32", op="attn", batch=16, q_lo=1, q_hi=1, kv_lo=512, kv_hi=8192, hkv=8, group=4,
             dim=128, page=64, type="f32", softcap=0.0, lens=2),
        # a scheduler's mixed step: decodes and short chunks together, odd lengths
        dict(name="attn mixed 24 seqs f32", op="attn", batch=24, q_lo=1, q_hi=263, kv_lo=300, kv_hi=3500, hkv=4, group=3,
             dim=64, page=24, type="f32", softcap=0.0, lens=3),
        # a long prompt's chunk behind what is cached of it
        dict(name="attn chunk 4096 of 16384", op="attn", batch=1, q_lo=4096, q_hi=4096, kv_lo=16384, kv_hi=16384, hkv=8,
             group=4, dim=128, page=128, type="f16", softcap=0.0, lens=4),
        # wide heads with a capped score, prompts of two users
        dict(name="attn softcap dim 256", op="attn", batch=2, q_lo=900, q_hi=1500, kv_lo=2000, kv_hi=5000, hkv=4, group=2,
             dim=256, page=32, type="f16", softcap=30.0, lens=5),
        # weights after the batched decode step
        dict(name="weights decode 16 seqs f32", op="weights", batch=16, q_lo=1, q_hi=1, kv_lo=512, kv_hi=8192, hkv=8,
             group=4, dim=128, page=64, type="f32", softcap=0.0, lens=2),
        # weights after a prompt's last chunk
        dict(name="weights chunk 2048 of 8192", op="weights", batch=1, q_lo=2048, q_hi=2048, kv_lo=8192, kv_hi=8192, hkv=8,
             group=4, dim=128, page=64, type="f16", softcap=0.0, lens=6),
        # a ragged batch cut down between two decode steps
        dict(name="evict 16 seqs to 1000", op="evict", batch=16, kv_lo=512, kv_hi=8192, hkv=8, dim=128, page=64, budget=1000,
             sink=4, recent=64, lens=2),
        # a long prompt cut down once
        dict(name="evict 32768 to 4096", op="evict", batch=1, kv_lo=32768, kv_hi=32768, hkv=8, dim=128, page=128,
             budget=4096, sink=16, recent=512, lens=7),
        # the decode step's 16 new tokens, one position axis
        dict(name="store 16 tokens", op="store", batch=16, q_lo=1, q_hi=1, kv_lo=512, kv_hi=8192, hkv=8, group=4, dim=128,
             page=64, type="f32", axes=1, pairs="halves", rot=128, lens=2),
        # a prompt of text and pictures: time, height and width
        dict(name="store 8000 tokens 3 axes", op="store", batch=3, q_lo=2000, q_hi=3000, kv_lo=3000, kv_hi=6000, hkv=8,
             group=4, dim=128, page=128, type="f32", axes=3, pairs="halves", rot=128, lens=8),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "weights", "evict", "store"])
    c = dict(op=op, dim=rng.choice([64, 128, 128, 256]), hkv=rng.choice([1, 2, 4, 5, 8]),
             page=rng.choice([8, 16, 24, 32, 64, 80, 128, 256]), batch=_log(rng, 1, 48), lens=rng.randrange(1 << 30))
    hi = _log(rng, 1, 20000)
    c["kv_lo"], c["kv_hi"] = max(1, int(hi * rng.uniform(0.05, 1.0))), hi
    if op == "evict":
        c["budget"] = max(1, int(hi * rng.uniform(0.05, 1.1)))
        c["sink"] = rng.randrange(0, c["budget"] // 4 + 1)
        c["recent"] = rng.randrange(0, c["budget"] // 2 + 1)
        while c["batch"] > 1 and c["batch"] * c["hkv"] * hi * c["dim"] > 1 << 28:
            c["batch"] //= 2
        return c
    c["group"] = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 16])
    c["type"] = rng.choice(["f16", "f32"])
    q = 1 if rng.random() < 0.4 else min(hi, _log(rng, 1, 4000))
    c["q_lo"], c["q_hi"] = max(1, int(q * rng.uniform(0.1, 1.0))), q
    if op == "store":
        c["rot"] = rng.choice([c["dim"], c["dim"], c["dim"] // 2])
        c["axes"] = rng.choice([1, 2, 3, 4])
        c["pairs"] = rng.choice(["halves", "adjacent"])
        while c["batch"] > 1 and c["batch"] * c["hkv"] * (hi + c["group"] * q) * c["dim"] > 1 << 28:
            c["batch"] //= 2
        return c
    c["softcap"] = rng.choice([0.0, 0.0, 0.0, 20.0, 50.0])
    most = 1 << 37 if op == "attn" else 1 << 36
    while c["hkv"] * c["group"] * c["batch"] * q * hi * c["dim"] > most:
        if c["batch"] > 1:
            c["batch"] //= 2
        else:
            q = (q + 1) // 2
            c["q_lo"], c["q_hi"] = min(c["q_lo"], q), q
    while c["batch"] > 1 and c["batch"] * c["hkv"] * hi * c["dim"] > 1 << 28:
        c["batch"] //= 2
    return c


def lengths(c):
    """(new tokens, cached tokens) of each sequence."""
    r = random.Random(c["lens"])
    kv = [r.randint(c["kv_lo"], c["kv_hi"]) for _ in range(c["batch"])]
    q = [min(r.randint(c["q_lo"], c["q_hi"]), n) for n in kv] if "q_lo" in c else [0] * c["batch"]
    return q, kv


def sections(c):
    """Frequencies of each position axis: the first one the most, as time beside height and width."""
    half, n = c["rot"] // 2, c["axes"]
    rest = [half // (n + 1)] * (n - 1)
    return [half - sum(rest)] + rest


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    q_len, kv_len = lengths(c)
    B, hkv, D, page = c["batch"], c["hkv"], c["dim"], c["page"]
    need = [-(-n // page) for n in kv_len]
    max_pages, n_pages = max(need), sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((B, max_pages), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    pool = lambda: torch.randn((n_pages, hkv, page, D), generator=g, device=dev, dtype=F16)  # noqa: E731
    starts = [0]
    for n in q_len:
        starts.append(starts[-1] + n)
    s = dict(case=c, k=pool(), v=pool(), table=table, kv_len=torch.tensor(kv_len, dtype=torch.int32, device=dev),
             q_start=torch.tensor(starts, dtype=torch.int32, device=dev), q_max=max(q_len), kv_max=max(kv_len))
    T, cap = starts[-1], max_pages * page
    if c["op"] == "evict":
        # accumulated weight: a few heavy tokens, many light ones
        s["weights"] = torch.randn((B, hkv, cap), generator=g, device=dev).mul_(2.0).exp_()
        s["weights_out"] = torch.zeros((B, hkv, cap), device=dev)
        s["new_len"] = torch.empty(B, dtype=torch.int32, device=dev)
        return s
    dt, hq = TYPES[c["type"]], hkv * c["group"]
    rows = lambda h: torch.randn((T, h, D), generator=g, device=dev).to(dt)  # noqa: E731
    if c["op"] == "store":
        s["q"], s["k_new"], s["v_new"] = rows(hq), rows(hkv), rows(hkv)
        s["q_out"] = torch.empty_like(s["q"])
        # positions: the first axis counts on, the others are places in pictures
        first = torch.randint(0, 200000, (1,), generator=g, device=dev)
        more = torch.randint(0, 1000, (c["axes"] - 1, T), generator=g, device=dev)
        s["positions"] = torch.cat([(first + torch.arange(T, device=dev))[None], more]).to(torch.int32)
        s["sections"], s["base"] = sections(c), 500000.0
        return s
    s["q"], s["scale"] = rows(hq), 1.5 / math.sqrt(D)
    if c["op"] == "weights":
        s["acc"] = torch.rand((B, hkv, cap), generator=g, device=dev)
        s["acc_out"] = torch.zeros((B, hkv, cap), device=dev)
        s["lse"] = flat_rows(s, torch.logsumexp(scores(s), dim=-1))
    return s


# ------------------------------------------------------------------ plain forms

def pages_of(s, pool):
    """The cached rows of each sequence in order: (batch, n_head_kv, slots, head_dim) f32, 0 past kv_len."""
    x = pool[s["table"].long().clamp(min=0)].permute(0, 2, 1, 3, 4)
    x = x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])[:, :, :s["kv_max"]]
    past = torch.arange(s["kv_max"], device=x.device)[None] >= s["kv_len"][:, None]
    return x.float().masked_fill(past[:, None, :, None], 0.0)


def new_rows(s):
    """For the padded layout (batch, q_max): each place's row among the new tokens, and whether it is one."""
    i = torch.arange(s["q_max"], device=s["q_start"].device)
    n = (s["q_start"][1:] - s["q_start"][:-1]).long()
    real = i[None] < n[:, None]
    return torch.where(real, s["q_start"][:-1].long()[:, None] + i[None], 0), real, n


def scores(s):
    """(batch, n_head_q, q_max, slots) scores, -inf where a slot is not seen."""
    c = s["case"]
    at, real, n = new_rows(s)
    q = s["q"].float()[at].transpose(1, 2)  # (batch, n_head_q, q_max, head_dim)
    k = pages_of(s, s["k"])
    q = q.reshape(q.shape[0], c["hkv"], -1, c["dim"])
    x = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"])
    x = x.reshape(x.shape[0], c["hkv"] * c["group"], s["q_max"], -1)
    if c["softcap"]:
        x = torch.tanh_(x.div_(c["softcap"])).mul_(c["softcap"])
    last = s["kv_len"].long()[:, None] - n[:, None] + torch.arange(s["q_max"], device=x.device)[None]
    seen = torch.arange(x.shape[-1], device=x.device) <= last[:, :, None]
    return x.masked_fill_(~(seen & real[:, :, None])[:, None], -math.inf)


def flat_rows(s, x):
    """(batch, heads, q_max, ...) in the padded layout -> (tokens, heads, ...)."""
    _, real, _ = new_rows(s)
    return x.transpose(1, 2)[real]


def attn(s):
    c = s["case"]
    x = scores(s)
    top = x.amax(dim=-1, keepdim=True).clamp(min=-1e30)
    p = x.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    v = pages_of(s, s["v"])
    o = torch.matmul(p.reshape(p.shape[0], c["hkv"], -1, p.shape[-1]), v).reshape(*p.shape[:3], c["dim"])
    o = o / total.clamp(min=1e-30)
    lse = (top + total.log())[..., 0]
    return {"out": flat_rows(s, o).to(s["q"].dtype), "lse": flat_rows(s, lse)}


def weights(s):
    c = s["case"]
    at, real, _ = new_rows(s)
    lse = s["lse"][at].transpose(1, 2)  # (batch, n_head_q, q_max)
    p = scores(s).sub_(lse[..., None]).exp_()
    new = p.reshape(p.shape[0], c["hkv"], -1, p.shape[-1]).sum(dim=2)
    out = s["acc_out"]
    seen = torch.arange(s["kv_max"], device=out.device)[None] < s["kv_len"][:, None]
    out[:, :, :s["kv_max"]] = torch.where(seen[:, None], s["acc"][:, :, :s["kv_max"]] + new, 0.0)
    return {"acc": out}


def evict(s):
    c = s["case"]
    w = s["weights"][:, :, :s["kv_max"]]
    B, H, L = w.shape
    slot = torch.arange(L, device=w.device)
    n = s["kv_len"].long()[:, None, None]
    size = torch.clamp(n, max=c["budget"])
    kept_for_sure = (slot < c["sink"]) | (slot >= n - c["recent"])
    key = torch.where(kept_for_sure, math.inf, w).masked_fill(slot >= n, -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    keep = torch.zeros((B, H, L), dtype=torch.bool, device=w.device).scatter_(2, order, slot.expand(B, H, L) < size)
    # kept tokens behind the new end, in order, go to the free slots before it, in order
    mover, hole = keep & (slot >= size), ~keep & (slot < size)
    rank = lambda m: torch.where(m, m.long().cumsum(2) - 1, L)  # noqa: E731
    from_of = torch.zeros((B, H, L + 1), dtype=torch.long, device=w.device).scatter_(2, rank(mover), slot.expand(B, H, L))
    source = torch.where(hole, from_of.gather(2, rank(hole).clamp(max=L)), slot.expand(B, H, L))
    b, h, to = hole.nonzero(as_tuple=True)
    frm = source[b, h, to]
    page = c["page"]
    tb = s["table"].long()
    p0, r0, p1, r1 = tb[b, frm // page], frm % page, tb[b, to // page], to % page
    s["k"][p1, h, r1] = s["k"][p0, h, r0]
    s["v"][p1, h, r1] = s["v"][p0, h, r0]
    kept = torch.full((B, H, c["budget"]), -1, dtype=torch.int32, device=w.device)
    m = min(L, c["budget"])
    live = slot[:m] < size
    kept[:, :, :m] = torch.where(live, source[:, :, :m], -1).to(torch.int32)
    # freed slots start again from nothing
    out = s["weights_out"]
    out[:, :, :L] = torch.where(slot < size, w.gather(2, source), 0.0)
    return {"k": s["k"], "v": s["v"], "kept": kept, "weights": out, "kv_len": size[:, 0, 0].to(torch.int32)}


def store(s):
    c = s["case"]
    half, dev = c["rot"] // 2, s["k"].device
    # angles of far positions need 64 bits
    freq = float(s["base"]) ** (-torch.arange(half, dtype=torch.float64, device=dev) * 2.0 / c["rot"])
    axis = torch.repeat_interleave(torch.arange(c["axes"], device=dev), torch.tensor(s["sections"], device=dev), output_size=half)
    angle = s["positions"].double()[axis].T * freq[None]  # (tokens, half)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x):
        x = x.float()
        if c["pairs"] == "halves":
            a, b, rest = x[..., :half], x[..., half:c["rot"]], x[..., c["rot"]:]
            return torch.cat([a * cos - b * sin, a * sin + b * cos, rest], dim=-1)
        a, b, rest = x[..., 0:c["rot"]:2], x[..., 1:c["rot"]:2], x[..., c["rot"]:]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
        return torch.cat([y, rest], dim=-1)

    token = torch.arange(s["q"].shape[0], device=dev)
    b = torch.searchsorted(s["q_start"].long()[1:].contiguous(), token, right=True)
    slot = s["kv_len"].long()[b] - s["q_start"].long()[b + 1] + token
    at, row = s["table"].long()[b, slot // c["page"]], slot % c["page"]
    s["k"][at, :, row] = turn(s["k_new"]).to(F16)
    s["v"][at, :, row] = s["v_new"].to(F16)
    s["q_out"].copy_(turn(s["q"]))
    return {"k": s["k"], "v": s["v"], "q": s["q_out"]}


# ------------------------------------------------------------------ this package's calls

def run_own(s):
    import mlz_b200 as m
    c = s["case"]
    if "cache" not in s:  # the handle that a program keeps beside its pools
        s["cache"] = m.PagedCache(s["k"], s["v"], s["table"], s["kv_len"], s["q_start"])
    cache = s["cache"]
    if c["op"] == "attn":
        out, lse = m.paged_attn(cache, s["q"], s["scale"], softcap=c["softcap"], return_lse=True)
        return {"out": out, "lse": lse}
    if c["op"] == "weights":
        return {"acc": m.paged_weights(cache, s["q"], s["lse"], s["scale"], softcap=c["softcap"], acc=s["acc"],
                                       out=s["acc_out"])}
    if c["op"] == "evict":
        kept, w, kv_len = m.paged_evict(cache, s["weights"], c["budget"], n_sink=c["sink"], n_recent=c["recent"],
                                        weights_out=s["weights_out"], kv_len_out=s["new_len"])
        return {"k": s["k"], "v": s["v"], "kept": kept, "weights": w, "kv_len": kv_len}
    m.paged_store(cache, s["k_new"], s["v_new"], q=s["q"], q_out=s["q_out"], positions=s["positions"],
                  sections=s["sections"], n_rot=c["rot"], pairs=c["pairs"], freq_base=s["base"])
    return {"k": s["k"], "v": s["v"], "q": s["q_out"]}


def run(state):
    if own:
        return run_own(state)
    return {"attn": attn, "weights": weights, "evict": evict, "store": store}[state["case"]["op"]](state)


# ------------------------------------------------------------------ work

def work(case):
    c = case
    q_len, kv_len = lengths(c)
    D, hkv, B = c["dim"], c["hkv"], c["batch"]
    if c["op"] == "evict":
        moved = 0.0
        for n in kv_len:
            size = min(n, c["budget"])
            sure = min(n, c["sink"]) + min(n, c["recent"])
            # of the tokens behind the new end: the recent ones, and those that win by weight
            behind = n - size
            rest = max(0, n - sure)
            p = max(0, size - sure) / rest if rest else 0.0
            moved += min(behind, c["recent"]) + p * max(0, behind - c["recent"])
        # weights read and written, kept list written, moved rows of K and V read and written
        return {"bytes": hkv * (8.0 * sum(kv_len) + 4.0 * B * c["budget"] + moved * D * 8), "flops": 0}
    e, hq, T = (2 if c["type"] == "f16" else 4), hkv * c["group"], sum(q_len)
    if c["op"] == "store":
        return {"bytes": T * D * (2.0 * hq * e + 2 * hkv * (e + 2)) + 4.0 * c["axes"] * T, "flops": 3.0 * T * c["rot"] * (hq + hkv)}
    seen = sum(a * (b - a) + a * (a + 1) / 2 for a, b in zip(q_len, kv_len))
    if c["op"] == "weights":
        return {"bytes": sum(kv_len) * hkv * (2.0 * D + 8) + T * hq * (D * e + 4.0), "flops": 2.0 * seen * hq * D}
    return {"bytes": sum(kv_len) * hkv * 4.0 * D + T * hq * (2.0 * D * e + 4), "flops": 4.0 * seen * hq * D}


# ------------------------------------------------------------------ 64-bit values

def exact(case, seed):
    """Each sequence and head by itself, in double precision, from the definition."""
    c, s = case, prepare(case, seed)
    q_len, kv_len = lengths(c)
    f64 = torch.float64
    page = c["page"]
    table = s["table"].tolist()
    spot = lambda b, i: (table[b][i // page], i % page)  # noqa: E731

    if c["op"] == "evict":
        kept = torch.full((c["batch"], c["hkv"], c["budget"]), -1, dtype=torch.int32)
        w, wout = s["weights"].cpu(), torch.zeros(s["weights"].shape)
        jobs = [[], [], [], [], []]
        for b, n in enumerate(kv_len):
            size = min(n, c["budget"])
            for h in range(c["hkv"]):
                row = w[b, h, :n].tolist()
                ranked = sorted(range(n), key=lambda i: (0 if i < c["sink"] or i >= n - c["recent"] else 1, -row[i], i))
                if size < n and any(i < c["sink"] or i >= n - c["recent"] for i in ranked[size:]):
                    return None
                stay = set(ranked[:size])
                movers = iter(sorted(i for i in stay if i >= size))
                for to in range(size):
                    frm = to if to in stay else next(movers)
                    kept[b, h, to], wout[b, h, to] = frm, row[frm]
                    if frm != to:
                        for j, x in zip(jobs, (*spot(b, frm), h, *spot(b, to))):
                            j.append(x)
        if jobs[0]:
            p0, r0, h, p1, r1 = (torch.tensor(j, device=s["k"].device) for j in jobs)
            for pool in (s["k"], s["v"]):
                pool[p1, h, r1] = pool[p0, h, r0].clone()
        return {"k": s["k"].double(), "v": s["v"].double(), "kept": kept, "weights": wout.double(),
                "kv_len": torch.tensor([min(n, c["budget"]) for n in kv_len], dtype=torch.int32)}

    if c["op"] == "store":
        half = c["rot"] // 2
        pos, angle = s["positions"].to(f64), torch.empty((s["q"].shape[0], half), dtype=f64, device=s["q"].device)
        j = 0
        for a, n in enumerate(s["sections"]):
            for _ in range(n):
                angle[:, j] = pos[a] * s["base"] ** (-2.0 * j / c["rot"])
                j += 1
        z = torch.polar(torch.ones_like(angle), angle)[:, None]

        def turn(x):
            y = x.to(f64).clone()
            first, second = (slice(0, half), slice(half, c["rot"])) if c["pairs"] == "halves" else (
                slice(0, c["rot"], 2), slice(1, c["rot"], 2))
            t = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * z
            y[..., first], y[..., second] = t.real, t.imag
            return y

        k, v, t = s["k"].to(f64), s["v"].to(f64), 0
        kn, vn = turn(s["k_new"]), s["v_new"].to(f64)
        for b, (a, n) in enumerate(zip(q_len, kv_len)):
            spots = torch.tensor([spot(b, n - a + i) for i in range(a)], device=k.device)
            k[spots[:, 0], :, spots[:, 1]] = kn[t:t + a]
            v[spots[:, 0], :, spots[:, 1]] = vn[t:t + a]
            t += a
        return {"k": k, "v": v, "q": turn(s["q"])}

    T, hq, g = s["q"].shape[0], c["hkv"] * c["group"], c["group"]
    out = torch.zeros((T, hq, c["dim"]), dtype=f64, device=s["q"].device)
    lse = torch.zeros((T, hq), dtype=f64, device=s["q"].device)
    acc = torch.zeros(s["acc"].shape, dtype=f64, device=s["q"].device) if c["op"] == "weights" else None
    t = 0
    for b, (a, n) in enumerate(zip(q_len, kv_len)):
        ids = torch.tensor(table[b][:-(-n // page)], device=s["q"].device)
        hidden = torch.arange(n, device=s["q"].device)[None] > (n - a + torch.arange(a, device=s["q"].device))[:, None]
        for h in range(c["hkv"]):
            k = s["k"][ids, h].reshape(-1, c["dim"])[:n].to(f64)
            v = s["v"][ids, h].reshape(-1, c["dim"])[:n].to(f64)
            for r in range(h * g, h * g + g):
                x = (s["q"][t:t + a, r].to(f64) @ k.T) * s["scale"]
                if c["softcap"]:
                    x = c["softcap"] * torch.tanh(x / c["softcap"])
                x[hidden] = -math.inf
                if acc is not None:
                    acc[b, h, :n] += torch.exp(x - s["lse"][t:t + a, r].to(f64)[:, None]).sum(dim=0)
                    continue
                lse[t:t + a, r] = torch.logsumexp(x, dim=-1)
                out[t:t + a, r] = torch.softmax(x, dim=-1) @ v
            if acc is not None:
                acc[b, h, :n] += s["acc"][b, h, :n].to(f64)
        t += a
    return {"acc": acc} if acc is not None else {"out": out, "lse": lse}
