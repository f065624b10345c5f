"""The batched-decode operators as measured programs.

Three operators over the KV cache of a batch of sequences: rotary positions
written into it (rope_append), attention of one token per sequence over a
prefix that all sequences share and each sequence's own rows
(attention_batch), and eviction of the rows with the least accumulated
attention weight (kv_evict).  `run` computes them in plain torch, or with
the library's kernels where `own` is true; `exact` computes them in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one token of one sequence enters its cache, every layer of every decode step
        {"name": "rope_token", "op": "rope", "dtype": "f32", "n_head": 28, "n_kv": 4, "head_dim": 128,
         "tokens": 1, "n_seq": 1, "max_ctx": 1024, "layout": "half", "rot": 128, "theta": 1e6,
         "scaling": "none", "factor": 1.0, "pos0": 511},
        # a batch of sequences far into a stretched context, the last tokens padding
        {"name": "rope_batch_parts", "op": "rope", "dtype": "bf16", "n_head": 28, "n_kv": 4, "head_dim": 128,
         "tokens": 67, "n_seq": 67, "max_ctx": 80, "layout": "half", "rot": 128, "theta": 1e6,
         "scaling": "parts", "factor": 4.0, "pos0": 100003},
        # a long prompt in one call, half of every head rotated, pairs side by side
        {"name": "rope_prompt", "op": "rope", "dtype": "f16", "n_head": 28, "n_kv": 4, "head_dim": 128,
         "tokens": 8191, "n_seq": 1, "max_ctx": 8192, "layout": "interleaved", "rot": 64, "theta": 1e4,
         "scaling": "linear", "factor": 2.0, "pos0": 0},
        # a single sequence, the cache length of the full decode token's benchmark
        {"name": "attn_single", "op": "attn", "dtype": "f32", "n_head": 28, "n_kv": 4, "head_dim": 128,
         "n_seq": 1, "prefix": 0, "len_lo": 812, "len_hi": 812, "max_ctx": 1024, "weights": False},
        # a batch of chats behind one system prompt, the cache in the decoder's own type
        {"name": "attn_chat_f32", "op": "attn", "dtype": "f32", "n_head": 28, "n_kv": 4, "head_dim": 128,
         "n_seq": 16, "prefix": 4093, "len_lo": 1, "len_hi": 700, "max_ctx": 768, "weights": False},
        # many samples of one long document
        {"name": "attn_document_bf16", "op": "attn", "dtype": "bf16", "n_head": 28, "n_kv": 4, "head_dim": 128,
         "n_seq": 64, "prefix": 16384, "len_lo": 0, "len_hi": 1000, "max_ctx": 1024, "weights": False},
        # long separate sequences whose rows are scored for eviction
        {"name": "attn_scored_f16", "op": "attn", "dtype": "f16", "n_head": 16, "n_kv": 8, "head_dim": 64,
         "n_seq": 8, "prefix": 0, "len_lo": 3001, "len_hi": 8191, "max_ctx": 8192, "weights": True},
        # the same in the decoder's type with a prefix, wide heads
        {"name": "attn_scored_f32", "op": "attn", "dtype": "f32", "n_head": 8, "n_kv": 4, "head_dim": 256,
         "n_seq": 5, "prefix": 333, "len_lo": 100, "len_hi": 2000, "max_ctx": 2048, "weights": True},
        # one sequence at its limit drops half of its rows
        {"name": "evict_single", "op": "evict", "dtype": "f32", "n_kv": 4, "head_dim": 128, "n_seq": 1,
         "max_ctx": 1024, "len_lo": 1024, "len_hi": 1024, "keep": 512, "n_sink": 4, "n_recent": 128},
        # a ragged batch, some sequences still short
        {"name": "evict_batch", "op": "evict", "dtype": "bf16", "n_kv": 4, "head_dim": 128, "n_seq": 32,
         "max_ctx": 4096, "len_lo": 1500, "len_hi": 4095, "keep": 2000, "n_sink": 4, "n_recent": 256},
        # long documents cut down to a short budget
        {"name": "evict_long", "op": "evict", "dtype": "f16", "n_kv": 8, "head_dim": 64, "n_seq": 2,
         "max_ctx": 32768, "len_lo": 30001, "len_hi": 32768, "keep": 4096, "n_sink": 16, "n_recent": 1024},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.4)))))


def draw(rng):
    op = rng.choice(["rope", "attn", "attn", "evict"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    n_kv = rng.choice([1, 2, 4, 8])
    head_dim = rng.choice([64, 128, 256]) if op != "rope" else rng.choice([32, 64, 128, 256])
    if n_kv * head_dim > 1024:
        n_kv = 1024 // head_dim
    group = rng.choice([1, 2, 4, 5, 7, 8])
    while n_kv * group * head_dim > 4096:
        group = max(1, group // 2)
    case = {"op": op, "dtype": dtype, "n_kv": n_kv, "head_dim": head_dim}
    if op == "rope":
        case["n_head"] = n_kv * group
        # no more elements than the long prompt's
        case["tokens"] = _log(rng, 1, min(8191, 8191 * 36 * 128 // (n_kv * (group + 2) * head_dim)))
        batch = rng.random() < 0.5 and case["tokens"] <= 512
        case["n_seq"] = case["tokens"] if batch else 1
        case["max_ctx"] = rng.randint(1, 64) if batch else case["tokens"] + rng.randint(0, 50)
        case["layout"] = rng.choice(["half", "interleaved"])
        case["rot"] = rng.choice([head_dim, head_dim // 2, head_dim // 4])
        case["theta"] = rng.choice([1e4, 5e5, 1e6])
        case["scaling"] = rng.choice(["none", "linear", "parts"])
        case["factor"] = 1.0 if case["scaling"] == "none" else rng.choice([2.0, 4.0, 8.0])
        case["pos0"] = _log(rng, 1, 200000) - 1
    elif op == "attn":
        case["n_head"] = n_kv * group
        case["n_seq"] = _log(rng, 1, 64)
        # no more products than the long document's (f32 costs several times as much each)
        cap = 14e9 / (4 if dtype == "f32" else 1) / (4 * n_kv * group * head_dim * case["n_seq"])
        case["prefix"] = _log(rng, 1, min(16384, int(cap))) if rng.random() < 0.7 else 0
        own_rows = max(2, min(8192, 49152 // case["n_seq"]))
        case["len_hi"] = _log(rng, 1, own_rows)
        case["len_lo"] = rng.randint(0, case["len_hi"]) if case["prefix"] else \
            rng.randint(min(1, case["len_hi"]), case["len_hi"])
        case["max_ctx"] = case["len_hi"] + rng.randint(0, 33)
        case["weights"] = rng.random() < 0.4
    else:
        case["n_seq"] = _log(rng, 1, 32)
        # no more cache than the ragged batch's
        rows = 32 * 4096 * 512 * 2 // (n_kv * head_dim * (4 if dtype == "f32" else 2) * case["n_seq"])
        case["max_ctx"] = _log(rng, 64, max(64, min(32768, rows)))
        case["len_hi"] = case["max_ctx"] - rng.randint(0, case["max_ctx"] // 8)
        case["len_lo"] = rng.randint(case["len_hi"] // 2, case["len_hi"])
        case["keep"] = rng.randint(max(1, case["len_hi"] // 10), max(1, case["len_hi"] * 9 // 10))
        case["n_sink"] = min(rng.choice([0, 1, 4]), case["keep"] // 2)
        case["n_recent"] = rng.randint(0, case["keep"] - case["n_sink"])
    return case


# ---- inputs -----------------------------------------------------------------
def _lens_of(case):
    """Lengths spread evenly over [len_lo, len_hi]; the seed orders them."""
    n, lo, hi = case["n_seq"], case["len_lo"], case["len_hi"]
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _keys(g, shape, dtype):
    """Keys as trained models have them: some channels with an offset or a
    wider range than the others, rows of differing size."""
    k = torch.randn(shape, device="cuda", generator=g)
    hd = shape[-1]
    off = torch.randn(hd, device="cuda", generator=g) * (torch.rand(hd, device="cuda", generator=g) < 0.1) * 3.0
    k = k * torch.exp(0.3 * torch.randn(shape[:-1] + (1,), device="cuda", generator=g)) + off
    return k.to(dtype)


def _freqs(case):
    """Angle per position of each rotated pair, in 64 bits."""
    rot, out = case["rot"], []
    for d in range(rot // 2):
        f = float(case["theta"]) ** (-2.0 * d / rot)
        if case["scaling"] == "linear":
            f = f / case["factor"]
        elif case["scaling"] == "parts":
            turns = case["ctx0"] * f / (2.0 * math.pi)
            g = min(1.0, max(0.0, (turns - 1.0) / (32.0 - 1.0)))
            f = f * (g + (1.0 - g) / case["factor"])
        out.append(f)
    return out


def _rope_case(case):
    c = dict(case)
    c["ctx0"] = 32768.0
    c["mscale"] = 1.125 if case["scaling"] == "parts" else 1.0
    return c


class State:
    pass


def prepare(case, seed):
    s = State()
    s.case = case
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    nk, hd, ns, mc = case["n_kv"], case["head_dim"], case["n_seq"], case["max_ctx"]
    if case["op"] == "rope":
        T, nh = case["tokens"], case["n_head"]
        s.c = _rope_case(case)
        s.qkv = torch.randn((T, (nh + 2 * nk) * hd), device="cuda", generator=g)
        shift = seed % 7
        if ns == 1:
            base = (mc - T) // 2
            s.pos = (torch.arange(T, device="cuda") + case["pos0"] + shift).to(torch.int32)
            s.slots = (torch.arange(T, device="cuda") + base).to(torch.int32)
        else:
            own_row = torch.randint(0, mc, (T,), device="cuda", generator=g)
            s.pos = (own_row + case["pos0"] + shift).to(torch.int32)
            s.slots = (torch.arange(T, device="cuda") * mc + own_row).to(torch.int32)
            s.slots[T - T // 8:] = -1      # padding of the batch: nothing is stored
        s.k = torch.randn((ns, mc, nk * hd), device="cuda", generator=g).to(dt)
        s.v = torch.randn((ns, mc, nk * hd), device="cuda", generator=g).to(dt)
    elif case["op"] == "attn":
        nh, L = case["n_head"], case["prefix"]
        s.q = (1.5 * torch.randn((ns, nh * hd), device="cuda", generator=g)).to(dt)
        s.k = _keys(g, (ns, mc, nk, hd), dt).reshape(ns, mc, nk * hd)
        s.v = torch.randn((ns, mc, nk * hd), device="cuda", generator=g).to(dt)
        s.pk = _keys(g, (L, nk, hd), dt).reshape(L, nk * hd) if L else None
        s.pv = torch.randn((L, nk * hd), device="cuda", generator=g).to(dt) if L else None
        order = torch.randperm(ns, device="cuda", generator=g)
        s.lens = torch.tensor(_lens_of(case), device="cuda", dtype=torch.int32)[order].contiguous()
        if case["weights"]:
            s.w0 = torch.rand((ns, nk, mc), device="cuda", generator=g).pow(6.0)
            s.w = s.w0.clone()
    else:
        s.k = torch.randn((ns, mc, nk * hd), device="cuda", generator=g).to(dt)
        s.v = torch.randn((ns, mc, nk * hd), device="cuda", generator=g).to(dt)
        order = torch.randperm(ns, device="cuda", generator=g)
        s.lens0 = torch.tensor(_lens_of(case), device="cuda", dtype=torch.int32)[order].contiguous()
        # accumulated weights: a few rows hold most of it, many hold exactly none
        w = torch.rand((ns, nk, mc), device="cuda", generator=g)
        s.w0 = torch.where(w < 0.05, torch.zeros_like(w), w.pow(8.0))
        s.pos0 = (torch.arange(mc, device="cuda", dtype=torch.int32) + seed % 3).expand(ns, nk, mc).contiguous()
        s.lens, s.w, s.pos = s.lens0.clone(), s.w0.clone(), s.pos0.clone()
    if own:
        import lalmodel_b200 as lb
        s.ctx = lb.Context(torch.cuda.current_device())
        s.cache = lb.KVBatch(s.k, s.v, nk, row_pos=getattr(s, "pos", None) if case["op"] == "evict" else None,
                             row_weight=getattr(s, "w", None))
        if case["op"] == "rope":
            c = s.c
            s.rope = lb.Rope(layout=c["layout"], rot_dim=c["rot"], theta=c["theta"], scaling=c["scaling"],
                             factor=c["factor"], orig_ctx=c["ctx0"], turns_fast=32.0, turns_slow=1.0,
                             mscale=c["mscale"])
            s.out = torch.empty((case["tokens"], case["n_head"] * hd), device="cuda", dtype=dt)
        elif case["op"] == "attn":
            s.ws = s.ctx.attention_batch_ws(s.cache, case["n_head"], prefix_len=case["prefix"],
                                            weights=case["weights"])
            s.out = torch.empty_like(s.q)
        else:
            s.ws = s.ctx.kv_evict_ws(s.cache, case["keep"])
    return s


# ---- the operators ------------------------------------------------------------
def _rope_rows(x, cos, sin, rot, layout):
    """x [T][heads][hd] fp32, cos/sin [T][1][rot/2]."""
    y = x.clone()
    if layout == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2] = a * cos - b * sin
        y[..., rot // 2:rot] = a * sin + b * cos
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2] = a * cos - b * sin
        y[..., 1:rot:2] = a * sin + b * cos
    return y


def _run_rope(s):
    c = s.c
    T, nh, nk, hd, rot, mc = c["tokens"], c["n_head"], c["n_kv"], c["head_dim"], c["rot"], c["max_ctx"]
    dt = s.k.dtype
    f = torch.tensor(_freqs(c), device="cuda", dtype=torch.float64)
    ang = s.pos.double()[:, None, None] * f
    cos, sin = (torch.cos(ang) * c["mscale"]).float(), (torch.sin(ang) * c["mscale"]).float()
    x = s.qkv.view(T, nh + 2 * nk, hd)
    qk = _rope_rows(x[:, :nh + nk], cos, sin, rot, c["layout"])
    q = qk[:, :nh].reshape(T, nh * hd).to(dt)
    # a token without a slot (padding) puts back the row it finds in its own sequence
    stored = (s.slots >= 0)[:, None]
    spare = torch.arange(T, device="cuda") * mc if c["n_seq"] > 1 else torch.zeros_like(s.slots).long()
    dst = torch.where(stored[:, 0], s.slots.long(), spare)
    for cache, new in ((s.k, qk[:, nh:]), (s.v, x[:, nh + nk:])):
        rows = cache.view(-1, nk * hd)
        rows[dst] = torch.where(stored, new.reshape(T, nk * hd).to(dt), rows[dst])
    return {"q": q, "k": s.k, "v": s.v}


def _run_attn(s):
    c = s.case
    ns, nh, nk, hd, L, mc = c["n_seq"], c["n_head"], c["n_kv"], c["head_dim"], c["prefix"], c["max_ctx"]
    g = nh // nk
    scale = 1.0 / math.sqrt(hd)
    q = s.q.float().view(ns, nk, g, hd)
    k = s.k.float().view(ns, mc, nk, hd).permute(0, 2, 1, 3)
    v = s.v.float().view(ns, mc, nk, hd).permute(0, 2, 1, 3)
    live = torch.arange(mc, device="cuda")[None, :] < s.lens[:, None]
    sc = torch.matmul(q, k.transpose(2, 3)) * scale
    sc = torch.where(live[:, None, None, :], sc, torch.full_like(sc, float("-inf")))
    if L:
        # the prefix once for all sequences: the queries of a KV head as one matrix
        qa = q.permute(1, 0, 2, 3).reshape(nk, ns * g, hd)
        kp = s.pk.float().view(L, nk, hd).permute(1, 2, 0)
        vp = s.pv.float().view(L, nk, hd).permute(1, 0, 2)
        sp = (torch.matmul(qa, kp) * scale).view(nk, ns, g, L).permute(1, 0, 2, 3)
        m = torch.maximum(sp.amax(-1, keepdim=True), sc.amax(-1, keepdim=True))
        ep, eo = torch.exp(sp - m), torch.exp(sc - m)
        den = ep.sum(-1, keepdim=True) + eo.sum(-1, keepdim=True)
        pp = (ep / den).permute(1, 0, 2, 3).reshape(nk, ns * g, L)
        po = eo / den
        o = torch.matmul(pp, vp).view(nk, ns, g, hd).permute(1, 0, 2, 3)
    else:
        eo = torch.exp(sc - sc.amax(-1, keepdim=True))
        po = eo / eo.sum(-1, keepdim=True)
        o = 0.0
    o = o + torch.matmul(po, torch.where(live[:, None, :, None], v, torch.zeros_like(v)))
    out = {"out": o.reshape(ns, nh * hd).to(s.q.dtype)}
    if c["weights"]:
        s.w.copy_(s.w0)
        s.w += po.sum(2)
        out["weights"] = s.w
    return out


def _run_evict(s):
    c = s.case
    ns, nk, hd, mc, keep = c["n_seq"], c["n_kv"], c["head_dim"], c["max_ctx"], c["keep"]
    s.w.copy_(s.w0)
    s.pos.copy_(s.pos0)
    s.lens.copy_(s.lens0)
    n = s.lens.long()[:, None, None]
    row = torch.arange(mc, device="cuda")[None, None, :]
    live = row < n
    last = torch.where(live, s.pos, torch.full_like(s.pos, -1)).amax(-1, keepdim=True)
    safe = live & ((s.pos < c["n_sink"]) | (s.pos > last - c["n_recent"]))
    key = torch.where(safe, torch.full_like(s.w, float("inf")), s.w)
    key = torch.where(live, key, torch.full_like(key, float("-inf")))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    sel = torch.zeros_like(live.expand(ns, nk, mc)).scatter(2, order, True) & live
    full = n > keep
    hole = full & ~sel & (row < keep)
    move = full & sel & (row >= keep)
    # the i-th hole takes the i-th kept row above the limit
    rank = torch.where(move, torch.cumsum(move, -1) - 1, torch.full_like(row, mc - 1))
    src = torch.zeros((ns, nk, mc), device="cuda", dtype=torch.long)
    src.scatter_(2, torch.where(move, rank, torch.full_like(rank, mc - 1)), row.expand(ns, nk, mc))
    take = torch.where(hole, src.gather(2, (torch.cumsum(hole, -1) - 1).clamp(min=0)), row.expand(ns, nk, mc))
    for t in (s.k, s.v):
        t4 = t.view(ns, mc, nk, hd)
        idx = take.permute(0, 2, 1)[:, :keep, :, None].expand(ns, keep, nk, hd)
        t4[:, :keep] = t4.gather(1, idx)
    gone = full & live & (row >= keep)
    s.w.copy_(torch.where(gone, torch.zeros_like(s.w), s.w.gather(2, take)))
    s.pos.copy_(s.pos.gather(2, take))
    s.lens.copy_(torch.minimum(s.lens, torch.full_like(s.lens, keep)))
    return {"k": s.k, "v": s.v, "row_pos": s.pos, "row_weight": s.w, "lens": s.lens}


def _run_own(s):
    c = s.case
    if c["op"] == "rope":
        q = s.ctx.rope_append(s.cache, s.qkv, s.pos, s.slots, c["n_head"], rope=s.rope, out=s.out)
        return {"q": q, "k": s.k, "v": s.v}
    if c["op"] == "attn":
        if c["weights"]:
            s.w.copy_(s.w0)
        o = s.ctx.attention_batch(s.cache, s.q, s.lens, c["n_head"], prefix_k=s.pk, prefix_v=s.pv,
                                  decay=1.0 if c["weights"] else None, ws=s.ws, out=s.out)
        return {"out": o, "weights": s.w} if c["weights"] else {"out": o}
    s.w.copy_(s.w0)
    s.pos.copy_(s.pos0)
    s.lens.copy_(s.lens0)
    s.ctx.kv_evict(s.cache, s.lens, c["keep"], n_sink=c["n_sink"], n_recent=c["n_recent"], ws=s.ws)
    return {"k": s.k, "v": s.v, "row_pos": s.pos, "row_weight": s.w, "lens": s.lens}


def run(state):
    if own:
        return _run_own(state)
    return {"rope": _run_rope, "attn": _run_attn, "evict": _run_evict}[state.case["op"]](state)


# ---- 64-bit definition ----------------------------------------------------------
def exact(case, seed):
    saved = globals()["own"]
    globals()["own"] = False
    try:
        s = prepare(case, seed)
    finally:
        globals()["own"] = saved
    nk, hd, ns, mc = case["n_kv"], case["head_dim"], case["n_seq"], case["max_ctx"]
    if case["op"] == "rope":
        c = s.c
        T, nh, rot = c["tokens"], c["n_head"], c["rot"]
        f = torch.tensor(_freqs(c), dtype=torch.float64, device="cuda")
        phase = torch.polar(torch.full((T, rot // 2), float(c["mscale"]), dtype=torch.float64, device="cuda"),
                            s.pos.double()[:, None] * f[None, :])
        x = s.qkv.double().view(T, nh + 2 * nk, hd)
        y = x.clone()
        if c["layout"] == "half":
            first, second = slice(0, rot // 2), slice(rot // 2, rot)
        else:
            first, second = slice(0, rot, 2), slice(1, rot, 2)
        for h in range(nh + nk):       # each pair as one complex number
            z = torch.complex(x[:, h, first].contiguous(), x[:, h, second].contiguous()) * phase
            y[:, h, first], y[:, h, second] = z.real, z.imag
        k, v = s.k.double().view(-1, nk * hd), s.v.double().view(-1, nk * hd)
        for cache, lo in ((k, nh), (v, nh + nk)):
            keepers = [(t, r) for t, r in enumerate(s.slots.tolist()) if r >= 0]
            if keepers:
                ts, rs = zip(*keepers)
                cache[list(rs)] = y[list(ts), lo:lo + nk].reshape(len(ts), nk * hd)
        return {"q": y[:, :nh].reshape(T, nh * hd), "k": k.view(ns, mc, nk * hd), "v": v.view(ns, mc, nk * hd)}
    if case["op"] == "attn":
        nh, L = case["n_head"], case["prefix"]
        g = nh // nk
        out = torch.zeros((ns, nh, hd), dtype=torch.float64, device="cuda")
        w = s.w0.double() if case["weights"] else None
        for b, n in enumerate(s.lens.tolist()):
            kb, vb = s.k[b, :n].double(), s.v[b, :n].double()
            if L:
                kb, vb = torch.cat([s.pk.double(), kb]), torch.cat([s.pv.double(), vb])
            for kvh in range(nk):
                col = slice(kvh * hd, (kvh + 1) * hd)
                qb = s.q[b].double().view(nh, hd)[kvh * g:(kvh + 1) * g]
                p = torch.softmax(qb @ kb[:, col].T / math.sqrt(hd), dim=1)
                out[b, kvh * g:(kvh + 1) * g] = p @ vb[:, col]
                if case["weights"]:
                    w[b, kvh, :n] += p[:, L:].sum(0)
        out = out.view(ns, nh * hd)
        return {"out": out, "weights": w} if case["weights"] else {"out": out}
    keep = case["keep"]
    k, v = s.k.cpu().view(ns, mc, nk, hd), s.v.cpu().view(ns, mc, nk, hd)
    pos, w, lens = s.pos0.cpu().clone(), s.w0.cpu().clone(), s.lens0.cpu().clone()
    for b in range(ns):
        n = int(lens[b])
        if n <= keep:
            continue
        for h in range(nk):
            p, wl = pos[b, h, :n].tolist(), w[b, h, :n].tolist()
            newest = max(p)
            rank = sorted(range(n), key=lambda i: (not (p[i] < case["n_sink"] or p[i] > newest - case["n_recent"]),
                                                   0.0 if (p[i] < case["n_sink"] or
                                                           p[i] > newest - case["n_recent"]) else -wl[i], i))
            kept = set(rank[:keep])
            holes = [i for i in range(keep) if i not in kept]
            movers = [i for i in range(keep, n) if i in kept]
            if holes:
                hi, mi = torch.tensor(holes), torch.tensor(movers)
                k[b, hi, h], v[b, hi, h] = k[b, mi, h], v[b, mi, h]
                pos[b, h, hi], w[b, h, hi] = pos[b, h, mi], w[b, h, mi]
            w[b, h, keep:n] = 0.0
        lens[b] = keep
    return {"k": k.reshape(ns, mc, nk * hd).double().cuda(), "v": v.reshape(ns, mc, nk * hd).double().cuda(),
            "row_pos": pos.cuda(), "row_weight": w.double().cuda(), "lens": lens.cuda()}


# ---- what a pass cannot do without ------------------------------------------------
def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    nk, hd, ns = case["n_kv"], case["head_dim"], case["n_seq"]
    if case["op"] == "rope":
        T, nh = case["tokens"], case["n_head"]
        stored = T if ns == 1 else T - T // 8
        return {"bytes": T * (nh + 2 * nk) * hd * 4 + es * hd * (T * nh + stored * 2 * nk) + 8 * T,
                "flops": 3 * T * (nh + nk) * case["rot"]}
    if case["op"] == "attn":
        nh, L, rows = case["n_head"], case["prefix"], sum(_lens_of(case))
        return {"bytes": es * hd * (2 * nk * (L + rows) + 2 * ns * nh) + 4 * ns +
                (8 * nk * rows if case["weights"] else 0),
                "flops": 4 * hd * nh * (ns * L + rows)}
    total, keep = 0, case["keep"]
    for n in _lens_of(case):
        if n <= keep:
            continue
        # rows above the limit that stay: the newest ones, and their share of the rest
        recent = min(case["n_recent"], n - keep)
        free = keep - case["n_sink"] - case["n_recent"]
        rest = n - case["n_sink"] - case["n_recent"]
        moved = recent + (free * (n - keep - recent) // rest if rest > 0 else 0)
        total += nk * (8 * n + moved * (4 * hd * es + 8) + 4 * (n - keep))
    return {"bytes": total + 8 * ns, "flops": 0}
