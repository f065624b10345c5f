"""The batched-decode operators (lalb_rope_append, lalb_attention_batch,
lalb_kv_evict) against their 64-bit restatements, their refusals, and a run of
them together."""
import ctypes

import numpy as np
import pytest
import torch

import _batch_ref as R
import _oracle as O
import lalmodel_b200 as lb
from lalmodel_b200 import _abi

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INVALID, UNSUPPORTED, BAD_ROW = -1, -4, 2


def half_step(dt):
    """Largest relative error of one rounding to dt."""
    return torch.finfo(dt).eps / 2


def rand(seed, *shape, dtype=torch.float32, sigma=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * sigma).to(dtype)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def within(got, ref, tol):
    err = (got.cpu().double() - ref).abs()
    assert bool(torch.isfinite(err).all())
    assert bool((err <= tol).all()), float((err - tol).max())


# ---- rotary append --------------------------------------------------------------------
def rope_tol(ref, mag, dt):
    # cos and sin: 2 units of 2^-24 from sincospif (1 ulp each side of 1), one
    # from the remainder's correction and one from mscale; the product and the
    # fma round once each: 6 x 2^-24 of |x0| + |x1|, then the store's rounding
    return 6 * 2.0 ** -24 * mag + half_step(dt) * (ref.abs() + 6 * 2.0 ** -24 * mag) + \
        (0 if dt == torch.float32 else 2.0 ** -25)


@pytest.mark.parametrize("dtype,layout,rot,scaling,T,nh,nk,hd", [
    ("f32", "half", 0, "none", 1, 28, 4, 128),
    ("f32", "half", 32, "linear", 5, 2, 2, 64),
    ("f16", "interleaved", 0, "parts", 3, 6, 3, 32),
    ("bf16", "half", 8, "none", 150, 1, 1, 32),        # more tokens than SMs: several per CTA
    ("bf16", "interleaved", 64, "parts", 301, 8, 1, 256),
    ("f32", "interleaved", 24, "linear", 2, 5, 5, 64),
    ("f16", "half", 256, "none", 149, 4, 4, 256),
    ("f32", "half", 0, "parts", 148, 71, 1, 64),
])
def test_rope_append(ctx, dtype, layout, rot, scaling, T, nh, nk, hd):
    dt = DT[dtype]
    n_seq, C = 4, (T + 3) // 4 + 2
    width = (nh + 2 * nk) * hd
    qkv = rand(T + nh, T, width + 8)
    pos = torch.randint(0, 200000, (T,), generator=torch.Generator().manual_seed(T)).to(torch.int32)
    slots = torch.randperm(n_seq * C, generator=torch.Generator().manual_seed(1))[:T].to(torch.int32)
    if T > 2:
        slots[1] = -1                                  # padding stores nothing
    k0, v0 = rand(7, n_seq, C, nk * hd, dtype=dt), rand(8, n_seq, C, nk * hd, dtype=dt)
    rp0 = torch.full((n_seq, nk, C), -5, dtype=torch.int32)
    rw0 = torch.full((n_seq, nk, C), 3.0)
    par = dict(theta=5e5, scaling=scaling, factor=4.0, orig_ctx=8192.0)
    ms = 1.25 if scaling == "parts" else 1.0
    cache = lb.KVBatch(k0.cuda(), v0.cuda(), nk, rp0.cuda(), rw0.cuda())
    rope = lb.Rope(layout=layout, rot_dim=rot, mscale=ms, **par)
    rows = qkv.cuda()[:, :width]                       # rows 8 elements apart
    q = ctx.rope_append(cache, rows, pos.cuda(), slots.cuda(), nh, rope)
    y, mag = R.rotate(qkv[:, :width].double().view(T, nh + 2 * nk, hd)[:, :nh + nk], pos,
                      R.freqs(rot or hd, **par), layout, ms)
    within(q, y[:, :nh].reshape(T, -1), rope_tol(y, mag, dt)[:, :nh].reshape(T, -1))
    tol = rope_tol(y, mag, dt)[:, nh:].reshape(T, -1)
    kf, vf = cache.k.cpu().view(-1, nk * hd), cache.v.cpu().view(-1, nk * hd)
    rp, rw = cache.row_pos.cpu(), cache.row_weight.cpu()
    stored = [t for t in range(T) if slots[t] >= 0]
    idx = slots[stored].long()
    within(kf[idx], y[stored, nh:].reshape(len(stored), -1), tol[stored])
    assert torch.equal(vf[idx], qkv[stored][:, (nh + nk) * hd:width].to(dt))
    others = torch.ones(n_seq * C, dtype=torch.bool)
    others[idx] = False
    assert torch.equal(kf[others], k0.view(-1, nk * hd)[others])
    assert torch.equal(vf[others], v0.view(-1, nk * hd)[others])
    for t in stored:
        b, j = divmod(int(slots[t]), C)
        rp0[b, :, j], rw0[b, :, j] = int(pos[t]), 0.0
    assert torch.equal(rp, rp0) and torch.equal(rw, rw0)


def test_rope_append_16_bit_rows_and_q_alone(ctx):
    nh, nk, hd, T = 3, 1, 64, 9
    x = rand(3, T, nh * hd, dtype=torch.bfloat16)
    k = torch.zeros(1, 4, hd, dtype=torch.bfloat16, device="cuda")
    cache = lb.KVBatch(k, k.clone(), nk)
    pos = torch.arange(T, dtype=torch.int32) * 1000
    q = ctx.rope_append(cache, x.cuda(), pos.cuda(), None, nh)
    y, mag = R.rotate(x.double().view(T, nh, hd), pos, R.freqs(hd), "half")
    within(q, y.reshape(T, -1), rope_tol(y, mag, torch.bfloat16).reshape(T, -1))
    assert not cache.k.any() and not cache.v.any()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_gradient_is_the_rotation_back(ctx, layout):
    """d<c, rope(x)>/dx is rope at the negated positions applied to c: against
    the formula's gradient in 64 bits and against differences."""
    nh, hd, T = 2, 32, 3
    cache = lb.KVBatch(torch.zeros(1, 1, 2 * hd, device="cuda"), torch.zeros(1, 1, 2 * hd, device="cuda"), 2)
    x, c = rand(5, T, nh * hd), rand(6, T, nh * hd)
    pos = ints(3, 77, 40001)
    rope = lb.Rope(layout=layout, rot_dim=16, theta=1e6, mscale=1.5)
    g = ctx.rope_append(cache, c.cuda(), (-pos).cuda(), None, nh, rope)
    f = R.freqs(16, theta=1e6)
    xd = x.double().view(T, nh, hd).requires_grad_()
    (R.rotate(xd, pos, f, layout, 1.5)[0] * c.double().view(T, nh, hd)).sum().backward()
    _, mag = R.rotate(c.double().view(T, nh, hd), pos, f, layout, 1.5)
    within(g, xd.grad.reshape(T, -1), rope_tol(xd.grad, mag, torch.float32).reshape(T, -1))
    # differences: the map is linear, so a step of 1 is exact up to rounding
    e = torch.zeros_like(x)
    for i in (0, 9, 33, 63):
        e[:, i] = 1.0
    step = (ctx.rope_append(cache, (x + e).cuda(), pos.cuda(), None, nh, rope).double()
            - ctx.rope_append(cache, x.cuda(), pos.cuda(), None, nh, rope).double()).cpu()
    diff = (step * c.double()).sum(1)
    want = (g.cpu().double() * e.double()).sum(1)
    # each side's roundings: 2 x 6 x 2^-24 of the magnitudes, and x + e rounds once
    bound = 16 * 2.0 ** -24 * (1.5 * 2 * ((x.abs() + 1).sum(1) * c.abs().max()).double() + mag.sum((1, 2)))
    assert bool(((diff - want).abs() <= bound).all())


def test_rope_append_bad_slot_is_reported(ctx):
    nk, hd = 1, 32
    k0 = rand(1, 2, 3, hd)
    cache = lb.KVBatch(k0.cuda(), k0.cuda(), nk)
    qkv = rand(2, 3, 3 * hd).cuda()
    ctx.rope_append(cache, qkv, ints(0, 1, 2).cuda(), ints(6, 2, 2 ** 31 - 1).cuda(), 1)
    assert ctx.device_status(reset=True) == BAD_ROW
    keep = [0, 1, 3, 4, 5]
    assert torch.equal(cache.k.cpu().view(6, hd)[keep], k0.view(6, hd)[keep])
    assert not torch.equal(cache.k.cpu().view(6, hd)[2], k0.view(6, hd)[2])
    assert ctx.rope_append(cache, qkv[:0], ints().cuda(), ints().cuda(), 1).shape == (0, hd)


# ---- attention ------------------------------------------------------------------------------
def score_step(top):
    """Bound on a score's error in natural units, from sum |q k| * scale:
    operands are exact (16 bits) or two fp16 parts, the high one on a grid of
    2^-11 of the largest of 16 rows, the rest within 2^-24 of it: 2 x 2^-23 of
    sum |q k| for the sizes tested; at most 16 large fp32 additions on the
    tensor cores (head_dim 256) within 2^-23 each, the 48 of the small products
    2^-10 of that; scale and shift round twice; twice all that: 64 x 2^-23."""
    return top * 64 * 2.0 ** -23


def attn_tol(ref, mag, top, dt, rows):
    """p is off by twice the score's error (its own and the maximum's) and by
    exp2's 2 ulp (2^-22); weights and values as two fp16 parts are within 3 x
    2^-22.  The tensor cores cut each addition off by up to 2^-23 of the sum:
    F32 makes 12 a tile of 64 rows, in runs of 4 tiles whose sums are then added
    in fp32 (one rounding per 256 rows); 16 bits makes 8 a tile.  8 more
    roundings join streams and partials.  16-bit outputs round by half a step
    (and their weights, as two parts, by its square)."""
    hd = ref.shape[1] // top.shape[1]
    t = top.repeat_interleave(hd, 1)
    adds = min(rows * 12 / 64, 48) + rows / 256 if dt == torch.float32 else rows * 8 / 64
    rel = 2 * score_step(t) + 2.0 ** -22 + 3 * 2.0 ** -22 + (adds + 8) * 2.0 ** -23
    if dt != torch.float32:
        rel = rel + half_step(dt) ** 2 * 4
    tiny = 0 if dt == torch.float32 else 2.0 ** -25
    return mag * rel * (1 + half_step(dt)) + half_step(dt) * ref.abs() + tiny


def run_attention(ctx, dtype, B, nh, nk, hd, L, lens, C, seed, weights=None, scale=None, stale=None, pad=0):
    dt = DT[dtype]
    q = rand(seed, B, nh * hd + pad, dtype=dt, sigma=1.5)[:, :nh * hd]
    k, v = rand(seed + 1, B, C, nk * hd, dtype=dt), rand(seed + 2, B, C, nk * hd, dtype=dt)
    pk = rand(seed + 3, L, nk * hd, dtype=dt) if L else None
    pv = rand(seed + 4, L, nk * hd, dtype=dt) if L else None
    kd, vd = k.clone(), v.clone()
    if stale is not None:      # rows behind a sequence hold anything
        for b in range(B):
            kd[b, max(0, int(lens[b])):] = stale
            vd[b, max(0, int(lens[b])):] = stale
    w0 = rand(seed + 5, B, nk, C).abs()
    cache = lb.KVBatch(kd.cuda(), vd.cuda(), nk, row_weight=w0.cuda() if weights is not None else None)
    base = rand(seed, B, nh * hd + pad, dtype=dt, sigma=1.5).cuda()
    out = ctx.attention_batch(cache, base[:, :nh * hd], lens.cuda(), nh, None if pk is None else pk.cuda(),
                              None if pv is None else pv.cuda(), scale=scale or 0.0, decay=weights)
    n = torch.where((lens < 0) | (lens > C), torch.zeros_like(lens), lens)
    ref, w, mag, top = R.attention(q, k, v, n, nh, nk, pk, pv, scale)
    rows = L + int(n.max()) if B else 0
    within(out, ref, attn_tol(ref, mag, top, dt, rows))
    assert not out.cpu()[(n == 0) & (L == 0)].any()
    if weights is not None:
        live = torch.arange(C)[None, None, :] < n[:, None, None]
        want = torch.where(live, weights * w0.double() + w, w0.double())
        step = score_step(top).view(B, nk, -1).amax(-1)[:, :, None]
        # the sum of exponentials is added up in fp32: a rounding per row of a
        # tile's 64 on each of its paths at most, one per tile and partial
        tol = torch.where(live, w * (2 * step + 2.0 ** -21 + (64 + rows / 64 + 8) * 2.0 ** -24)
                          + 3 * 2.0 ** -24 * want.abs() + 1e-38, torch.zeros_like(want))
        within(cache.row_weight, want, tol)
    return out, cache


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B,nh,nk,hd,L,lens,C", [
    (1, 28, 4, 128, 0, [1], 1),                 # the first token
    (1, 28, 4, 128, 0, [815], 1024),
    (3, 4, 4, 64, 65, [0, 63, 64], 64),         # plain heads, lengths around a tile
    (2, 6, 2, 32, 129, [7, 200], 201),
    (5, 8, 2, 256, 31, [0, 1, 33, 64, 130], 130),
    (4, 16, 1, 128, 300, [128, 129, 0, 5], 140),
    (19, 14, 2, 64, 1000, list(range(0, 190, 10)), 190),   # 133 rows of queries per KV head
    (2, 130, 1, 64, 77, [100, 3], 128),         # more q heads on a KV head than one tile holds
    (40, 8, 4, 128, 700, [3] * 40, 8),
])
def test_attention_batch(ctx, dtype, B, nh, nk, hd, L, lens, C):
    run_attention(ctx, dtype, B, nh, nk, hd, L, ints(*lens), C, seed=B * 100 + hd, stale=float("nan"))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,decay", [(128, 1.0), (64, 0.5), (256, 0.0), (32, 1.0)])
def test_attention_batch_weights(ctx, dtype, hd, decay):
    run_attention(ctx, dtype, 4, 6, 2, hd, 100, ints(0, 1, 70, 333), 333, seed=hd, weights=decay,
                  stale=float("nan"))
    run_attention(ctx, dtype, 2, 3, 3, hd, 0, ints(64, 400), 400, seed=hd + 1, weights=decay)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_batch_empty_and_bad_lengths(ctx, dtype):
    """No rows at all gives 0; a length outside the cache counts as 0 and is reported."""
    run_attention(ctx, dtype, 3, 4, 2, 64, 0, ints(0, 5, 0), 8, seed=1, stale=float("inf"))
    assert ctx.device_status() == 0
    run_attention(ctx, dtype, 3, 4, 2, 64, 0, ints(-1, 5, 9), 8, seed=2, weights=1.0)
    assert ctx.device_status(reset=True) == BAD_ROW
    run_attention(ctx, dtype, 2, 4, 2, 64, 40, ints(-7, 2 ** 31 - 1), 8, seed=3)
    assert ctx.device_status(reset=True) == BAD_ROW


def test_attention_batch_scale_and_strided_rows(ctx):
    run_attention(ctx, "f32", 3, 4, 2, 64, 50, ints(10, 20, 30), 32, seed=11, scale=0.37, pad=64)
    run_attention(ctx, "bf16", 3, 4, 2, 64, 50, ints(10, 20, 30), 32, seed=12, scale=-0.2, pad=8)


@pytest.mark.parametrize("mag", [1e-12, 1e-4, 3e4, 1e9])
def test_attention_batch_f32_ranges(ctx, mag):
    """fp32 values far from 1, and rows whose sizes differ by 2^20, through
    the fp16 parts."""
    B, nh, nk, hd, L, C = 2, 4, 2, 128, 90, 80
    q, k, v = rand(1, B, nh * hd), rand(2, B, C, nk * hd), rand(3, B, C, nk * hd) * mag
    pk, pv = rand(4, L, nk * hd), rand(5, L, nk * hd) * mag
    size = torch.exp2(torch.randint(-20, 1, (B, C, 1), generator=torch.Generator().manual_seed(6)).float())
    v *= size
    k *= size.flip(1)
    lens = ints(80, 41)
    kc = (k / mag).cuda()           # q k stays of order 1
    cache = lb.KVBatch(kc, v.cuda(), nk)
    out = ctx.attention_batch(cache, (q * mag).cuda(), lens.cuda(), nh, (pk / mag).cuda(), pv.cuda())
    ref, _, m, top = R.attention((q * mag), kc.cpu(), v, lens, nh, nk, (pk / mag), pv)
    within(out, ref, attn_tol(ref, m, top, torch.float32, L + 80))


@pytest.mark.parametrize("dtype,hd,nk,nh,B,L,C", [
    ("f32", 32, 8, 8, 2, 12000, 40),      # several sums of O per segment, few rows
    ("f32", 128, 1, 8, 20, 40000, 9),     # .. and 160 rows of queries
    ("f32", 256, 2, 2, 3, 20000, 70),     # one stream of tiles
    ("bf16", 64, 4, 8, 3, 30000, 70),
])
def test_attention_batch_long(ctx, dtype, hd, nk, nh, B, L, C):
    run_attention(ctx, dtype, B, nh, nk, hd, L, ints(*[(7 * b + 3) % (C + 1) for b in range(B)]), C, seed=hd, weights=1.0)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_batch_many_sequences(ctx, dtype):
    """More sequences than a CTA keeps lengths of, most of them short, some empty."""
    B, C = 700, 130
    lens = torch.tensor([(b * 37) % 9 if b % 50 else C - b % 3 for b in range(B)], dtype=torch.int32)
    run_attention(ctx, dtype, B, 2, 1, 64, 65, lens, C, seed=5, weights=0.5, stale=float("nan"))


def test_attention_batch_two_calls_at_once(ctx):
    """Two streams, a workspace each, the same cache."""
    B, nh, nk, hd, C, L = 6, 8, 2, 128, 500, 3000
    k, v = rand(1, B, C, nk * hd), rand(2, B, C, nk * hd)
    pk, pv, lens = rand(3, L, nk * hd), rand(4, L, nk * hd), ints(500, 3, 0, 77, 128, 499)
    cache = lb.KVBatch(k.cuda(), v.cuda(), nk)
    qs = [rand(10 + i, B, nh * hd) for i in range(2)]
    dev = [q.cuda() for q in qs]
    pkd, pvd, ld = pk.cuda(), pv.cuda(), lens.cuda()
    ws = [ctx.attention_batch_ws(cache, nh, L) for _ in range(2)]
    outs = [torch.empty_like(d) for d in dev]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                ctx.attention_batch(cache, dev[i], ld, nh, pkd, pvd, ws=ws[i], out=outs[i])
    torch.cuda.synchronize()
    for i in range(2):
        ref, _, mag, top = R.attention(qs[i], k, v, lens, nh, nk, pk, pv)
        within(outs[i], ref, attn_tol(ref, mag, top, torch.float32, L + C))


def test_attention_batch_large_scores(ctx):
    """Scores in the hundreds: one row takes all the weight, whichever tile it is in."""
    for dtype in ("f32", "bf16"):
        dt = DT[dtype]
        B, nh, nk, hd, L, C = 2, 2, 1, 64, 500, 300
        q = rand(1, B, nh * hd, dtype=dt, sigma=8.0)
        k, v = rand(2, B, C, hd, dtype=dt, sigma=8.0), rand(3, B, C, hd, dtype=dt)
        pk, pv = rand(4, L, hd, dtype=dt, sigma=8.0), rand(5, L, hd, dtype=dt)
        lens = ints(300, 17)
        out = ctx.attention_batch(lb.KVBatch(k.cuda(), v.cuda(), nk), q.cuda(), lens.cuda(), nh, pk.cuda(), pv.cuda())
        ref, _, mag, top = R.attention(q, k, v, lens, nh, nk, pk, pv)
        within(out, ref, attn_tol(ref, mag, top, dt, L + 300))


def test_attention_batch_repeats_bit_for_bit(ctx):
    a, _ = run_attention(ctx, "f32", 6, 8, 2, 64, 3000, ints(0, 9, 500, 77, 64, 1), 500, seed=21, weights=1.0)
    for _ in range(3):
        b, _ = run_attention(ctx, "f32", 6, 8, 2, 64, 3000, ints(0, 9, 500, 77, 64, 1), 500, seed=21, weights=1.0)
        assert torch.equal(a, b)


def test_attention_batch_captured_on_another_stream(ctx):
    """One graph replayed with other lengths and queries, on a stream of its own."""
    nh, nk, hd, L, C, B = 8, 2, 128, 200, 300, 4
    k, v = rand(1, B, C, nk * hd, dtype=torch.bfloat16), rand(2, B, C, nk * hd, dtype=torch.bfloat16)
    pk, pv = rand(3, L, nk * hd, dtype=torch.bfloat16), rand(4, L, nk * hd, dtype=torch.bfloat16)
    cache = lb.KVBatch(k.cuda(), v.cuda(), nk, row_weight=torch.zeros(B, nk, C, device="cuda"))
    q, lens, pkd, pvd = torch.zeros(B, nh * hd, dtype=torch.bfloat16, device="cuda"), ints(1, 2, 3, 4).cuda(), \
        pk.cuda(), pv.cuda()
    ws = ctx.attention_batch_ws(cache, nh, L, True)
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        def call():
            ctx.attention_batch(cache, q, lens, nh, pkd, pvd, decay=0.0, ws=ws, out=out)
        call()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            call()
        for n in ([300, 0, 64, 129], [5, 299, 1, 0]):
            qh = rand(sum(n), B, nh * hd, dtype=torch.bfloat16)
            q.copy_(qh)
            lens.copy_(ints(*n))
            ws.fill_(0xff)               # nothing in the workspace is kept between calls
            graph.replay()
            s.synchronize()
            ref, w, mag, top = R.attention(qh, k, v, ints(*n), nh, nk, pk, pv)
            within(out, ref, attn_tol(ref, mag, top, torch.bfloat16, L + 300))
            for b in range(B):
                assert abs(float(cache.row_weight[b, :, :n[b]].sum()) - float(w[b].sum())) < 1e-3
    graph.reset()


# ---- eviction ----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,B,nk,hd,C,lens,keep,sink,recent", [
    ("f32", 1, 4, 128, 1024, [1024], 512, 4, 128),
    ("bf16", 4, 2, 64, 700, [700, 300, 301, 0], 300, 0, 0),
    ("f16", 3, 1, 256, 130, [130, 129, 128], 1, 0, 1),
    ("f32", 2, 3, 32, 97, [97, 50], 49, 20, 29),            # protected rows fill the budget
    ("bf16", 1, 1, 32, 9000, [8999], 8000, 16, 100),
    ("f16", 2, 2, 64, 2, [2, 1], 1, 0, 0),
    ("bf16", 1, 2, 32, 60000, [59999], 4097, 5, 1000),      # keys formed again in every pass
])
def test_kv_evict(ctx, dtype, B, nk, hd, C, lens, keep, sink, recent):
    dt = DT[dtype]
    k, v = rand(1, B, C, nk * hd, dtype=dt), rand(2, B, C, nk * hd, dtype=dt)
    g = torch.Generator().manual_seed(C)
    # positions in any order, as they are after an earlier eviction; weights with ties, zeros, NaN
    pos = torch.stack([torch.randperm(2 * C, generator=g)[:C] for _ in range(B * nk)]).view(B, nk, C).to(torch.int32)
    w = (torch.rand(B, nk, C, generator=g) * 16).floor() / 16
    w[torch.rand(B, nk, C, generator=g) < 0.05] = float("nan")
    w[torch.rand(B, nk, C, generator=g) < 0.05] = -0.0
    lens = ints(*lens)
    cache = lb.KVBatch(k.cuda(), v.cuda(), nk, pos.cuda(), w.cuda())
    ld = lens.cuda()
    ctx.kv_evict(cache, ld, keep, sink, recent)
    rl, rp, rw, moves = R.evict(lens, pos, w, keep, sink, recent)
    assert torch.equal(ld.cpu(), rl)
    assert torch.equal(cache.row_pos.cpu(), rp)
    assert torch.equal(cache.row_weight.cpu().view(torch.int32), rw.view(torch.int32))
    for got, t in ((cache.k, k), (cache.v, v)):
        assert torch.equal(got.cpu().view(torch.int16), R.apply_moves(t, moves, nk).view(torch.int16))


def test_kv_evict_weights_of_every_kind(ctx):
    """Infinities, negatives and subnormals rank as numbers do."""
    C, keep = 64, 7
    w = torch.tensor([float("inf"), -float("inf"), 1e-45, -1e-45, 0.0, -0.0, 3.4e38, -3.4e38] * 8).view(1, 1, C)
    pos = torch.arange(C, dtype=torch.int32).view(1, 1, C)
    k = rand(4, 1, C, 32)
    cache = lb.KVBatch(k.cuda(), k.cuda(), 1, pos.cuda(), w.cuda())
    lens = ints(C).cuda()
    ctx.kv_evict(cache, lens, keep)
    _, rp, _, moves = R.evict(ints(C), pos, w, keep, 0, 0)
    assert torch.equal(cache.row_pos.cpu(), rp)
    assert torch.equal(cache.k.cpu(), R.apply_moves(k, moves, 1))


def test_kv_evict_bad_length_is_reported_and_left(ctx):
    C = 20
    k, pos = rand(4, 3, C, 32), torch.arange(C, dtype=torch.int32).expand(3, 1, C).contiguous()
    w = rand(5, 3, 1, C).abs()
    cache = lb.KVBatch(k.cuda(), k.cuda(), 1, pos.cuda(), w.cuda())
    lens = ints(21, 20, -3)
    ld = lens.cuda()
    ctx.kv_evict(cache, ld, 10)
    assert ctx.device_status(reset=True) == BAD_ROW
    assert ld.cpu().tolist() == [21, 10, -3]
    assert torch.equal(cache.k.cpu()[[0, 2]], k[[0, 2]]) and torch.equal(cache.row_weight.cpu()[[0, 2]], w[[0, 2]])
    # nothing can be too long for a budget of the whole cache, but a bad length is still reported
    before = cache.k.clone()
    ctx.kv_evict(cache, ints(20, 21, 0).cuda(), 20)
    assert ctx.device_status(reset=True) == BAD_ROW
    assert torch.equal(cache.k, before)


def test_two_graphs_share_a_workspace(ctx):
    """A step of attention whose output replaces its queries, and an eviction,
    each in a graph, replayed in turn over one workspace."""
    nh, nk, hd, L, C, B, keep = 6, 2, 64, 130, 200, 3, 90
    k, v = rand(1, B, C, nk * hd), rand(2, B, C, nk * hd)
    pk, pv = rand(3, L, nk * hd), rand(4, L, nk * hd)
    pos = torch.arange(C, dtype=torch.int32).expand(B, nk, C).contiguous()
    cache = lb.KVBatch(k.cuda(), v.cuda(), nk, pos.cuda(), torch.zeros(B, nk, C, device="cuda"))
    q, lens, pkd, pvd = torch.zeros(B, nh * hd, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda"), \
        pk.cuda(), pv.cuda()
    ws = max(ctx.attention_batch_ws(cache, nh, L, True), ctx.kv_evict_ws(cache, keep), key=lambda t: t.numel())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        calls = (lambda: ctx.attention_batch(cache, q, lens, nh, pkd, pvd, decay=1.0, ws=ws, out=q),
                 lambda: ctx.kv_evict(cache, lens, keep, n_sink=2, n_recent=5, ws=ws))
        graphs = []
        for call in calls:
            call()
            s.synchronize()
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=s):
                call()
        for i, n in enumerate(([200, 90, 120], [91, 0, 200], [1, 150, 89])):
            qh = rand(50 + i, B, nh * hd)
            q.copy_(qh)
            lens.copy_(ints(*n))
            before = (cache.k.cpu(), cache.v.cpu(), cache.row_weight.cpu())
            graphs[0].replay()
            s.synchronize()
            ref, w, mag, top = R.attention(qh, *before[:2], ints(*n), nh, nk, pk, pv)
            within(q, ref, attn_tol(ref, mag, top, torch.float32, L + C))
            got = cache.row_weight.cpu()
            step = score_step(top).view(B, nk, -1).amax(-1)[:, :, None]
            within(got, before[2].double() + w,                 # run_attention's bound
                   w * (2 * step + 2.0 ** -21 + (64 + (L + C) / 64 + 8) * 2.0 ** -24)
                   + 3 * 2.0 ** -24 * (before[2].double() + w))
            rl, rp, rw, moves = R.evict(ints(*n), cache.row_pos.cpu(), got, keep, 2, 5)
            graphs[1].replay()
            s.synchronize()
            assert torch.equal(lens.cpu(), rl) and torch.equal(cache.row_pos.cpu(), rp)
            assert torch.equal(cache.row_weight.cpu(), rw)
            assert torch.equal(cache.k.cpu(), R.apply_moves(before[0], moves, nk))
            assert torch.equal(cache.v.cpu(), R.apply_moves(before[1], moves, nk))
    for g in graphs:
        g.reset()


# ---- refusals --------------------------------------------------------------------------------------
def test_batch_refusals(ctx):
    hd, nk, B, C = 64, 2, 2, 16
    k = torch.zeros(B, C, nk * hd, device="cuda")
    rp = torch.zeros(B, nk, C, dtype=torch.int32, device="cuda")
    rw = torch.zeros(B, nk, C, device="cuda")
    cache = lb.KVBatch(k, k.clone(), nk, rp, rw)
    bare = lb.KVBatch(k, k.clone(), nk)
    lens, q = ints(1, 1).cuda(), torch.zeros(B, 4 * hd, device="cuda")
    qkv, pos, slots = torch.zeros(B, 8 * hd, device="cuda"), ints(0, 1).cuda(), ints(0, 16).cuda()

    def refuses(status, fn, *a, **kw):
        with pytest.raises(lb.LalbError) as e:
            fn(*a, **kw)
        assert e.value.status == status, str(e.value)

    # rotary parameters
    for bad in (dict(theta=1.0), dict(theta=float("inf")), dict(theta=float("nan")), dict(mscale=float("nan")),
                dict(scaling="linear", factor=0.0), dict(scaling="parts", factor=2.0),
                dict(scaling="parts", factor=2.0, orig_ctx=100.0, turns_fast=1.0, turns_slow=1.0)):
        refuses(INVALID, ctx.rope_append, cache, qkv, pos, slots, 4, lb.Rope(**bad))
    for rot in (12, 72, -8):
        refuses(UNSUPPORTED, ctx.rope_append, cache, qkv, pos, slots, 4, lb.Rope(rot_dim=rot))
    refuses(INVALID, lb.Rope, layout="thirds")
    # tensors
    refuses(INVALID, ctx.rope_append, cache, qkv.half(), pos, slots, 4)
    refuses(INVALID, ctx.rope_append, cache, qkv[:, 1:], pos, slots, 4)
    refuses(INVALID, ctx.rope_append, cache, qkv, pos.long(), slots, 4)
    refuses(INVALID, ctx.rope_append, cache, qkv, pos.cpu(), slots, 4)
    refuses(INVALID, ctx.attention_batch, cache, q.half(), lens, 4)
    refuses(INVALID, ctx.attention_batch, cache, q[:1], lens, 4)
    refuses(INVALID, ctx.attention_batch, cache, q, lens[:1], 4)
    refuses(INVALID, ctx.attention_batch, cache, q, lens, 4, prefix_k=k[0])
    refuses(INVALID, ctx.attention_batch, bare, q, lens, 4, decay=1.0)
    refuses(INVALID, ctx.attention_batch, cache, q, lens, 4, decay=float("nan"))
    refuses(INVALID, ctx.attention_batch, cache, q, lens, 4, scale=float("inf"))
    refuses(INVALID, ctx.attention_batch, cache, q, lens, 4, scale=3e38)
    refuses(INVALID, ctx.attention_batch, cache, torch.zeros(B, 3 * hd, device="cuda"), lens, 3)
    refuses(INVALID, ctx.attention_batch, cache, q, lens, 4, ws=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    refuses(INVALID, ctx.kv_evict, bare, lens, 8)
    for keep, sink, recent in ((0, 0, 0), (17, 0, 0), (8, 5, 4), (8, -1, 0), (8, 0, -1)):
        refuses(INVALID, ctx.kv_evict, cache, lens, keep, sink, recent)
    # head_dim the kernels do not handle
    odd = lb.KVBatch(torch.zeros(1, 4, 48, device="cuda"), torch.zeros(1, 4, 48, device="cuda"), 1)
    refuses(UNSUPPORTED, ctx.attention_batch, odd, torch.zeros(1, 48, device="cuda"), ints(1).cuda(), 1)
    # the C entry points: null, misaligned and short arguments
    L, d = _abi.lib(), ctypes.byref(cache.desc)
    attn, rope = _abi.AttnBatchDesc(4, 0.0, 0, None, None, 0, 0.0), lb.Rope().desc
    ws, p, s = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda"), lb._p, lb._stream()
    off = ctypes.c_void_p(q.data_ptr() + 4)
    assert L.lalb_attention_batch(ctx.h, d, ctypes.byref(attn), None, 256, p(lens), p(ws), p(q), s) == INVALID
    assert L.lalb_attention_batch(ctx.h, d, ctypes.byref(attn), off, 256, p(lens), p(ws), p(q), s) == INVALID
    assert L.lalb_attention_batch(ctx.h, d, ctypes.byref(attn), p(q), 255, p(lens), p(ws), p(q), s) == INVALID
    assert L.lalb_attention_batch(ctx.h, d, ctypes.byref(attn), p(q), 256, p(lens), off, p(q), s) == INVALID
    assert L.lalb_rope_append(ctx.h, ctypes.byref(rope), d, 4, p(qkv), 0, 511, 2, p(pos), p(slots), p(q), s) == INVALID
    assert L.lalb_rope_append(ctx.h, ctypes.byref(rope), d, 4, p(qkv), 0, 512, -1, p(pos), p(slots), p(q), s) == INVALID
    assert L.lalb_kv_evict(ctx.h, d, p(lens), 8, 0, 0, None, s) == INVALID
    assert L.lalb_kv_evict(None, d, p(lens), 8, 0, 0, p(ws), s) == INVALID
    assert ctx.device_status() == 0


# ---- together ------------------------------------------------------------------------------------------
def test_far_rows(ctx):
    """Rows whose offsets pass 2^31 elements (2^32 bytes)."""
    nk, hd, B, C = 8, 128, 3, 1100000
    k = torch.empty(B, C, nk * hd, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    rp = torch.zeros(B, nk, C, dtype=torch.int32, device="cuda")
    cache = lb.KVBatch(k, v, nk, rp, torch.zeros(B, nk, C, device="cuda"))
    T = 70
    qkv = rand(1, T, 3 * nk * hd)
    pos = torch.arange(T, dtype=torch.int32)
    ctx.rope_append(cache, qkv.cuda(), pos.cuda(), (2 * C + pos).to(torch.int32).cuda(), nk)
    kb, vb = k[2:, :T].cpu(), v[2:, :T].cpu()
    y, mag = R.rotate(qkv.double().view(T, 3 * nk, hd)[:, nk:2 * nk], pos, R.freqs(hd), "half")
    within(kb[0], y.reshape(T, -1), rope_tol(y, mag, torch.bfloat16).reshape(T, -1))
    q = rand(2, B, nk * hd, dtype=torch.bfloat16)
    lens = ints(0, 0, T)
    out = ctx.attention_batch(cache, q.cuda(), lens.cuda(), nk, decay=1.0)
    ref, _, m, top = R.attention(q[2:], kb, vb, ints(T), nk, nk)
    within(out[2:], ref, attn_tol(ref, m, top, torch.bfloat16, T))
    w = cache.row_weight[2:, :, :T].cpu()
    ld = lens.cuda()
    ctx.kv_evict(cache, ld, 20, 2, 8)
    _, _, _, moves = R.evict(ints(T), rp[2:, :, :T].cpu() * 0 + pos.expand(1, nk, T), w, 20, 2, 8)
    assert ld.cpu().tolist() == [0, 0, 20]
    assert torch.equal(k[2:, :T].cpu(), R.apply_moves(kb, moves, nk))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_batch_decode_run(ctx, dtype):
    """Steps of a layer as a serving loop makes them: a prompt becomes the
    shared prefix, then each step's qkv product goes through the rotary append
    and the attention, with an eviction between steps; every step against the
    64-bit restatement of the rows the cache holds."""
    dt = DT[dtype]
    nh, nk, hd, hidden, B, C, keep = 4, 2, 64, 256, 3, 48, 24
    width = (nh + 2 * nk) * hd
    W = torch.from_numpy(O.q4k_quantize(O.normal(width * hidden, seed=5, sigma=0.05).reshape(width, hidden))).cuda()
    rope = lb.Rope(theta=1e4, rot_dim=32, layout="interleaved")
    # the prefix: a prompt of 150 tokens into a cache of its own
    L = 150
    x = torch.from_numpy(O.normal(L * hidden, seed=6).reshape(L, hidden)).cuda()
    pre = lb.KVBatch(torch.zeros(1, L, nk * hd, dtype=dt, device="cuda"),
                     torch.zeros(1, L, nk * hd, dtype=dt, device="cuda"), nk)
    at = torch.arange(L, dtype=torch.int32, device="cuda")
    ctx.rope_append(pre, ctx.matmul_q4_k_prefill(W, width, hidden, x), at, at, nh, rope)
    cache = lb.KVBatch(torch.zeros(B, C, nk * hd, dtype=dt, device="cuda"),
                       torch.zeros(B, C, nk * hd, dtype=dt, device="cuda"), nk,
                       torch.zeros(B, nk, C, dtype=torch.int32, device="cuda"),
                       torch.zeros(B, nk, C, device="cuda"))
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    first = torch.arange(B, dtype=torch.int32, device="cuda") * C
    weights = torch.zeros(B, nk, C, dtype=torch.float64)
    for step in range(60):
        x = torch.from_numpy(O.normal(B * hidden, seed=100 + step).reshape(B, hidden)).cuda()
        qkv = ctx.matmul_q4_k_prefill(W, width, hidden, x)
        q = ctx.rope_append(cache, qkv, torch.full_like(lens, L + step), first + lens, nh, rope)
        lens += 1
        out = ctx.attention_batch(cache, q, lens, nh, pre.k[0], pre.v[0], decay=1.0)
        n = lens.cpu()
        ref, w, mag, top = R.attention(q.cpu(), cache.k.cpu(), cache.v.cpu(), n, nh, nk, pre.k[0].cpu(),
                                       pre.v[0].cpu())
        within(out, ref, attn_tol(ref, mag, top, dt, L + C))
        assert bool((cache.row_weight.cpu()[:, :, n[0]:] == 0).all())
        if int(n[0]) == C:
            before = (n, cache.row_pos.cpu(), cache.row_weight.cpu(), cache.k.cpu(), cache.v.cpu())
            ctx.kv_evict(cache, lens, keep, n_sink=0, n_recent=8)
            rl, rp, rw, moves = R.evict(*before[:3], keep, 0, 8)
            assert torch.equal(lens.cpu(), rl) and torch.equal(cache.row_pos.cpu(), rp)
            assert torch.equal(cache.row_weight.cpu(), rw)
            assert torch.equal(cache.k.cpu(), R.apply_moves(before[3], moves, nk))
            assert torch.equal(cache.v.cpu(), R.apply_moves(before[4], moves, nk))
    assert ctx.device_status() == 0
    assert int(cache.row_pos[:, :, :int(lens[0])].max()) == L + 59
