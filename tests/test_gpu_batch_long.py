"""The batched-decode operators over long rows and many steps: every form of
the eviction's selection, sums that are put away many times, row weights that
gather over a decode."""
import pytest
import torch

import _batch_ref as R
import lalmodel_b200 as lb
from test_gpu_batch import score_step
from test_gpu_batch_values import F32_NORM, head_errors

pytestmark = pytest.mark.gpu


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("B,nk,C,long,keep,sink,recent", [
    # keys of a CTA in shared memory: a cluster of 2 and of 4
    (10, 4, 17000, {0: 16999, 3: 17000, 9: 12001}, 9000, 4, 500),
    (2, 2, 60000, {0: 59999, 1: 33000}, 4097, 5, 1000),
    # more rows of a CTA than fit there: the keys formed again in every pass, by one
    # CTA of more pairs than leave room for clusters, and by a cluster of 4
    (19, 4, 46500, {0: 46500, 7: 46100, 18: 45000}, 20000, 16, 3000),
    (1, 1, 190001, {0: 189990}, 100003, 0, 7),
    # .. where all the weights are equal, so that whole CTAs are ties
    (1, 1, 190001, {0: 190001}, 95001, 3, 0),
])
def test_kv_evict_long(ctx, B, nk, C, long, keep, sink, recent):
    hd, dt = 32, torch.float16
    g = torch.Generator().manual_seed(C + keep)
    k = torch.randn(B, C, nk * hd, generator=torch.Generator("cuda").manual_seed(C), device="cuda").to(dt)
    v = torch.randn(B, C, nk * hd, generator=torch.Generator("cuda").manual_seed(B), device="cuda").to(dt)
    pos = torch.stack([torch.randperm(2 * C, generator=g)[:C] for _ in range(B * nk)]).view(B, nk, C).to(torch.int32)
    w = (torch.rand(B, nk, C, generator=g) * 4096).floor() / 4096
    if sink == 3:
        w = torch.full_like(w, 0.25)
    lens = torch.tensor([long.get(b, keep - b) for b in range(B)], dtype=torch.int32)
    before = (k.clone(), v.clone())
    cache = lb.KVBatch(k, v, nk, pos.cuda(), w.cuda())
    ld = lens.cuda()
    ctx.kv_evict(cache, ld, keep, sink, recent)
    rl, rp, rw, moves = R.evict(lens, pos, w, keep, sink, recent)
    assert torch.equal(ld.cpu(), rl)
    assert torch.equal(cache.row_pos.cpu(), rp)
    assert torch.equal(cache.row_weight.cpu(), rw)
    for got, t in ((cache.k, before[0]), (cache.v, before[1])):
        rows = t.view(B, C, nk, hd)
        for (b, h), pairs in moves.items():
            if pairs:
                d, s = torch.tensor(pairs, device="cuda").T
                rows[b, d, h] = rows[b, s, h]
        assert torch.equal(got, t)
    assert ctx.device_status() == 0


@pytest.mark.parametrize("hd,nk,nh,L", [
    (64, 1, 8, 250000),      # 26 tiles a CTA: three sums in memory of each of two streams
    (128, 1, 8, 250000),
    (256, 1, 4, 100000),     # two halves of the value columns, 21 tiles a CTA, one stream: five
    (128, 1, 20, 120000),    # .. more than 16 query rows
])
def test_f32_sums_over_many_tiles(ctx, hd, nk, nh, L):
    k, v, q = rand(hd, L, nk * hd), rand(hd + 1, L, nk * hd), rand(hd + 2, 1, nh * hd)
    own = rand(hd + 3, 1, 5, nk * hd)
    lens = torch.tensor([5], dtype=torch.int32)
    out = ctx.attention_batch(lb.KVBatch(own.cuda(), own.cuda(), nk), q.cuda(), lens.cuda(), nh, k.cuda(), v.cuda())
    ref = R.attention(q, own, own, lens, nh, nk, k, v)[0]
    err = head_errors(out.cpu().view(1, nh, hd), ref.view(1, nh, hd))
    assert float(err.max()) <= F32_NORM, err


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_row_weights_gather_over_a_decode(ctx, dtype):
    """row_weight through appends (0), steps of attention (decay 1) and
    evictions (moved with their rows), against the 64-bit weights of every
    step added up."""
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    nh, nk, hd, B, C, keep, L = 4, 2, 64, 3, 48, 24, 70
    pk, pv = rand(1, L, nk * hd, dtype=dt), rand(2, L, nk * hd, dtype=dt)
    cache = lb.KVBatch(torch.zeros(B, C, nk * hd, dtype=dt, device="cuda"),
                       torch.zeros(B, C, nk * hd, dtype=dt, device="cuda"), nk,
                       torch.zeros(B, nk, C, dtype=torch.int32, device="cuda"),
                       torch.zeros(B, nk, C, device="cuda"))
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    first = torch.arange(B, dtype=torch.int32, device="cuda") * C
    want, tol = torch.zeros(B, nk, C, dtype=torch.float64), torch.zeros(B, nk, C, dtype=torch.float64)
    rope, evictions = lb.Rope(theta=1e4), 0
    for step in range(100):
        qkv = rand(100 + step, B, (nh + 2 * nk) * hd).cuda()
        q = ctx.rope_append(cache, qkv, torch.full_like(lens, L + step), first + lens, nh, rope)
        at = int(lens[0])
        want[:, :, at] = tol[:, :, at] = 0.0
        lens += 1
        ctx.attention_batch(cache, q, lens, nh, pk.cuda(), pv.cuda(), decay=1.0)
        _, w, _, top = R.attention(q.cpu(), cache.k.cpu(), cache.v.cpu(), lens.cpu(), nh, nk, pk, pv)
        # a weight: twice the score's error, the sum of exponentials (a rounding per
        # row of a tile on each of its paths, per tile and partial); then the addition
        s = score_step(top).view(B, nk, -1).amax(-1)[:, :, None]
        want += w
        tol += w * (2 * s + 2.0 ** -21 + (64 + (L + C) / 64 + 8) * 2.0 ** -24) + 3 * 2.0 ** -24 * want
        got = cache.row_weight.cpu()
        assert bool(((got - want).abs() <= tol).all()), (step, float(((got - want).abs() - tol).max()))
        if at + 1 == C:
            _, _, _, moves = R.evict(lens.cpu(), cache.row_pos.cpu(), got, keep, 0, 8)
            ctx.kv_evict(cache, lens, keep, n_sink=0, n_recent=8)
            for (b, g), pairs in moves.items():
                for d, s in pairs:
                    want[b, g, d], tol[b, g, d] = want[b, g, s], tol[b, g, s]
            want[:, :, keep:] = tol[:, :, keep:] = 0.0
            assert bool(((cache.row_weight.cpu() - want).abs() <= tol).all())
            evictions += 1
    # full after 48 rows, then after every 24 more: steps 48, 72 and 96
    assert evictions == 3 and ctx.device_status() == 0
