"""lalb_attention_batch on values of very different sizes and on values that
are not finite: what one head, sequence or row holds must not reach another."""
import math

import pytest
import torch

import _batch_ref as R
import lalmodel_b200 as lb

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

# F32, ||error|| / ||out|| of one head's row, for scores of order 1 (|s| <= 4
# over a thousand rows).  The tensor cores cut each addition off by 2^-24 of
# the running sum on average.  Scores: 16 large additions at most (head_dim
# 256), sums that grow from 0 to s, |s| 2 in the root mean square of the rows
# that matter: 16 * 2^-24 * 2 = 1.9e-6.  Outputs: 12 additions a tile, four
# tiles to a sum that grows from 0: 48 / 2 * 2^-24 = 1.4e-6; rounding of
# streams, partials and 22-bit parts: 10 * 2^-24 = 0.6e-6.
F32_NORM = 4e-6


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


class Case:
    """A batch with a prefix: sequences and heads of a small attention call."""

    def __init__(self, dtype, B, nh, nk, hd, L, lens, seed):
        dt = DT[dtype]
        self.B, self.nh, self.nk, self.hd, self.lens = B, nh, nk, hd, ints(*lens)
        C = max(lens) + 3
        self.q = rand(seed, B, nh * hd, dtype=dt)
        self.k, self.v = rand(seed + 1, B, C, nk * hd, dtype=dt), rand(seed + 2, B, C, nk * hd, dtype=dt)
        self.pk = rand(seed + 3, L, nk * hd, dtype=dt) if L else None
        self.pv = rand(seed + 4, L, nk * hd, dtype=dt) if L else None
        self.w = None

    def run(self, ctx, decay=None):
        w = None if decay is None else torch.zeros(self.B, self.nk, self.k.shape[1], device="cuda")
        cache = lb.KVBatch(self.k.cuda(), self.v.cuda(), self.nk, row_weight=w)
        out = ctx.attention_batch(cache, self.q.cuda(), self.lens.cuda(), self.nh,
                                  None if self.pk is None else self.pk.cuda(),
                                  None if self.pv is None else self.pv.cuda(), decay=decay)
        self.w = None if w is None else w.cpu()
        return out.cpu().view(self.B, self.nh, self.hd)

    def exact(self):
        out = R.attention(self.q, self.k, self.v, self.lens, self.nh, self.nk, self.pk, self.pv)[0]
        return out.view(self.B, self.nh, self.hd)


def head_errors(got, ref):
    """||error|| / ||ref|| of each (sequence, head)."""
    return (got.double() - ref).norm(dim=-1) / ref.norm(dim=-1)


# (B, nh, nk, L, lens): query rows of a prefix unit above and up to 16
MANY, FEW = (5, 8, 2, 333, (200, 70, 0, 64, 1)), (3, 4, 2, 70, (40, 130, 9))


@pytest.mark.parametrize("shape", [MANY, FEW])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_f32_one_sequences_queries_leave_the_others(ctx, hd, shape):
    """One sequence's queries 2^12, 2^30 or 1e30 times larger, or infinite; the
    others' outputs stay as exact as they are without."""
    B, nh, nk, L, lens = shape
    for big in (2.0 ** 12, 2.0 ** 30, 1e30, float("inf")):
        c = Case("f32", B, nh, nk, hd, L, lens, seed=hd + B)
        ref = c.exact()
        c.q[1] *= big
        others = [b for b in range(B) if b != 1]
        err = head_errors(c.run(ctx), ref)[others]
        assert float(err.max()) <= F32_NORM, (big, err)
    assert ctx.device_status() == 0


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_f32_heads_of_different_size(ctx, hd):
    """Every other head's queries 2^10 times larger: the heads beside them, in
    the prefix's units and in each sequence's own, stay as exact."""
    c = Case("f32", 4, 8, 2, hd, 150, (90, 0, 33, 128), seed=hd)
    c.q.view(c.B, c.nh, hd)[:, ::2] *= 2.0 ** 10
    err = head_errors(c.run(ctx), c.exact())[:, 1::2]
    assert float(err.max()) <= F32_NORM, err


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("factor", [64.0, 1024.0])
def test_f32_outlier_keys_and_channels(ctx, hd, factor):
    """One key in eight many times larger, pointing away from the queries (it
    takes no weight); then one channel of all keys larger and of all queries
    smaller.  Either way the scores that matter are those without."""
    c = Case("f32", 4, 8, 2, hd, 150, (90, 3, 33, 250), seed=hd + 1)
    c.q = c.q.abs() * 0.5
    for k in (c.pk, c.k.view(-1, 2 * hd)):
        k[::8] = -factor * k[::8].abs()
    err = head_errors(c.run(ctx), c.exact())
    assert float(err.max()) <= F32_NORM, err
    c = Case("f32", 4, 8, 2, hd, 150, (90, 3, 33, 250), seed=hd + 2)
    c.q.view(-1, hd)[:, 5] /= factor
    for k in (c.pk, c.k):
        k.view(-1, hd)[:, 5] *= factor
    err = head_errors(c.run(ctx), c.exact())
    assert float(err.max()) <= F32_NORM, err


def check_heads(got, ref, bad, dtype):
    """Heads in `bad` [B][nh] are NaN throughout, the others as exact as ever:
    F32 by F32_NORM, 16 bits by one rounding of every element."""
    assert bool(torch.isnan(got[bad]).all())
    err = head_errors(got, ref)[~bad]
    tol = F32_NORM if dtype == "f32" else torch.finfo(DT[dtype]).eps / 2
    assert bool((err <= tol).all()), err


ALONE = (3, 4, 2, 0, (65, 1, 130))       # no prefix


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [MANY, FEW, ALONE])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_nan_query_stays_in_its_head(ctx, dtype, hd, shape):
    B, nh, nk, L, lens = shape
    c = Case(dtype, B, nh, nk, hd, L, lens, seed=hd + 10)
    ref, bad = c.exact(), torch.zeros(B, nh, dtype=torch.bool)
    for b, h in ((0, 1), (B - 1, nh - 1)):
        c.q.view(B, nh, hd)[b, h, hd // 2 + b] = float("nan")
        bad[b, h] = True
    check_heads(c.run(ctx, decay=0.0), ref, bad, dtype)
    # the weights that such a head adds to are NaN, all others numbers
    group = bad.view(B, nk, nh // nk).any(-1)
    for b in range(B):
        assert torch.equal(torch.isnan(c.w[b, :, :lens[b]]).all(-1), group[b] | (torch.tensor(lens[b]) == 0))
        assert bool(torch.isfinite(c.w[b][~group[b]]).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [MANY, FEW, ALONE])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_nan_key_reaches_the_heads_that_read_it(ctx, dtype, hd, shape):
    """A NaN in a row's key, the only row of a sequence and the ends of tiles
    among them: every head that reads it is NaN, and no other."""
    B, nh, nk, L, lens = shape
    group = nh // nk
    for b in range(B):
        for j in sorted({0, 63, 64, lens[b] - 1}):
            if not 0 <= j < lens[b]:
                continue
            c = Case(dtype, B, nh, nk, hd, L, lens, seed=hd + 11)
            ref, bad = c.exact(), torch.zeros(B, nh, dtype=torch.bool)
            c.k[b, j, (nk - 1) * hd + 3] = float("nan")
            bad[b, (nk - 1) * group:] = True
            check_heads(c.run(ctx), ref, bad, dtype)
    if L:
        c = Case(dtype, B, nh, nk, hd, L, lens, seed=hd + 12)
        ref, bad = c.exact(), torch.zeros(B, nh, dtype=torch.bool)
        c.pk[L - 1, 0] = float("nan")
        bad[:, :group] = True
        check_heads(c.run(ctx), ref, bad, dtype)
    assert ctx.device_status() == 0


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [MANY, FEW, ALONE])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("what", ["inf", "-inf", "nan"])
def test_value_that_is_not_finite_stays_in_its_column(ctx, dtype, hd, shape, what):
    B, nh, nk, L, lens = shape
    group, col, bad = nh // nk, 7, float(what)
    rest = torch.ones(hd, dtype=torch.bool)
    rest[col] = False
    tol = F32_NORM if dtype == "f32" else torch.finfo(DT[dtype]).eps / 2
    for where in ("own", "prefix") if L else ("own",):
        c = Case(dtype, B, nh, nk, hd, L, lens, seed=hd + 13)
        ref = c.exact()
        spoiled = torch.zeros(B, nh, dtype=torch.bool)
        if where == "own":
            for b, j in ((0, lens[0] - 1), (1, 0)):
                c.v[b, j, (nk - 1) * hd + col] = bad
                spoiled[b, (nk - 1) * group:] = True
        else:
            c.pv[L // 2, col] = bad
            spoiled[:, :group] = True
        got = c.run(ctx)
        assert not bool(torch.isfinite(got[spoiled][:, col]).any())
        assert bool((head_errors(got[..., rest], ref[..., rest]) <= tol).all())
        assert bool((head_errors(got, ref)[~spoiled] <= tol).all())


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_infinite_keys(ctx, hd):
    """F32: the heads that read one are NaN, the others as exact as without.
    16 bits: a score of -inf is a weight of 0."""
    for dtype in ("f32", "f16", "bf16"):
        B, nh, nk, L, lens = MANY
        c = Case(dtype, B, nh, nk, hd, L, lens, seed=hd + 14)
        c.q.view(B, nh, hd)[..., 2] = 0.5
        bad = torch.zeros(B, nh, dtype=torch.bool)
        ref = c.exact()
        for b, j in ((0, 199), (1, 0)):
            c.k[b, j, 2] = -float("inf")
            bad[b, :nh // nk] = True
        if dtype != "f32":
            ref, bad = c.exact(), torch.zeros_like(bad)
        check_heads(c.run(ctx), ref, bad, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("shape", [MANY, FEW, ALONE])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_scores_of_minus_infinity_throughout(ctx, dtype, hd, shape):
    """Rows of which every score is -inf: NaN as the softmax of them is (0 is
    for a sequence without rows); beside a prefix with other scores, nothing."""
    B, nh, nk, L, lens = shape
    c = Case(dtype, B, nh, nk, hd, L, lens, seed=hd + 15)
    c.q.view(B, nh, hd)[..., 2] = 0.5
    c.k[1, :, 2] = -float("inf")
    ref, bad = c.exact(), torch.zeros(B, nh, dtype=torch.bool)
    bad[1, :nh // nk] = L == 0
    check_heads(c.run(ctx, decay=0.0), ref, bad, dtype)
    w = c.w[1, 0, :lens[1]]
    assert bool((w == 0).all() if L else torch.isnan(w).all()), w
    if L and 0 in lens:
        b = lens.index(0)
        c.pk[:, 2] = -float("inf")
        bad[1, :nh // nk] = bad[b, :nh // nk] = True
        check_heads(c.run(ctx), c.exact(), bad, dtype)


def test_bf16_outputs_are_the_nearest(ctx):
    """How many outputs are not the exact result's nearest bf16.  An error e
    moves an output x off its nearest with probability e / step(x), steps
    being 2^-8 to 2^-7 of |x|: 185 e / |x| on average.  Outputs are sums of
    values of either sign, normal about 0 with deviation s, and an error is of
    s's size, not of |x|'s: the mean of 1 / |x| over |x| > d is
    sqrt(2 / pi) (ln(s / d) + 0.06) / s, 6.1 / s for the d = 5e-4 s below which
    every output is off.  So 185 * 6.1 = 1130 of e / s.  Weights as two rounded
    bf16 parts are within 2^-18 of a weight, 1.7e-6 on average; scores (8
    additions cut off at 2^-24 of 4, and the shift's rounding), the
    exponential (2^-22) and a tile's 8 additions add 1.5e-6 at most:
    1130 * 3.3e-6 = 3.8e-3.  A first part cut off instead of rounded, within
    2^-16, is above that: 1130 * 6.8e-6 for the weights alone at their bound,
    4.3e-3 as measured."""
    c = Case("bf16", 64, 8, 2, 128, 0, (64,) * 64, seed=77)
    got, ref = c.run(ctx), c.exact()
    off = (got != ref.to(torch.bfloat16)).double().mean()
    assert float(off) <= 3.8e-3, float(off)
