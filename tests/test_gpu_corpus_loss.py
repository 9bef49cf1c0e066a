"""Softmax losses over a whole corpus and their gradients (include/cgvec_train.h) against their definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

from _util import pkg

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24


def _half_step(dt):
    return torch.finfo(TYPES[dt]).eps / 2


def _unit(x):
    return x / x.norm(dim=1, keepdim=True).clamp_min(1e-30)


def _problem(b, n, d, k, dt, seed, toward=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows = _unit(torch.randn((n, d), generator=gen, device="cuda"))
    ids = torch.randint(0, n, (b, k), generator=gen, device="cuda")
    q = torch.randn((b, d), generator=gen, device="cuda")
    q = _unit(_unit(q) + (rows[ids].mean(dim=1) * 1.5 if toward else 0))
    sc = torch.rand((b, k), generator=gen, device="cuda").sort(dim=1, descending=True).values
    g = torch.rand((b,), generator=gen, device="cuda") + 0.25
    return q.to(TYPES[dt]), rows.to(TYPES[dt]), ids, sc, g


def _reference(q, r, ids, sc, g, scale, tscale):
    """The definition, 64 bits; also what the tolerances need. Queries without a listed row count as zero vectors."""
    b, n = q.shape[0], r.shape[0]
    valid = (ids >= 0) & (ids < n)
    if sc is None:
        w = valid.double()
    else:
        t = torch.where(valid, sc.double() * tscale, torch.full_like(sc, -math.inf, dtype=torch.float64))
        top = t.amax(dim=1, keepdim=True)
        w = torch.where(torch.isinf(top), torch.zeros_like(t), torch.exp(t - top))
    some = w.sum(dim=1) > 0
    w = w / w.sum(dim=1, keepdim=True).clamp_min(1e-300)
    q = torch.where(some[:, None], q.double(), torch.zeros_like(q, dtype=torch.float64))
    r = r.double()
    s = scale * torch.matmul(q, r.t())
    lse = torch.logsumexp(s, dim=1)
    picked = torch.gather(s, 1, ids.clamp(0, n - 1))
    loss = torch.where(some, (torch.special.xlogy(w, w) + torch.where(w > 0, w * (lse[:, None] - picked), torch.zeros_like(w))).sum(dim=1), torch.zeros_like(lse))
    P = torch.exp(s - lse[:, None]) * some[:, None]
    W = torch.zeros_like(s).scatter_add_(1, ids.clamp(0, n - 1), w)
    G = (P - W) * (g.double() * scale)[:, None]
    M = (P + W) * (g.double().abs() * abs(scale))[:, None]
    return dict(loss=loss, dq=G @ r, dr=torch.matmul(G.t(), q), mq=M @ r.abs(), mr=torch.matmul(M.t(), q.abs()), lse=lse, some=some,
                norm=q.norm(dim=1) * r.norm(dim=1).max(), q=q, r=r, w=w)


def _check(got_loss, got_dq, got_dr, ref, d, n, scale, dt, g, u=None):
    # A score is a sum of d products in f32: partial sums stay below |q| |r|, each addition rounds by at most 2^-24 of one, signs
    # at random: 4 sqrt(d) of them (and the product's own, and the factor's). log-sum-exp: the exponentials' arguments are rounded
    # once more (2^-24 of the score), exp2 itself is good to 2^-22, their sum has errors like 4 sqrt(n) * 2^-24.
    ds = U * abs(scale) * (4 * math.sqrt(d) + 12) * ref["norm"] + U * 2 * ref["lse"].abs()
    rel = 2 * ds + U * (4 * math.sqrt(n) + 16)
    lim = rel + U * (ref["loss"].abs() + 8)
    err = (got_loss.double() - ref["loss"]).abs()
    assert bool((err <= lim).all()), ("loss", float((err / lim).max()))
    u = u or max(_half_step(dt), 2.0 ** -22)      # G is rounded to the type (f32: three planes, 2^-24 of a product left out twice)
    per = rel.max() + u + U * (4 * math.sqrt(max(n, got_loss.numel())) + 8)
    # fp16: entries of G below 2^-14 of the scaled range lose digits: an absolute 2^-38 of the largest factor
    # every type: a softmax value below 2^-126, the smallest normal f32, is zero - its entry of G is off by 2^-126 |dloss * scale|
    sub = (2.0 ** -37 if dt == "fp16" else 2.0 ** -126) * float((g * scale).abs().max())
    tiny = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "fp16": 2.0 ** -24}[dt]
    for name, got, want, mag, other in (("dq", got_dq, ref["dq"], ref["mq"], ref["r"]), ("dr", got_dr, ref["dr"], ref["mr"], ref["q"])):
        if got is None:
            continue
        lim = mag * per + want.abs() * _half_step(dt) * 1.001 + sub * other.abs().sum(dim=0)[None] + tiny
        err = (got.double() - want).abs()
        assert got.dtype == TYPES[dt] and got.shape == want.shape
        assert bool((err <= lim).all()), (name, float((err / lim).max()))
        # and far closer than that on the whole: roundings are independent
        if want.norm() > 1e-3 * mag.norm():
            assert float((got.double() - want).norm() / want.norm()) <= 3 * _half_step(dt) + 4 * float(per - u) * float(mag.norm() / want.norm()) + 1e-6


SHAPES = [(1, 1, 1, 1), (1, 2, 64, 1), (2, 3, 8, 3), (3, 257, 63, 2), (32, 1000, 384, 1), (64, 256, 64, 5), (65, 300, 65, 1), (128, 777, 96, 4),
          (130, 2000, 128, 10), (257, 1023, 200, 37), (300, 5000, 768, 1), (40, 600, 1536, 256), (1000, 3000, 64, 3)]


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("b,n,d,k", SHAPES)
def test_losses_and_gradients(b, n, d, k, dt):
    m = pkg()
    q, r, ids, sc, g = _problem(b, n, d, k, dt, b + n + d)
    if b > 8:
        ids[b // 3] = -1                                     # queries that take no part
        ids[b - 1] = n
    if k > 2:
        ids[0, 1:] = -1                                      # a list of one, a list that ends early
        sc[0, 1:] = -math.inf
        sc[min(1, b - 1), k // 2:] = -math.inf
        ids[b // 2, 1] = ids[b // 2, 0]                      # the same row twice
    scale, tscale = 12.0, 9.0
    q.requires_grad_()
    r.requires_grad_()
    ref = _reference(q.detach(), r.detach(), ids, sc, g, scale, tscale)
    loss = m.corpus_distillation(q, r, ids, sc, scale=scale, teacher_scale=tscale)
    assert loss.dtype == torch.float32 and loss.shape == (b,)
    dq, dr = torch.autograd.grad(loss, (q, r), g)
    _check(loss.detach(), dq, dr, ref, d, n, scale, dt, g)
    assert bool((loss[~ref["some"]] == 0).all()) and bool((dq[~ref["some"]] == 0).all())
    again = m.corpus_distillation(q, r, ids, sc, scale=scale, teacher_scale=tscale)
    assert torch.equal(loss, again)                          # the same bits every time
    assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(again, (q, r), g), (dq, dr)))
    t = ids[:, 0].contiguous()
    ref = _reference(q.detach(), r.detach(), t[:, None], None, g, scale, 1.0)
    loss = m.corpus_cross_entropy(q, r, t, scale=scale)
    dq, dr = torch.autograd.grad(loss, (q, r), g)
    _check(loss.detach(), dq, dr, ref, d, n, scale, dt, g)


@pytest.mark.parametrize("b,n,d,k,dt", [(20, 6000, 8192, 1, "f32"), (2900, 20_000, 64, 2, "f32"), (2000, 70_001, 64, 1, "bf16"), (70, 300_000, 40, 3, "fp16"),
                                        (5000, 30_011, 72, 1, "fp16")])
def test_corpus_in_pieces(b, n, d, k, dt):
    """Corpora that are gone through in several pieces, in place and through the padded copy."""
    m = pkg()
    q, r, ids, sc, g = _problem(b, n, d, k, dt, 77)
    q.requires_grad_()
    r.requires_grad_()
    ref = _reference(q.detach(), r.detach(), ids, sc, g, 8.0, 3.0)
    loss = m.corpus_distillation(q, r, ids, sc, scale=8.0, teacher_scale=3.0)
    dq, dr = torch.autograd.grad(loss, (q, r), g)
    _check(loss.detach(), dq, dr, ref, d, n, 8.0, dt, g)


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("b,n,d,k", [(300, 20_000, 72, 2), (430, 17_001, 96, 3), (640, 12_000, 63, 1), (700, 20_000, 40, 20), (3000, 6000, 64, 1),
                                     (65_950, 300, 16, 1)])
def test_batches_in_columns_of_two_widths(b, n, d, k, dt):
    """Batches whose last column of tiles is narrower than the others, up to more columns than the card has CUs."""
    m = pkg()
    q, r, ids, sc, g = _problem(b, n, d, k, dt, b + 1)
    ids[b - 1] = n - 1
    ids[b - 2] = -1
    q.requires_grad_()
    r.requires_grad_()
    ref = _reference(q.detach(), r.detach(), ids, sc, g, 8.0, 3.0)
    loss = m.corpus_distillation(q, r, ids, sc, scale=8.0, teacher_scale=3.0)
    dq, dr = torch.autograd.grad(loss, (q, r), g)
    _check(loss.detach(), dq, dr, ref, d, n, 8.0, dt, g)
    assert bool((dq[b - 2] == 0).all())


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("b,n,d,k", [(33, 500, 64, 1), (70, 3000, 123, 2), (1000, 700, 40, 1), (100, 2000, 8, 10), (812, 20_000, 64, 2), (200, 30_000, 72, 30)])
def test_listed_entries_lose_nothing_to_16_bits(b, n, d, k, dt):
    """The queries' gradient, in small problems the corpus' too: only what the rows outside the list add is rounded to 16 bits on its way. dloss is
    the same for all queries, so that the listed entries and their roundings are nearly alike."""
    m = pkg()
    q, r, ids, sc, _ = _problem(b, n, d, k, dt, b + n)
    ids[5] = -1
    if k > 2:
        ids[0, 2] = ids[0, 1]
    g = torch.full((b,), 1.013, device="cuda")
    q.requires_grad_()
    ref = _reference(q.detach(), r, ids, sc, g, 8.0, 1.0)
    (dq,) = torch.autograd.grad(m.corpus_distillation(q, r, ids, sc, scale=8.0, teacher_scale=1.0), (q,), g)
    P = torch.exp(8.0 * torch.matmul(ref["q"], ref["r"].t()) - ref["lse"][:, None]) * ref["some"][:, None]
    P.scatter_(1, ids.clamp(0, n - 1), 0.0)                  # (5: a query without a list has no gradient at all)
    u = _half_step(dt)
    ds = U * 8.0 * (4 * math.sqrt(d) + 12) * ref["norm"] + U * 2 * ref["lse"].abs()
    per = float((2 * ds + U * (4 * math.sqrt(n) + 16)).max()) + u * u + U * (4 * math.sqrt(max(n, b)) + 8)
    lim = (P * g[:, None].double() * 8.0) @ ref["r"].abs() * u + ref["mq"] * per + ref["dq"].abs() * u * 1.001
    lim = lim + (2.0 ** -37 if dt == "fp16" else 2.0 ** -126) * 8.2 * ref["r"].abs().sum(dim=0)[None] + (2.0 ** -24 if dt == "fp16" else 2.0 ** -126)
    err = (dq.double() - ref["dq"]).abs()
    assert bool((err <= lim).all()), float((err / lim).max())
    if b * k <= 1024 and n <= 5000:                          # small problems: the corpus' gradient as well
        r.requires_grad_()
        (dr,) = torch.autograd.grad(m.corpus_distillation(q, r, ids, sc, scale=8.0, teacher_scale=1.0), (r,), g)
        lim = (P * g[:, None].double() * 8.0).t() @ ref["q"].abs() * u + ref["mr"] * per + ref["dr"].abs() * u * 1.001
        lim = lim + (2.0 ** -37 if dt == "fp16" else 2.0 ** -126) * 8.2 * ref["q"].abs().sum(dim=0)[None] + (2.0 ** -24 if dt == "fp16" else 2.0 ** -126)
        err = (dr.double() - ref["dr"]).abs()
        assert bool((err <= lim).all()), float((err / lim).max())


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("b,n,d,k", [(1, 1, 8, 1), (1, 40, 17, 3), (3, 326, 123, 1), (8, 5000, 96, 256), (31, 20_000, 64, 2), (32, 60_000, 200, 5)])
def test_few_queries_lose_nothing_to_16_bits(b, n, d, k, dt):
    """Up to 32 queries: G is kept in two 16-bit parts, off by half a step of half a step; only the results' own rounding is left."""
    m = pkg()
    q, r, ids, sc, g = _problem(b, n, d, k, dt, b + n)
    if b > 3:
        ids[2] = -1
    if k > 2:
        ids[0, 2] = ids[0, 1]
    for h in (g, torch.where(torch.arange(b, device="cuda") % 2 == 0, g, g * 2.0 ** -6)):
        q.requires_grad_(), r.requires_grad_()
        ref = _reference(q.detach(), r.detach(), ids, sc, h, 8.0, 3.0)
        loss = m.corpus_distillation(q, r, ids, sc, scale=8.0, teacher_scale=3.0)
        dq, dr = torch.autograd.grad(loss, (q, r), h)
        _check(loss.detach(), dq, dr, ref, d, n, 8.0, dt, h, u=_half_step(dt) ** 2)
        (only,) = torch.autograd.grad(m.corpus_distillation(q, r.detach(), ids, sc, scale=8.0, teacher_scale=3.0), (q,), h)
        assert torch.equal(only, dq)


@pytest.mark.parametrize("b,n,d,dt", [(3, 700_001, 200, "bf16"), (100, 300_000, 456, "fp16"), (190, 130_001, 1040, "bf16"), (250, 270_000, 520, "fp16")])
def test_a_corpus_that_no_cache_holds(b, n, d, dt):
    """One column of tiles over more than 256 MiB of rows."""
    m = pkg()
    q, r, ids, sc, g = _problem(b, n, d, 2, dt, 9)
    ids[b - 1] = n - 1
    ref = _reference(q, r, ids, sc, g, 8.0, 3.0)
    loss = m.corpus_distillation(q, r, ids, sc, scale=8.0, teacher_scale=3.0)
    _check(loss, None, None, ref, d, n, 8.0, dt, g)
    assert torch.equal(loss, m.corpus_distillation(q, r, ids, sc, scale=8.0, teacher_scale=3.0))


def test_a_million_queries_with_long_lists():
    """More than 2^32 threads' worth of lists."""
    m = pkg()
    b, n, d, k = 2 ** 20 + 7, 20, 8, 256
    q, r, ids, sc, g = _problem(b, n, d, k, "bf16", 5)
    ids[b - 1, 1:] = -1
    ids[b - 2] = -1
    q.requires_grad_()
    r.requires_grad_()
    ref = _reference(q.detach(), r.detach(), ids, sc, g, 8.0, 3.0)
    loss = m.corpus_distillation(q, r, ids, sc, scale=8.0, teacher_scale=3.0)
    dq, dr = torch.autograd.grad(loss, (q, r), g)
    _check(loss.detach(), dq, dr, ref, d, n, 8.0, "bf16", g)
    del ref, q, r, ids, sc, g, loss, dq, dr
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dt", list(TYPES))
def test_one_gradient_at_a_time(dt):
    m = pkg()
    q, r, ids, sc, g = _problem(70, 900, 128, 3, dt, 5)
    both = torch.autograd.grad(m.corpus_distillation(q.requires_grad_(), r.requires_grad_(), ids, sc, scale=5.0), (q, r), g)
    (dq,) = torch.autograd.grad(m.corpus_distillation(q, r.detach(), ids, sc, scale=5.0), (q,), g)
    (dr,) = torch.autograd.grad(m.corpus_distillation(q.detach(), r, ids, sc, scale=5.0), (r,), g)
    assert torch.equal(dq, both[0]) and torch.equal(dr, both[1])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_small_losses_keep_their_digits(dt):
    """A query that finds its row: the loss is far below the scores' rounding, and so is the gradient."""
    m = pkg()
    q, r, ids, _, g = _problem(40, 500, 64, 1, dt, 6)
    q = r[ids[:, 0]].clone()
    scale = 40.0
    ref = _reference(q, r, ids, None, g, scale, 1.0)
    # 64 bits lose such a loss too where it is a difference of two scores: log1p of the others' sum does not
    diff = scale * torch.matmul(q.double(), r.double().t())
    diff = diff - torch.gather(diff, 1, ids)
    ref["loss"] = torch.log1p(torch.exp(diff).scatter_(1, ids, 0.0).sum(dim=1))
    assert float(ref["loss"].max()) < 1e-7
    loss = m.corpus_cross_entropy(q.requires_grad_(), r, ids[:, 0], scale=scale)
    # tail = log1p(sum of exp(s - s_target)): its relative error is that of the exponentials
    lim = (2 * U * scale * (4 * 8 + 12) * ref["norm"] + U * 2 * scale * 2 + U * 120) * ref["loss"]
    assert bool(((loss.detach().double() - ref["loss"]).abs() <= lim).all())
    (dq,) = torch.autograd.grad(loss, (q,), g)
    assert float((dq.double() - ref["dq"]).norm() / ref["dq"].norm()) <= 4 * _half_step(dt) + 2e-4


@pytest.mark.parametrize("dt", list(TYPES))
def test_strides_and_alignment(dt):
    m = pkg()
    for d in (64, 70):
        q, r, ids, sc, g = _problem(33, 300, d, 2, dt, 7)
        want = m.corpus_distillation(q.requires_grad_(), r.requires_grad_(), ids, sc, scale=6.0)
        grads = torch.autograd.grad(want, (q, r), g)
        wq, wr = torch.zeros((33, d + 40), device="cuda", dtype=q.dtype), torch.zeros((300, d + 40), device="cuda", dtype=q.dtype)
        for a in (0, 1, 8, 24):
            wq[:, a:a + d], wr[:, a:a + d] = q.detach(), r.detach()
            vq, vr = wq[:, a:a + d].detach().requires_grad_(), wr[:, a:a + d].detach().requires_grad_()
            got = m.corpus_distillation(vq, vr, ids.int(), sc.double(), scale=6.0)
            assert torch.equal(got, want)
            assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(got, (vq, vr), g), grads))
        tq, tr = q.detach().t().contiguous().t(), r.detach().t().contiguous().t()      # columns contiguous
        assert torch.equal(m.corpus_distillation(tq, tr, ids, sc, scale=6.0), want)
        one = m.corpus_distillation(q[:1].expand(33, d), r, ids[:1].expand(33, 2), sc[:1].expand(33, 2), scale=6.0)
        assert bool((one == want[0]).all())
        (dg,) = torch.autograd.grad(m.corpus_distillation(q, r, ids, sc, scale=6.0).sum(), (q,))     # an expanded incoming gradient
        (dg1,) = torch.autograd.grad(m.corpus_distillation(q, r, ids, sc, scale=6.0), (q,), torch.ones_like(g))
        assert torch.equal(dg, dg1)


def test_gradients_by_differences():
    m = pkg()
    q, r, ids, sc, g = _problem(9, 40, 24, 4, "f32", 8)
    args = (ids, sc)
    kw = dict(scale=3.0, teacher_scale=2.0)
    dq, dr = torch.autograd.grad(m.corpus_distillation(q.requires_grad_(), r.requires_grad_(), *args, **kw), (q, r), g)

    def f(qq, rr):
        return float((m.corpus_distillation(qq.detach(), rr.detach(), *args, **kw).double() * g.double()).sum())

    h = 2.0 ** -6
    for i, e in ((0, 0), (8, 23), (4, 7)):
        for x, grad in ((q, dq), (r, dr)):
            up, down = x.detach().clone(), x.detach().clone()
            up[i, e] += h
            down[i, e] -= h
            num = (f(up, r) - f(down, r)) / (2 * h) if x is q else (f(q, up) - f(q, down)) / (2 * h)
            # central difference: h^2 / 6 times a third derivative (scale^3 |row|^3, 9 queries), and the losses' own rounding
            assert abs(num - float(grad[i, e])) <= h * h / 6 * 27 * 2 * 9 * 1.25 * 0.5 + 9 * 40 * U / h


def test_values_that_must_not_spread():
    """NaN and Inf in queries that take no part, and behind masked entries of a list, reach nothing."""
    m = pkg()
    for dt in TYPES:
        q, r, ids, sc, g = _problem(66, 400, 72, 3, dt, 9)
        ids[5], ids[60] = -1, 400
        sc[7, 1:] = -math.inf
        sc[9] = -math.inf
        clean = m.corpus_distillation(q.requires_grad_(), r.requires_grad_(), ids, sc, scale=4.0)
        want = torch.autograd.grad(clean, (q, r), g)
        bad, g2, sc2 = q.detach().clone(), g.clone(), sc.clone()
        bad[5], bad[60, 3], bad[9, 0] = math.nan, math.inf, -math.inf
        g2[5], g2[9] = math.nan, math.inf
        sc2[5], sc2[60] = math.nan, math.inf                 # scores beside ids that are no rows
        bad.requires_grad_()
        got = m.corpus_distillation(bad, r, ids, sc2, scale=4.0)
        assert torch.equal(got, clean)
        assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(got, (bad, r), g2), want))
        bad = q.detach().clone()
        bad[3, 1] = math.nan                                 # one that does: its own loss, and every gradient of a row
        got = m.corpus_distillation(bad, r, ids, sc, scale=4.0)
        keep = torch.arange(66, device="cuda") != 3
        assert bool(torch.isnan(got[3])) and torch.equal(got[keep], clean[keep])
        nan = sc.clone()
        nan[11, 2] = math.nan
        got = m.corpus_distillation(q, r, ids, nan, scale=4.0)
        keep = torch.arange(66, device="cuda") != 11
        assert bool(torch.isnan(got[11])) and torch.equal(got[keep], clean[keep])


def test_large_scores():
    """Scores of some thousands: the sum of exp lies far beyond f32, the loss does not."""
    m = pkg()
    q, r, ids, sc, g = _problem(20, 600, 64, 2, "f32", 10)
    for scale in (3000.0, -3000.0):
        ref = _reference(q, r, ids, sc, g, scale, 1.0)
        loss = m.corpus_distillation(q.requires_grad_(), r.requires_grad_(), ids, sc, scale=scale)
        dq, dr = torch.autograd.grad(loss, (q, r), g)
        _check(loss.detach(), dq, dr, ref, 64, 600, scale, "f32", g)


def test_empty_forms():
    m = pkg()
    r = torch.randn((10, 16), device="cuda", requires_grad=True)
    q = torch.empty((0, 16), device="cuda", requires_grad=True)
    loss = m.corpus_cross_entropy(q, r, torch.empty((0,), dtype=torch.int64, device="cuda"))
    assert loss.shape == (0,)
    dq, dr = torch.autograd.grad(loss.sum(), (q, r))
    assert dq.shape == (0, 16) and bool((dr == 0).all())
    q = torch.randn((5, 16), device="cuda", requires_grad=True)
    loss = m.corpus_cross_entropy(q, r, torch.full((5,), -1, device="cuda"))
    dq, dr = torch.autograd.grad(loss.sum(), (q, r))
    assert bool((loss == 0).all()) and bool((dq == 0).all()) and bool((dr == 0).all())
    one = m.corpus_cross_entropy(q, r[:1], torch.zeros(5, dtype=torch.int64, device="cuda"), scale=7.0)   # a corpus of one row
    assert bool((one == 0).all())


def test_refusals():
    m = pkg()
    q, r = torch.zeros((3, 8), device="cuda"), torch.zeros((6, 8), device="cuda")
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    ids, sc = torch.zeros((3, 2), dtype=torch.int64, device="cuda"), torch.zeros((3, 2), device="cuda")
    inv, dim, non = m.cgvec.CGV_ERR_INVALID_ARG, m.cgvec.CGV_ERR_DIM_MISMATCH, m.cgvec.CGV_ERR_NONFINITE
    for code, call in ((inv, lambda: m.corpus_cross_entropy(q.cpu(), r, t)), (inv, lambda: m.corpus_cross_entropy(q, r.cpu(), t)), (inv, lambda: m.corpus_cross_entropy(q, r, t.cpu())),
                       (inv, lambda: m.corpus_cross_entropy(q.half(), r, t)), (inv, lambda: m.corpus_cross_entropy(q.double(), r.double(), t)),
                       (dim, lambda: m.corpus_cross_entropy(q[:, :7], r, t)), (dim, lambda: m.corpus_cross_entropy(q, r, t[:2])), (dim, lambda: m.corpus_cross_entropy(q, r, ids)),
                       (inv, lambda: m.corpus_cross_entropy(q, r[:0], t)), (inv, lambda: m.corpus_cross_entropy(q, r, t.float())),
                       (non, lambda: m.corpus_cross_entropy(q, r, t, scale=math.nan)), (non, lambda: m.corpus_distillation(q, r, ids, sc, teacher_scale=math.inf)),
                       (dim, lambda: m.corpus_distillation(q, r, ids, sc[:, :1])), (inv, lambda: m.corpus_distillation(q, r, ids, sc.cpu())),
                       (inv, lambda: m.corpus_distillation(q, r, ids[:, :0], sc[:, :0])), (inv, lambda: m.corpus_distillation(q, r, ids, ids)),
                       (inv, lambda: m.corpus_distillation(q, r, torch.zeros((3, 257), dtype=torch.int64, device="cuda"), torch.zeros((3, 257), device="cuda")))):
        with pytest.raises(m.CgvError) as ei:
            call()
        assert ei.value.code == code


def test_streams_and_graphs():
    m = pkg()
    q, r, ids, sc, g = _problem(100, 3000, 128, 4, "bf16", 11)
    q.requires_grad_()
    r.requires_grad_()

    def step():
        loss = m.corpus_distillation(q, r, ids, sc, scale=9.0)
        return (loss, *torch.autograd.grad(loss, (q, r), g))

    want = [x.detach().clone() for x in step()]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = step()
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            res = step()
        graphs.append((cg, res))
    gen = torch.Generator(device="cuda").manual_seed(12)
    for it in range(4):
        with torch.no_grad():
            q.copy_(_unit(torch.randn((100, 128), generator=gen, device="cuda")))
            ids.copy_(torch.randint(-1, 3000, (100, 4), generator=gen, device="cuda"))
            for _, res in graphs:
                [x.zero_() for x in res]
        want = step()
        torch.cuda.synchronize()
        for cg, _ in graphs:
            cg.replay()
        torch.cuda.synchronize()
        for _, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, want)), it


def test_two_threads():
    import threading
    m = pkg()
    probs = [_problem(40 + 30 * i, 2000, 96, 2, "bf16", 20 + i) for i in range(3)]

    def step(p):
        q, r, ids, sc, g = p
        q, r = q.detach().requires_grad_(), r.detach().requires_grad_()
        loss = m.corpus_distillation(q, r, ids, sc, scale=6.0)
        return (loss.detach(), *torch.autograd.grad(loss, (q, r), g))

    want = [step(p) for p in probs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(8):
                got = step(probs[i])
                st.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)
    th = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    [t.start() for t in th]
    [t.join() for t in th]
    assert not bad


def test_trained_then_served():
    """The operators as they are used together: a table is looked up and trained against a corpus, a search's answers teach a
    narrower model, the trained rows are searched and scored in 4 bits."""
    m = pkg()
    gen = torch.Generator(device="cuda").manual_seed(13)
    n, d, b, k = 2000, 64, 128, 10
    rows = _unit(torch.randn((n, d), generator=gen, device="cuda")).requires_grad_()
    table = _unit(torch.randn((500, d), generator=gen, device="cuda")).requires_grad_()
    words = torch.randint(0, 500, (b, 6), generator=gen, device="cuda")
    target = torch.randint(0, n, (b,), generator=gen, device="cuda")

    def losses(tab, rr):
        q = m.lookup_rows(tab, words, scale=6.0 ** -0.5).sum(dim=1)
        return m.corpus_cross_entropy(q, rr, target, scale=10.0)

    loss = losses(table, rows)
    dt, dr = torch.autograd.grad(loss.mean(), (table, rows))
    # against torch's own operators in 64 bits
    t64, r64 = table.detach().double().requires_grad_(), rows.detach().double().requires_grad_()
    q64 = (t64[words] * 6.0 ** -0.5).sum(dim=1)
    l64 = torch.nn.functional.cross_entropy(torch.matmul(q64, r64.t()) * 10.0, target, reduction="none")
    e = torch.autograd.grad(l64.mean(), (t64, r64))
    assert float((loss.detach() - l64.detach()).abs().max()) <= 2e-5
    for got, want in zip((dt, dr), e):
        assert float((got.double() - want).norm() / want.norm()) <= 2e-5
    with torch.no_grad():
        table -= dt
        rows -= dr
    ix = m.HipKnnIndex(d, metric="dot", dtype="f32")
    q4 = m.Int4ScanIndex(d, group=32)
    try:
        ix.add(rows.detach())
        q4.add(rows.detach())
        q = m.lookup_rows(table.detach(), words, scale=6.0 ** -0.5).sum(dim=1)
        ids, sc = ix.search(q, k)
        small_q = q[:, :32].clone().requires_grad_()
        small_r = rows.detach()[:, :32].clone().requires_grad_()
        kd = m.corpus_distillation(small_q, small_r, ids, sc, scale=2.0, teacher_scale=2.0)
        grads = torch.autograd.grad(kd.sum(), (small_q, small_r))
        assert bool(torch.isfinite(kd).all()) and all(bool(torch.isfinite(x).all()) for x in grads)
        ref = _reference(small_q.detach(), small_r.detach(), ids, sc, torch.ones(b, device="cuda"), 2.0, 2.0)
        assert float((kd.detach().double() - ref["loss"]).abs().max()) <= 1e-4
        approx = q4.scores(q)
        exact = q.double() @ rows.detach().double().t()
        # an element is off by half a scale at most: amax of its group / 14, but for the scale's own rounding
        group = rows.detach().view(n, d // 32, 32).abs().amax(dim=2).double() / 14 * 1.01
        lim = q.double().abs().view(b, d // 32, 32).sum(dim=2) @ group.t() + 1e-5
        assert bool(((approx.double() - exact).abs() <= lim).all())
    finally:
        ix.close()
        q4.close()
