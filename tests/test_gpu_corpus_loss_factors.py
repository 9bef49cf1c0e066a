"""Gradients of softmax losses whose queries weigh very differently (weighted losses, an outlier, losses near zero): a query's gradient has the
digits of its type whatever the others' factors are."""
import math

import pytest
import torch

from _util import pkg

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24


def _unit(x):
    return x / x.norm(dim=1, keepdim=True).clamp_min(1e-30)


def _definition(q, r, ids, w, g, scale):
    """64 bits; the anchor's entry - softmax of the heaviest listed row less its weight - without the difference of two numbers near 1."""
    q, r = q.double(), r.double()
    s = scale * torch.matmul(q, r.t())
    lse = torch.logsumexp(s, dim=1)
    P = torch.exp(s - lse[:, None])
    W = torch.zeros_like(s).scatter_add_(1, ids, w)
    G = P - W
    if ids.shape[1] == 1:
        G.scatter_(1, ids, -P.scatter(1, ids, 0.0).sum(dim=1, keepdim=True))
    c = g.double()[:, None] * scale
    return dict(dq=(G * c) @ r, dr=(G * c).t() @ q, G=(G * c).abs(), lse=lse, q=q.abs(), r=r.abs())


def _limits(ref, dt, d, n, b, scale, few):
    # an entry of G: its own rounding to 16 bits (up to 32 queries: two parts), the score's and the logarithm's error, exp2 - as a share of it
    u = torch.finfo(TYPES[dt]).eps / 2
    norm = (ref["q"].pow(2).sum(dim=1).sqrt() * ref["r"].pow(2).sum(dim=1).sqrt().max()).max()
    ds = float(U * abs(scale) * (4 * math.sqrt(d) + 12) * norm + 2 * U * ref["lse"].abs().max())
    part = 2 * ds + (u * u if few and dt != "f32" else max(u, 2.0 ** -22)) + U * (4 * math.sqrt(max(n, b)) + 32)
    # entries far below the query's largest lose digits in fp16: an absolute 2^-25 where the largest is 2^13 at least
    sub = ref["G"].amax(dim=1, keepdim=True) * (2.0 ** -38 if dt == "fp16" else 0.0) + 2.0 ** -126
    G = ref["G"] * part + sub
    tiny = 2.0 ** -24 if dt == "fp16" else 2.0 ** -126
    out = u * 1.001
    # fp16: queries stand beside their powers of two for the corpus' gradient: what underflows there is 2^-38 of the largest entry of all
    lost = float(ref["G"].max()) * 2.0 ** -37 * ref["q"].amax() * b if dt == "fp16" else 0.0
    return G @ ref["r"] + ref["dq"].abs() * out + tiny, G.t() @ ref["q"] + ref["dr"].abs() * out + tiny + lost


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("b,n,d,k", [(20, 30_000, 64, 1), (300, 30_000, 64, 1), (300, 30_000, 72, 3), (77, 3000, 123, 2), (700, 60_000, 256, 1)])
def test_factors_from_one_to_a_millionth(b, n, d, k, dt):
    m = pkg()
    gen = torch.Generator(device="cuda").manual_seed(b + d)
    # rows with something in common: the corpus' share of a gradient is as large as the listed rows'
    rows = _unit(torch.randn((n, d), generator=gen, device="cuda") / math.sqrt(d) + 1.5 * _unit(torch.randn((1, d), generator=gen, device="cuda"))).to(TYPES[dt])
    q = _unit(torch.randn((b, d), generator=gen, device="cuda")).to(TYPES[dt])
    ids = torch.stack([torch.randperm(n, generator=gen, device="cuda")[:k] for _ in range(b)])
    g = 1024.0 * 10.0 ** (-6.0 * torch.rand((b,), generator=gen, device="cuda"))
    g[0], g[1], g[2] = 1024.0, 1024.0e-6, 0.0
    scale = 2.0
    w = torch.full((b, k), 1.0 / k, dtype=torch.float64, device="cuda")
    sc = torch.zeros((b, k), device="cuda")
    q.requires_grad_(), rows.requires_grad_()
    ref = _definition(q.detach(), rows.detach(), ids, w, g, scale)
    dq, dr = torch.autograd.grad(m.corpus_distillation(q, rows, ids, sc, scale=scale), (q, rows), g)
    lq, lr = _limits(ref, dt, d, n, b, scale, b <= 32)
    for name, got, want, lim in (("dq", dq, ref["dq"], lq), ("dr", dr, ref["dr"], lr)):
        err = (got.double() - want).abs()
        assert bool((err <= lim).all()), (name, float((err / lim).max()))
    # row by row, and far closer than the worst signs allow: a query's gradient is as good as if it stood alone
    e = (dq.double() - ref["dq"]).norm(dim=1) / ref["dq"].norm(dim=1).clamp_min(1e-30)
    assert float(e[g > 0].max()) <= 6 * torch.finfo(TYPES[dt]).eps + 2e-5, float(e[g > 0].max())
    assert bool((dq[2] == 0).all())
    alone = torch.autograd.grad(m.corpus_distillation(q, rows, ids, sc, scale=scale), (q,), torch.where(torch.arange(b, device="cuda") == 1, g, torch.zeros_like(g)))[0]
    assert torch.equal(alone[1], dq[1])                      # whatever the others' factors are


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("b", [20, 40])
def test_small_losses_keep_their_digits_in_both_gradients(b, dt):
    """Queries that find their rows, losses below 1e-7 (and factors as a loss scaler gives them)."""
    m = pkg()
    gen = torch.Generator(device="cuda").manual_seed(6)
    n, d, scale = 500, 64, 40.0
    rows = _unit(torch.randn((n, d), generator=gen, device="cuda")).to(TYPES[dt])
    ids = torch.randperm(n, generator=gen, device="cuda")[:b, None]
    q = rows[ids[:, 0]].clone()
    g = 2.0 ** 20 * (0.5 + torch.rand((b,), generator=gen, device="cuda"))
    q.requires_grad_(), rows.requires_grad_()
    ref = _definition(q.detach(), rows.detach(), ids, torch.ones((b, 1), dtype=torch.float64, device="cuda"), g, scale)
    loss = m.corpus_cross_entropy(q, rows, ids[:, 0], scale=scale)
    assert float(loss.detach().max()) < 1e-7
    dq, dr = torch.autograd.grad(loss, (q, rows), g)
    lq, lr = _limits(ref, dt, d, n, b, scale, b <= 32)
    for name, got, want, lim in (("dq", dq, ref["dq"], lq), ("dr", dr, ref["dr"], lr)):
        err = (got.double() - want).abs()
        assert bool((err <= lim).all()), (name, float((err / lim).max()))
    listed = ids[:, 0]
    assert float((dr.double() - ref["dr"])[listed].norm() / ref["dr"][listed].norm()) <= 3 * torch.finfo(TYPES[dt]).eps + 2e-4
