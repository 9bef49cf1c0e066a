"""The softmax sum over a corpus whose scores are mostly alike: every addition then rounds the same way, and nothing averages out. The limits
hold for the worst signs."""
import pytest
import torch

from _util import pkg

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24


def _limit(most, loss):
    # What a loss may be off by, natural units, if every score is exact before the factor: the factor in f32, its product and the difference
    # to the maximum round by 2^-24 of at most 2 |s| + 2 each (the maximum is an integer power of two above all); exp2 is good to 2^-22; a
    # lane adds 16 values four times over and those four, the tiles' sums lose nothing; two halves, one rounding of the pair, the loss' own
    return U * (6 * most + 6 + 4 + 19 + 4 + loss.abs())


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("b,n", [(40, 90_000), (1024, 1_000_000), (33_000, 300_000)])
def test_a_corpus_of_equal_rows(b, n, dt):
    """All rows but ten are the same (a collapsed or untrained corpus): from one share of it per query up to many."""
    m = pkg()
    gen = torch.Generator(device="cuda").manual_seed(b)
    few, d = 10, 16

    def eighths(*shape):
        return torch.randint(-8, 9, shape, generator=gen, device="cuda").double() / 8       # products and sums of these are exact

    q, same, others = eighths(b, d), eighths(1, d), eighths(few, d) * 1.5
    target = torch.randint(0, n, (b,), generator=gen, device="cuda")
    target[: b // 2] %= few
    rows = same.to(TYPES[dt]).expand(n, d).contiguous()
    rows[:few] = others.to(TYPES[dt])
    s = torch.cat([torch.matmul(q, others.t()), torch.matmul(q, same.t())], dim=1)           # [b, 11], the last for all equal rows
    top = s.amax(dim=1, keepdim=True)
    count = torch.ones(few + 1, dtype=torch.float64, device="cuda")
    count[few] = n - few
    lse = top[:, 0] + torch.log((torch.exp(s - top) * count).sum(dim=1))
    want = lse - torch.gather(s, 1, target.clamp(max=few)[:, None])[:, 0]
    got = m.corpus_cross_entropy(q.to(TYPES[dt]), rows, target, scale=1.0)
    err, lim = (got.double() - want).abs(), _limit(s.abs().amax(dim=1), want)
    assert bool((err <= lim).all()), float((err / lim).max())


@pytest.mark.parametrize("b,n", [(64, 200_000), (33_000, 200_000)])
def test_scores_that_rise_along_the_corpus(b, n):
    """A corpus in order of its scores: the running maximum moves with every tile, by ever the same little."""
    m = pkg()
    rows = (torch.arange(n, device="cuda").double() * 2.0 ** -18)[:, None]                   # exact in f32, as are eighths of them
    factor = torch.tensor([0.125, 0.5, 1.0, 1.5, 3.0, 6.0, -2.0, 0.0], dtype=torch.float64, device="cuda")
    s = torch.matmul(factor[:, None], rows.t())
    lse = torch.logsumexp(s, dim=1)
    which = torch.arange(b, device="cuda") % 8
    target = torch.randint(0, n, (b,), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    want = lse[which] - factor[which] * rows[target, 0]
    got = m.corpus_cross_entropy(factor[which].float()[:, None], rows.float(), target, scale=1.0)
    err, lim = (got.double() - want).abs(), _limit(s.abs().amax(dim=1)[which], want)
    assert bool((err <= lim).all()), float((err / lim).max())


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-45, -1e-30])
def test_a_factor_of_nothing(scale, dt):
    """Every row weighs the same: the loss is the logarithm of their number, also where the heaviest listed row is left out of the sum."""
    m = pkg()
    gen = torch.Generator(device="cuda").manual_seed(3)
    for b, n in ((5, 1), (40, 700), (300, 30_001)):
        q, r = (torch.randn((s, 24), generator=gen, device="cuda").to(TYPES[dt]) for s in (b, n))
        t = torch.randint(0, n, (b,), generator=gen, device="cuda")
        want = torch.full((b,), float(n), dtype=torch.float64, device="cuda").log()
        got = m.corpus_cross_entropy(q, r, t, scale=scale)
        assert bool(((got.double() - want).abs() <= _limit(torch.full_like(want, 1e-27), want)).all())
