"""The 4-bit scan at both ends of its scales' range: a score that f32 can hold comes out, whatever the group sums on the way would reach."""
import numpy as np
import pytest

from _util import pkg

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24


def _bf16(x):
    """Values that bf16 holds, given as f32 -> their 16 bits."""
    u = np.asarray(x, np.float32).view(np.uint32)
    assert not (u & 0xFFFF).any()
    return (u >> 16).astype(np.uint16)


def _pack(c):
    if c.shape[1] % 2:
        c = np.concatenate([c, np.full((c.shape[0], 1), 8, c.dtype)], axis=1)
    return (c[:, 0::2] | (c[:, 1::2] << 4)).astype(np.uint8)


@pytest.mark.parametrize("qdt", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("n,d,group,mq", [(50, 96, 32, 1), (333, 200, 64, 4), (1000, 1100, 128, 17), (17, 8192, 64, 2)])
def test_scales_over_the_range_of_bf16(n, d, group, mq, qdt):
    import torch
    m = pkg()
    rng = np.random.default_rng(n + d)
    ng = -(-d // group)
    c = rng.integers(0, 16, (n, d))
    e = rng.integers(-126, 128, (n, 1)) + np.zeros((1, ng), np.int64)         # from the smallest normal f32 to the largest
    e[: n // 2] -= rng.integers(0, 20, (n // 2, ng))                          # and groups of one row apart
    e = np.clip(e, -133, 127)
    s = np.ldexp(np.where(e < -126, 1.0, rng.choice([1.0, 1.5, 1.9921875], (n, ng))), e).astype(np.float32)
    val = (c - 8) * np.repeat(s.astype(np.float64), group, axis=1)[:, :d]
    big = np.abs(val).max()
    ix = m.Int4ScanIndex(d, group=group, scales="bf16")
    try:
        ix.add_q4(_pack(c), _bf16(s))
        for size in (2.0 ** -12, 2.0 ** -3, 1.0, 2.0 ** 10) + ((2.0 ** -60, 2.0 ** 60) if qdt != "float16" else ()):
            x = torch.from_numpy((rng.uniform(0.5, 1.0, (mq, d)) * rng.choice([-1.0, 1.0], (mq, d)) * size).astype(np.float32)).cuda().to(getattr(torch, qdt))
            ref = x.double().cpu().numpy() @ val.T
            lim = (d + 4) * EPS * (np.abs(x.double().cpu().numpy()) @ np.abs(val).T) + 2.0 ** -140
            got = ix.scores(x).cpu().numpy().astype(np.float64)
            fits = np.abs(ref) + lim < np.finfo(np.float32).max
            with np.errstate(invalid="ignore"):
                ok = np.abs(got - ref) <= lim
            assert ok[fits].all(), (size, int((~ok[fits]).sum()), int(fits.sum()))
            over = np.abs(ref) - lim > float(np.finfo(np.float32).max) * 1.001
            assert (got[over] == np.sign(ref[over]) * np.inf).all()
            if qdt == "float32":
                host = ix.scores(x.cpu().numpy()).astype(np.float64)
                assert np.array_equal(host, got)
        bad = torch.ones((3, d), device="cuda", dtype=getattr(torch, qdt))
        bad[1, d // 2] = float("inf")
        got = ix.scores(bad)
        assert bool(torch.isnan(got[1]).all()) and not bool(torch.isnan(got[[0, 2]]).any())
        assert big > 2.0 ** 100
    finally:
        ix.close()


def test_rows_quantised_from_large_values():
    """add() takes rows of any finite size with bf16 scales, and finds them again."""
    import torch
    m = pkg()
    rng = np.random.default_rng(5)
    rows = (rng.standard_normal((300, 64)) * 1e37).astype(np.float32)
    ix = m.Int4ScanIndex(64, group=32, scales="bf16")
    try:
        ix.add(rows)
        val = np.stack([ix.get_row(i) for i in range(300)]).astype(np.float64)
        x = (rng.standard_normal((5, 64)) * 1e-3).astype(np.float32)
        ref = x.astype(np.float64) @ val.T
        lim = 68 * EPS * (np.abs(x).astype(np.float64) @ np.abs(val).T)
        assert np.all(np.abs(ix.scores(x) - ref) <= lim)
        y = torch.from_numpy(x).cuda()
        out = ix.scores(y)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            again = ix.scores(y)
        for _ in range(3):
            again.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(again, out)
    finally:
        ix.close()
