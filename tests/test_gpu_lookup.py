"""Rows of a table by id and the table's gradient (include/cgvec_train.h) against their definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

from _util import pkg

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "fp16": 2.0 ** -24}     # a step of the subnormal numbers


def _step(dt):
    return torch.finfo(TYPES[dt]).eps / 2


def _table(gen, n, d, dt):
    return torch.randn((n, d), generator=gen, device="cuda").to(TYPES[dt])


def _expect_rows(table, ids, scale):
    there = (ids >= 0) & (ids < table.shape[0])
    out = torch.zeros((ids.numel(), table.shape[1]), dtype=torch.float64, device="cuda")
    out[there.flatten()] = table.double()[ids.flatten()[there.flatten()]] * scale
    return out


def _check_rows(got, table, ids, scale, dt):
    ref = _expect_rows(table, ids, scale)
    # one product in f32, then one rounding to the type
    lim = ref.abs() * (_step(dt) + 2.0 ** -24) * 1.0001 + TINY[dt]
    err = (got.double().view(ref.shape) - ref).abs()
    assert bool((err <= lim).all()), float((err / lim).max())


def _check_grad(got, dout, ids, n, scale, dt):
    d = dout.shape[-1]
    ids, dout = ids.flatten().cpu(), dout.reshape(-1, d).cpu()      # sums in 64 bits, on the CPU: rows that many ids share are quick there
    there = (ids >= 0) & (ids < n)
    ref = torch.zeros((n, d), dtype=torch.float64).index_add_(0, ids[there], dout[there].double() * scale).cuda()
    mag = torch.zeros((n, d), dtype=torch.float64).index_add_(0, ids[there], dout[there].double().abs() * abs(scale)).cuda()
    cnt = torch.bincount(ids[there], minlength=n).double().cuda()
    # k - 1 additions and one product in f32, then one rounding to the type
    lim = mag * (cnt[:, None] * 2.0 ** -24) * 1.0001 + ref.abs() * _step(dt) * 1.0001 + TINY[dt]
    assert got.shape == (n, d) and got.dtype == TYPES[dt]
    err = (got.double() - ref).abs()
    assert bool((err <= lim).all()), float((err / lim).max())
    assert bool((got[cnt == 0] == 0).all())


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n,d,k", [(1, 1, 1), (3, 8, 5), (40, 16, 256), (40, 16, 257), (3, 8, 2048), (90_000, 24, 2047), (100, 7, 64), (1000, 64, 513), (511, 100, 1000), (70, 384, 512), (5000, 768, 2049),
                                   (300_000, 16, 70_000), (40, 1536, 9000), (2, 32, 30_000), (9, 8192, 40)])
def test_forward_and_gradient(n, d, k, dt):
    m = pkg()
    gen = torch.Generator(device="cuda").manual_seed(n + d + k)
    scale = 0.37
    table = _table(gen, n, d, dt).requires_grad_()
    ids = torch.randint(0, n, (k,), generator=gen, device="cuda")
    if k > 4:
        ids[1], ids[k // 2], ids[k - 1] = -1, n, 2 ** 62        # padding and strangers
        ids[2] = -(2 ** 63)
    out = m.lookup_rows(table, ids, scale=scale)
    assert out.shape == (k, d) and out.dtype == TYPES[dt]
    _check_rows(out.detach(), table.detach(), ids, scale, dt)
    dout = _table(gen, k, d, dt)
    if k > 4:
        dout[1] = float("nan")                                  # rows that no id names do not reach the gradient
        dout[k - 1] = float("inf")
    (grad,) = torch.autograd.grad(out, (table,), dout)
    clean = torch.where(((ids >= 0) & (ids < n))[:, None], dout, torch.zeros_like(dout))
    _check_grad(grad, clean, ids, n, scale, dt)
    again = m.lookup_rows_grad(dout, ids, n, scale=scale)
    assert torch.equal(again, grad)                              # the same bits every time


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("k", [400, 4000, 100_003])
def test_frequent_ids(k, dt):
    """Ids that repeat as words do, one of them in more than a third of all places; runs of every length around the pieces'."""
    m = pkg()
    gen = torch.Generator(device="cuda").manual_seed(k)
    n, d = 5000, 72
    ids = (torch.exp(torch.rand(k, generator=gen, device="cuda", dtype=torch.float64) * math.log(n)).long() - 1).clamp(0, n - 1)
    ids[torch.rand(k, generator=gen, device="cuda") < 0.4] = 4321
    dout = _table(gen, k, d, dt)
    _check_grad(m.lookup_rows_grad(dout, ids, n, scale=2.0), dout, ids, n, 2.0, dt)
    srt = ids.sort().values
    _check_grad(m.lookup_rows_grad(dout, srt, n, scale=2.0), dout, srt, n, 2.0, dt)
    one = torch.full((k,), n - 1, device="cuda")
    _check_grad(m.lookup_rows_grad(dout, one, n, scale=-1.0), dout, one, n, -1.0, dt)
    runs = torch.arange(k, device="cuda") // 31                  # runs of 31: every piece's ends fall inside one
    _check_grad(m.lookup_rows_grad(dout, runs, int(runs[-1]) + 1, scale=1.0), dout, runs, int(runs[-1]) + 1, 1.0, dt)


def test_sums_are_f32():
    """70 000 equal bf16 rows: a bf16 sum would stop growing at 256 summands."""
    m = pkg()
    dout = torch.ones((70_000, 8), device="cuda", dtype=torch.bfloat16)
    ids = torch.zeros(70_000, dtype=torch.int64, device="cuda")
    assert float(m.lookup_rows_grad(dout, ids, 1)[0, 0]) == float(torch.tensor(70_000.0).bfloat16())


@pytest.mark.parametrize("dt", list(TYPES))
def test_strides_shapes_and_alignment(dt):
    m = pkg()
    gen = torch.Generator(device="cuda").manual_seed(5)
    n, d = 300, 64
    wide = _table(gen, n, d + 24, dt)
    ids = torch.randint(-1, n, (3, 5, 7), generator=gen, device="cuda")
    for a in (0, 1, 8, 16):                                      # aligned and unaligned column windows of a wider table
        view = wide[:, a:a + d]
        out = m.lookup_rows(view, ids, scale=1.5)
        assert out.shape == (3, 5, 7, d)
        _check_rows(out, view, ids, 1.5, dt)
    t = wide[:, :d].t().contiguous().t()                         # columns contiguous instead of rows
    assert torch.equal(m.lookup_rows(t, ids), m.lookup_rows(wide[:, :d], ids))
    assert torch.equal(m.lookup_rows(wide[:1].expand(n, -1)[:, :d], ids), m.lookup_rows(wide[:1].repeat(n, 1)[:, :d], ids))
    flat = torch.empty(n * d + 1, device="cuda", dtype=TYPES[dt])  # rows that start between two 16-byte addresses
    flat[1:] = wide[:, :d].reshape(-1)
    assert torch.equal(m.lookup_rows(flat[1:].view(n, d), ids.int()), m.lookup_rows(wide[:, :d], ids))
    table = wide[:, :d].contiguous().requires_grad_()
    out = m.lookup_rows(table, ids)
    dout = _table(gen, 105, d, dt).view(3, 5, 7, d)
    for g in (dout, dout.transpose(0, 1).contiguous().transpose(0, 1), dout[..., :1].expand(3, 5, 7, d)):
        (grad,) = torch.autograd.grad(out, (table,), g, retain_graph=True)
        _check_grad(grad, g, ids, n, 1.0, dt)
    dflat = torch.empty(105 * d + 1, device="cuda", dtype=TYPES[dt])
    dflat[1:] = dout.reshape(-1)
    assert torch.equal(m.lookup_rows_grad(dflat[1:].view(3, 5, 7, d), ids, n), m.lookup_rows_grad(dout, ids, n))


def test_gradient_by_differences():
    m = pkg()
    gen = torch.Generator(device="cuda").manual_seed(6)
    table = _table(gen, 20, 12, "f32").requires_grad_()
    ids = torch.tensor([3, 3, 7, -1, 19, 0, 3], device="cuda")
    w = _table(gen, 7, 12, "f32")
    (grad,) = torch.autograd.grad((m.lookup_rows(table, ids, scale=2.5) * w).sum(), (table,))
    for r, c in ((3, 0), (7, 11), (19, 5), (0, 3), (1, 1)):
        up, down = table.detach().clone(), table.detach().clone()
        up[r, c] += 0.5
        down[r, c] -= 0.5
        # linear in the table: the difference is the gradient but for the rounding of the outputs
        f = [float((m.lookup_rows(x, ids, scale=2.5).double() * w.double()).sum()) for x in (up, down)]
        assert abs((f[0] - f[1]) - float(grad[r, c])) <= 2.0 ** -20


def test_empty_and_single():
    m = pkg()
    table = torch.randn((5, 16), device="cuda", requires_grad=True)
    none = torch.empty((0,), dtype=torch.int64, device="cuda")
    out = m.lookup_rows(table, none)
    assert out.shape == (0, 16)
    (g,) = torch.autograd.grad(out.sum(), (table,))
    assert g.shape == (5, 16) and bool((g == 0).all())
    assert m.lookup_rows(table, torch.tensor(3, device="cuda")).shape == (16,)
    assert bool((m.lookup_rows(torch.empty((0, 16), device="cuda"), torch.tensor([0, -1], device="cuda")) == 0).all())
    assert m.lookup_rows_grad(torch.ones((2, 16), device="cuda"), torch.tensor([0, 1], device="cuda"), 0).shape == (0, 16)
    gone = torch.full((600,), -1, device="cuda")
    assert bool((m.lookup_rows_grad(torch.full((600, 16), float("nan"), device="cuda"), gone, 5) == 0).all())


def test_refusals():
    m = pkg()
    t = torch.zeros((4, 8), device="cuda")
    ids = torch.zeros(2, dtype=torch.int64, device="cuda")
    inv, dim, non = m.cgvec.CGV_ERR_INVALID_ARG, m.cgvec.CGV_ERR_DIM_MISMATCH, m.cgvec.CGV_ERR_NONFINITE
    for code, call in ((inv, lambda: m.lookup_rows(t.cpu(), ids)), (inv, lambda: m.lookup_rows(t, ids.cpu())), (inv, lambda: m.lookup_rows(t.double(), ids)),
                       (inv, lambda: m.lookup_rows(t, ids.float())), (dim, lambda: m.lookup_rows(t[0], ids)), (non, lambda: m.lookup_rows(t, ids, scale=math.inf)),
                       (inv, lambda: m.lookup_rows(torch.zeros((4, 8193), device="cuda"), ids)), (inv, lambda: m.lookup_rows(t[:, :0], ids)),
                       (dim, lambda: m.lookup_rows_grad(t, ids, 4)), (inv, lambda: m.lookup_rows_grad(t[:2], ids, -1)),
                       (inv, lambda: m.lookup_rows_grad(t[:2].double(), ids, 4)), (non, lambda: m.lookup_rows_grad(t[:2], ids, 4, scale=math.nan))):
        with pytest.raises(m.CgvError) as ei:
            call()
        assert ei.value.code == code


def test_streams_and_graphs():
    m = pkg()
    gen = torch.Generator(device="cuda").manual_seed(7)
    n, d, k = 4000, 96, 3000
    table = _table(gen, n, d, "bf16")
    ids = torch.randint(-1, n, (k,), generator=gen, device="cuda")
    dout = _table(gen, k, d, "bf16")
    want = (m.lookup_rows(table, ids, scale=3.0), m.lookup_rows_grad(dout, ids, n, scale=3.0))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = (m.lookup_rows(table, ids, scale=3.0), m.lookup_rows_grad(dout, ids, n, scale=3.0))
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):                                           # two graphs: their workspaces are their own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = (m.lookup_rows(table, ids, scale=3.0), m.lookup_rows_grad(dout, ids, n, scale=3.0))
        graphs.append((g, res))
    for it in range(4):
        ids.copy_(torch.randint(-1, n, (k,), generator=gen, device="cuda"))
        dout.copy_(_table(gen, k, d, "bf16"))
        want = (m.lookup_rows(table, ids, scale=3.0), m.lookup_rows_grad(dout, ids, n, scale=3.0))
        torch.cuda.synchronize()
        for g, res in graphs:
            [r.zero_() for r in res]
        for g, res in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, want)), it


def test_rows_behind_the_hits_of_a_search():
    """What a search returns goes in as it is: its ids, with the -1 that pads short lists."""
    m = pkg()
    rng = np.random.default_rng(8)
    rows = rng.standard_normal((7, 32)).astype(np.float32)
    ix = m.HipKnnIndex(32, dtype="f32")
    try:
        ix.add(rows)
        q = torch.from_numpy(rng.standard_normal((4, 32)).astype(np.float32)).cuda()
        ids, _ = ix.search(q, 10)                                # 7 rows: three places of ten are padding
        out = m.lookup_rows(torch.from_numpy(rows).cuda(), ids)
        assert out.shape == (4, 10, 32)
        assert torch.equal(out[:, :7].cpu(), torch.from_numpy(rows)[ids[:, :7].cpu()]) and bool((out[:, 7:] == 0).all())
    finally:
        ix.close()


def test_more_elements_than_a_direction_of_a_launch():
    """More than 2^32 threads' worth of single elements: rows of three 16-bit elements cannot be read in wider vectors."""
    m = pkg()
    gen = torch.Generator(device="cuda").manual_seed(8)
    k, n = 1_431_655_800, 1000
    table = _table(gen, n, 3, "bf16")
    ids = torch.arange(k, device="cuda").remainder_(n + 1)            # n itself: no row
    out = m.lookup_rows(table, ids, scale=2.0)
    at = torch.cat([torch.randint(0, k, (100_000,), generator=gen, device="cuda"), torch.arange(k - 1000, k, device="cuda")])
    want = torch.where((ids[at] < n)[:, None], table[ids[at].clamp_max(n - 1)] * 2.0, torch.zeros((), dtype=table.dtype, device="cuda"))
    assert torch.equal(out[at], want)
    del out, ids
    for few in (40, 600):                                             # one launch, and sorted
        some = torch.cat([torch.randint(0, k, (few - 2,), generator=gen, device="cuda"), torch.tensor([0, k - 1], device="cuda")])
        dout = _table(gen, few, 3, "bf16")
        g = m.lookup_rows_grad(dout, some, k)
        assert some.unique().numel() == few and torch.equal(g[some], dout)
        g[some] = 0
        assert not bool(g.view(torch.int16)[:1 << 28].any()) and not bool(g.view(torch.int16)[-(1 << 28):].any())
        del g
    torch.cuda.empty_cache()
