"""What the operators beside the search promise at their edges: NaN and Inf that take part, a caller's earlier errors, host forms that work piece by
piece, and how exact the corpus' gradient is on both sides of the rule that makes the listed entries' rounding good."""
import math
import mmap

import numpy as np
import pytest
import torch

from _util import pkg

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24


def _unit(x):
    return x / x.norm(dim=1, keepdim=True).clamp_min(1e-30)


def _problem(b, n, d, k, dt, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q, r = (_unit(torch.randn((s, d), generator=gen, device="cuda")).to(TYPES[dt]) for s in (b, n))
    ids = torch.stack([torch.randperm(n, generator=gen, device="cuda")[:k] for _ in range(b)])
    g = torch.rand((b,), generator=gen, device="cuda") + 0.25
    return q, r, ids, torch.zeros((b, k), device="cuda"), g


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("b,n,d", [(20, 700, 64), (66, 400, 72), (300, 40_000, 64)])
def test_a_query_with_nan_that_takes_part(b, n, d, dt):
    """Its own loss and gradient, and every row of the corpus' gradient; no other query's loss or gradient."""
    m = pkg()
    q, r, ids, sc, g = _problem(b, n, d, 3, dt, 9)
    clean = m.corpus_distillation(q.requires_grad_(), r.requires_grad_(), ids, sc, scale=4.0)
    want = torch.autograd.grad(clean, (q, r), g)
    for value in (math.nan, math.inf):
        bad = q.detach().clone()
        bad[3, 1] = value
        bad.requires_grad_()
        loss = m.corpus_distillation(bad, r, ids, sc, scale=4.0)
        dq, dr = torch.autograd.grad(loss, (bad, r), g)
        keep = torch.arange(b, device="cuda") != 3
        assert not bool(torch.isfinite(loss[3])) and torch.equal(loss[keep], clean[keep])
        assert not bool(torch.isfinite(dq[3]).any()) and torch.equal(dq[keep], want[0][keep])
        assert bool(torch.isnan(dr).any(dim=1).all())


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("b,n,d", [(20, 700, 64), (66, 403, 70), (300, 40_000, 64)])
def test_a_corpus_row_with_nan_or_inf(b, n, d, dt):
    """Every query that takes part; a query without a list stays at 0."""
    m = pkg()
    q, r, ids, sc, g = _problem(b, n, d, 3, dt, 10)
    row = n - 1 if n < 1000 else 12_345
    ids[ids == row] = 0
    ids[5] = -1
    there = torch.arange(b, device="cuda") != 5
    others = torch.arange(n, device="cuda") != row
    without = m.corpus_distillation(q, r[others].contiguous(), torch.where(ids > row, ids - 1, ids), sc, scale=4.0)
    for value in (math.nan, math.inf):
        bad = r.clone()
        bad[row, 2] = value
        bad.requires_grad_()
        loss = m.corpus_distillation(q.requires_grad_(), bad, ids, sc, scale=4.0)
        dq, dr = torch.autograd.grad(loss, (q, bad), g)
        loss = loss.detach()
        assert float(loss[5]) == 0.0 and bool((dq[5] == 0).all())
        if math.isnan(value):
            assert bool(torch.isnan(loss[there]).all()) and bool(torch.isnan(dq[there]).all())
        else:       # a score of -Inf has no weight; f32 rows are split into parts, of which Inf leaves NaN
            against = there & (q.detach()[:, 2] < 0)
            assert not bool(torch.isfinite(loss[there & ~against]).any())
            if dt != "f32":
                assert bool(((loss - without)[against].abs() <= 1e-5).all())
        q = q.detach()


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("b,n,d,k,made_good", [(512, 4000, 64, 2, True), (513, 4000, 64, 2, False), (70, 3000, 123, 14, True), (70, 3000, 123, 15, False),
                                               (500, 10_000, 512, 2, True), (500, 20_000, 512, 2, False), (40, 30_000, 1024, 25, False),
                                               (1024, 65_000, 1024, 2, False), (1024, 70_001, 1024, 2, True), (1030, 90_112, 768, 88, True), (1030, 90_111, 768, 88, False),
                                               (2100, 300_007, 112, 3, True), (66_000, 2000, 528, 1, True), (40, 900_000, 2000, 1, True)])
def test_the_corpus_gradient_on_both_sides_of_its_rule(b, n, d, k, made_good, dt):
    """Where the listed entries' rounding is made good only the results' own and the unlisted entries' remain; elsewhere each entry is off by half a
    step of its type at most, which is all that is promised."""
    m = pkg()
    q, r, ids, sc, _ = _problem(b, n, d, k, dt, b + n)
    g = torch.full((b,), 1.013, device="cuda")
    ids[:, 0] = torch.where(torch.arange(b, device="cuda") % 7 == 3, ids[0, 0], ids[:, 0])          # a row that many queries list
    ids[b - 1, 0] = n - 1
    r.requires_grad_()
    (dr,) = torch.autograd.grad(m.corpus_distillation(q, r, ids, sc, scale=8.0), (r,), g)
    q64, r64 = q.double(), r.detach().double()
    s = 8.0 * torch.matmul(q64, r64.t())
    lse = torch.logsumexp(s, dim=1)
    P = torch.exp(s - lse[:, None])
    G = P.clone().scatter_add_(1, ids, torch.full(ids.shape, -1.0 / k, dtype=torch.float64, device="cuda"))
    want = (G * 8.0 * g[:, None].double()).t() @ q64
    u = torch.finfo(TYPES[dt]).eps / 2
    ds = float(U * 8.0 * (4 * math.sqrt(d) + 12) * 1.1 + 2 * U * lse.abs().max())
    per = 2 * ds + U * (4 * math.sqrt(max(n, b)) + 40)
    tiny = 2.0 ** -24 if dt == "fp16" else 2.0 ** -126
    mag = G.abs() * 8.2
    if made_good:
        mag = mag * (u * u + per) + (P * 8.2).scatter(1, ids, 0.0) * u
    else:
        mag = mag * (u + per)
    lim = (mag + 8.2 * 2.0 ** -38).t() @ q64.abs() + want.abs() * u * 1.001 + tiny
    err = (dr.double() - want).abs()
    assert bool((err <= lim).all()), float((err / lim).max())
    # the norm: the result's own rounding is u / sqrt(3) of it on the average; an entry's rounding adds as much at most, twice at the worst
    assert float(err.norm() / want.norm()) <= (0.75 if made_good else 1.7) * u + per


def test_an_earlier_error_of_the_caller_is_not_reported_as_theirs():
    m = pkg()
    rng = np.random.default_rng(3)
    rows = rng.standard_normal((2000, 64)).astype(np.float32)
    mm = mmap.mmap(-1, 4096)
    addr = np.frombuffer(mm, dtype=np.uint8).ctypes.data

    def leave_an_error():
        assert int(torch.cuda.cudart().cudaHostUnregister(addr)) != 0

    r = torch.from_numpy(rows).cuda()
    ids = torch.randint(0, 2000, (700,), device="cuda")
    dout = torch.randn((700, 64), device="cuda")
    q = torch.randn((40, 64), device="cuda")
    torch.cuda.synchronize()
    L = m.training.lib()
    st = torch.cuda.current_stream().cuda_stream
    out = torch.empty((700, 64), device="cuda")
    table = torch.empty((2000, 64), device="cuda")
    loss, saved = torch.empty(40, device="cuda"), torch.empty(40 * 3, dtype=torch.float64, device="cuda")
    g, dq, dr = torch.ones(40, device="cuda"), torch.empty_like(q), torch.empty_like(r)
    ws = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    lws = L.cgv_lookup_grad_workspace(700, 2000, 64)
    fws, bws = L.cgv_corpus_loss_workspace(40, 2000, 64, 1, 0), L.cgv_corpus_loss_grad_workspace(40, 2000, 64, 1, 0)
    assert max(lws, fws, bws) <= ws.numel()
    p = torch.Tensor.data_ptr
    for call in (lambda: L.cgv_lookup_rows_dev(0, p(r), 0, 2000, 64, 64, p(ids), 700, 1.0, p(out), st),
                 lambda: L.cgv_lookup_grad_dev(0, p(dout), 0, p(ids), 700, 2000, 64, 1.0, p(table), p(ws), lws, st),
                 lambda: L.cgv_corpus_loss_dev(0, p(q), 64, p(r), 64, 0, 40, 2000, 64, p(ids), None, 1, 1.0, 1.0, p(loss), p(saved), p(ws), fws, st),
                 lambda: L.cgv_corpus_loss_grad_dev(0, p(q), 64, p(r), 64, 0, 40, 2000, 64, p(ids), None, 1, 1.0, 1.0, p(saved), p(g), p(dq), p(dr), p(ws), bws, st)):
        leave_an_error()
        assert call() == 0
    assert torch.equal(out, r[ids])
    assert bool(torch.isfinite(loss).all()) and bool(torch.isfinite(dr).all())
    leave_an_error()
    ix = m.Int4ScanIndex(64)
    try:
        for rr in (rows, r):
            leave_an_error()
            ix.add(rr)
        leave_an_error()
        host = ix.scores(rows[:3])
        qd = r[:3].clone()
        leave_an_error()
        got = ix.scores(qd)
        leave_an_error()
        assert np.array_equal(ix.get_row(5), ix.get_row(2005))
        leave_an_error()
        ix.reserve(100_000)
        assert np.array_equal(got.cpu().numpy(), host)
    finally:
        leave_an_error()
        ix.close()
    torch.cuda.synchronize()


def test_host_rows_that_come_in_pieces():
    """Rows, codes and scores of more than the staging buffer's 256 and 512 MiB: the same as from the device."""
    m = pkg()
    gen = torch.Generator(device="cuda").manual_seed(4)
    n, d = 8300, 8192                                        # 8192 rows fill a piece
    rows = torch.randn((n, d), generator=gen, device="cuda")
    x = torch.randn((2, d), generator=gen, device="cuda")
    one, two = m.Int4ScanIndex(d, group=128), m.Int4ScanIndex(d, group=128)
    try:
        one.add(rows)
        two.add(rows.cpu().numpy())
        assert len(two) == n and torch.equal(one.scores(x), two.scores(x))
    finally:
        one.close(), two.close()
    del rows
    n, d = 100_000, 5376                                     # 2688 + 336 bytes of codes and scales a row: 88 768 rows a piece
    codes = torch.randint(0, 256, (n, d // 2), generator=gen, device="cuda", dtype=torch.uint8)
    scales = (torch.rand((n, d // 32), generator=gen, device="cuda") + 0.5).half()
    x = torch.randn((2, d), generator=gen, device="cuda")
    one, two = m.Int4ScanIndex(d, group=32), m.Int4ScanIndex(d, group=32)
    try:
        one.add_q4(codes, scales)
        two.add_q4(codes.cpu(), scales.cpu())
        assert len(two) == n and torch.equal(one.scores(x), two.scores(x))
    finally:
        one.close(), two.close()
    del codes, scales
    n, d, mq = 600_000, 32, 229                              # 223 queries' scores fill the buffer
    ix = m.Int4ScanIndex(d, group=32)
    try:
        ix.add(torch.randn((n, d), generator=gen, device="cuda"))
        x = torch.randn((mq, d), generator=gen, device="cuda")
        want = ix.scores(x)
        assert np.array_equal(ix.scores(x.cpu().numpy()), want.cpu().numpy())
    finally:
        ix.close()


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_sorted_entries_repeat_and_replay(dt):
    """The corpus' gradient of a large problem: the same bits every time, captured on two graphs with lists that change between replays."""
    m = pkg()
    b, n, d, k = 1024, 70_001, 1024, 3
    q, r, ids, sc, g = _problem(b, n, d, k, dt, 21)
    q.requires_grad_(), r.requires_grad_()

    def step():
        loss = m.corpus_distillation(q, r, ids, sc, scale=8.0)
        return (loss.detach(), *torch.autograd.grad(loss, (q, r), g))

    want = step()
    assert all(torch.equal(x, y) for x, y in zip(step(), want))
    graphs = []
    for _ in range(2):
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            res = step()
        graphs.append((cg, res))
    gen = torch.Generator(device="cuda").manual_seed(22)
    for _ in range(3):
        ids.copy_(torch.randint(-2, n + 2, (b, k), generator=gen, device="cuda"))
        ids[::5] = ids[0, 0]
        for _, res in graphs:
            [x.zero_() for x in res]
        want = step()
        torch.cuda.synchronize()
        for cg, _ in graphs:
            cg.replay()
        torch.cuda.synchronize()
        for _, res in graphs:
            assert all(torch.equal(x, y) for x, y in zip(res, want))
