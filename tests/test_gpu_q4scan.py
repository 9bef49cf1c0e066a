"""The 4-bit scan (include/cgvec_q4.h) against its definition in 64 bits."""
import numpy as np
import pytest

from _util import pkg

pytestmark = pytest.mark.gpu

# a score is a sum of d products in f32: each product and each addition is off by at most half a step (2^-24 relative), the
# query's own split into parts by less; |error| <= (d + 4) * 2^-24 * sum |x * value|
EPS = 2.0 ** -24


def _to16(x, scales):
    """f32 -> (the 16 bits, their f32 value), round to nearest even."""
    x = np.asarray(x, np.float32)
    if scales == "fp16":
        h = x.astype(np.float16)
        return h.view(np.uint16), h.astype(np.float32)
    u = x.view(np.uint32).astype(np.uint64)
    u = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return u, (u.astype(np.uint32) << 16).view(np.float32)


def _quantise(rows, group, scales):
    n, d = rows.shape
    ng = -(-d // group)
    x = np.zeros((n, ng * group), np.float32)
    x[:, :d] = rows
    x = x.reshape(n, ng, group)
    bits, s = _to16(np.abs(x).max(axis=2) / np.float32(7.0), scales)
    sv = s[:, :, None]
    c = np.where(sv > 0, np.clip(np.rint(x / np.where(sv > 0, sv, 1).astype(np.float32)), -8, 7), 0).astype(np.int64) + 8
    return c.reshape(n, ng * group)[:, :d], bits, s


def _pack(c):
    n, d = c.shape
    if d % 2:
        c = np.concatenate([c, np.full((n, 1), 5, c.dtype)], axis=1)    # the odd last nibble is ignored
    return (c[:, 0::2] | (c[:, 1::2] << 4)).astype(np.uint8)


def _values(c, s, group):
    return (c - 8) * np.repeat(s.astype(np.float64), group, axis=1)[:, :c.shape[1]]


def _check(got, x, val):
    ref = x.astype(np.float64) @ val.T
    lim = (val.shape[1] + 4) * EPS * (np.abs(x).astype(np.float64) @ np.abs(val).T) + 1e-300
    assert got.shape == ref.shape
    assert np.all(np.abs(got - ref) <= lim), float((np.abs(got - ref) / lim).max())


def _rows(rng, n, d):
    x = rng.standard_normal((n, d)).astype(np.float32)
    return x / np.linalg.norm(x, axis=1, keepdims=True).astype(np.float32)


CASES = [(1, 1, 32), (15, 31, 32), (16, 33, 64), (17, 128, 128), (1000, 100, 32), (333, 257, 64), (4097, 384, 32), (2050, 768, 64),
         (700, 1000, 128), (129, 1536, 128), (20, 8192, 64)]


@pytest.mark.parametrize("scales", ["fp16", "bf16"])
@pytest.mark.parametrize("n,d,group", CASES)
def test_scores_and_quantiser(n, d, group, scales):
    m = pkg()
    rng = np.random.default_rng(n * 7 + d)
    rows = _rows(rng, n, d)
    if n > 5:
        rows[3] = 0.0                                  # a zero row: every scale is 0
        rows[4, : d // 2 + 1] *= 1e-3
    c, bits, s = _quantise(rows, group, scales)
    val = _values(c, s, group)
    ix = m.Int4ScanIndex(d, group=group, scales=scales)
    try:
        cut = n // 3
        ix.add(rows[:cut] if cut else rows[:0])        # quantised on the device ...
        ix.add_q4(_pack(c[cut:]), bits[cut:])          # ... and brought along, in the middle of a tile
        assert len(ix) == n
        for i in {0, n // 3 - 1 if n > 3 else 0, n // 3, n - 1, min(3, n - 1)}:
            assert np.array_equal(ix.get_row(i).astype(np.float64), val[i]), i
        for mq in (1, 2, 3, 4, 5, 9, 16, 33):
            x = _rows(rng, mq, d) * np.float32(3.7)
            _check(ix.scores(x), x, val)
        x = _rows(rng, 1, d)[0]
        one = ix.scores(x)
        assert one.shape == (n,)
        _check(one[None], x[None], val)
    finally:
        ix.close()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("mq", [1, 3, 4, 15, 16, 17, 40])
def test_device_queries(dtype, mq):
    import torch
    m = pkg()
    rng = np.random.default_rng(mq)
    n, d, group = 3001, 200, 64
    rows = _rows(rng, n, d)
    c, bits, s = _quantise(rows, group, "fp16")
    ix = m.Int4ScanIndex(d, group=group)
    try:
        ix.add(torch.from_numpy(rows).cuda())
        x = torch.from_numpy(_rows(rng, mq, d)).cuda().to(getattr(torch, dtype))
        got = ix.scores(x)
        assert got.dtype == torch.float32 and got.is_cuda
        _check(got.cpu().numpy(), x.float().cpu().numpy(), _values(c, s, group))
        wide = torch.zeros((mq, d + 8), device="cuda", dtype=x.dtype)        # a strided view of a wider tensor
        wide[:, 3:3 + d] = x
        assert torch.equal(ix.scores(wide[:, 3:3 + d]), got)
        assert torch.equal(ix.scores(x), got)                                # the same call gives the same bits
        st = torch.cuda.Stream()                                             # on another stream than the tensors' own
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            other = ix.scores(x)
        st.synchronize()
        assert torch.equal(other, got)
    finally:
        ix.close()


def test_wide_ranges_of_queries_and_scales():
    """Elements of one query from 2^-60 to 2^60, scales over the range of bf16: the error bound is the same."""
    m = pkg()
    rng = np.random.default_rng(8)
    n, d, group = 200, 96, 32
    c = rng.integers(0, 16, (n, d))
    bits, s = _to16(np.exp2(rng.integers(-40, 40, (n, d // group))).astype(np.float32) * 1.3, "bf16")
    ix = m.Int4ScanIndex(d, group=group, scales="bf16")
    try:
        ix.add_q4(_pack(c), bits)
        x = (rng.standard_normal((6, d)) * np.exp2(rng.integers(-60, 60, (6, 1)))).astype(np.float32)
        x[1] = 0.0
        x[2, 5:] = 0.0
        _check(ix.scores(x), x, _values(c, s, group))
        # elements of one query far below its largest: each counts with an absolute error of 2^-37 of the largest at most
        y = (rng.standard_normal((3, d)) * np.exp2(-rng.integers(0, 60, (3, d)))).astype(np.float32)
        got, val = ix.scores(y), _values(c, s, group)
        ref = y.astype(np.float64) @ val.T
        lim = (d + 4) * EPS * (np.abs(y).astype(np.float64) @ np.abs(val).T) + 2.0 ** -37 * np.abs(y).max(axis=1)[:, None] * np.abs(val).sum(axis=1)[None]
        assert np.all(np.abs(got - ref) <= lim)
    finally:
        ix.close()


def test_non_finite_queries_are_nan_for_themselves_only():
    import torch
    m = pkg()
    rng = np.random.default_rng(9)
    rows = _rows(rng, 100, 70)
    ix = m.Int4ScanIndex(70)
    try:
        ix.add(rows)
        x = _rows(rng, 7, 70)
        clean = ix.scores(x)
        bad = x.copy()
        bad[2, 5], bad[4, 0], bad[6, 69] = np.nan, np.inf, -np.inf
        got = ix.scores(bad)
        assert np.isnan(got[[2, 4, 6]]).all()
        assert np.array_equal(got[[0, 1, 3, 5]], clean[[0, 1, 3, 5]])
        assert np.isnan(ix.scores(torch.from_numpy(bad).cuda().half()).cpu().numpy()[[2, 4, 6]]).all()
    finally:
        ix.close()


def test_refusals_and_empty_forms():
    import torch
    m = pkg()
    rng = np.random.default_rng(10)
    rows = _rows(rng, 40, 64)
    ix = m.Int4ScanIndex(64, group=32)
    try:
        assert len(ix) == 0 and ix.scores(rows[:3]).shape == (3, 0)
        ix.add(rows[:0])
        ix.add(rows)
        keep = ix.scores(rows[:2])
        assert ix.scores(rows[:0]).shape == (0, 40)
        assert tuple(ix.scores(torch.empty((0, 64), device="cuda")).shape) == (0, 40)
        bad = rows.copy()
        bad[7, 3] = np.inf
        for r in (bad, torch.from_numpy(bad).cuda()):
            with pytest.raises(m.CgvError) as ei:
                ix.add(r)
            assert ei.value.code == m.cgvec.CGV_ERR_NONFINITE and "not applied" in str(ei.value)
        big = rows.copy()
        big[7, 3] = 1e6                                       # 1e6 / 7 is beyond fp16
        with pytest.raises(m.CgvError) as ei:
            ix.add(big)
        assert ei.value.code == m.cgvec.CGV_ERR_INVALID_ARG
        c, bits, _ = _quantise(rows, 32, "fp16")
        bits = bits.copy()
        bits[1, 1] = 0x7C00
        with pytest.raises(m.CgvError) as ei:
            ix.add_q4(_pack(c), bits)
        assert ei.value.code == m.cgvec.CGV_ERR_NONFINITE
        for call in (lambda: ix.add(rows[:, :63]), lambda: ix.scores(rows[:, :63]), lambda: ix.add_q4(_pack(c)[:, :31], bits),
                     lambda: ix.add_q4(_pack(c), bits[:, :1]), lambda: ix.scores(torch.zeros((2, 65), device="cuda"))):
            with pytest.raises(m.CgvError) as ei:
                call()
            assert ei.value.code == m.cgvec.CGV_ERR_DIM_MISMATCH
        for call in (lambda: ix.scores(torch.zeros((2, 64), device="cuda", dtype=torch.float64)), lambda: ix.get_row(-1),
                     lambda: ix.add_q4(_pack(c).astype(np.int8), bits),
                     lambda: ix.add_q4(torch.zeros((1, 32), dtype=torch.uint8, device="cuda"), torch.zeros((1, 2), dtype=torch.bfloat16, device="cuda"))):
            with pytest.raises(m.CgvError) as ei:
                call()
            assert ei.value.code == m.cgvec.CGV_ERR_INVALID_ARG
        with pytest.raises(m.CgvError) as ei:
            ix.get_row(40)
        assert ei.value.code == m.cgvec.CGV_ERR_OUT_OF_RANGE
        assert len(ix) == 40 and np.array_equal(ix.scores(rows[:2]), keep)
        ix.add(rows)                                          # and rows after a refused add
        assert np.array_equal(ix.scores(rows[:2])[:, 40:], keep)
    finally:
        ix.close()


def test_captured_and_replayed():
    import torch
    m = pkg()
    rng = np.random.default_rng(11)
    ix = m.Int4ScanIndex(300, group=64)
    try:
        ix.reserve(6000)
        ix.add(_rows(rng, 5000, 300))
        x = torch.from_numpy(_rows(rng, 5, 300)).cuda()
        eager = ix.scores(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ix.scores(x)
        for k in range(4):
            x.copy_(torch.from_numpy(_rows(rng, 5, 300)))
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            eager = ix.scores(x)
            assert torch.equal(out, eager), k
        with pytest.raises(m.CgvError, match="captured"):
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                h = torch.cuda.CUDAGraph()
                h.capture_begin()
                try:
                    ix.add(x)
                finally:
                    h.capture_end()
        assert len(ix) == 5000
    finally:
        ix.close()


def test_two_threads_score_one_index():
    import threading
    import torch
    m = pkg()
    rng = np.random.default_rng(12)
    rows = _rows(rng, 20_000, 128)
    ix = m.Int4ScanIndex(128)
    try:
        ix.add(rows)
        qs = [_rows(rng, 3, 128) for _ in range(4)]
        want = [ix.scores(q) for q in qs]
        bad = []

        def work(i):
            for _ in range(10):
                if not np.array_equal(ix.scores(qs[i]), want[i]):
                    bad.append(i)
                with torch.cuda.stream(torch.cuda.Stream()):
                    t = ix.scores(torch.from_numpy(qs[i]).cuda())
                    if not np.array_equal(t.cpu().numpy(), want[i]):
                        bad.append(-i)
        th = [threading.Thread(target=work, args=(i,)) for i in range(4)]
        [t.start() for t in th]
        [t.join() for t in th]
        assert not bad
    finally:
        ix.close()


def test_replays_after_the_corpus_has_moved():
    import torch
    m = pkg()
    rng = np.random.default_rng(13)
    rows = _rows(rng, 70_000, 200)
    ix = m.Int4ScanIndex(200)
    try:
        ix.add(rows[:40])
        x = torch.from_numpy(_rows(rng, 2, 200)).cuda()
        g = torch.cuda.CUDAGraph()
        ix.scores(x)
        with torch.cuda.graph(g):
            out = ix.scores(x)
        at = 40
        for n in (3000, 20_000, 46_960):                   # each beyond what the buffers hold
            ix.add(rows[at:at + n])
            at += n
            x.copy_(torch.from_numpy(_rows(rng, 2, 200)))
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            now = ix.scores(x)
            assert now.shape == (2, at) and torch.equal(out, now[:, :40])
    finally:
        ix.close()


def test_scores_of_the_first_rows():
    import ctypes as C
    m = pkg()
    rng = np.random.default_rng(14)
    ix = m.Int4ScanIndex(96, group=32)
    try:
        ix.add(_rows(rng, 1000, 96))
        x = _rows(rng, 3, 96)
        want = ix.scores(x)
        L, p = m.q4scan.lib(), lambda a: a.ctypes.data_as(C.c_void_p)
        for n in (0, 1, 15, 16, 17, 999, 1000):
            out = np.full((3, n + 1), 7.0, np.float32)
            assert L.cgv_q4_scores_f32(ix._h, p(x), 3, n, p(out)) == 0
            assert np.array_equal(out.ravel()[:3 * n].reshape(3, n), want[:, :n]) and np.all(out.ravel()[3 * n:] == 7.0)
        out = np.zeros((3, 1001), np.float32)
        assert L.cgv_q4_scores_f32(ix._h, p(x), 3, 1001, p(out)) == m.cgvec.CGV_ERR_OUT_OF_RANGE
        assert L.cgv_q4_scores_dev(ix._h, p(x), 0, 3, 1001, p(out), None, 0, None) == m.cgvec.CGV_ERR_OUT_OF_RANGE
    finally:
        ix.close()


def test_scoring_while_another_thread_adds():
    import threading
    import torch
    m = pkg()
    rng = np.random.default_rng(15)
    rows = _rows(rng, 60_000, 64)
    x = torch.from_numpy(_rows(rng, 2, 64)).cuda()
    ix = m.Int4ScanIndex(64)
    got = []
    try:
        ix.add(rows[:100])

        def add():
            for a in range(100, 60_000, 5990):
                ix.add(rows[a:a + 5990])
        t = threading.Thread(target=add)
        t.start()
        while True:
            last = not t.is_alive()
            got.append(ix.scores(x))
            if last:
                break
        t.join()
        torch.cuda.synchronize()
        assert got[-1].shape == (2, 60_000)
        assert all(torch.equal(s, got[-1][:, :s.shape[1]]) for s in got)
    finally:
        ix.close()
