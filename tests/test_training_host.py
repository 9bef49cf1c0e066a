"""Refusals of include/cgvec_train.h that need no GPU, and the workspaces' sizes."""
import ctypes as C
import math

import pytest
import torch

from _util import pkg


def test_lookup_checks_its_arguments_first():
    m = pkg()
    L = m.training.lib()
    p = C.c_void_p(4096)                       # never read: every call below is refused before
    inv, non = m.cgvec.CGV_ERR_INVALID_ARG, m.cgvec.CGV_ERR_NONFINITE

    def rows(dtype=0, n=10, d=8, stride=8, ids=p, k=3, scale=1.0, out=p, table=p):
        return L.cgv_lookup_rows_dev(0, table, dtype, n, d, stride, ids, k, scale, out, None)

    assert rows(dtype=3) == inv and rows(dtype=4) == inv and rows(d=0) == inv and rows(d=8193, stride=9000) == inv and rows(stride=7) == inv
    assert rows(n=2 ** 31) == inv and rows(k=2 ** 31) == inv and rows(scale=math.nan) == non and rows(scale=math.inf) == non
    assert rows(ids=None) == inv and rows(out=None) == inv and rows(table=None) == inv
    assert rows(k=0) == 0

    def grad(dtype=0, n=10, d=8, ids=p, k=3, scale=1.0, dout=p, out=p, ws=None, nb=0):
        return L.cgv_lookup_grad_dev(0, dout, dtype, ids, k, n, d, scale, out, ws, nb, None)

    assert grad(dtype=3) == inv and grad(d=0) == inv and grad(n=2 ** 31) == inv and grad(k=2 ** 31) == inv and grad(scale=math.nan) == non
    assert grad(ids=None) == inv and grad(out=None) == inv and grad(dout=None) == inv
    need = L.cgv_lookup_grad_workspace(5000, 10, 8)
    assert need > 0 and grad(k=5000, ws=p, nb=need - 1) == inv and grad(k=5000, ws=None, nb=need) == inv
    assert grad(k=5000, ws=C.c_void_p(4096 + 8), nb=need) == inv     # not aligned
    assert grad(n=0) == 0


def test_lookup_workspace():
    m = pkg()
    L = m.training.lib()
    assert L.cgv_lookup_grad_workspace(256, 1000, 64) == 0          # few ids need none
    for k, n, d in ((513, 1, 1), (65_536, 100_000, 768), (2 ** 31 - 1, 2 ** 31 - 1, 8192)):
        b = L.cgv_lookup_grad_workspace(k, n, d)
        assert b >= 16 * k + 8 * n
    assert L.cgv_lookup_grad_workspace(5, 2 ** 31, 64) == 0


def test_corpus_loss_checks_its_arguments_first():
    m = pkg()
    L = m.training.lib()
    p, odd = C.c_void_p(4096), C.c_void_p(4096 + 2)      # never read: every call below is refused before
    inv, non = m.cgvec.CGV_ERR_INVALID_ARG, m.cgvec.CGV_ERR_NONFINITE

    def fwd(q=p, qs=64, r=p, rs=64, dtype=1, b=5, n=10, d=64, ids=p, ts=p, k=2, scale=1.0, tscale=1.0, loss=p, saved=p, ws=p, nb=1 << 40):
        return L.cgv_corpus_loss_dev(0, q, qs, r, rs, dtype, b, n, d, ids, ts, k, scale, tscale, loss, saved, ws, nb, None)

    def bwd(q=p, qs=64, r=p, rs=64, dtype=1, b=5, n=10, d=64, ids=p, ts=p, k=2, scale=1.0, tscale=1.0, saved=p, dl=p, dq=p, dr=p, ws=p, nb=1 << 40):
        return L.cgv_corpus_loss_grad_dev(0, q, qs, r, rs, dtype, b, n, d, ids, ts, k, scale, tscale, saved, dl, dq, dr, ws, nb, None)

    for f in (fwd, bwd):
        for kw in (dict(dtype=3), dict(dtype=4), dict(d=0), dict(d=8193, qs=9000, rs=9000), dict(qs=63), dict(rs=63), dict(n=0), dict(n=2 ** 31 - 1),
                   dict(b=2 ** 24 + 1), dict(k=0), dict(k=257), dict(q=None), dict(r=None), dict(ids=None), dict(saved=None), dict(ws=None), dict(nb=255),
                   dict(ws=C.c_void_p(4096 + 64)), dict(r=odd), dict(rs=65), dict(rs=2 ** 22 + 8)):
            assert f(**kw) == inv, kw
        for kw in (dict(scale=math.nan), dict(scale=math.inf), dict(tscale=-math.inf)):
            assert f(**kw) == non, kw
    assert fwd(loss=None) == inv and bwd(dl=None) == inv
    assert fwd(b=0) == 0 and bwd(dq=None, dr=None) == 0
    if m.device_count() == 0:                            # no queries, a corpus' gradient to clear: gets as far as the device
        assert bwd(b=0) == m.cgvec.CGV_ERR_HIP


def test_corpus_loss_workspaces():
    m = pkg()
    L = m.training.lib()
    for f in (L.cgv_corpus_loss_workspace, L.cgv_corpus_loss_grad_workspace):
        assert f(0, 10, 64, 1, 0) == 0 and f(5, 0, 64, 1, 0) == 0 and f(5, 10, 64, 257, 0) == 0 and f(5, 10, 64, 1, 3) == 0
        for b, n, d, k, dt in ((1, 1, 1, 1, 0), (1024, 1_000_000, 768, 1, 1), (2 ** 20, 2 ** 31 - 2, 8192, 256, 2)):
            assert f(b, n, d, k, dt) > 2 * b * d
    # the corpus' size does not show: neither scores nor gradients of scores are kept
    big, small = (L.cgv_corpus_loss_grad_workspace(1024, n, 768, 1, 1) for n in (100_000_000, 1_000_000))
    assert big == small < 1 << 30


def test_cpu_tensors_are_refused():
    m = pkg()
    with pytest.raises(m.CgvError, match="no CPU fallback"):
        m.corpus_cross_entropy(torch.zeros((3, 4)), torch.zeros((5, 4)), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(m.CgvError, match="no CPU fallback"):
        m.lookup_rows(torch.zeros((3, 4)), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(m.CgvError, match="no CPU fallback"):
        m.lookup_rows_grad(torch.zeros((3, 4)), torch.zeros(3, dtype=torch.int64), 5)
