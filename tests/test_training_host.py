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
    assert L.cgv_lookup_grad_workspace(512, 1000, 64) == 0          # few ids need none
    for k, n, d in ((513, 1, 1), (65_536, 100_000, 768), (2 ** 31 - 1, 2 ** 31 - 1, 8192)):
        b = L.cgv_lookup_grad_workspace(k, n, d)
        assert b >= 16 * k + 8 * n
    assert L.cgv_lookup_grad_workspace(5, 2 ** 31, 64) == 0


def test_cpu_tensors_are_refused():
    m = pkg()
    with pytest.raises(m.CgvError, match="no CPU fallback"):
        m.lookup_rows(torch.zeros((3, 4)), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(m.CgvError, match="no CPU fallback"):
        m.lookup_rows_grad(torch.zeros((3, 4)), torch.zeros(3, dtype=torch.int64), 5)
