"""The 4-bit scan's refusals that need no GPU (include/cgvec_q4.h)."""
import ctypes as C

import numpy as np
import pytest

from _util import pkg


def test_create_checks_its_arguments():
    m = pkg()
    L = m.q4scan.lib()
    h = C.c_void_p()
    bad = m.cgvec.CGV_ERR_INVALID_ARG
    for dim, group, sdt in ((0, 64, 2), (8193, 64, 2), (64, 0, 2), (64, 16, 2), (64, 48, 2), (64, 256, 2), (64, 64, 0), (64, 64, 3), (64, 64, 9)):
        assert L.cgv_q4_create(dim, group, sdt, 0, C.byref(h)) == bad, (dim, group, sdt)
        assert not h.value
    assert L.cgv_q4_create(64, 64, 2, 0, None) == bad
    for kw in (dict(dim=64, scales="f32"), dict(dim=-1), dict(dim=64, group=-32)):
        with pytest.raises(m.CgvError) as ei:
            m.Int4ScanIndex(**kw)
        assert ei.value.code == bad


def test_null_handles():
    m = pkg()
    L = m.q4scan.lib()
    bad = m.cgvec.CGV_ERR_INVALID_ARG
    x = np.zeros(64, np.float32)
    p = x.ctypes.data_as(C.c_void_p)
    assert L.cgv_q4_count(None) == 0 and L.cgv_q4_destroy(None) == 0
    assert L.cgv_q4_reserve(None, 5) == bad
    assert L.cgv_q4_add_f32(None, p, 1) == bad and L.cgv_q4_add_f32_dev(None, p, 1, None) == bad
    assert L.cgv_q4_add_codes(None, p, p, 1) == bad and L.cgv_q4_add_codes_dev(None, p, p, 1, None) == bad
    assert L.cgv_q4_get_row_f32(None, 0, p) == bad
    assert L.cgv_q4_scores_f32(None, p, 1, 1, p) == bad and L.cgv_q4_scores_dev(None, p, 0, 1, 1, p, None, 0, None) == bad
    assert L.cgv_q4_scores_workspace(None, 0, 5) == 0


def test_fails_loudly_without_gpu():
    m = pkg()
    if m.device_count() > 0:
        pytest.skip("GPU present")
    with pytest.raises(m.CgvError, match="no CPU fallback"):
        m.Int4ScanIndex(128)
