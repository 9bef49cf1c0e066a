"""A HIP call of the CALLER that failed before (here: unregistering host memory that was never registered; elsewhere a
hipHostRegister that the system refuses) leaves an error unread in the runtime. The library's own calls that follow succeed."""
import mmap

import numpy as np
import pytest

from _util import pkg

pytestmark = pytest.mark.gpu


def test_an_earlier_error_of_the_caller_is_not_reported_as_ours(oracle):
    import torch
    m = pkg()
    rng = np.random.default_rng(3)
    rows = rng.standard_normal((2000, 64)).astype(np.float32)
    q = rng.standard_normal((9, 64)).astype(np.float32)
    mm = mmap.mmap(-1, 4096)
    addr = np.frombuffer(mm, dtype=np.uint8).ctypes.data

    def leave_an_error():
        assert int(torch.cuda.cudart().cudaHostUnregister(addr)) != 0

    torch.zeros(1, device="cuda")
    for dtype, odt in (("bf16", 1), ("f32", 0)):
        leave_an_error()
        ix = m.HipKnnIndex(64, dtype=dtype)
        try:
            leave_an_error()
            ix.add(rows)
            leave_an_error()
            idx, sc = ix.search(q, 5)
            ri, rs = oracle.batch_top_k(q, rows, 5, dtype=odt)
            assert np.array_equal(idx, ri) and np.array_equal(sc, rs)
        finally:
            ix.close()
    ix8 = m.Int8ScanIndex(64)
    try:
        leave_an_error()
        ix8.add(rows)
        leave_an_error()
        assert len(ix8.search_optimized(q[0], 5)) == 5
    finally:
        ix8.close()
    leave_an_error()
    assert m.quantize_u8(rows).shape == rows.shape
    torch.cuda.synchronize()
