"""A handle that is created, filled and searched while the caller's default stream is busy: its streams do not wait for that one, so nothing that
the handle needs may be enqueued there."""
import numpy as np
import pytest

from _util import pkg

pytestmark = pytest.mark.gpu


def test_a_handle_made_while_the_default_stream_works(oracle):
    import torch
    m = pkg()
    rng = np.random.default_rng(4)
    rows = rng.standard_normal((3000, 64)).astype(np.float32)
    q = rng.standard_normal((7, 64)).astype(np.float32)
    want = {d: oracle.batch_top_k(q, rows, 5, dtype=o) for d, o in (("f32", 0), ("bf16", 1))}
    q4 = m.Int4ScanIndex(64)
    q4.add(rows)
    scores = q4.scores(q)
    q4.close()
    a = torch.randn((8192, 8192), device="cuda")
    for dtype in ("bf16", "f32", "bf16", "f32"):
        # what a handle before left where the next one's flags and norms will be
        old = m.HipKnnIndex(64, dtype=dtype)
        old.add(rows * 1e3)
        old.search(q, 5)
        old.close()
        torch.cuda.synchronize()
        for _ in range(12):
            b = a @ a                                       # some 80 ms of the default stream
        ix = m.HipKnnIndex(64, dtype=dtype)
        q4 = m.Int4ScanIndex(64)
        try:
            ix.add(rows)
            q4.add(rows)
            idx, sc = ix.search(q, 5)
            assert np.array_equal(idx, want[dtype][0]) and np.array_equal(sc, want[dtype][1])
            assert np.array_equal(q4.scores(q), scores)
            torch.cuda.synchronize()
            idx, sc = ix.search(q, 5)
            assert np.array_equal(idx, want[dtype][0]) and np.array_equal(sc, want[dtype][1])
        finally:
            ix.close(), q4.close()
        del b
