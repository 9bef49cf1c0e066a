"""Forward-mode tangents: the operators have none, and say so instead of dropping them."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from _util import pkg

pytestmark = pytest.mark.gpu


def test_tangents_are_refused():
    m = pkg()
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, r, tab = (torch.randn(s, generator=gen, device="cuda") for s in ((4, 16), (30, 16), (20, 16)))
    ids = torch.randint(0, 20, (4, 2), generator=gen, device="cuda")
    sc = torch.rand((4, 2), generator=gen, device="cuda")
    dout = torch.randn((4, 2, 16), generator=gen, device="cuda")
    ix = m.Int4ScanIndex(16, group=32)
    try:
        ix.add(r)
        calls = [(tab, lambda x: m.lookup_rows(x, ids)), (dout, lambda x: m.lookup_rows_grad(x, ids, 20)),
                 (q, lambda x: m.corpus_cross_entropy(x, r, ids[:, 0])), (r, lambda x: m.corpus_cross_entropy(q, x, ids[:, 0])),
                 (q, lambda x: m.corpus_distillation(x, r, ids, sc)), (r, lambda x: m.corpus_distillation(q, x, ids, sc)),
                 (sc, lambda x: m.corpus_distillation(q, r, ids, x)), (q, ix.scores), (q[0].clone(), ix.scores)]
        for x, call in calls:
            want = call(x)
            with fwd.dual_level():
                assert torch.equal(call(x), want)                       # a level alone changes nothing
                for leaf in (x, x.clone().requires_grad_()):
                    with pytest.raises(m.CgvError, match="forward-mode") as ei:
                        call(fwd.make_dual(leaf, torch.ones_like(x)))
                    assert ei.value.code == m.cgvec.CGV_ERR_INVALID_ARG
        q.requires_grad_(), tab.requires_grad_()
        for x, call, g in ((tab, lambda: m.lookup_rows(tab, ids), dout), (q, lambda: m.corpus_cross_entropy(q, r, ids[:, 0]), sc[:, 0].clone())):
            with fwd.dual_level(), pytest.raises(m.CgvError, match="forward-mode"):       # of the incoming gradient
                torch.autograd.grad(call(), (x,), fwd.make_dual(g, torch.ones_like(g)))
    finally:
        ix.close()
