"""What the training operators refuse before anything runs: inputs that are no matrices."""
import pytest
import torch

from _util import pkg


@pytest.mark.parametrize("where", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_inputs_that_are_no_matrices(where):
    m = pkg()
    bad, dim = m.cgvec.CGV_ERR_INVALID_ARG, m.cgvec.CGV_ERR_DIM_MISMATCH
    rows, ids = torch.zeros((6, 8), device=where), torch.zeros((3,), dtype=torch.int64, device=where)
    lists, sc = ids[:, None], torch.zeros((3, 1), device=where)
    for q, code in ((torch.tensor(1.0, device=where), dim), (torch.zeros(8, device=where), dim), (torch.zeros((3, 8, 1), device=where), dim), ([[0.0] * 8] * 3, bad), (None, bad)):
        for call in (lambda: m.corpus_cross_entropy(q, rows, ids), lambda: m.corpus_distillation(q, rows, lists, sc)):
            with pytest.raises(m.CgvError) as ei:
                call()
            assert ei.value.code == (bad if where == "cpu" else code)
    for r, code in ((rows[0], dim), (rows[0, 0], dim), (None, bad)):
        with pytest.raises(m.CgvError) as ei:
            m.corpus_cross_entropy(torch.zeros((3, 8), device=where), r, ids)
        assert ei.value.code == (bad if where == "cpu" else code)
