"""Lists of matrices longer than one call takes: refused as a whole, before anything of them is stepped."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_bad_matrix_behind_the_first_chunk_leaves_the_list_alone():
    from recsys_amd import ops
    ws = [torch.randn(4, 5, device="cuda") for _ in range(30)] + [torch.randn(16385, 2, device="cuda")]
    gs, ms = [torch.randn_like(w) for w in ws], [torch.zeros_like(w) for w in ws]
    before = [w.clone() for w in ws]
    with pytest.raises(RuntimeError, match="16384"):
        ops.muon_step(ws, gs, ms, [0.1] * 31)
    with pytest.raises(ValueError, match="steps"):
        ops.muon_step(ws[:30], gs[:30], ms[:30], [0.1] * 30, steps=33)
    out = [torch.full_like(w, 7.0) for w in ws]
    with pytest.raises(RuntimeError, match="16384"):
        ops.orthogonalize(gs, out=out)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ws, before))
    assert not any(m.any() for m in ms) and all((o == 7.0).all() for o in out)
    ops.muon_step(ws[:30], gs[:30], ms[:30], [0.1] * 30)
    torch.cuda.synchronize()
    assert not any(torch.equal(a, b) for a, b in zip(ws[:30], before))
