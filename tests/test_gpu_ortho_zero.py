"""Newton-Schulz of matrices of zeros, with eps = 0 as well, beside others of the list."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", [0.0, 1e-7])
def test_zeros_give_zeros(eps):
    from recsys_amd import ops
    shapes = [(8, 300), (64, 128), (300, 400), (1, 1), (500, 500)]
    for zeros in ((0, 1, 2, 3, 4), (1, 4), (0, 2, 3)):
        mats = [torch.zeros(s, device="cuda") if i in zeros else torch.randn(s, device="cuda") for i, s in enumerate(shapes)]
        out = ops.orthogonalize(mats, eps=eps)
        for i, o in enumerate(out):
            assert torch.isfinite(o).all()
            assert bool(o.any()) == (i not in zeros), i
        bad = [m.clone() for m in mats]
        bad[4][3, 3] = float("nan")
        assert ops.orthogonalize(bad, eps=eps)[4].isnan().all()
