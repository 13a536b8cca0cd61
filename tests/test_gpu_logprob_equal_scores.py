"""Rows of many nearly equal scores: additions to a lane's sum that all round the same way.  u = 2^-24.

Tolerance: an exponential is good to 2 u, its argument (below 1) to u; 16 of them are joined in four roundings and added with the
rounding kept (2 u); lanes, wavefronts and splits join in a tree of at most 16; the logarithm and the row's offset cost 4 u of
their size."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("R,V", [(1100, 1_000_003), (1, 200_000_003)])
def test_sums_of_nearly_equal_scores(R, V):
    from recsys_amd import autograd as rxa
    g = torch.Generator(device="cuda").manual_seed(1)
    for spread in (1e-6, 1e-5, 1e-4, 0.3):
        l = torch.rand(R, V, generator=g, device="cuda").mul_(-spread)
        l += 0.25
        l[:, ::4096] = 0.25
        out = rxa.log_probs(l, torch.zeros(R, dtype=torch.int64, device="cuda"))
        want = torch.cat([torch.logsumexp(l[i:i + 32].double(), 1) for i in range(0, R, 32)])
        tol = (3 + 4 + 2 + 16) * U + 4 * U * want.abs()
        err = (out.lse.double() - want).abs()
        assert (err <= tol).all(), (spread, float((err / tol).max()), float(err.max()))
        del l
