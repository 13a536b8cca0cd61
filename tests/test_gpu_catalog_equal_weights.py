"""Catalogue softmax: sums over many items of nearly the same probability.  u = 2^-24."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias", [False, True])
def test_sums_of_nearly_equal_weights(dtype, bias):
    """65536 rows leave a wavefront 100 003 items to add up, whose weights differ by less than the sum's last step: additions that all
    round the same way.  Tolerance: the scores' error (below (D / 2 + 16) u of a size of 0.1), 2 u of an exponential, 16 weights
    joined in five roundings, their sums with the rounding kept, and 4 u of the logarithm's value (12)."""
    from recsys_amd import autograd as rxa
    R, V, D = 65536, 100_003, 32
    gen = torch.Generator(device="cuda").manual_seed(6)
    for std in (0.003, 0.02):
        x = (torch.randn(R, D, generator=gen, device="cuda") * std).to(dtype)
        t = (torch.randn(V, D, generator=gen, device="cuda") * std).to(dtype)
        b = torch.full((V,), 0.3, device="cuda") if bias else None
        y = torch.randint(0, V, (R,), generator=gen, device="cuda")
        _, lse = rxa.catalog_logprob(x, t, y, bias=b)
        some = torch.arange(0, R, 97, device="cuda")
        want = torch.logsumexp(x[some].double() @ t.double().t() + (0.0 if b is None else b.double()), 1)
        assert float((lse[some].double() - want).abs().max()) <= (32 * 0.1 + 2 + 8 + 4 * 12) * U
        xr = x.detach().clone().requires_grad_(True)      # with the means
        _, lse = rxa.catalog_logprob(xr, t, y, bias=b)
        assert float((lse[some].detach().double() - want).abs().max()) <= (32 * 0.1 + 2 + 8 + 4 * 12) * U
