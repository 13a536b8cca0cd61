"""Catalogue softmax: rows whose log-probability carries no gradient, with targets that are next to impossible.  Such a row
adds nothing through its target.  Reference and tolerances of test_gpu_catalog; a mask of -1e9 or below has weight 0 on both sides, so that the
reference takes it as -inf."""
import pytest
import torch

from test_gpu_catalog import INF, _check, _make, _ref, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [-100.0, -1e4, -1e9, -1e30, torch.finfo(torch.float32).min])
def test_zero_gradient_of_a_masked_target(mask, dtype):
    for R, V, D in ((200, 700, 20), (70, 3706, 64), (130, 90, 130)):
        x, t, y, b = _make(R, V, D, dtype, True, R)
        b[0] = mask
        b[V // 2] = mask
        y[y == 0] = 1
        y[y == V // 2] = 1
        y[::3] = 0                               # padding: the masked item
        y[1::7] = V // 2
        g = torch.randn(R, device="cuda") / R
        g[(y == 0) | (y == V // 2)] = 0
        for gl in (torch.zeros(R, device="cuda"), torch.randn(R, device="cuda") / R):
            got = _run(x, t, y, b, g, gl)
            bb = b.clone()
            if mask < -1e3:
                bb[b == mask] = -INF
            ref, tol = _ref(x, t, y, bb, g, gl)
            assert all(torch.isfinite(v).all() for v in got)
            live = torch.isfinite(ref[0])
            ref[0], tol[0] = torch.where(live, ref[0], got[0].detach().double()), torch.where(live, tol[0], torch.zeros_like(tol[0]))
            _check(got, ref, tol)
            if mask < -1e3:
                assert not got[3][0].any() and not got[3][V // 2].any() and not got[4][0].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_only_the_lse_carries_a_gradient(dtype):
    """Scores spread over hundreds: most targets have no weight at all."""
    for bias in (False, True):
        x, t, y, b = _make(150, 400, 40, dtype, bias, 11, scale=40.0)
        g, gl = torch.zeros(150, device="cuda"), torch.randn(150, device="cuda")
        got = _run(x, t, y, b, g, gl)
        assert all(v is None or torch.isfinite(v).all() for v in got)
        ref, tol = _ref(x, t, y, b, g, gl)
        _check(got, ref, tol)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_next_to_nothing(dtype):
    """Gradients of 1e-30 .. 1e-37, targets without weight among them: finite, and in proportion to those of 1."""
    x, t, y, b = _make(100, 300, 24, dtype, True, 12, scale=20.0)
    g = torch.rand(100, device="cuda") + 0.5
    zero = torch.zeros_like(g)
    one = _run(x, t, y, b, g, zero)
    for size in (2.0 ** -100, 2.0 ** -118, 2.0 ** -123):
        got = _run(x, t, y, b, g * size, zero)
        for p, q, terms in zip(got[2:], one[2:], (100, 100, 100)):
            assert torch.isfinite(p).all()
            # |g| is part of a weight's exponent, which is below 256 in log2 units with steps of 2^-16 there: three additions are
            # off by 3 * 2^-17 ln 2 < 2^-15 of the weight.  Terms below the smallest normal number are held as zero.  Each of the
            # two bf16 results is off by half a step.
            step = 2.0 ** -14 + (2 * 2.0 ** -8 if dtype == torch.bfloat16 else 0.0)
            lim = step * q.double().abs() * size + 2.0 ** -126 * 100 * 4 * float(x.abs().max())
            assert ((p.double() - q.double() * size).abs() <= lim).all()
