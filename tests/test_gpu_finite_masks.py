"""Rows beyond 1024 columns with finite masks of any size, and with all scores far from zero: the results are those of the
definition in fp64 on the same numbers, as for narrow rows.

Tolerances: those of test_gpu_logprob (its ``_tol`` and ``_ref_grad``), which count 8 u of a result's own size; a masked score has
weight exp(-1e9) = 0 on both sides.  A weight below the smallest normal number, 2^-126 = e^-87.3, is held as zero: its whole gradient,
that many times |g_lse| + sum |g| + |g_H| (88 + H), is left out.  A log-probability beyond the largest fp32 number (rows of
+-2.3e38) is -inf, as rounding has it."""
import pytest
import torch

from test_gpu_logprob import INF, _compare, _ref, _ref_grad

pytestmark = pytest.mark.gpu


def _gradients(logits, targets, lengths, only_logprob):
    from recsys_amd import autograd as rxa
    R, T = targets.shape
    x = logits.clone().requires_grad_(True)
    out = rxa.log_probs(x, targets, lengths=lengths)
    gen = torch.Generator(device="cuda").manual_seed(R)
    g = torch.randn(R, T, device="cuda", generator=gen)
    gh, gl = (torch.zeros(R, device="cuda") if only_logprob else torch.randn(R, device="cuda", generator=gen) for _ in range(2))
    dl, = torch.autograd.grad(out[:1] if only_logprob else out[:3], x, (g,) if only_logprob else (g, gh, gl))
    ref, noise = _ref_grad(logits, targets, lengths, g, gh, gl)
    H = out.entropy.detach()
    tiny = 2.0 ** -126 * (gl.abs() + g.abs().sum(1) + gh.abs() * (88 + H)).double().cpu()[:, None]
    tol = noise + (2.0 ** -8 * (ref.abs() + noise) if logits.dtype == torch.bfloat16 else 0) + tiny
    err = (dl.double().cpu() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())


def _both(logits, k):
    from recsys_amd import autograd as rxa
    R, V = logits.shape
    targets = torch.stack([torch.zeros(R, dtype=torch.int64), torch.full((R,), V - 1), torch.full((R,), V // 2)], 1).cuda()
    ref = list(_ref(logits, targets, None, k)[0])
    ref[:4] = [torch.where(v.float() == -INF, torch.full_like(v, -INF), v) for v in ref[:4]]
    _compare(rxa.log_probs(logits, targets, k=k), ref, V)
    for only_logprob in (True, False):
        _gradients(logits, targets, None, only_logprob)


@pytest.mark.parametrize("V", [1000, 1500, 9001, 30000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masks_of_any_size(V, dtype):
    lowest = torch.finfo(dtype).min
    for mask in (-1e7, -2e7, -1e8, -1e9, -1e10, -1e12, -1e18, -1e20, -1e24, -1e30, -1e35, -1e36, -1e37, -9e37, -1e38, lowest / 2, lowest):
        gen = torch.Generator(device="cuda").manual_seed(V)
        base = torch.randn(7, V, generator=gen, device="cuda") * 2
        u = torch.rand(7, V, generator=gen, device="cuda")
        base[0] = mask
        base[1, u[1] < 0.5] = mask
        base[2, u[2] < 0.99] = mask
        base[3, 1:] = mask                       # nothing left but the first, the last, one in the middle
        base[4, :-1] = mask
        base[5, :V // 2] = mask
        base[5, V // 2 + 1:] = mask
        base[6, u[6] < 0.9] = mask
        base[6, u[6] > 0.95] = -INF
        _both(base.to(dtype), 12)


@pytest.mark.parametrize("V", [1500, 30000, 200003])
def test_scores_far_from_zero(V):
    """Rows around an offset, also where the steps of fp32 there are 1 .. 2^60, rows of two levels, and rows that rise."""
    gen = torch.Generator(device="cuda").manual_seed(V)
    for at in (1.6e7, 1.6777e7, 1.6778e7, 1e8, 1e10, 1e25, 1e37, 2.3e38):
        base = torch.randn(6, V, generator=gen, device="cuda") * 3
        for r, sign in ((0, 1.0), (1, -1.0)):
            base[r] = sign * at + base[r]
            base[r + 2] = torch.where(torch.rand(V, generator=gen, device="cuda") < 0.5, sign * at + base[r + 2], -sign * at + base[r + 2])
        base[4] = -at * (1 + torch.arange(V, device="cuda") * 2.0 ** -22)
        base[5] = at * (1 + torch.arange(V, device="cuda") * 2.0 ** -22)
        _both(base, 7)


def test_splits_that_hold_masks_only():
    """A row over several workgroups: all but one see nothing but masks, of two sizes."""
    for V in (70001, 1000003):
        for mask in (-1e9, -1e30, -1e38):
            base = torch.full((2, V), mask, device="cuda")
            base[:, ::3] = 2 * mask
            base[0, V - 3000:] = torch.linspace(-5, 5, 3000, device="cuda")
            _both(base, 50)
