"""Catalogue softmax: gradients of rows that are nearly sure of their target, where g (t_y - mean) and g (1 - p_y) cancel.

dx = g sum_{v != y} p_v (t_y - t_v): every weight p_v may be off by its score's error (relative ``ew``) and, bf16, by its rounding (2^-8);
sums and products in fp32 add (V / 2 + 64) u of the terms' size, whose vectors meet separately, and bf16 rounds the result
(2^-8).  All of it is in proportion to 1 - p_y.  The table's gradient is a sum over rows of c p_v x and, for the target, g (1 - p_y) x, each
of them off by ``ew`` and the bf16 rounding of its weight, with (R / 2 + 64) u for the sum."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _confident(R, V, D, dtype, want, seed, offset=0.0):
    """Rows along their target's vector, as long as it takes for p_y to come near ``want``; ``offset``: what all items share."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = (torch.randn(V, D, generator=gen, device="cuda") / math.sqrt(D) + offset).to(dtype)
    y = torch.randint(0, V, (R,), generator=gen, device="cuda")
    T = t.double()
    way = T[y] - T.mean(0) + 0.1 * torch.randn(R, D, generator=gen, device="cuda", dtype=torch.float64) / math.sqrt(D)
    lo, hi = torch.zeros(R, 1, dtype=torch.float64, device="cuda"), torch.full((R, 1), 200.0, dtype=torch.float64, device="cuda")
    for _ in range(50):
        mid = (lo + hi) / 2
        p = torch.softmax(mid * way @ T.t(), 1).gather(1, y[:, None])
        lo, hi = torch.where(p < want, mid, lo), torch.where(p < want, hi, mid)
    return (hi * way).to(dtype), t, y


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("want", [0.5, 0.9, 0.99, 0.999, 0.9999])
@pytest.mark.parametrize("R,V,D,offset", [(300, 1000, 64, 0.0), (130, 5003, 128, 0.0), (40, 200, 20, 0.5), (64, 20011, 200, 0.0), (600, 90, 32, -1.0)])
def test_gradient_of_x(R, V, D, offset, want, dtype):
    from recsys_amd import autograd as rxa
    x, t, y = _confident(R, V, D, dtype, want, R + V, offset)
    gen = torch.Generator(device="cuda").manual_seed(1)
    g = torch.randn(R, generator=gen, device="cuda")
    for bias in (None, torch.zeros(V, device="cuda")):
        leaves = [v.detach().clone().requires_grad_(True) for v in (x, t) + (() if bias is None else (bias,))]
        lp, _ = rxa.catalog_logprob(leaves[0], leaves[1], y, bias=None if bias is None else leaves[2])
        grads = torch.autograd.grad(lp, leaves, g)
        X, T = x.double(), t.double()
        s = X @ T.t()
        p = torch.softmax(s, 1)
        rows = torch.arange(R, device="cuda")
        rest = p.clone()
        rest[rows, y] = 0
        G, q = g.double()[:, None], rest.sum(1, keepdim=True)
        ref = G * (q * T[y] - rest @ T)
        apart = torch.stack([(rest[i, :, None] * (T[y[i]] - T).abs()).sum(0) for i in range(R)]) * G.abs()
        whole = G.abs() * (q * T[y].abs() + rest @ T.abs())
        size = (X.abs() @ T.abs().t()).max(1, keepdim=True).values
        big = X.abs().max() * T.abs().sum(1).max() + T.abs().max() * X.abs().sum(1, keepdim=True)
        ew = 4 * ((D / 2 + 16) * U * size + 2.0 ** -39 * big) + 8 * U * (s.abs().max(1, keepdim=True).values + 8)
        r = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
        # fp32: planes of weights (2^-36 of the largest beside them) and of vectors (2^-22)
        planes = 0.0 if dtype == torch.bfloat16 else 2.0 ** -36 * G.abs() * T.abs().sum(0) + 16 * U * whole
        tol = apart * (r + ew) + whole * (min(V, 4096) / 2 + 64) * U + r * ref.abs() * (1 + r) + planes
        err = (grads[0].double() - ref).abs()
        assert (err <= tol).all(), (float((err / tol).max()), float((err.norm(dim=1) / ref.norm(dim=1)).max()))
        if dtype == torch.bfloat16 and offset == 0.0:      # the same in one number: 2^-8 for the weights and as much for the result
            assert float((err.norm(dim=1) / ref.norm(dim=1)).max()) <= 2.0 ** -7
        W = -G * rest
        W[rows, y] = (G * q)[:, 0]
        ref, size = W.t() @ X, W.abs().t() @ X.abs()
        tol = (W.abs() * (ew + r)).t() @ X.abs() + size * ((R / 2 + 64) * U + (16 * U if r == 0 else 0.0)) + r * ref.abs() * (1 + r) + 3 * 2.0 ** -126 * X.abs().sum(0)
        if r == 0:
            tol = tol + 2.0 ** -36 * W.abs().max(0).values[:, None] * X.abs().sum(0) + 2.0 ** -39 * X.abs().max() * W.abs().sum(0)[:, None]
        err = (grads[1].double() - ref).abs()
        assert (err <= tol).all(), ("table", float((err / tol).max()))
        if bias is not None:
            err = (grads[2].double() - W.sum(0)).abs()
            tol = (W.abs() * ew).sum(0) + W.abs().sum(0) * 64 * U + 3 * 2.0 ** -126 * R
            assert (err <= tol).all(), ("bias", float((err / tol).max()))
        only = leaves[1].detach().clone().requires_grad_(True)      # without the means
        lp, _ = rxa.catalog_logprob(x, only, y, bias=bias)
        dt, = torch.autograd.grad(lp, only, g)
        err = (dt.double() - ref).abs()
        tol = (W.abs() * (ew + r)).t() @ X.abs() + size * ((R / 2 + 64) * U + (16 * U if r == 0 else 0.0)) + r * ref.abs() * (1 + r) + 3 * 2.0 ** -126 * X.abs().sum(0)
        if r == 0:
            tol = tol + 2.0 ** -36 * W.abs().max(0).values[:, None] * X.abs().sum(0) + 2.0 ** -39 * X.abs().max() * W.abs().sum(0)[:, None]
        assert (err <= tol).all(), ("table alone", float((err / tol).max()))


def test_with_a_gradient_of_the_lse_as_well():
    """g = g_lse: the means drop out, and dx = g t_y; g_lse alone: the mean with the target in it."""
    from recsys_amd import autograd as rxa
    for dtype in (torch.float32, torch.bfloat16):
        x, t, y = _confident(200, 700, 48, dtype, 0.99, 4)
        y[::5] = -1
        g = torch.randn(200, device="cuda")
        leaf = x.detach().clone().requires_grad_(True)
        lp, lse = rxa.catalog_logprob(leaf, t, y)
        p = torch.softmax(x.double() @ t.double().t(), 1)
        mean, size = p @ t.double(), p @ t.double().abs()
        ty = torch.where((y >= 0)[:, None], t[y.clamp(min=0)].double(), torch.zeros_like(mean))
        r = (2.0 ** -8 if dtype == torch.bfloat16 else 0.0) + 2.0 ** -15
        for a, b, want in ((1.0, 1.0, torch.where((y >= 0)[:, None], ty, mean)), (0.0, 1.0, mean)):
            dx, = torch.autograd.grad((lp, lse), leaf, (a * g, b * g), retain_graph=True)
            want = g.double()[:, None] * want
            assert ((dx.double() - want).abs() <= r * (g.double().abs()[:, None] * (size + ty.abs()) + want.abs())).all()
