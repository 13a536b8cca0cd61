"""Catalogue softmax over tables that are zero or nearly so: all items equally likely, many of them.  u = 2^-24."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _grads(x, t, y, b, g, gl):
    from recsys_amd import autograd as rxa
    leaves = [v.detach().clone().requires_grad_(True) for v in (x, t)] + ([] if b is None else [b.detach().clone().requires_grad_(True)])
    lp, lse = rxa.catalog_logprob(leaves[0], leaves[1], y, bias=None if b is None else leaves[2])
    return (lp, lse) + tuple(torch.autograd.grad((lp, lse), leaves, (g, gl)))


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("size", [0.0, 1e-30, 1e-24, 1e-20])
def test_tables_of_nothing(size, bias):
    """p = 1 / V to fp32 (scores are below 1e-18).  Each of the results' sums has at most 16 chains of equal, exact terms."""
    V, D, R = 200_003, 24, 9
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(R, D, generator=gen, device="cuda")
    t = torch.randn(V, D, generator=gen, device="cuda") * size
    b = torch.zeros(V, device="cuda") if bias else None
    y = torch.randint(0, V, (R,), generator=gen, device="cuda")
    y[3] = -1
    g, gl = torch.randn(R, generator=gen, device="cuda"), torch.randn(R, generator=gen, device="cuda")
    got = _grads(x, t, y, b, g, gl)
    lse = math.log(V)
    assert ((got[1].double() - lse).abs() <= 64 * U).all()
    lp = torch.where(y < 0, 0.0, -lse).double()
    assert ((got[0].double() - lp).abs() <= 64 * U).all()
    G = torch.where(y < 0, torch.zeros_like(g), g).double()
    c = gl.double() - G
    X, T = x.double(), t.double()
    dx = G[:, None] * T[y.clamp(min=0)] + c[:, None] * T.mean(0)
    lim = (G.abs()[:, None] * T[y.clamp(min=0)].abs() + c.abs()[:, None] * T.abs().mean(0)) * 2.0 ** -18 + 3 * 2.0 ** -126
    assert ((got[2].double() - dx).abs() <= lim).all()
    dt = (c[:, None] * X).sum(0).expand(V, D) / V
    ab = ((c.abs()[:, None] * X.abs()).sum(0) / V).expand(V, D)
    hot, hab = torch.zeros(V, D, dtype=torch.float64, device="cuda"), torch.zeros(V, D, dtype=torch.float64, device="cuda")
    hot.index_add_(0, y.clamp(min=0), G[:, None] * X)
    hab.index_add_(0, y.clamp(min=0), (G[:, None] * X).abs())
    assert ((got[3].double() - dt - hot).abs() <= 128 * U * (ab + hab)).all()
    if bias:
        db = torch.zeros(V, dtype=torch.float64, device="cuda").index_add_(0, y.clamp(min=0), G) + c.sum() / V
        assert ((got[4].double() - db).abs() <= 128 * U * (G.abs().sum() * (db.abs() > 1e-3) + c.abs().sum() / V)).all()


def test_a_zero_table_can_be_trained():
    """Its first step moves it: a dead row would leave it at zero."""
    from recsys_amd import autograd as rxa
    t = torch.zeros(150_000, 16, device="cuda", requires_grad=True)
    x = torch.randn(300, 16, device="cuda")
    lp, _ = rxa.catalog_logprob(x, t, torch.arange(300, device="cuda"))
    d, = torch.autograd.grad(-lp.mean(), t)
    assert torch.isfinite(lp).all() and (d[:300].abs().sum(1) > 0).all() and (d[300:].abs().sum(1) > 0).all()


def test_many_rows_of_zeros():
    """Rows of zeros stream through the table's pass by the hundred thousand beside ordinary ones."""
    R, V, D = 400_000, 300, 8
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(R, D, generator=gen, device="cuda")
    x[1000:] = 0
    t, b = torch.randn(V, D, generator=gen, device="cuda"), torch.randn(V, generator=gen, device="cuda")
    y = torch.randint(0, V, (R,), generator=gen, device="cuda")
    g, gl = torch.randn(R, generator=gen, device="cuda"), torch.randn(R, generator=gen, device="cuda")
    got = _grads(x, t, y, b, g, gl)
    s = x.double() @ t.double().t() + b.double()
    p = torch.softmax(s, 1)
    c = gl.double() - g.double()
    w = p * c[:, None]
    aw = w.abs()
    w[torch.arange(R, device="cuda"), y] += g.double()
    aw[torch.arange(R, device="cuda"), y] += g.double().abs()
    assert ((got[1].double() - torch.logsumexp(s, 1)).abs() <= 512 * U).all()
    # weights good to 512 u (their scores are below 16, of 8 products); the sums over 400 000 rows keep what additions lose
    assert ((got[4].double() - w.sum(0)).abs() <= 600 * U * aw.sum(0)).all()
    assert ((got[3].double() - w.t() @ x.double()).abs() <= 1200 * U * (aw.t() @ x.double().abs())).all()
