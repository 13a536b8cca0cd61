"""Newton-Schulz orthogonalisation (rx_orthogonalize) against the iteration in fp64.

A step amplifies an error along a small singular value by up to a = 3.44 and none by more than 4 (the largest slope of
a s + b s^3 + c s^5 on [0, 1.2]), so no fixed multiple of 2^-24 describes the result: it is held to the error of the same
iteration in plain fp32, whose products round K times per entry where these round 3 K / 16 times after plane products
that hold a term to 12 u (two planes hold an operand to 2^-22 = 4 u, the product left out is below 4 u), times 4, plus 64 u
of the result's norm: five steps at 12 u, for lists where the plain form happens to round to nothing."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ABC = (3.4445, -4.7750, 2.0315)


def _iterate(G, steps, dtype, abc=ABC, eps=1e-7):
    X = G.to(dtype)
    flip = X.shape[0] > X.shape[1]
    if flip:
        X = X.t()
    X = X / (X.pow(2).sum().sqrt() + eps)
    for _ in range(steps):
        A = X @ X.t()
        X = abc[0] * X + (abc[1] * A + abc[2] * (A @ A)) @ X
    return (X.t() if flip else X).contiguous()


def _grad(m, n, seed):
    g = torch.Generator().manual_seed(seed)
    r = max(1, min(m, n) // 6)
    low = (torch.randn(m, r, generator=g) * torch.logspace(0, -2, r)) @ torch.randn(r, n, generator=g)
    return ((low + 0.2 * torch.randn(m, n, generator=g)) * 1e-3).cuda()


def _check(mats, outs, steps=5, abc=ABC):
    for G, o in zip(mats, outs):
        ref = _iterate(G.cpu().double(), steps, torch.float64, abc)
        plain = _iterate(G.cpu(), steps, torch.float32, abc).double()
        err, base, norm = (o.cpu().double() - ref).norm(), (plain - ref).norm(), ref.norm()
        assert err <= 4 * base + 64 * U * norm, (tuple(G.shape), float(err / norm), float(base / norm))


SHAPES = [[(1, 1)], [(1, 64), (64, 1), (5, 3)], [(64, 128), (32, 64), (32, 64), (1, 64)], [(845, 13), (63, 257), (300, 7), (129, 130)],
          [(16, 16), (17, 17), (96, 96), (97, 97)], [(96, 260), (260, 96), (2000, 8), (3, 2500)], [(128, 128), (64, 700)],
          [(200, 1000), (1000, 200), (65, 64)], [(432, 432), (256, 512)], [(2100, 2200)], [(500, 64)] * 30]


@pytest.mark.parametrize("shapes", SHAPES, ids=lambda s: "_".join(f"{m}x{n}" for m, n in s[:4]))
def test_lists_of_matrices(shapes):
    from recsys_amd import ops
    mats = [_grad(m, n, 7 * i + m + n) for i, (m, n) in enumerate(shapes)]
    keep = [m.clone() for m in mats]
    outs = ops.orthogonalize(mats)
    assert all(torch.equal(a, b) for a, b in zip(mats, keep))
    _check(mats, outs)
    again = ops.orthogonalize(mats, out=[torch.full_like(m, float("nan")) for m in mats])
    assert all(torch.equal(a, b) for a, b in zip(outs, again))
    if len(shapes) <= 4:          # a matrix does not depend on its company, as long as the list keeps to one tile size
        for m, o in zip(mats, outs):
            alone, = ops.orthogonalize([m])
            assert (alone.cpu().double() - o.cpu().double()).norm() <= 8e-6 * o.cpu().double().norm()


def test_thin_matrices_on_either_side_of_a_workgroups_memory():
    """Up to 16 rows beside a matrix of the large path: those that fit a workgroup's memory and those that do not."""
    from recsys_amd import ops
    shapes = [(150, 140), (16, 2300), (16, 2600), (2700, 16), (9, 4400), (5000, 9), (1, 16384), (2, 16384), (16384, 3)]
    mats = [_grad(m, n, 31 * i + m) for i, (m, n) in enumerate(shapes)]
    _check(mats, ops.orthogonalize(mats))
    for m in mats:
        _check([m], ops.orthogonalize([m]))


def test_steps_and_coefficients():
    from recsys_amd import ops
    mats = [_grad(40, 90, 1), _grad(150, 140, 2)]
    for steps, abc in ((1, ABC), (3, (1.5, -0.5, 0.0)), (8, (2.0, -1.5, 0.5))):
        _check(mats, ops.orthogonalize(mats, steps=steps, coeffs=abc), steps, abc)


def test_scale_zero_and_nonfinite():
    from recsys_amd import ops
    for shape in ((30, 50), (300, 200)):
        G = _grad(*shape, 3)
        base, = ops.orthogonalize([G])
        for s in (1e12, 1e4):               # eps stands against the norm; above it the scale drops out, to rounding
            other, = ops.orthogonalize([G * s])
            assert (other.double() - base.double()).norm() <= 1e-4 * base.double().norm()
        big, = ops.orthogonalize([torch.full(shape, 3e38, device="cuda")])          # squares beyond fp32
        assert torch.isfinite(big).all()
        zero, bad, fine = ops.orthogonalize([torch.zeros(shape, device="cuda"), torch.full(shape, float("nan"), device="cuda"), G])
        assert not zero.any() and bad.isnan().all() and torch.isfinite(fine).all()


def test_singular_values_come_near_one():
    from recsys_amd import ops
    for shape in ((60, 120), (400, 250)):
        G = _grad(*shape, 4)
        out, = ops.orthogonalize([G])
        s = torch.linalg.svdvals(out.cpu().double())
        s0 = torch.linalg.svdvals(G.cpu().double())
        assert ((s > 0.6) & (s < 1.25))[s0 > 1e-2 * s0.norm()].all()


def test_recorded_and_replayed():
    from recsys_amd import ops
    mats = [_grad(64, 128, 1), _grad(200, 170, 2), _grad(7, 300, 3)]
    outs = [torch.empty_like(m) for m in mats]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.orthogonalize(mats, out=outs)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.orthogonalize(mats, out=outs)
    for seed in range(3):
        for i, m in enumerate(mats):
            m.copy_(_grad(*m.shape, 50 + seed + i))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, ops.orthogonalize(mats)))


def test_refusals():
    from recsys_amd import ops
    G = _grad(8, 9, 1)
    for args, kw, kind in (([G.cpu()], {}, ValueError), ([G.double()], {}, TypeError), ([G.t()], {}, ValueError), ([G[0]], {}, ValueError),
                           ([G[:0]], {}, ValueError), ([G], dict(steps=0), ValueError), ([G], dict(steps=33), ValueError),
                           ([G], dict(coeffs=(1.0, 2.0)), ValueError), ([G], dict(out=[]), ValueError),
                           ([G], dict(out=[torch.empty(9, 8, device="cuda")]), ValueError), ([G], dict(out=[G]), RuntimeError),
                           ([torch.zeros(16385, 1, device="cuda")], {}, RuntimeError)):
        with pytest.raises(kind):
            ops.orthogonalize(args, **kw)
    assert ops.orthogonalize([]) == []
