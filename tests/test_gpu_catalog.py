"""Softmax over a whole catalogue (rx_catalog_*) against the definition in fp64.

Tolerances, u = 2^-24.  A score is a sum of D products, computed as three plane products accumulated in fp32 (two planes
hold an operand to 2^-22 = 4 u and the product left out is below 4 u of a term: 12 u; scale and bias round a few times more,
and 3 D / 8 additions cover the accumulation): |ds| <= (D / 2 + 16) u sum_d |x_d t_d| =: delta.
lse moves by at most max delta, plus the sum of V weights in chains of at most ``_seq`` additions: (_seq + 32) u, plus
4 u |lse|.  A weight p carries the relative error delta + 4 u (|lse| + |s| + 8).  A gradient entry is a sum of weights
times vector entries; with M = sum |weight * entry| it may be off by M times the weights' error plus (terms / 2 + 32) u for
the plane products.  bf16: the weights are rounded once (2^-8 of each term) and so is the result (2^-8 of the value).
Weights and planes of weights below the smallest normal number, 2^-126, are held as zero: at most three times 2^-126 per
term, whatever the term's size.  fp32: the second product's weights are fp16 pairs under a reference that takes the largest of
a vector's weights to at least 2^11, and the lower of a pair has steps of 2^-24, so that a weight is off by up to 2^-25, 2^-36 of
the largest, on top of its relative error.  Likewise an element of x or the table: scaled so that the largest of its vector, or of
64 neighbours, is at least 2^14, it is off by up to 2^-25, 2^-39 of that one, on top of its relative 4 u."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U, INF = 2.0 ** -24, float("inf")
BF = 2.0 ** -8


def _make(R, V, D, dtype, bias, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, D, generator=g).mul(scale).to(dtype).cuda()
    t = (torch.randn(V, D, generator=g) * (2 / math.sqrt(D))).to(dtype).cuda()
    b = torch.randn(V, generator=g).cuda() if bias else None
    y = torch.randint(0, V, (R,), generator=g).cuda()
    return x, t, y, b


def _ref(x, t, y, b, g=None, gl=None):
    """(values, tolerances) of logprob, lse and, with gradients, dx, dt, db."""
    R, D = x.shape
    V, bf = t.shape[0], x.dtype == torch.bfloat16
    X, T = x.detach().double(), t.detach().double()
    B = torch.zeros(V, dtype=torch.float64, device=x.device) if b is None else b.detach().double()
    s = X @ T.t() + B
    size = X.abs() @ T.abs().t() + torch.where(B.abs() < 1e30, B.abs(), torch.zeros_like(B))
    m = s.max(1, keepdim=True).values
    m = torch.where(m == -INF, torch.zeros_like(m), m)
    e = (s - m).exp()
    z = e.sum(1, keepdim=True)
    empty = z[:, 0] == 0
    lse = (m + z.log())[:, 0]
    logp = (s - m) - z.log()
    p = torch.where(empty[:, None], torch.zeros_like(e), e / z)
    none = y < 0
    yy = y.clamp(min=0)
    lp = logp.gather(1, yy[:, None])[:, 0]
    lp = torch.where(s.gather(1, yy[:, None])[:, 0] == -INF, torch.full_like(lp, -INF), lp)
    lp = torch.where(none, torch.zeros_like(lp), lp)
    delta = (D / 2 + 16) * U * torch.where(torch.isfinite(s), size, torch.zeros_like(size)).max(1).values
    px, pt = (X.abs().max(), T.abs().max()) if not bf else (0.0, 0.0)
    delta = delta + 2.0 ** -39 * (px * T.abs().sum(1).max() + pt * X.abs().sum(1))
    seq = max(64, V / 64)
    big = torch.where(torch.isfinite(lse), lse.abs(), torch.zeros_like(lse))
    t_lse = delta + (seq + 32) * U + 4 * U * big
    t_lp = 2 * t_lse + 4 * U * torch.where(torch.isfinite(lp), lp.abs(), torch.zeros_like(lp))
    out, tol = [lp, lse], [t_lp, t_lse]
    if g is None:
        return out, tol
    live = ~none & ~empty & (B[yy] > -INF)
    G = torch.where(live, g.double(), torch.zeros_like(lp))
    c = torch.where(empty, torch.zeros_like(lp), gl.double() - G)
    w = p * c[:, None]
    hot = torch.zeros_like(w)
    hot[torch.arange(R, device=x.device), yy] = G
    W = w + hot
    ew = t_lse + delta + 4 * U * (big + size.max(1).values + 8)          # relative error of a row's weights
    dx, dt, db = W @ T, W.t() @ X, W.sum(0)
    aw = w.abs()
    mx, mt = aw @ T.abs() + hot.abs() @ T.abs(), aw.t() @ X.abs() + hot.abs().t() @ X.abs()
    acc_x, acc_t = (V / 2 + 64) * U if V < 4096 else (2048 + 64) * U, (R / 2 + 64) * U
    r = BF if bf else 0.0
    tx = mx * (acc_x + r) + (aw * ew[:, None]) @ T.abs()
    tt = mt * (acc_t + r) + (aw * ew[:, None]).t() @ X.abs()
    tb = (aw.sum(0) + hot.abs().sum(0)) * acc_t + (aw * ew[:, None]).sum(0)
    out += [dx, dt, db]
    tiny = 3 * 2.0 ** -126
    if not bf:
        big = torch.maximum(aw, hot.abs())
        tx = tx + 2.0 ** -36 * aw.max(1, keepdim=True).values * T.abs().sum(0) + 2.0 ** -39 * pt * aw.sum(1, keepdim=True)
        tt = tt + 2.0 ** -36 * big.max(0).values[:, None] * X.abs().sum(0) + 2.0 ** -39 * px * (aw + hot.abs()).sum(0)[:, None]
    tol += [tx + r * dx.abs() + tiny * T.abs().sum(0), tt + r * dt.abs() + tiny * X.abs().sum(0), tb + tiny * R]
    return out, tol


def _check(got, ref, tol):
    names = ("logprob", "lse", "dx", "dt", "db")
    for n, a, e, t in zip(names, got, ref, tol):
        if a is None:
            continue
        a = a.detach().double()
        assert a.shape == e.shape, n
        fin = torch.isfinite(e)
        assert torch.equal(a[~fin], e[~fin]) or torch.equal(a[~fin].isnan(), e[~fin].isnan()), n
        err = (a - e).abs()[fin]
        assert (err <= t[fin]).all(), (n, float((err / t[fin]).max()), float(err.max()))


def _run(x, t, y, b, g, gl):
    from recsys_amd import autograd as rxa
    leaves = [v.detach().clone().requires_grad_(True) for v in (x, t)] + ([b.detach().clone().requires_grad_(True)] if b is not None else [])
    lp, lse = rxa.catalog_logprob(leaves[0], leaves[1], y, bias=leaves[2] if b is not None else None)
    grads = torch.autograd.grad((lp, lse), leaves, (g, gl))
    return (lp, lse) + tuple(grads) + ((None,) if b is None else ())


SIZES = [(1, 1, 1), (1, 2, 3), (7, 3706, 16), (3, 31, 31), (33, 64, 32), (130, 65, 33), (129, 1000, 64), (64, 129, 65), (257, 300, 100),
         (20, 5003, 128), (150, 200, 130), (5, 700, 200), (300, 129, 256), (1, 20011, 64), (1000, 40, 48), (2000, 3, 8), (513, 1029, 7)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V,D", SIZES)
def test_values_and_gradients(R, V, D, dtype):
    from recsys_amd import autograd as rxa
    for bias in (False, True):
        x, t, y, b = _make(R, V, D, dtype, bias, R + 3 * V + 7 * D)
        y[::4] = -1
        g = torch.randn(R, device="cuda") / R
        gl = torch.randn(R, device="cuda") / R
        gl[::5] = g[::5]                         # c = 0 where there is a target
        got = _run(x, t, y, b, g, gl)
        ref, tol = _ref(x, t, y, b, g, gl)
        _check(got, ref, tol)
        again = _run(x, t, y, b, g, gl)
        assert all(p is None or torch.equal(p, q) for p, q in zip(got, again))
        with torch.no_grad():                    # without the expectations
            lp, lse = rxa.catalog_logprob(x, t, y, bias=b)
        _check((lp, lse), ref[:2], tol[:2])


def test_every_row_wants_the_same_item():
    for dtype in (torch.float32, torch.bfloat16):
        x, t, y, b = _make(900, 70, 40, dtype, True, 3)
        y[:] = 69
        g = -torch.rand(900, device="cuda")
        gl = torch.zeros(900, device="cuda")
        ref, tol = _ref(x, t, y, b, g, gl)
        _check(_run(x, t, y, b, g, gl), ref, tol)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_items_and_large_scores(dtype):
    R, V, D = 70, 500, 24
    lowest = torch.finfo(torch.float32).min
    for case in range(6):
        x, t, y, b = _make(R, V, D, dtype, True, case, scale=30.0 if case == 5 else 1.0)
        if case == 0:
            b[torch.rand(V, device="cuda") < 0.6] = -INF
        elif case == 1:
            b[:] = -INF
        elif case == 2:
            b[torch.rand(V, device="cuda") < 0.6] = lowest
        elif case == 3:
            b[:] = lowest
        elif case == 4:
            b[:] = -INF
            b[77] = 0.5
        g, gl = torch.randn(R, device="cuda"), torch.randn(R, device="cuda")
        got = _run(x, t, y, b, g, gl)
        if case == 3:            # every score is the lowest value: the items are equally likely, whatever x says
            assert ((got[0] + math.log(V)).abs() < 1e-3).all()
            w = (gl - g)[:, None].double() / V + torch.nn.functional.one_hot(y, V) * g[:, None].double()
            assert ((got[3].double() - w.t() @ x.double()).abs() <= (2 * BF if dtype == torch.bfloat16 else 1e-5) * (w.abs().t() @ x.double().abs())).all()
            continue
        ref, tol = _ref(x, t, y, b, g, gl)
        if case == 2:            # the target's own log-probability there is the mask's value: relative to it
            off = b[y] == lowest
            assert (got[0][off] < -1e38).all()
            ref[0], tol[0] = ref[0].clone(), tol[0].clone()
            ref[0][off] = got[0][off].double()
        _check(got, ref, tol)
        if case == 1:
            assert (got[1] == -INF).all() and (got[0] == -INF).all() and not any(v.any() for v in got[2:])


def test_sharp_softmax_beside_targets_of_small_elements():
    """Scores of several tens: an item's gradient is its target row's share plus weights 2^-20 of it times larger elements."""
    for seed in range(30):
        x, t, y, b = _make(16, 1710, 74, torch.float32, True, 400 + seed, scale=4.0)
        x[:, ::5] *= 1e-4
        g = torch.Generator().manual_seed(seed)
        g, gl = torch.randn(16, generator=g).cuda(), torch.zeros(16, device="cuda")
        ref, tol = _ref(x, t, y, b, g, gl)
        _check(_run(x, t, y, b, g, gl), ref, tol)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [20, 64, 200])
def test_items_that_are_out_may_hold_anything(dtype, D):
    """The results are those of a table with zeros there: the same bits, a zero gradient."""
    x, t, y, b = _make(150, 700, D, dtype, True, 5)
    out = torch.rand(700, device="cuda") < 0.3
    b[out] = -INF
    t[out] = 0
    g, gl = torch.randn(150, device="cuda"), torch.randn(150, device="cuda")
    clean = _run(x, t, y, b, g, gl)
    t[out] = torch.tensor([float("nan"), INF, -INF, 3e38], device="cuda").to(dtype)[torch.randint(0, 4, (int(out.sum()), 1), device="cuda")]
    for a, c in zip(_run(x, t, y, b, g, gl), clean):
        assert torch.equal(a, c)
    assert not clean[3][out].any() and not clean[4][out].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V,D", [(150, 700, 20), (65, 90, 64), (200, 3000, 190), (7, 40, 3)])
def test_padded_rows_may_hold_anything(R, V, D, dtype):
    """Rows without a target: zero gradient for them, the same bits for the others and the table as with zeros there."""
    for bias in (False, True):
        x, t, y, b = _make(R, V, D, dtype, bias, R + V)
        pad = torch.rand(R, device="cuda") < 0.3
        pad[-2:] = True
        y[pad] = -1
        x[pad] = 0
        g, gl = torch.randn(R, device="cuda"), torch.zeros(R, device="cuda")
        clean = _run(x, t, y, b, g, gl)
        x[pad] = torch.tensor([float("nan"), INF, -INF, 3e38], device="cuda").to(dtype)[torch.randint(0, 4, (int(pad.sum()), 1), device="cuda")]
        got = _run(x, t, y, b, g, gl)
        assert torch.equal(got[0], clean[0]) and torch.equal(got[1][~pad], clean[1][~pad])
        for p, q in zip(got[2:], clean[2:]):
            assert p is None or torch.equal(p, q)
        assert not got[2][pad].any()


def test_a_nan_row_keeps_to_itself_in_the_forward_pass():
    from recsys_amd import autograd as rxa
    x, t, y, b = _make(100, 300, 20, torch.float32, False, 1)
    good, _ = rxa.catalog_logprob(x, t, y)
    x[41, 3] = float("nan")
    lp, lse = rxa.catalog_logprob(x, t, y)
    keep = torch.arange(100, device="cuda") != 41
    assert torch.equal(lp[keep], good[keep]) and lp[41].isnan() and lse[41].isnan()


def test_gradients_against_differences():
    x, t, y, b = _make(5, 37, 6, torch.float32, True, 2)
    y[1] = -1
    g, gl = torch.randn(5, device="cuda"), torch.randn(5, device="cuda")
    got = _run(x, t, y, b, g, gl)

    def f(X, T, B):
        s = X @ T.t() + B
        lse = torch.logsumexp(s, 1)
        lp = torch.where(y >= 0, s.gather(1, y.clamp(min=0)[:, None])[:, 0] - lse, torch.zeros_like(lse))
        return float((lp * g.double()).sum() + (lse * gl.double()).sum())

    base = [x.double(), t.double(), b.double()]
    for k, grad in enumerate(got[2:5]):
        flat = grad.reshape(-1)
        for i in range(0, flat.numel(), max(1, flat.numel() // 40)):
            d = []
            for s in (1e-5, -1e-5):
                v = [q.clone() for q in base]
                v[k].reshape(-1)[i] += s
                d.append(f(*v))
            want = (d[0] - d[1]) / 2e-5          # 1e-10 third-order terms, 1e-16 / 1e-5 of rounding
            assert abs(float(flat[i]) - want) <= 2e-6 * (1 + abs(want)), (k, i)


def test_strided_operands_and_partial_gradients():
    from recsys_amd import autograd as rxa
    for dtype in (torch.float32, torch.bfloat16):
        x, t, y, b = _make(65, 210, 20, dtype, True, 4)
        bx = torch.full((65, 37), float("nan"), dtype=dtype, device="cuda")
        bt = torch.full((210, 29), float("nan"), dtype=dtype, device="cuda")
        for off in (0, 1, 4):
            bx[:, off:off + 20] = x
            bt[:, off:off + 20] = t
            g = torch.randn(65, device="cuda")
            vx, vt = bx[:, off:off + 20].detach().requires_grad_(True), bt[:, off:off + 20].detach().requires_grad_(True)
            vb = b.clone().requires_grad_(True)
            lp, lse = rxa.catalog_logprob(vx, vt, y, bias=vb)
            dx, dt, db = torch.autograd.grad(lp, (vx, vt, vb), g)
            ref, tol = _ref(x, t, y, b, g, torch.zeros_like(g))
            _check((lp, lse, dx, dt, db), ref, tol)
        for want in ((True, False, False), (False, True, False), (False, False, True), (True, False, True)):
            leaves = [v.detach().clone().requires_grad_(w) for v, w in zip((x, t, b), want)]
            lp, _ = rxa.catalog_logprob(leaves[0], leaves[1], y, bias=leaves[2])
            got = torch.autograd.grad(lp, [v for v in leaves if v.requires_grad], g)
            for v, k in zip(got, [i for i in range(3) if want[i]]):
                assert ((v.double() - ref[2 + k]).abs() <= tol[2 + k]).all()


def test_recorded_and_replayed_on_another_stream():
    from recsys_amd import ops
    ops.set_index_check("deferred")
    try:
        for dtype, bias in ((torch.float32, True), (torch.bfloat16, False)):
            x, t, y, b = _make(140, 1500, 32, dtype, bias, 9)
            g, gl = torch.randn(140, device="cuda"), torch.randn(140, device="cuda")
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                _run(x, t, y, b, g, gl)
                stream.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    rec = _run(x, t, y, b, g, gl)
            torch.cuda.current_stream().wait_stream(stream)
            for seed in range(3):
                nx, nt, ny, nb = _make(140, 1500, 32, dtype, bias, 20 + seed)
                x.copy_(nx); t.copy_(nt); y.copy_(ny); g.normal_()
                if bias:
                    b.copy_(nb)
                torch.cuda.synchronize()
                graph.replay()
                eager = _run(x, t, y, b, g, gl)
                torch.cuda.synchronize()
                assert all(p is None or torch.equal(p, q) for p, q in zip(rec, eager))
        ops.raise_if_index_error()
    finally:
        ops.set_index_check("sync")


def test_refusals():
    from recsys_amd import autograd as rxa, ops
    x, t, y, b = _make(6, 40, 12, torch.float32, True, 5)
    for bad in (40, -2, 1 << 40):
        yy = y.clone()
        yy[2] = bad
        with pytest.raises(IndexError):
            rxa.catalog_logprob(x, t, yy, bias=b)
    ops.raise_if_index_error()
    for args, kind in (((x.bfloat16(), t, y), TypeError), ((x.double(), t.double(), y), TypeError), ((x[:, :11], t, y), ValueError),
                       ((x, t, y[:5]), ValueError), ((x, t, y.int()), TypeError), ((x, t.t(), y), ValueError),
                       ((torch.zeros(2, 257, device="cuda"), torch.zeros(3, 257, device="cuda"), y[:2]), ValueError)):
        with pytest.raises(kind):
            rxa.catalog_logprob(*args)
    with pytest.raises(ValueError):
        rxa.catalog_logprob(x, t, y, bias=b[:39])
    with pytest.raises(TypeError):
        rxa.catalog_logprob(x, t, y, bias=b.double())
    leaf = t.clone().requires_grad_(True)
    lp, _ = rxa.catalog_logprob(x[:0], leaf, y[:0])
    d, = torch.autograd.grad(lp.sum(), leaf)
    assert lp.shape == (0,) and d.shape == t.shape and not d.any()
