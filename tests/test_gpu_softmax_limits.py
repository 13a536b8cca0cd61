"""Calls at the edges of the softmax operators: offsets past 32 bits, the widest row distance, two streams at once, recording
while an eager graph of the same leaves is alive.  u = 2^-24."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF = 2.0 ** -8


@pytest.fixture
def deferred():
    from recsys_amd import ops
    ops.set_index_check("deferred")
    yield
    ops.raise_if_index_error()
    ops.set_index_check("sync")


def test_scores_past_32_bits():
    """Two bf16 rows of 1.2e9 columns, zero but for one score of the second: sum exp = V - 1 + e^30.  Each of at most 256 x 256
    chains adds fewer than 2^15 exact ones in fp32 (steps of at most 2^-9 of one: below 2^-24 of the sum each, (2^15 + 32) u in
    all), and e^30 is good to 40 u."""
    from recsys_amd import autograd as rxa
    V, far = 1_200_000_000, 1_199_999_990
    x = torch.zeros(2, V, dtype=torch.bfloat16, device="cuda")
    x[1, far] = 30.0
    x.requires_grad_(True)
    y = torch.tensor([V - 1, far], device="cuda")
    out = rxa.log_probs(x, y, k=2)
    lse = torch.tensor([math.log(V), math.log(V - 1 + math.exp(30))], dtype=torch.float64)
    tol = (2 ** 15 + 80) * U
    assert ((out.lse.double().cpu() - lse).abs() <= tol).all()
    assert ((out.logprob.double().cpu() - (torch.tensor([0.0, 30.0]) - lse)).abs() <= 2 * tol).all()
    with torch.no_grad():
        top = rxa.log_probs(x, y, k=2).top_index
    assert top.tolist() == [[0, 1], [far, 0]]
    d, = torch.autograd.grad(out.logprob.sum(), x)
    for r, c in ((0, V - 1), (0, V - 2), (1, far), (1, far + 1), (1, 0)):
        want = (1.0 if c == int(y[r]) else 0.0) - math.exp(float(x[r, c].detach()) - float(lse[r]))
        assert abs(float(d[r, c]) - want) <= BF * abs(want) + 2 * tol * math.exp(float(x[r, c].detach()) - float(lse[r])), (r, c)


def test_catalogue_past_32_bits():
    """A table of 20 million rows of 128, zero but for a few: lse = log(V - 3 + sum of the few)."""
    from recsys_amd import autograd as rxa
    V, D = 20_000_000, 128
    t = torch.zeros(V, D, device="cuda")
    few = torch.tensor([5, 17_000_003, V - 1], device="cuda")
    g = torch.Generator().manual_seed(1)
    t[few] = torch.randn(3, D, generator=g).cuda()
    x = torch.randn(3, D, generator=g).cuda().requires_grad_(True)
    y = torch.tensor([V - 1, 17_000_003, 9], device="cuda")
    t.requires_grad_(True)
    lp, lse = rxa.catalog_logprob(x, t, y)
    s = x.detach().double() @ t.detach()[few].double().t()
    size = x.detach().double().abs() @ t.detach()[few].double().abs().t()
    want = (s.exp().sum(1) + (V - 3)).log()
    tol = (V / 512 / 64 + 64) * U + (D / 2 + 16) * U * size.max()       # a chain of a split adds one tile's 32 lanes at a time
    assert ((lse.double() - want).abs() <= tol + 8 * U * want).all()
    dx, dt = torch.autograd.grad(lp.sum(), (x, t))
    p = (s - want[:, None]).exp()
    X = x.detach().double()
    hot = (y[:, None] == few[None, :]).double()
    wx = t.detach()[y].double() - p @ t.detach()[few].double()
    assert ((dx.double() - wx).abs() <= 64 * U * (1 + t.detach().abs().max()) + tol).all()
    wt = (hot - p).t() @ X
    lim = (hot + p).t() @ X.abs()
    assert ((dt[few].double() - wt).abs() <= (tol + 512 * U) * lim + 3 * 2.0 ** -126).all()
    q = torch.exp(-want)                                                # every zero row: -sum_r p_r x_r, and row 2's target there
    assert ((dt[V - 2].double() + (q[:, None] * X).sum(0)).abs() <= (tol + 512 * U) * (q[:, None] * X.abs()).sum(0) + 3 * 2.0 ** -126).all()
    assert ((dt[9].double() - X[2] + (q[:, None] * X).sum(0)).abs() <= (tol + 512 * U) * (X[2].abs() + (q[:, None] * X.abs()).sum(0))).all()


def test_rows_far_apart():
    """Rows at the largest distance, and one element more refused."""
    from recsys_amd import autograd as rxa
    D, far = 21, 1 << 22
    big = torch.full((70, far + 1), float("nan"), device="cuda")
    x, t = torch.randn(9, D, device="cuda"), torch.randn(70, D, device="cuda")
    y = torch.arange(9, device="cuda")
    want = rxa.catalog_logprob(x, t, y)
    view = big.as_strided((70, D), (far, 1))
    view.copy_(t)
    got = rxa.catalog_logprob(x, view, y)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match="apart"):
        rxa.catalog_logprob(x, big[:, :D], y)


def test_two_streams_at_once(deferred):
    from recsys_amd import autograd as rxa
    torch.manual_seed(3)
    jobs = []
    for i in range(6):
        jobs.append((torch.randn(50 + i, 20000, device="cuda"), torch.randint(0, 20000, (50 + i,), device="cuda"),
                     torch.randn(50 + i, 48, device="cuda"), torch.randn(20000, 48, device="cuda")))

    def work(l, y, x, t):
        l, x, t = (v.detach().requires_grad_(True) for v in (l, x, t))
        out = rxa.log_probs(l, y)
        lp, lse = rxa.catalog_logprob(x, t, y)
        return (*out[:3], lp, lse, *torch.autograd.grad((out.logprob.sum() + lp.sum(),), (l, x, t)))

    alone = [work(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i, j in enumerate(jobs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(work(*j))
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_recording_beside_a_live_eager_graph_is_refused(deferred):
    """The refusal comes in the forward call, before anything of the backward pass is recorded."""
    from recsys_amd import autograd as rxa
    x = torch.randn(6, 16, device="cuda", requires_grad=True)
    t = torch.randn(40, 16, device="cuda", requires_grad=True)
    l = torch.randn(6, 40, device="cuda", requires_grad=True)
    y = torch.arange(6, device="cuda")
    calls = (lambda: rxa.catalog_logprob(x, t, y)[0], lambda: rxa.log_probs(l, y).logprob)
    for call in calls:
        kept = call()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        torch.cuda.synchronize()
        del kept
        leaf = l if call is calls[1] else x
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            d, = torch.autograd.grad(call().sum(), leaf)
        for _ in range(3):
            graph.replay()
            e, = torch.autograd.grad(call().sum(), leaf)
            torch.cuda.synchronize()
            assert torch.equal(d, e)


def test_adam_takes_the_matrices_muon_does_not():
    from recsys_amd.optim import FusedOptimizer

    class Wide(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.a = torch.nn.Parameter(torch.randn(20000, 3, device="cuda"))
            self.b = torch.nn.Parameter(torch.randn(40, 30, device="cuda"))

        def sparse_parameters(self):
            return []

    m = Wide()
    opt = FusedOptimizer(m, dense_kind="muon", lr=0.01)
    assert not opt._is_muon(m.a) and opt._is_muon(m.b)
    sign = torch.where(torch.rand_like(m.a) < 0.5, -1.0, 1.0)
    m.a.grad, m.b.grad = sign * (0.5 + torch.rand_like(m.a)), torch.randn_like(m.b)
    before = m.a.detach().clone()
    opt.step()
    torch.cuda.synchronize()
    step = (before - m.a.detach()) * m.a.grad.sign()
    assert ((step - 0.01).abs() <= 1e-4).all()          # Adam's first step: lr sign(g), less 2e-8 of it for adam_eps


def test_recordings_of_kernels_with_much_shared_memory(deferred):
    """Launches that ask for more than 64 KiB of LDS, recorded, replayed three times beside eager calls."""
    from recsys_amd import autograd as rxa, ops
    torch.manual_seed(5)
    mats = [torch.randn(90, 300, device="cuda"), torch.randn(700, 650, device="cuda"), torch.randn(16, 2200, device="cuda")]
    y = torch.randint(0, 900, (70,), device="cuda")
    b = torch.randn(900, device="cuda")

    def step(x, t):
        x, t = x.detach().requires_grad_(True), t.detach().requires_grad_(True)
        lp, lse = rxa.catalog_logprob(x, t, y, bias=b)
        return (lp, lse, *torch.autograd.grad(lp.sum() + 0.5 * lse.sum(), (x, t)), *ops.orthogonalize(mats[:1]), *ops.orthogonalize(mats))

    for D, dtype in ((256, torch.float32), (190, torch.float32), (256, torch.bfloat16), (128, torch.float32)):
        x, t = torch.randn(70, D, device="cuda").to(dtype), (0.1 * torch.randn(900, D, device="cuda")).to(dtype)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(x, t)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                rec = step(x, t)
        torch.cuda.current_stream().wait_stream(stream)
        for _ in range(3):
            x.copy_(torch.randn(70, D, device="cuda"))
            for m in mats:
                m.normal_()
            torch.cuda.synchronize()
            graph.replay()
            eager = step(x, t)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(rec, eager))
