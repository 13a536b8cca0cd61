"""The softmax objectives, the Muon step and the catalogue ranking as the framework's own paths use them: model losses,
FusedOptimizer, recorded train loops, recommend()."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DIMS = dict(n_users=60, n_items=150, n_occupations=5, max_timestamp_rank=30)


def _model(name, dim=24, seed=0, **kw):
    import inspect
    from recsys_amd.models import matrix_factorization as mf, neuralcf as ncf
    cls = getattr(mf, name, None) or getattr(ncf, name)
    torch.manual_seed(seed)
    args = {k: v for k, v in dict(DIMS, embedding_dim=dim, **kw).items() if k in inspect.signature(cls.__init__).parameters}
    m = cls(**args)
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() == 2 and p.shape[1] > 1:
                p.mul_(0.5)
    return m.cuda().train()


def _batch(B=90, N=6, seed=0):
    g = torch.Generator().manual_seed(seed)
    b = {"user_code": torch.randint(0, 60, (B,), generator=g), "item_code": torch.randint(0, 150, (B, N), generator=g),
         "user_occupation": torch.randint(0, 5, (B,), generator=g), "item_timestamp_rank": torch.randint(0, 30, (B,), generator=g),
         "label": torch.zeros(B, N, dtype=torch.float64)}
    b["label"][:, 0] = 1
    return {k: v.cuda() for k, v in b.items()}


@pytest.mark.parametrize("name", ["VanillaMF", "BiasMF", "TemporalMF", "GMF", "MLP", "NeuMF", "FactorizationMachine"])
def test_softmax_loss_is_the_log_softmax_of_the_models_scores(name):
    """Value and gradients against autograd through the model's own scores in torch."""
    m = _model(name, dropout=0.0)
    b = _batch()
    b["target"] = torch.randint(0, 4, (90,), device="cuda")
    b["list_length"] = torch.randint(4, 7, (90,), device="cuda")
    want = m(b)
    hidden = torch.arange(6, device="cuda")[None] >= b["list_length"][:, None]
    ref = -torch.log_softmax(want.double().masked_fill(hidden, -math.inf), 1).gather(1, b["target"][:, None]).mean()
    gref = torch.autograd.grad(ref, list(m.parameters()), allow_unused=True)
    m.set_objective("softmax")
    loss = m.loss(b)
    got = torch.autograd.grad(loss, list(m.parameters()), allow_unused=True)
    assert loss.dtype == torch.float64
    # the two share the scores: 6 scores per row and the mean of 90 rows, both in fp32
    assert abs(loss.item() - ref.item()) <= 64 * U * (1 + abs(ref.item()))
    for (n, _), a, e in zip(m.named_parameters(), got, gref):
        assert (a is None) == (e is None), n
        # dL/dscore agrees to 16 u; both then pass through the same kernels (fp32 sums, either order of operations).
        # The terms of a gradient sum up to at most 2 in size (a row's sum of |1 - p| and p, averaged), times the score's
        # slope, which is below 2 here: a gradient that cancels to zero, like a bias's, keeps 16 u * 4 of rounding.
        if a is not None:
            assert (a - e).abs().max() <= 2e-5 * e.abs().max() + 64 * U, n


@pytest.mark.parametrize("name", ["VanillaMF", "BiasMF", "SideFeaturesMF", "TemporalMF", "GMF"])
def test_catalog_loss_is_the_softmax_over_every_item(name):
    m = _model(name, seed=1)
    b = _batch(seed=1)
    every = dict(b, item_code=torch.arange(150, device="cuda").expand(90, 150).contiguous(), target=b["item_code"][:, 0].contiguous())
    with torch.no_grad():
        full = m(every).double()
    ref = -torch.log_softmax(full, 1).gather(1, every["target"][:, None]).mean()
    m.set_objective("softmax")
    gref = torch.autograd.grad(m.loss(every), list(m.parameters()), allow_unused=True)
    m.set_objective("catalog")
    loss = m.loss(b)
    got = torch.autograd.grad(loss, list(m.parameters()), allow_unused=True)
    assert abs(loss.item() - ref.item()) <= 256 * U * (1 + abs(ref.item()))
    for (n, _), a, e in zip(m.named_parameters(), got, gref):
        if a is None:            # constants of a row: their gradient is a sum that cancels
            assert e is None or e.abs().max() <= 1e-5, n
        else:
            assert (a - e).abs().max() <= 5e-5 * e.abs().max() + 1e-9, n


def test_objectives_are_refused_where_they_do_not_apply():
    m = _model("MLP")
    with pytest.raises(ValueError):
        m.set_objective("catalog")
    with pytest.raises(ValueError):
        m.set_objective("hinge")
    with pytest.raises(ValueError):
        m.catalog_loss(_batch())
    m.set_objective("softmax")
    one = _batch(N=1)
    with pytest.raises(ValueError):
        m.loss(one)
    with pytest.raises(ValueError):
        m.loss(dict(one, item_code=one["item_code"][:, 0].contiguous()), pointwise=True)
    wide = _model("VanillaMF", dim=260).set_objective("catalog")
    with pytest.raises(ValueError):
        wide.loss(_batch())


@pytest.mark.parametrize("clip", [None, 0.05])
@pytest.mark.parametrize("kind", ["sgd", "adagrad"])
def test_fused_optimizer_steps_the_whole_item_table(kind, clip):
    """The catalogue gradient touches every item row; the fused sparse rule then equals the dense torch optimizer."""
    from recsys_amd.optim import FusedOptimizer
    ref, m = _model("BiasMF", seed=2).set_objective("catalog"), _model("BiasMF", seed=2).set_objective("catalog")
    opt = FusedOptimizer(m, kind=kind, lr=0.3, clip_norm=clip)
    live = [p for n, p in ref.named_parameters() if n not in ("user_bias", "bias")]
    topt = torch.optim.SGD(live, lr=0.3) if kind == "sgd" else torch.optim.Adagrad(live, lr=0.3, eps=1e-10)
    for s in range(3):
        b = _batch(seed=s)
        topt.zero_grad()
        ref.loss(b).backward()
        if clip is not None:
            torch.nn.utils.clip_grad_norm_(live, clip)
        topt.step()
        opt.zero_grad()
        m.loss(b).backward()
        opt.step()
        touched = torch.zeros(60, dtype=torch.bool)
        touched[b["user_code"].cpu()] = True
    for (n, p), q in zip(ref.named_parameters(), m.parameters()):
        # three steps of the same fp32 gradients; Adagrad's first steps move by lr g / |g|, so entries whose gradient is
        # rounding noise are left out of its comparison
        d = (p - q).abs()
        if kind == "adagrad":
            assert d.median() <= 1e-5 and (d > 1e-3).float().mean() < 0.01, n
        else:
            assert d.max() <= 1e-5 * p.abs().max(), n


# ------------------------------------------------------------------ Muon
def _newton_schulz(G):
    X = G.t() if G.shape[0] > G.shape[1] else G
    X = X / (X.pow(2).sum().sqrt() + 1e-7)
    for _ in range(5):
        A = X @ X.t()
        X = 3.4445 * X + (-4.7750 * A + 2.0315 * (A @ A)) @ X
    return X.t() if G.shape[0] > G.shape[1] else X


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("with_scale", [True, False])
def test_muon_step_against_its_formula(nesterov, with_scale):
    from recsys_amd import ops
    shapes = [(64, 128), (128, 48), (130, 200), (300, 97), (2, 2)]
    g = torch.Generator().manual_seed(1)
    ws = [torch.randn(s, generator=g).cuda() for s in shapes]
    ms = [torch.zeros(s).cuda() for s in shapes]
    lrs = [0.1, 0.2, 0.05, 0.02, 0.3]
    w64, m64 = [w.double().cpu() for w in ws], [m.double().cpu() for m in ms]
    scale = torch.tensor([0.4], device="cuda") if with_scale else None
    for _ in range(3):
        gs = [torch.randn(s, generator=g).cuda() for s in shapes]
        ops.muon_step(ws, gs, ms, lrs, momentum=0.9, nesterov=nesterov, scale=scale)
        for i in range(len(shapes)):
            gr = gs[i].double().cpu() * (float(scale) if with_scale else 1.0)
            m64[i] = 0.9 * m64[i] + gr
            w64[i] = w64[i] - lrs[i] * _newton_schulz(gr + 0.9 * m64[i] if nesterov else m64[i])
    for w, m, rw, rm, lr in zip(ws, ms, w64, m64, lrs):
        assert (m.cpu().double() - rm).abs().max() <= 8 * U * (1 + rm.abs().max())
        # Gaussian matrices: the directions with the smallest singular values carry errors up to 485 u relative to the norm
        assert (w.cpu().double() - rw).norm() <= 3 * lr * 2000 * U * rw.norm() + 8 * U * rw.norm()


def test_muon_refusals():
    from recsys_amd import ops
    w, g, m = (torch.randn(8, 9, device="cuda") for _ in range(3))
    for args, kind in ((([w], [g], [w], [0.1]), RuntimeError), (([w], [g], [g], [0.1]), RuntimeError), (([w, w], [g, g], [m, m], [0.1, 0.1]), RuntimeError),
                       (([w], [g], [m], []), ValueError), (([w], [g[:7]], [m], [0.1]), ValueError), (([w.double()], [g], [m], [0.1]), TypeError),
                       (([w.cpu()], [g], [m], [0.1]), ValueError), (([w[0]], [g], [m], [0.1]), ValueError)):
        with pytest.raises(kind):
            ops.muon_step(*args)
    with pytest.raises(ValueError):
        ops.muon_step([w], [g], [m], [0.1], scale=torch.ones(2, device="cuda"))
    ops.muon_step([], [], [], [])


def test_muon_through_the_optimizer():
    """Matrices by Muon, the one-row layer and the biases by Adam, the tables by their sparse rule."""
    from recsys_amd.optim import FusedOptimizer
    m = _model("MLP", seed=3, dropout=0.0).set_objective("softmax")
    opt = FusedOptimizer(m, kind="sgd", lr=0.02, dense_kind="muon", adam_lr=1e-3, clip_norm=0.1)
    w = {n: p.detach().double().cpu() for n, p in m.named_parameters()}
    mom = {n: torch.zeros_like(v) for n, v in w.items()}
    av = {n: [torch.zeros_like(v), torch.zeros_like(v)] for n, v in w.items()}
    for t in range(1, 4):
        b = _batch(seed=t)
        twin = _model("MLP", seed=3, dropout=0.0).set_objective("softmax")
        twin.load_state_dict(m.state_dict())
        twin.loss(b).backward()
        gr = {n: p.grad.double().cpu() for n, p in twin.named_parameters()}
        s = min(1.0, 0.1 / (math.sqrt(sum(float(v.pow(2).sum()) for v in gr.values())) + 1e-6))
        opt.zero_grad()
        m.loss(b).backward()
        opt.step()
        for n, v in gr.items():
            v = v * s
            if "embedding" in n:
                w[n] = w[n] - 0.02 * v
            elif v.dim() == 2 and min(v.shape) >= 2:
                mom[n] = 0.95 * mom[n] + v
                w[n] = w[n] - 0.02 * math.sqrt(max(1.0, v.shape[0] / v.shape[1])) * _newton_schulz(v + 0.95 * mom[n])
            else:
                a = av[n]
                a[0], a[1] = 0.9 * a[0] + 0.1 * v, 0.999 * a[1] + 0.001 * v * v
                w[n] = w[n] - 1e-3 * (a[0] / (1 - 0.9 ** t)) / ((a[1] / (1 - 0.999 ** t)).sqrt() + 1e-8)
        for n, p in m.named_parameters():
            d = (p.detach().double().cpu() - w[n])
            # an update whose gradient is rank-deficient (few distinct rows) has directions made of rounding noise alone;
            # what counts is the step's size, 0.02 per singular direction
            assert d.norm() <= 2e-3 * 0.02 * math.sqrt(min(d.shape) if d.dim() == 2 else d.numel()) * t + 1e-6 * w[n].norm(), (t, n)
            w[n] = p.detach().double().cpu()
    assert opt.step_count == 3
    with pytest.raises(ValueError):
        FusedOptimizer(m, kind="dense_adam", dense_kind="muon")


# ------------------------------------------------------------------ all of it in the train loop
@pytest.mark.parametrize("case", ["mf_catalog_sgd", "side_catalog_adagrad", "neumf_softmax_muon", "mlp_softmax_muon"])
def test_train_epochs_as_graph_replays_equal_eager_ones(case):
    from recsys_amd import ops
    from recsys_amd.dataset import ImplicitData, synthetic_ml1m_data
    from recsys_amd.models import matrix_factorization as mf, neuralcf as ncf
    from recsys_amd.optim import FusedOptimizer
    from recsys_amd.utils import LoopGraph, train_epoch
    d = synthetic_ml1m_data(seed=3, n_users=400, n_items=300, n_occupations=7, n_train=12000, pool=60, n_test_codes=50)
    results = []
    for graphed in (False, True):
        data = ImplicitData(d, device="cuda", train_batch_size=500, seed=9)
        torch.manual_seed(0)
        kw = dict(n_users=data.n_users, n_items=data.n_items, embedding_dim=16)
        if case.startswith("mf"):
            model = mf.VanillaMF(**kw)
        elif case.startswith("side"):
            model = mf.SideFeaturesMF(n_occupations=data.n_occupations, **kw)
        else:
            model = (ncf.NeuMF if case.startswith("neumf") else ncf.MLP)(dropout=0.0, **kw)
        model = model.cuda().train().set_objective("catalog" if "catalog" in case else "softmax")
        opt = FusedOptimizer(model, kind="adagrad" if "adagrad" in case else "sgd", lr=0.05, clip_norm=1.0,
                             dense_kind="muon" if "muon" in case else None, **(dict(adam_lr=1e-3) if "muon" in case else {}))
        step = LoopGraph(model, opt) if graphed else None
        ops.set_index_check("deferred")
        try:
            sums = [float(train_epoch(model, opt, data.create_negative_sampled_train_dataloader(), 1.0, step).item()) for _ in range(2)]
            ops.raise_if_index_error()
        finally:
            ops.set_index_check("sync")
        results.append((sums, {k: v.detach().clone() for k, v in model.state_dict().items()}))
    assert results[0][0] == results[1][0] and all(math.isfinite(v) for v in results[0][0])
    for k, v in results[0][1].items():
        assert torch.equal(v, results[1][1][k]), k


def test_train_loop_runs_with_the_new_objectives(capsys):
    from recsys_amd.dataset import ImplicitData, synthetic_ml1m_data
    from recsys_amd.models.matrix_factorization import BiasMF
    from recsys_amd.models.neuralcf import NeuMF
    from recsys_amd.optim import FusedOptimizer
    from recsys_amd.utils import recommend, train_loop
    d = synthetic_ml1m_data(seed=3, n_users=400, n_items=300, n_occupations=7, n_train=12000, pool=60, n_test_codes=50)
    for cls, objective, dense in ((BiasMF, "catalog", None), (NeuMF, "softmax", "muon")):
        data = ImplicitData(d, device="cuda", train_batch_size=256, test_batch_size=128)
        torch.manual_seed(0)
        model = cls(data.n_users, data.n_items, 16).cuda().set_objective(objective)
        opt = FusedOptimizer(model, kind="adagrad", lr=0.02, clip_norm=1.0, dense_kind=dense)
        hist = train_loop(model, data, opt, num_epochs=2, clip_norm=1.0, k=10, graph=True)
        assert all(math.isfinite(h[0]) for h in hist)
        codes, logprob, entropy = recommend(model, {"user_code": torch.arange(5, device="cuda"), "item_code": torch.arange(300, device="cuda").expand(5, 300).contiguous()}, k=7)
        assert codes.shape == (5, 7) and (codes >= 0).all() and torch.isfinite(logprob).all() and (entropy > 0).all()


# ------------------------------------------------------------------ recommend
def test_recommend_over_the_catalogue_and_over_lists():
    from recsys_amd.utils import recommend
    m = _model("VanillaMF", seed=5).eval()
    users = torch.arange(40, device="cuda")
    scores = m({"user_code": users, "item_code": None}).detach()
    seen = torch.randint(-1, 150, (40, 9), generator=torch.Generator().manual_seed(1)).cuda()
    for exclude in (None, seen):
        z = scores.clone()
        if exclude is not None:
            for r in range(40):
                z[r, exclude[r][exclude[r] >= 0]] = -math.inf
        codes, logprob, entropy = recommend(m, {"user_code": users, "item_code": None}, k=12, exclude=exclude)
        val, idx = torch.sort(z, dim=1, descending=True, stable=True)
        assert torch.equal(codes, idx[:, :12])
        want = torch.log_softmax(z.double(), 1)
        assert (logprob - want.gather(1, codes)).abs().max() <= 1e-5
        H = -(want.exp() * want.clamp(min=-1e4)).sum(1)
        assert (entropy - H).abs().max() <= 1e-5
    lists = _batch(B=40, N=8, seed=3)
    codes, _, _ = recommend(m, lists, k=10)
    assert (codes[:, 8:] == -1).all()
    best = m(lists).argmax(1, keepdim=True)
    assert torch.equal(codes[:, :1], lists["item_code"].gather(1, best))
    with pytest.raises(IndexError):
        recommend(m, {"user_code": users, "item_code": None}, k=3, exclude=torch.full((40, 1), 150))
    with pytest.raises(ValueError):
        recommend(m, {"user_code": users, "item_code": None}, k=3, exclude=seen[:3])
