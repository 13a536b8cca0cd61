"""GMF under the catalogue objective in recorded train loops: every replay gives the bits of the eager step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [500, 1024, 4096])
def test_replays_equal_eager_steps(batch):
    from recsys_amd import ops
    from recsys_amd.dataset import ImplicitData, synthetic_ml1m_data
    from recsys_amd.models.neuralcf import GMF
    from recsys_amd.optim import FusedOptimizer
    from recsys_amd.utils import LoopGraph, train_epoch
    d = synthetic_ml1m_data(seed=3, n_users=400, n_items=300, n_occupations=7, n_train=12 * batch, pool=60, n_test_codes=50)
    results = []
    for graphed in (False, True):
        data = ImplicitData(d, device="cuda", train_batch_size=batch, seed=9)
        torch.manual_seed(0)
        model = GMF(n_users=data.n_users, n_items=data.n_items, embedding_dim=64).cuda().train().set_objective("catalog")
        opt = FusedOptimizer(model, kind="sgd", lr=0.5, clip_norm=1.0)
        step = LoopGraph(model, opt) if graphed else None
        ops.set_index_check("deferred")
        try:
            sums = []
            for _ in range(3):
                sums.append(float(train_epoch(model, opt, data.create_negative_sampled_train_dataloader(), 1.0, step).item()))
                torch.randn(1 << 20, device="cuda").sum().item()        # the program's own work between the replays
            ops.raise_if_index_error()
        finally:
            ops.set_index_check("sync")
        results.append((sums, {k: v.detach().clone() for k, v in model.state_dict().items()}))
    assert results[0][0] == results[1][0] and all(math.isfinite(v) for v in results[0][0])
    for k, v in results[0][1].items():
        assert torch.equal(v, results[1][1][k]), k


@pytest.mark.parametrize("objective", ["catalog", "softmax"])
@pytest.mark.parametrize("name", ["VanillaMF", "BiasMF", "SideFeaturesMF", "TemporalMF", "GMF"])
def test_a_recorded_gradient_holds_kernels_only(name, objective):
    """No memset node (type 2 of hipGraphNodeType) at a batch where torch's reductions record one."""
    import ctypes as C
    import inspect
    from recsys_amd import ops
    from recsys_amd.models import matrix_factorization as mf, neuralcf as ncf
    ops.set_index_check("deferred")
    try:
        cls = getattr(mf, name, None) or getattr(ncf, name)
        dims = dict(n_users=400, n_items=300, n_occupations=7, max_timestamp_rank=30, embedding_dim=64)
        m = cls(**{k: v for k, v in dims.items() if k in inspect.signature(cls.__init__).parameters}).cuda().set_objective(objective)
        B = 8192
        b = {"user_code": torch.randint(0, 400, (B,), device="cuda"), "item_code": torch.randint(0, 300, (B, 5), device="cuda"),
             "user_occupation": torch.randint(0, 7, (B,), device="cuda"), "item_timestamp_rank": torch.randint(0, 30, (B,), device="cuda")}
        step = lambda: torch.autograd.grad(m.loss(b), list(m.parameters()), allow_unused=True)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
            stream.synchronize()
            graph = torch.cuda.CUDAGraph(keep_graph=True)
            with torch.cuda.graph(graph, stream=stream):
                step()
        hip, n, raw = C.CDLL("libamdhip64.so"), C.c_size_t(0), C.c_void_p(graph.raw_cuda_graph())
        assert hip.hipGraphGetNodes(raw, None, C.byref(n)) == 0
        nodes, kind = (C.c_void_p * n.value)(), C.c_int(-1)
        assert hip.hipGraphGetNodes(raw, nodes, C.byref(n)) == 0
        kinds = set()
        for node in nodes:
            assert hip.hipGraphNodeGetType(C.c_void_p(node), C.byref(kind)) == 0
            kinds.add(kind.value)
        assert kinds == {0}, kinds
        ops.raise_if_index_error()
    finally:
        ops.set_index_check("sync")


def test_the_weights_gradient_is_the_sum_over_the_batch():
    """dw = sum_b g_b u_b over 3000 rows, against fp64: (3000 / 2 + 64) u of the terms' size at most."""
    from recsys_amd import autograd as rxa
    g = torch.Generator().manual_seed(2)
    for B, D in ((1, 5), (3000, 64), (777, 33), (5, 256)):
        e, w, go = (torch.randn(s, generator=g).cuda() for s in ((B, D), (1, D), (B, D)))
        le, lw = e.clone().requires_grad_(True), w.clone().requires_grad_(True)
        out = rxa.scale_columns(le, lw)
        assert torch.equal(out, e * w)
        de, dw = torch.autograd.grad(out, (le, lw), go)
        assert torch.equal(de, go * w)
        t = (go * e).double()
        assert ((dw.double() - t.sum(0)).abs() <= (B / 2 + 64) * 2.0 ** -24 * t.abs().sum(0)).all() and dw.shape == (1, D)
        only, = torch.autograd.grad(rxa.scale_columns(e, lw).sum(), lw)
        assert (only - e.sum(0)).abs().max() <= (B / 2 + 64) * 2.0 ** -24 * e.abs().sum(0).max()
